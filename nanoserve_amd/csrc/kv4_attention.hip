// Paged attention over the cache held in 4 bits (record layout: kv4.h).
//
// Same rows, masks and results as the 16-bit op (paged_attention.hip): query
// row j of a sequence with context length L and query length ql sees keys
// 0 .. L - ql + j, KV head of query head h is h / (Hq / Hkv), softmax and sums
// in float32, a row without keys is zero.  With a row of K or V stored as
// scale s, offset b and codes c,
//     q . k_t    = s_t (q . c_t) + b_t sum(q)
//     sum p_t v_t = sum (p_t s_t) c_t + sum p_t b_t
// so the products run on the codes and a token's scale and offset enter once
// per score, never per element.
#include <math.h>

#include "kv4.h"

namespace ns {
namespace {

struct Kv4AttnParams {
  char* out;
  const char* query;
  const char* k_cache;
  const char* v_cache;
  const void* bt;
  int64_t bt_stride;
  const void* seq_lens;
  const void* qsl;        // query offsets (not read for decode-only batches)
  int bt64, sl64, qsl64, decode_only;
  int num_seqs, num_heads, num_kv_heads, group, head_dim, block_size;
  int64_t num_tokens, num_blocks, record;
  int64_t max_ctx;        // keys a row may have: max_seq_len rounded to blocks, within the table
  float scale;
};

struct Rows {
  int64_t row0, ql, len;  // first query row, query rows, context length
};

__device__ __forceinline__ Rows rows_of(const Kv4AttnParams& p, int s) {
  Rows r;
  if (p.decode_only) {
    r.row0 = s;
    r.ql = 1;
  } else {
    r.row0 = load_index(p.qsl, s, p.qsl64);
    r.ql = load_index(p.qsl, s + 1, p.qsl64) - r.row0;
    // Offsets that leave the query tensor are never followed.
    if (r.row0 < 0 || r.ql < 0 || r.row0 + r.ql > p.num_tokens) r.ql = 0;
  }
  r.len = load_index(p.seq_lens, s, p.sl64);
  r.len = r.len < 0 ? 0 : (r.len < p.max_ctx ? r.len : p.max_ctx);
  return r;
}

// ---- any shape: one wave per (token row, query head) ------------------------
//
// One key per lane: the lane's dot product of the query (in LDS, float32) with
// the key's codes joins the wave's running maximum and sum; then every lane
// adds the chunk's weighted values into the output dims it owns, one key at a
// time.  Plain: the serving shapes run the matrix-core kernel.
// DL: output dims per lane (head_dim <= 64 * DL).
template <class DT, int DL>
__global__ __launch_bounds__(64) void kv4_attention_generic_kernel(Kv4AttnParams p) {
  __shared__ float q_lds[64 * DL];
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y;
  const int D = p.head_dim, half = D / 2, bs = p.block_size;
  const int kvh = h / p.group;

  // The row's sequence: the last s with query_start_loc[s] <= t.
  int s = static_cast<int>(t);
  if (!p.decode_only) {
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (load_index(p.qsl, mid, p.qsl64) <= t) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
  }
  const Rows r = rows_of(p, s);
  if (t < r.row0 || t >= r.row0 + r.ql) return;  // a row of no sequence is left as it is
  const int64_t limit = r.len - r.ql + (t - r.row0);  // the row's last key
  const int64_t nkeys = limit < 0 ? 0 : (limit + 1 < r.len ? limit + 1 : r.len);

  const char* qrow = p.query + (t * p.num_heads + h) * D * 2;
  float qsum = 0.f;
  for (int d = lane; d < 64 * DL; d += 64) {
    const float q = d < D ? Half<DT>::to_f32(reinterpret_cast<const uint16_t*>(qrow)[d]) : 0.f;
    q_lds[d] = q;
    qsum += q;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) qsum += __shfl_xor(qsum, off);
  __syncthreads();

  const int64_t bt_row = static_cast<int64_t>(s) * p.bt_stride;
  float m = -INFINITY, l = 0.f, o[DL];
#pragma unroll
  for (int j = 0; j < DL; ++j) o[j] = 0.f;
  int bad = 0;
  for (int64_t c0 = 0; c0 < nkeys; c0 += 64) {
    const int64_t key = c0 + lane;
    int64_t rec = 0;  // this lane's key: its record and place in it
    int tk = 0;
    bool ok = false;
    if (key < nkeys) {
      const int64_t blk = load_index(p.bt, bt_row + key / bs, p.bt64);
      tk = static_cast<int>(key % bs);
      if (blk < 0 || blk >= p.num_blocks) {
        bad = 1;
      } else {
        ok = true;
        rec = (blk * p.num_kv_heads + kvh) * p.record;
      }
    }
    float sc = -INFINITY, vs = 0.f, vb = 0.f;
    if (ok) {
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(p.k_cache + rec + bs * half + 4 * tk);
      const uint32_t vp = *reinterpret_cast<const uint32_t*>(p.v_cache + rec + bs * half + 4 * tk);
      const uint32_t* kw = reinterpret_cast<const uint32_t*>(p.k_cache + rec + tk * half);
      float acc = 0.f;
      for (int w = 0; w < D / 8; ++w) {
        const uint32_t x = kw[w];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          acc = __builtin_fmaf(q_lds[8 * w + e], static_cast<float>((x >> (4 * e)) & 15u), acc);
      }
      sc = (kv4_scale<DT>(kp) * acc + kv4_offset<DT>(kp) * qsum) * p.scale;
      vs = kv4_scale<DT>(vp);
      vb = kv4_offset<DT>(vp);
    }
    float cm = sc;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) cm = fmaxf(cm, __shfl_xor(cm, off));
    const float m_new = fmaxf(m, cm);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = expf(m - m_use);
    const float pk = ok ? expf(sc - m_use) : 0.f;
    float ps = pk;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ps += __shfl_xor(ps, off);
    l = l * alpha + ps;
    m = m_new;
#pragma unroll
    for (int j = 0; j < DL; ++j) o[j] *= alpha;
    const int nk = nkeys - c0 < 64 ? static_cast<int>(nkeys - c0) : 64;
    const uint32_t rec_lo = static_cast<uint32_t>(rec), rec_hi = static_cast<uint32_t>(rec >> 32);
    for (int kk = 0; kk < nk; ++kk) {
      const float w = __shfl(pk, kk);
      if (w == 0.f) continue;  // uniform: the weight is broadcast
      const float ws = w * __shfl(vs, kk), wb = w * __shfl(vb, kk);
      const int kt = __shfl(tk, kk);
      const int64_t kr = static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(__shfl(rec_hi, kk))) << 32) |
                                              static_cast<uint32_t>(__shfl(rec_lo, kk)));
      const uint8_t* vrow = reinterpret_cast<const uint8_t*>(p.v_cache) + kr + (kt >> 2) * (4 * half) + kv4_v_pos(kt);
#pragma unroll
      for (int j = 0; j < DL; ++j) {
        const int d = lane + 64 * j;
        if (d < D) {
          const float c = static_cast<float>((vrow[4 * (d >> 1)] >> (4 * (d & 1))) & 15);
          o[j] = __builtin_fmaf(ws, c, o[j]) + wb;
        }
      }
    }
  }
  bad = __builtin_amdgcn_ballot_w64(bad != 0) != 0;

  char* orow = p.out + (t * p.num_heads + h) * D * 2;
  const float inv = l > 0.f ? 1.f / l : l;  // no key: zero; a NaN stays one
#pragma unroll
  for (int j = 0; j < DL; ++j) {
    const int d = lane + 64 * j;
    if (d < D)
      reinterpret_cast<uint16_t*>(orow)[d] =
          static_cast<uint16_t>(bad ? Half<DT>::nan : Half<DT>::from_f32(o[j] * inv));
  }
}

template <class DT>
hipError_t launch_generic(const Kv4AttnParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.num_tokens), static_cast<unsigned>(p.num_heads));
  void* args[] = {const_cast<Kv4AttnParams*>(&p)};
  const void* fn = p.head_dim <= 64    ? reinterpret_cast<const void*>(&kv4_attention_generic_kernel<DT, 1>)
                   : p.head_dim <= 128 ? reinterpret_cast<const void*>(&kv4_attention_generic_kernel<DT, 2>)
                                       : reinterpret_cast<const void*>(&kv4_attention_generic_kernel<DT, 4>);
  return hipLaunchKernel(fn, grid, dim3(64), args, 0, stream);
}

bool misaligned(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

}  // namespace
}  // namespace ns

extern "C" int ns_paged_attention_int4(void* out, const void* query,
                                       const void* k_cache, const void* v_cache,
                                       const void* block_tables, int64_t block_table_stride,
                                       int64_t block_table_width, int block_tables_is_int64,
                                       const void* seq_lens, int seq_lens_is_int64,
                                       const void* query_start_loc, int query_start_loc_is_int64,
                                       int num_seqs, int64_t num_tokens, int max_query_len, int max_seq_len,
                                       int is_decode_only,
                                       int num_heads, int num_kv_heads, int head_dim,
                                       int block_size, int64_t num_blocks,
                                       float scale, int dtype, void* stream) {
  using namespace ns;
  if (num_seqs < 0 || num_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      head_dim <= 0 || block_size <= 0 || num_blocks <= 0 || max_seq_len < 0 || !(fabsf(scale) < INFINITY))
    return NS_ERR_INVALID_ARG;
  if (dtype != NS_DTYPE_F16 && dtype != NS_DTYPE_BF16) return NS_ERR_UNSUPPORTED;
  if (!kv4_shape_ok(head_dim, block_size)) return NS_ERR_UNSUPPORTED;
  if (num_seqs == 0 || num_tokens == 0) return NS_OK;
  if (!out || !query || !k_cache || !v_cache || !block_tables || !seq_lens) return NS_ERR_INVALID_ARG;
  if (is_decode_only ? num_tokens != num_seqs : !query_start_loc) return NS_ERR_INVALID_ARG;
  if (!is_decode_only && max_query_len <= 0) return NS_ERR_INVALID_ARG;
  if (block_table_width <= 0 || block_table_stride < block_table_width) return NS_ERR_INVALID_ARG;
  if (misaligned(out, 16) || misaligned(query, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16) ||
      misaligned(block_tables, block_tables_is_int64 ? 8 : 4) || misaligned(seq_lens, seq_lens_is_int64 ? 8 : 4) ||
      misaligned(query_start_loc, query_start_loc_is_int64 ? 8 : 4))
    return NS_ERR_INVALID_ARG;
  if (num_tokens > 0x7FFFFFFF || num_heads > 65535) return NS_ERR_UNSUPPORTED;
  Kv4AttnParams p;
  p.out = static_cast<char*>(out);
  p.query = static_cast<const char*>(query);
  p.k_cache = static_cast<const char*>(k_cache);
  p.v_cache = static_cast<const char*>(v_cache);
  p.bt = block_tables;
  p.bt_stride = block_table_stride;
  p.seq_lens = seq_lens;
  p.qsl = query_start_loc;
  p.bt64 = block_tables_is_int64 ? 1 : 0;
  p.sl64 = seq_lens_is_int64 ? 1 : 0;
  p.qsl64 = query_start_loc_is_int64 ? 1 : 0;
  p.decode_only = is_decode_only ? 1 : 0;
  p.num_seqs = num_seqs;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_tokens = num_tokens;
  p.num_blocks = num_blocks;
  p.record = kv4_record_bytes(block_size, head_dim);
  const int64_t ctx = (static_cast<int64_t>(max_seq_len) + block_size - 1) / block_size * block_size;
  const int64_t table = block_table_width * static_cast<int64_t>(block_size);
  p.max_ctx = ctx < table ? ctx : table;
  p.scale = scale;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = dtype == NS_DTYPE_F16 ? launch_generic<F16>(p, st) : launch_generic<BF16>(p, st);
  return e == hipSuccess ? NS_OK : NS_ERR_HIP;
}
