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
  int64_t max_ctx;        // keys a row may have: max_seq_len, within the table
  float scale;
  // Matrix-core kernels: a row's keys are cut into nsplit ranges of split
  // tokens (a multiple of 32).  With more than one, range i of row r and head h
  // leaves its maximum (log2 units), sum and unnormalised output at index
  // (r * num_heads + h) * nsplit + i of part_m, part_l and part_o.
  int nsplit, split;
  int every_row;          // the column kernel takes one-row sequences too
  float* part_m;
  float* part_l;
  float* part_o;
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

// ---- head sizes 64 and 128, blocks of whole 16-token tiles --------------------
//
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16, straight from the
// cache: a lane's part of a 16-token tile is one load (8 or 16 bytes), a mask
// turns its words into operands (kv4.h), and nothing passes through LDS.  Both
// model dtypes run in float16: the codes are exact there, the query is brought
// into its range by a power of two per column (exact but for elements 2^-29 of
// the column's largest, whose error is below 2^-40 of it), and the probabilities
// keep 11 bits where bfloat16 would keep 8.
//
// A score is y = s_t (q.c_t) + b_t sum(q), its logarithm to base 2 is y times a
// column's factor, which the exponential's own fused multiply-add applies.  The
// operand of the second product is p s_t, rounded once to float16: p is kept
// 2^14 times its value, s_t divided by a power of two above the largest scale
// that the wave has met (the accumulators follow when that grows, exactly), so
// a product lies below 2^14 and keeps its 11 bits down to 2^-28 of the largest.
// sum p and sum p b_t are float32.
//
// The result layout of the first product, tokens 4 g + r of column lane % 16 in
// lane group g, is the operand layout of the second.

// The operands of one step of 32 tokens: a lane's words of the two tiles.
template <int D>
struct Step {
  uint32_t k[2][D / 32], v[2][D / 32];
  u32x4 kp[2], vp[2];  // parameter words of tokens 4 g .. 4 g + 3 of each tile
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const char* p) {
  if constexpr (N == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    w[0] = x[0];
    w[1] = x[1];
  } else {
    static_assert(N == 4, "head sizes 64 and 128");
    const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = x[i];
  }
}

// Where the wave's tiles lie: lane l holds tile l & 1 of step l / 2 of a window
// of 32 steps, as the byte offset of its codes and, from there, of its
// parameter words (bit 0 of which marks a block id outside the cache).
struct Window {
  uint32_t lo, hi;
  int par;
};

__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

constexpr float kCodeUnit = 16777216.f;  // 2^24: an even dim's code as a half's bits is code / 2^24
constexpr float kLift = 14.f;            // p is kept 2^14 times its value

// One wave's state: NT tiles of 16 columns, D output dims each.
template <class DT, int D, int NT>
struct Wave {
  half8 q[NT][D / 32];
  float cf[NT], qs[NT];       // log2 units per score unit; sum(q) in score units
  float m[NT], l[NT], b[NT];  // maximum (log2), sum p (this lane's tokens), sum p b_t (likewise)
  floatx4 acc[NT][D / 16];
  float sigma, inv_sigma;     // the scales' power of two
  uint32_t top;               // largest parameter word that needs no larger sigma

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      l[n] = b[n] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[n][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    sigma = inv_sigma = 1.f;
    top = 0xFFFFu;
  }

  // Column n's query row, as the operand that meets the codes: lane group g
  // holds dims (D / 4) g .. + D / 4, eight of them per 32-dim step in the order
  // of a word's masked nibbles, odd dims a sixteenth of their value.
  __device__ __forceinline__ void load_query(int n, const char* row, int g, float scale) {
    float x[D / 4], big = 0.f;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      const u32x4 r = *reinterpret_cast<const u32x4*>(row + (g * (D / 4) + 8 * w) * 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[8 * w + 2 * e] = Half<DT>::to_f32(r[e] & 0xFFFFu);
        x[8 * w + 2 * e + 1] = Half<DT>::to_f32(r[e] >> 16);
        big = fmaxf(big, fmaxf(fabsf(x[8 * w + 2 * e]), fabsf(x[8 * w + 2 * e + 1])));
      }
    }
    big = group4_max(big);
    // The largest becomes 2^14 .. 2^15 (a column of zeros or non-finite values as it comes).
    int e = static_cast<int>(__float_as_uint(big) >> 23) - 127;
    e = 14 - e;
    e = e < -113 ? -113 : e > 100 ? 100 : e;
    if (!(big > 0.f) || !(big < INFINITY)) e = 0;
    float f = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    cf[n] = fabsf(scale) * 1.4426950408889634f * (kCodeUnit / f);
    if (scale < 0.f) f = -f;  // a negative scale turns the query around, exactly
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      x[i] *= f;
      sum += x[i];
    }
    qs[n] = group4_sum(sum) * (1.f / kCodeUnit);
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float unit = (i & 1) ? 0.0625f : 1.f;
        q[n][w][2 * i] = static_cast<_Float16>(x[8 * w + i] * unit);
        q[n][w][2 * i + 1] = static_cast<_Float16>(x[8 * w + i + 4] * unit);
      }
    }
  }

  // Two codes in each word: four operand registers from a word's eight codes.
  static __device__ __forceinline__ half8 k_operand(uint32_t w) {
    const uint32_t y = w >> 8;
    return __builtin_bit_cast(half8, u32x4{w & 0x000F000Fu, w & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u});
  }
  static __device__ __forceinline__ half8 v_operand(uint32_t a, uint32_t b, uint32_t mask) {
    return __builtin_bit_cast(half8, u32x4{a & mask, (a >> 8) & mask, b & mask, (b >> 8) & mask});
  }

  // A larger scale has come: the next power of two above it, the accumulators along.
  __device__ __forceinline__ void raise_sigma(uint32_t w) {
    w = max(w, static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), 16)));
    w = max(w, static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), 32)));
    const uint32_t bits = __float_as_uint(kv4_scale<DT>(w));
    float next = __uint_as_float((bits & 0x7F800000u) + 0x00800000u);
    if constexpr (DT::code == NS_DTYPE_F16) {
      next = fmaxf(next, 6.103515625e-05f);  // subnormal scales share 2^-14
      top = w | 0x03FFFFFFu;
    } else {
      top = w | 0x007FFFFFu;
    }
    const float ratio = sigma / next;
    sigma = next;
    inv_sigma = 1.f / next;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[n][i] *= ratio;
  }

  // One step over tokens tok .. tok + 31.  MASK: some column does not see all of
  // them; column n sees tokens up to limit[n], none of the wave's sees past last.
  template <bool MASK>
  __device__ __forceinline__ void step(const Step<D>& d, int tok, int g, const int (&limit)[NT], int last) {
    floatx4 s[NT][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const half8 a = k_operand(d.k[j][w]);
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][j] = mfma16x16x32(F16{}, a, q[n][w], s[n][j]);
      }
    }
    float vs[2][4], vb[2][4];
    uint32_t big = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        uint32_t w = d.vp[j][r];
        if (MASK && tok + 16 * j + 4 * g + r > last) w = 0;  // what lies there is nobody's
        big = max(big, w);
        vs[j][r] = kv4_scale<DT>(w);
        vb[j][r] = kv4_offset<DT>(w);
      }
    }
    if (__builtin_amdgcn_ballot_w64(big > top)) raise_sigma(big);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) vs[j][r] *= inv_sigma;

    half8 pv[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top_y = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t w = d.kp[j][r];
          const float y = __builtin_fmaf(kv4_scale<DT>(w), s[n][j][r], kv4_offset<DT>(w) * qs[n]);
          s[n][j][r] = y;
          if (MASK) top_y = fmaxf(top_y, tok + 16 * j + 4 * g + r <= limit[n] ? y : -INFINITY);
          else top_y = fmaxf(top_y, y);
        }
      }
      float x = top_y * cf[n];
      if (MASK && top_y == -INFINITY) x = -INFINITY;  // a factor of zero
      const float m_new = fmaxf(m[n], group4_max_swap(x));
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      if (__builtin_amdgcn_ballot_w64(m_new > m[n])) {
        const float alpha = fast_exp2(m[n] - m_use);
        l[n] *= alpha;
        b[n] *= alpha;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[n][i] *= alpha;
        m[n] = m_new;
      }
      const float shift = kLift - m_use;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float p = fast_exp2(__builtin_fmaf(s[n][j][r], cf[n], shift));
          float off = vb[j][r];
          if (MASK) {
            // A masked place may hold anything: neither its score nor its row enters.
            const bool seen = tok + 16 * j + 4 * g + r <= limit[n];
            p = seen ? p : 0.f;
            off = seen ? off : 0.f;
          }
          l[n] += p;
          b[n] = __builtin_fmaf(p, off, b[n]);
          pv[n][4 * j + r] = static_cast<_Float16>(p * vs[j][r]);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const half8 a = v_operand(d.v[0][w], d.v[1][w], odd ? 0x00F000F0u : 0x000F000Fu);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][2 * w + odd] = mfma16x16x32(F16{}, a, pv[n], acc[n][2 * w + odd]);
      }
    }
  }

  // Unnormalised output dim (D / 4) g + (D / 16) r + i of column n.
  __device__ __forceinline__ float value(int n, int r, int i, float b_sum) const {
    return acc[n][i][r] * (sigma * ((i & 1) ? kCodeUnit / 16.f : kCodeUnit)) + b_sum;
  }
};

// Tokens [first, end) of sequence s in steps `stride` tokens apart, into w.
// Tokens from end on and past a column's limit are masked; tiles past the
// wave's last token are never looked up.
template <class DT, int D, int NT>
__device__ __forceinline__ void run_keys(Wave<DT, D, NT>& w, const Kv4AttnParams& p, int s, int kvh, int lane,
                                         int first, int end, int stride, const int (&limit)[NT], int all_see,
                                         int last) {
  if (first >= end) return;
  const int g = lane >> 4, col = lane & 15;
  const int steps = (end - first + stride - 1) / stride;
  const int tpb = p.block_size >> 4;
  const int tile_last = last >> 4;
  const int64_t bt_row = static_cast<int64_t>(s) * p.bt_stride;
  const int code_bytes = p.block_size * (D / 2);
  const int k_off = col * (D / 2) + g * (D / 8), v_off = g * (2 * D) + col * (D / 8), p_off = g * 16;
  Window win;
  auto fill = [&](int i) {
    int tile = (first + (i + (lane >> 1)) * stride) / 16 + (lane & 1);
    tile = tile < tile_last ? tile : tile_last;
    const int at = tile / tpb, in = tile - at * tpb;
    int64_t id = load_index(p.bt, bt_row + at, p.bt64);
    const bool bad = id < 0 || id >= p.num_blocks;
    id = bad ? 0 : id;
    const int64_t off = (id * p.num_kv_heads + kvh) * p.record + in * (8 * D);
    win.lo = static_cast<uint32_t>(off);
    win.hi = static_cast<uint32_t>(off >> 32);
    win.par = (code_bytes + in * (64 - 8 * D)) | (bad ? 1 : 0);
  };
  auto load = [&](Step<D>& d, int i) {
    if ((i & 31) == 0) fill(i);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int from = 2 * (i & 31) + j;
      const uint64_t off = (static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(win.hi), from))) << 32) |
                           static_cast<uint32_t>(lane_value(static_cast<int>(win.lo), from));
      const int par = lane_value(win.par, from);
      const char* kb = p.k_cache + off;
      const char* vb = p.v_cache + off;
      load_words(d.k[j], kb + k_off);
      load_words(d.v[j], vb + v_off);
      d.kp[j] = *reinterpret_cast<const u32x4*>(kb + (par & ~1) + p_off);
      d.vp[j] = *reinterpret_cast<const u32x4*>(vb + (par & ~1) + p_off);
      if (par & 1) {  // a block outside the cache: every row of it is NaN
        const uint32_t nan = Half<DT>::nan;
        d.kp[j] = u32x4{nan, nan, nan, nan};
        d.vp[j] = u32x4{0u, 0u, 0u, 0u};
      }
    }
  };
  auto compute = [&](const Step<D>& d, int i) {
    const int tok = first + i * stride;
    if (tok + 31 <= all_see && tok + 32 <= end) w.template step<false>(d, tok, g, limit, last);
    else w.template step<true>(d, tok, g, limit, last);
  };
  Step<D> a, b;
  load(a, 0);
  for (int i = 0; i < steps; i += 2) {
    if (i + 1 < steps) load(b, i + 1);
    compute(a, i);
    if (i + 1 < steps) {
      if (i + 2 < steps) load(a, i + 2);
      compute(b, i + 1);
    }
  }
}

// A column's D / 4 consecutive results of this lane, as the output's dtype.
template <class DT, int D>
__device__ __forceinline__ void store_row(char* dst, const float (&x)[D / 4]) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = Half<DT>::from_f32(x[8 * i + 2 * e]) | (Half<DT>::from_f32(x[8 * i + 2 * e + 1]) << 16);
    *reinterpret_cast<u32x4*>(dst + 16 * i) = v;
  }
}

// Rows of one-row sequences: a workgroup takes a range of one (sequence, KV
// head)'s keys for the group's query heads (up to 16 columns), its four waves
// every fourth step of it, and merges the four states through LDS.
template <class DT, int D>
__global__ __launch_bounds__(256) void kv4_decode_kernel(Kv4AttnParams p) {
  __shared__ float sm[4][16], sl[4][16];
  __shared__ float so[4][16][D + 4];  // the four floats keep the 16 columns' stores on different banks
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int pairs = p.num_seqs * p.num_kv_heads;
  const int range = blockIdx.x / pairs, pair = blockIdx.x - range * pairs;
  const int s = pair / p.num_kv_heads, kvh = pair - s * p.num_kv_heads;
  const Rows rows = rows_of(p, s);
  if (rows.ql != 1) return;
  const int len = static_cast<int>(rows.len);
  const int t0 = range * p.split;
  if (t0 >= len && range > 0) return;  // the merge reads ranges that hold keys
  const int t1 = p.nsplit > 1 && len - t0 > p.split ? t0 + p.split : len;

  Wave<DT, D, 1> w;
  w.init();
  const int head = kvh * p.group + (col < p.group ? col : p.group - 1);
  w.load_query(0, p.query + (rows.row0 * p.num_heads + head) * (D * 2), g, p.scale);
  const int limit[1] = {t1 - 1};
  run_keys(w, p, s, kvh, lane, t0 + 32 * wave, t1, 128, limit, t1 - 1, len - 1);
  const float l = group4_sum(w.l[0]), b = group4_sum(w.b[0]);
  if (g == 0) {
    sm[wave][col] = w.m[0];
    sl[wave][col] = l;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
#pragma unroll
    for (int i = 0; i < D / 16; i += 4) {
      floatx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = w.value(0, r, i + e, b);
      *reinterpret_cast<floatx4*>(&so[wave][col][(D / 4) * g + (D / 16) * r + i]) = v;
    }
  }
  __syncthreads();

  // Column threadIdx.x / 16, D / 16 dims of it.
  const int c = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16);
  if (c >= p.group) return;
  float m = fmaxf(fmaxf(sm[0][c], sm[1][c]), fmaxf(sm[2][c], sm[3][c]));
  const float m_use = m == -INFINITY ? 0.f : m;
  float sum = 0.f, o[D / 16];
#pragma unroll
  for (int e = 0; e < D / 16; ++e) o[e] = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float f = fast_exp2(sm[v][c] - m_use);
    sum = __builtin_fmaf(f, sl[v][c], sum);
#pragma unroll
    for (int e = 0; e < D / 16; ++e) o[e] = __builtin_fmaf(f, so[v][c][d0 + e], o[e]);
  }
  const int64_t h = kvh * p.group + c;
  if (p.nsplit > 1) {
    const int64_t at = (static_cast<int64_t>(s) * p.num_heads + h) * p.nsplit + range;
    if (d0 == 0) {
      p.part_m[at] = m;
      p.part_l[at] = sum;
    }
#pragma unroll
    for (int e = 0; e < D / 16; ++e) p.part_o[at * D + d0 + e] = o[e];
  } else {
    const float inv = sum > 0.f ? 1.f / sum : sum;  // no key: zero; a NaN stays one
    uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (rows.row0 * p.num_heads + h) * D + d0;
#pragma unroll
    for (int e = 0; e < D / 16; e += 2)
      *reinterpret_cast<uint32_t*>(dst + e) =
          Half<DT>::from_f32(o[e] * inv) | (Half<DT>::from_f32(o[e + 1] * inv) << 16);
  }
}

// Rows of longer queries: a wave takes 16 NT flattened (query row, head) columns
// of one (sequence, KV head) over a range of its keys; the workgroup's four
// waves lie side by side and walk the same keys, which the first of them to
// come brings into the cache.  No wave waits for another.
template <class DT, int D, int NT>
__global__ __launch_bounds__(256) void kv4_columns_kernel(Kv4AttnParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int pairs = p.num_seqs * p.num_kv_heads;
  const int part = blockIdx.x / pairs, pair = blockIdx.x - part * pairs;
  const int block = part / p.nsplit, range = part - block * p.nsplit;
  const int s = pair / p.num_kv_heads, kvh = pair - s * p.num_kv_heads;
  const Rows rows = rows_of(p, s);
  const int ql = static_cast<int>(rows.ql), len = static_cast<int>(rows.len);
  if (ql < (p.every_row ? 1 : 2)) return;
  const int cols = ql * p.group;
  // The last columns, which see the most keys, first.
  const int blocks = (cols + 64 * NT - 1) / (64 * NT);
  if (block >= blocks) return;
  const int base = ((blocks - 1 - block) * 4 + wave) * (16 * NT);
  if (base >= cols) return;
  const int end_col = base + 16 * NT < cols ? base + 16 * NT : cols;
  const int all_see = len - ql + base / p.group;               // the first column's last key
  const int last = len - ql + (end_col - 1) / p.group;         // the last column's
  const int t0 = range * p.split;
  if (t0 > last && range > 0) return;  // the merge reads ranges that hold keys
  int t1 = last + 1;
  if (p.nsplit > 1 && t1 - t0 > p.split) t1 = t0 + p.split;

  Wave<DT, D, NT> w;
  w.init();
  int limit[NT];
  int64_t row[NT];
  int head[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    int f = base + 16 * n + col;
    f = f < cols ? f : cols - 1;  // a column past the last repeats it and is not stored
    const int j = f / p.group;
    row[n] = rows.row0 + j;
    head[n] = kvh * p.group + (f - j * p.group);
    limit[n] = len - ql + j;
    w.load_query(n, p.query + (row[n] * p.num_heads + head[n]) * (D * 2), g, p.scale);
  }
  run_keys(w, p, s, kvh, lane, t0, t1, 32, limit, all_see, last);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float l = group4_sum(w.l[n]), b = group4_sum(w.b[n]);
    if (base + 16 * n + col >= cols) continue;
    float x[D / 4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < D / 16; ++i) x[(D / 16) * r + i] = w.value(n, r, i, b);
    const int64_t at = row[n] * p.num_heads + head[n];
    if (p.nsplit > 1) {
      if (g == 0) {
        p.part_m[at * p.nsplit + range] = w.m[n];
        p.part_l[at * p.nsplit + range] = l;
      }
      float* dst = p.part_o + (at * p.nsplit + range) * D + g * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 4; i += 4)
        *reinterpret_cast<floatx4*>(dst + i) = floatx4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    } else {
      const float inv = l > 0.f ? 1.f / l : l;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) x[i] *= inv;
      store_row<DT, D>(p.out + (at * D + g * (D / 4)) * 2, x);
    }
  }
}

// Joins the ranges of a row, in order: one wave per (row, query head).  DECODE:
// row r of the partials is sequence r's only row; else it is query row r.
template <class DT, int D, bool DECODE>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Kv4AttnParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = at / p.num_heads;
  int s = static_cast<int>(r);
  if (DECODE) {
    if (s >= p.num_seqs) return;
  } else {
    if (r >= p.num_tokens) return;
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (load_index(p.qsl, mid, p.qsl64) <= r) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
  }
  const Rows rows = rows_of(p, s);
  int64_t keys = rows.len;
  int64_t row = rows.row0;
  if (DECODE) {
    if (rows.ql != 1) return;
  } else {
    if (r < rows.row0 || r >= rows.row0 + rows.ql || rows.ql < (p.every_row ? 1 : 2)) return;
    row = r;
    keys = rows.len - rows.ql + (r - rows.row0) + 1;
  }
  const int n = keys <= 0 ? 0 : static_cast<int>((keys + p.split - 1) / p.split);
  const float* pm = p.part_m + at * p.nsplit;
  const float* pl = p.part_l + at * p.nsplit;
  const float* po = p.part_o + at * p.nsplit * D;
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, pm[i]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  const float m_use = m == -INFINITY ? 0.f : m;
  float sum = 0.f, o[D / 64];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float f = fast_exp2(pm[i] - m_use);
    sum = __builtin_fmaf(f, pl[i], sum);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = __builtin_fmaf(f, po[static_cast<int64_t>(i) * D + (D / 64) * lane + e], o[e]);
  }
  const float inv = sum > 0.f ? 1.f / sum : sum;
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (row * p.num_heads + (at - r * p.num_heads)) * D + (D / 64) * lane;
  if constexpr (D == 64) {
    *dst = static_cast<uint16_t>(Half<DT>::from_f32(o[0] * inv));
  } else {
    *reinterpret_cast<uint32_t*>(dst) = Half<DT>::from_f32(o[0] * inv) | (Half<DT>::from_f32(o[1] * inv) << 16);
  }
}

// How a call is cut.  Host arithmetic on sizes only.
struct Cut {
  bool fast, decode, columns;     // matrix-core kernels; which of them
  bool every_row;
  int nt;                         // column tiles per wave
  int dec_split, dec_n;           // tokens per range and ranges of one-row sequences
  int col_split, col_n;           // ... of longer queries
  int64_t col_blocks;             // column blocks of the longest query
  size_t dec_bytes, col_bytes;    // partials
};

int round_up(int64_t x, int to) { return static_cast<int>((x + to - 1) / to * to); }

Cut cut_of(int num_seqs, int64_t num_tokens, int max_query_len, int max_seq_len, int64_t context, int decode_only,
           int num_heads, int num_kv_heads, int head_dim, int block_size) {
  Cut c = {};
  c.fast = (head_dim == 64 || head_dim == 128) && block_size % 16 == 0;
  if (!c.fast) return c;
  const int group = num_heads / num_kv_heads;
  c.every_row = group > 16;
  c.decode = !c.every_row;
  c.columns = !decode_only || c.every_row;
  c.nt = 2;
  const int longest = max_seq_len > 0 ? max_seq_len : 1;
  const int64_t all = static_cast<int64_t>(num_seqs) * longest;
  const int64_t tokens = (context > 0 && context < all ? context : all) * num_kv_heads;
  const int row_bytes = (head_dim + 2) * 4;
  if (c.decode) {
    c.dec_split = round_up(tokens / 1024, 128);
    c.dec_split = c.dec_split < 256 ? 256 : c.dec_split;
    c.dec_n = (longest + c.dec_split - 1) / c.dec_split;
    c.dec_bytes = c.dec_n > 1 ? static_cast<size_t>(num_seqs) * num_heads * c.dec_n * row_bytes : 0;
  }
  if (c.columns) {
    const int ql = decode_only ? 1 : max_query_len;
    c.col_blocks = (static_cast<int64_t>(ql) * group + 64 * c.nt - 1) / (64 * c.nt);
    // Workgroups that there are at most, by the rows of the batch.
    int64_t groups = num_tokens * group / (64 * c.nt);
    groups = (groups < 1 ? 1 : groups) * num_kv_heads;
    int64_t want = 512 / groups;
    want = want < 1 ? 1 : want;
    c.col_split = round_up((longest + want - 1) / want, 32);
    c.col_split = c.col_split < 256 ? 256 : c.col_split;
    c.col_n = (longest + c.col_split - 1) / c.col_split;
    c.col_bytes = c.col_n > 1 ? static_cast<size_t>(num_tokens) * num_heads * c.col_n * row_bytes : 0;
  }
  return c;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

hipError_t launch(const void* fn, int64_t blocks, Kv4AttnParams& p, hipStream_t st) {
  if (blocks <= 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  void* args[] = {&p};
  return hipLaunchKernel(fn, dim3(static_cast<unsigned>(blocks)), dim3(256), args, 0, st);
}

template <class DT, int D>
hipError_t launch_fast(Kv4AttnParams p, const Cut& c, char* workspace, hipStream_t st) {
  const int64_t pairs = static_cast<int64_t>(p.num_seqs) * p.num_kv_heads;
  auto partials = [&](char* at, int64_t rows, int n) {
    const int64_t cells = rows * p.num_heads * n;
    p.part_o = reinterpret_cast<float*>(at);
    p.part_m = p.part_o + cells * D;
    p.part_l = p.part_m + cells;
  };
  hipError_t e = hipSuccess;
  if (c.columns) {
    p.nsplit = c.col_n;
    p.split = c.col_split;
    p.every_row = c.every_row ? 1 : 0;
    partials(workspace + align256(c.dec_bytes), p.num_tokens, c.col_n);
    e = launch(reinterpret_cast<const void*>(&kv4_columns_kernel<DT, D, 2>), pairs * c.col_blocks * c.col_n, p, st);
    if (e == hipSuccess && c.col_n > 1)
      e = launch(reinterpret_cast<const void*>(&kv4_merge_kernel<DT, D, false>), (p.num_tokens * p.num_heads + 3) / 4, p, st);
    if (e != hipSuccess) return e;
  }
  if (c.decode) {
    p.nsplit = c.dec_n;
    p.split = c.dec_split;
    partials(workspace, p.num_seqs, c.dec_n);
    e = launch(reinterpret_cast<const void*>(&kv4_decode_kernel<DT, D>), pairs * c.dec_n, p, st);
    if (e == hipSuccess && c.dec_n > 1)
      e = launch(reinterpret_cast<const void*>(&kv4_merge_kernel<DT, D, true>),
                 (static_cast<int64_t>(p.num_seqs) * p.num_heads + 3) / 4, p, st);
  }
  return e;
}

bool misaligned(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

}  // namespace
}  // namespace ns

extern "C" size_t ns_paged_attention_int4_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                                        int block_size, int max_seq_len, int max_query_len,
                                                        int64_t num_tokens, int64_t context_tokens,
                                                        int is_decode_only) {
  using namespace ns;
  if (num_seqs <= 0 || num_tokens <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      max_seq_len < 0 || !kv4_shape_ok(head_dim, block_size))
    return 0;
  const Cut c = cut_of(num_seqs, num_tokens, max_query_len, max_seq_len, context_tokens, is_decode_only, num_heads,
                       num_kv_heads, head_dim, block_size);
  return align256(c.dec_bytes) + align256(c.col_bytes);
}

extern "C" int ns_paged_attention_int4(void* out, const void* query,
                                       const void* k_cache, const void* v_cache,
                                       const void* block_tables, int64_t block_table_stride,
                                       int64_t block_table_width, int block_tables_is_int64,
                                       const void* seq_lens, int seq_lens_is_int64,
                                       const void* query_start_loc, int query_start_loc_is_int64,
                                       int num_seqs, int64_t num_tokens, int max_query_len, int max_seq_len,
                                       int64_t context_tokens, int is_decode_only,
                                       int num_heads, int num_kv_heads, int head_dim,
                                       int block_size, int64_t num_blocks,
                                       float scale, int dtype,
                                       void* workspace, size_t workspace_bytes, void* stream) {
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
  // Rows, heads and columns are counted in 32 bits.
  if (num_heads > 65535 || num_tokens > 0x7FFFFFFF / num_heads || num_seqs > 0x7FFFFFFF / num_heads)
    return NS_ERR_UNSUPPORTED;
  const Cut cut = cut_of(num_seqs, num_tokens, max_query_len, max_seq_len, context_tokens, is_decode_only, num_heads,
                         num_kv_heads, head_dim, block_size);
  const size_t need = align256(cut.dec_bytes) + align256(cut.col_bytes);
  if (need > 0 && (!workspace || workspace_bytes < need || misaligned(workspace, 256))) return NS_ERR_WORKSPACE;
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
  const int64_t table = block_table_width * static_cast<int64_t>(block_size);
  p.max_ctx = max_seq_len < table ? max_seq_len : table;
  p.scale = scale;
  p.nsplit = 1;
  p.split = 0;
  p.every_row = 0;
  p.part_m = p.part_l = p.part_o = nullptr;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e;
  if (!cut.fast) {
    e = dtype == NS_DTYPE_F16 ? launch_generic<F16>(p, st) : launch_generic<BF16>(p, st);
  } else {
    char* ws = static_cast<char*>(workspace);
    if (dtype == NS_DTYPE_F16)
      e = head_dim == 64 ? launch_fast<F16, 64>(p, cut, ws, st) : launch_fast<F16, 128>(p, cut, ws, st);
    else
      e = head_dim == 64 ? launch_fast<BF16, 64>(p, cut, ws, st) : launch_fast<BF16, 128>(p, cut, ws, st);
  }
  return e == hipSuccess ? NS_OK : NS_ERR_HIP;
}
