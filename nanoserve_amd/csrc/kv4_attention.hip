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

// A context's keys are cut into ranges of `tokens` (a multiple of 32), up to n of
// them.  Where there is more than one, m, range i of row j and head h of the
// sequence leaves its maximum (log2 units), sum and unnormalised output at index
// first * num_heads + (j * num_heads + h) * m + i of the three: a sequence has
// rows * m cells of num_heads results, and only sequences that are split have
// any, from `first` on.  There are `cells` of them.  The lengths that were
// expected need no more; where the device's would, every workgroup takes ranges
// twice as long until they fit, and the join is told.
struct Place {
  int first, tokens;
};
struct Ranges {
  int n, tokens, cells;
  float* maxima;
  float* sums;
  float* outputs;
  Place* places;  // [num_seqs], of the sequences of the part; where n > 1

  // Ranges of a context: one where it is empty or nothing is split.
  __device__ __forceinline__ int of(int len, int each) const {
    return n == 1 || len <= each ? 1 : (len + each - 1) / each;
  }
};
constexpr int kManyCells = 1 << 24;  // more than any workspace has; sums of 64 stay within 32 bits
__device__ __forceinline__ int cells_of(int ql, int ranges) {
  const int64_t n = static_cast<int64_t>(ql) * ranges;
  return ranges == 1 ? 0 : n < kManyCells ? static_cast<int>(n) : kManyCells;
}

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
  // Matrix-core kernels.
  Ranges one, more;       // of one-row sequences; of longer queries
  int every_row;          // the column part takes one-row sequences too
  int column_groups;      // workgroups of the column part, in front of the others
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

// The sequence of query row t: the last s with query_start_loc[s] <= t, where there
// are offsets (a decode-only batch has none: its rows are its sequences).
__device__ __forceinline__ int sequence_of(const Kv4AttnParams& p, int64_t t) {
  if (p.decode_only) return static_cast<int>(t);
  int lo = 0, hi = p.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (load_index(p.qsl, mid, p.qsl64) <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
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

  const int s = sequence_of(p, t);
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
// S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16, 32 tokens a step.  Codes
// and parameter words arrive in LDS by LDS-DMA, which holds no registers in
// flight: into a ring of each wave's own (one-row sequences; no wave waits for
// another) or into chunks that a workgroup shares (longer queries).  A lane's part
// of a tile is one LDS read (8 or 16 bytes), and a mask turns its words into
// operands (kv4.h).  Both model dtypes run in float16: the codes are exact there, the query is brought
// into its range by a power of two for the columns that share a workgroup: the
// largest element becomes 2^14 at least (of 2^-86 and more), so all are exact but
// those below 2^-24 of it in odd dims, which are stored as a sixteenth, and below
// 2^-28 in even ones; their error is at most 2^-35 of it.  (bfloat16 rows beyond
// 2^16 are divided by a power of their own besides, and the largest becomes 2^13
// at least: 2^-23, 2^-27 and 2^-34 of a row's own largest.)  The
// probabilities keep 11 bits where bfloat16 would keep 8.
//
// A score in log2 units is two fused multiply-adds, s_t (q.c_t) + (b_t sum(q) -
// reference), with the softmax scale in s_t and b_t: the reference is the
// maximum of an earlier step, and only when some score of a step passes it by
// 2^8 is the column's maximum taken over its lanes and the reference moved.
// The operand of the second product is p s_t, rounded once to float16: s_t is
// divided by a power of two above the largest scale that the wave has met (the
// accumulators follow when that grows, exactly), so a product lies below 2^14
// and keeps its 11 bits down to 2^-20 of the largest.  sum p and sum p (b_t +
// 8 s_t) are float32, and one more product, with a tile of eights, gives 8 times
// the sum of the rounded p s_t to take off again: a rounding then acts on a code's
// distance from the middle, half as far as its distance from 0.
//
// Bound: one-row sequences by the cache's stream (64 contexts around 4K, four KV
// heads of 128: 53 us, 4.0 TB/s of codes and parameters) or, where that is short, by
// the chain of lengths, block ids and tiles; longer queries by vector issue, 80% of
// the cycles at head size 128: ~205 operations and 16 exponentials a step of 32
// columns, 80 of them unpacking, beside 34 matrix products (35%).
//
// The result layout of the first product, tokens 4 g + r of column lane % 16 in
// lane group g, is the operand layout of the second.

// A step's place in the ring: codes of two tiles of K, of V, then the parameter
// words of both tiles of K and of V.
template <int D>
struct Slot {
  static constexpr int v = 16 * D, par = 32 * D, bytes = 32 * D + 256;
  static constexpr int loads = D == 128 ? 5 : 3;  // vector memory operations that fill it
};

using floatx2 = float __attribute__((ext_vector_type(2)));

// A step's parameters as float32: lane l makes the two of token l % 32 of K
// (l < 32) or V, and each lane reads back those of tokens 4 g .. 4 g + 3 of both
// tiles.  (Each lane converting the eight words that it needs itself was 72 of
// the ~330 vector instructions of a step of 32 columns.)
struct alignas(16) Params {
  float of[64][2];  // K: s_t, b_t in log2 units; V (from 32 on): s_t, b_t + 8 s_t
};

// A lane's words of the two tiles of K or V.
template <int D>
struct Tiles {
  uint32_t w[2][D / 32];

  // code_off: the lane's bytes in a tile.
  __device__ __forceinline__ void read_codes(const char* codes, int code_off) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const char* at = codes + j * (8 * D) + code_off;
      if constexpr (D == 64) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(at);
        w[j][0] = x[0];
        w[j][1] = x[1];
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j][i] = x[i];
      }
    }
  }
};

// Where the wave's tiles lie: lane l holds tile l & 1 of step l / 2 of a window
// of 32 steps, as the addresses of its codes in K and V and, from there, the
// distance to its parameter words.
struct Window {
  uint32_t k_lo, k_hi, v_lo, v_hi;
  int par;
};

__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ const char* lane_pointer(uint32_t lo, uint32_t hi, int lane) {
  return reinterpret_cast<const char*>(
      (static_cast<uint64_t>(static_cast<uint32_t>(lane_value(static_cast<int>(hi), lane))) << 32) |
      static_cast<uint32_t>(lane_value(static_cast<int>(lo), lane)));
}
// Until at most N of the wave's vector memory operations are pending.
template <int N>
__device__ __forceinline__ void vector_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// What a block id outside the cache reads instead: rows of K that are NaN (an
// offset of NaN, so every score with them is), rows of V without any.
constexpr int kPageWords = 512;  // a tile's codes at head size 128 are 1 KiB, parameters start at 0
struct Page {
  uint32_t w[kPageWords];
};
constexpr Page page_of(uint32_t x) {
  Page p = {};
  for (int i = 0; i < kPageWords; ++i) p.w[i] = x;
  return p;
}
__device__ const Page kNanF16 = page_of(Half<F16>::nan);
__device__ const Page kNanBF16 = page_of(Half<BF16>::nan);
__device__ const Page kZeros = page_of(0);

// The wave's largest, on every lane.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t w) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) w = max(w, static_cast<uint32_t>(__shfl_xor(static_cast<int>(w), off)));
  return w;
}

constexpr float kCodeUnit = 16777216.f;  // 2^24: an even dim's code as a half's bits is code / 2^24
// p is kept relative to a reference that is at most kSlack binades below the
// column's running maximum and lifted by kLift, so that the largest lies in
// [2^kLift, 2^(kLift + kSlack)] and fits a half: the reference (and with it the
// accumulators) moves only when a score passes it by that much.
constexpr float kLift = 6.f, kSlack = 8.f;
constexpr float kEven = 65536.f;  // more than any float16

// One wave's state: NT tiles of 16 columns, D output dims each.
template <class DT, int D, int NT>
struct Wave {
  half8 q[NT][D / 32];
  float cf;                   // log2 units per score unit
  float qs[NT];               // sum(q) in score units
  float m[NT], ref[NT];       // reference (log2 units); kLift - reference
  float l[NT], b[NT];         // sum p (this lane's tokens), sum p (b_t + 8 s_t) (likewise)
  floatx4 acc[NT][D / 16];
  floatx4 mid[NT];            // the same of a dim whose every code is 8
  bool uneven;                // some column's q was divided by far[column], in LDS, beforehand
  const float* far;
  float sigma, inv_sigma;     // the scales' power of two
  uint32_t top;               // largest parameter word that needs no larger sigma

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      ref[n] = INFINITY;
      l[n] = b[n] = 0.f;
      mid[n] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[n][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    }
    sigma = inv_sigma = 1.f;
    top = 0xFFFFu;
  }

  // The columns' query rows, as the operands that meet the codes: lane group g
  // holds dims (D / 4) g .. + D / 4, eight of them per 32-dim step in the order
  // of a word's masked nibbles, odd dims a sixteenth of their value.
  // all: the largest of those who share parameters, from this wave's.  spare: 16 NT
  // floats of LDS, this wave's.
  template <class All>
  __device__ __forceinline__ void load_queries(const char* const (&row)[NT], int g, float scale, float* spare,
                                               All all) {
    // Without their signs, halves are ordered as their bits are.
    using u16x2 = unsigned short __attribute__((ext_vector_type(2)));
    uint32_t x[NT][D / 8];
    u16x2 bits = {0, 0};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const u32x4 r = *reinterpret_cast<const u32x4*>(row[n] + (g * (D / 4) + 8 * w) * 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[n][4 * w + e] = r[e];
          bits = __builtin_elementwise_max(bits, __builtin_bit_cast(u16x2, r[e] & 0x7FFF7FFFu));
        }
      }
    }
    uint32_t most = max(static_cast<uint32_t>(bits[0]), static_cast<uint32_t>(bits[1]));
    const uint32_t inf = DT::code == NS_DTYPE_F16 ? 0x7C00u : 0x7F80u;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(most >= inf) != 0, 0)) {
      most = 0;  // of the finite elements
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const uint32_t lo = x[n][i] & 0x7FFFu, hi = (x[n][i] >> 16) & 0x7FFFu;
          most = max(most, max(lo < inf ? lo : 0u, hi < inf ? hi : 0u));
        }
      }
    }
    float big = Half<DT>::to_f32(most);
    // A bfloat16 query may hold a row so large that the others would vanish beside
    // it in float16: columns past kEven are divided by a power of two of their own,
    // which their scores are given back.
    uneven = false;
    far = spare;
    if constexpr (DT::code != NS_DTYPE_F16) {
      uneven = __builtin_amdgcn_ballot_w64(big > kEven) != 0;
      if (__builtin_expect(uneven, 0)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const uint32_t lo = x[n][i] & 0x7FFFu, hi = (x[n][i] >> 16) & 0x7FFFu;
            top = max(top, max(lo < inf ? lo : 0u, hi < inf ? hi : 0u));
          }
          top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
          top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
          const float above = Half<DT>::to_f32(top) * (2.f / kEven);
          const float by = above > 2.f ? __uint_as_float(__float_as_uint(above) & 0x7F800000u) : 1.f;
          spare[16 * n + (threadIdx.x & 15)] = by;  // the same from a column's four lanes
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            const float lo = Half<DT>::to_f32(x[n][i] & 0xFFFFu) / by, hi = Half<DT>::to_f32(x[n][i] >> 16) / by;
            x[n][i] = Half<DT>::from_f32(lo) | (Half<DT>::from_f32(hi) << 16);
          }
        }
        big = fminf(big, kEven);
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor(big, off));
    big = all(big);
    // The largest finite element (or kEven) becomes 2^14 .. 2^15.
    int e = 14 - (static_cast<int>(__float_as_uint(big) >> 23) - 127);
    e = e < -113 ? -113 : e > 100 ? 100 : e;
    float f = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    cf = fabsf(scale) * 1.4426950408889634f * (kCodeUnit / f);
    if (scale < 0.f) f = -f;  // a negative scale turns the query around, exactly
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = Half<DT>::to_f32(x[n][4 * w + i] & 0xFFFFu) * f;
          v[2 * i + 1] = Half<DT>::to_f32(x[n][4 * w + i] >> 16) * f;
          sum += v[2 * i] + v[2 * i + 1];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float unit = (i & 1) ? 0.0625f : 1.f;
          q[n][w][2 * i] = static_cast<_Float16>(v[i] * unit);
          q[n][w][2 * i + 1] = static_cast<_Float16>(v[i + 4] * unit);
        }
      }
      qs[n] = group4_sum(sum) * (1.f / kCodeUnit);
      if (DT::code != NS_DTYPE_F16 && __builtin_expect(uneven, 0)) qs[n] *= far[16 * n + (threadIdx.x & 15)];
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
    w = wave_max_u32(w);
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
    for (int n = 0; n < NT; ++n) {
      mid[n] *= ratio;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[n][i] *= ratio;
    }
  }

  // Makes a slot's parameters; its tokens from `valid` on are nobody's.
  __device__ __forceinline__ void convert(char* slot, Params& params, int lane, int valid) const {
    uint32_t& at = *reinterpret_cast<uint32_t*>(slot + Slot<D>::par + lane * 4);
    uint32_t word = at;
    const bool of_v = lane >= 32;
    if (valid < 32) {
      if ((lane & 31) >= valid) word = 0;
      at = word;
    }
    const float sc = kv4_scale<DT>(word), of = kv4_offset<DT>(word);
    *reinterpret_cast<floatx2*>(params.of[lane]) =
        floatx2{of_v ? sc : sc * cf, of_v ? __builtin_fmaf(8.f, sc, of) : of * cf};
  }

  // One step over tokens tok .. tok + 31.  MASK: some column does not see all of
  // them; column n sees tokens up to limit[n].
  template <bool MASK>
  __device__ __forceinline__ void step(const char* slot, const Params& params, int lane, int tok, int g,
                                       const int (&limit)[NT]) {
    Tiles<D> k, v;
    const uint32_t big = *reinterpret_cast<const uint32_t*>(slot + Slot<D>::par + 128 + (lane & 31) * 4);
    // K for D = 128 and V lie in lane order; a tile of K at D = 64 row after row.
    k.read_codes(slot, D == 128 ? lane * 16 : (lane & 15) * 32 + g * 8);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(big > top) != 0, 0)) raise_sigma(big);
    floatx4 s[NT][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][j] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const half8 a = k_operand(k.w[j][w]);
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][j] = mfma16x16x32(F16{}, a, q[n][w], s[n][j]);
      }
    }
    floatx4 ks[2], kb[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int at = 16 * j + 4 * g;
      const floatx4 a = *reinterpret_cast<const floatx4*>(params.of[at]);
      const floatx4 b = *reinterpret_cast<const floatx4*>(params.of[at + 2]);
      ks[j] = floatx4{a[0], a[2], b[0], b[2]};
      kb[j] = floatx4{a[1], a[3], b[1], b[3]};
    }

    float x[NT][2][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      auto seen = [&](int j, int r) { return !MASK || tok + 16 * j + 4 * g + r <= limit[n]; };
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[n][j][r] = __builtin_fmaf(ks[j][r], s[n][j][r], __builtin_fmaf(kb[j][r], qs[n], ref[n]));
          most = fmaxf(most, seen(j, r) ? x[n][j][r] : -INFINITY);
        }
      }
      const bool anew = __builtin_amdgcn_ballot_w64(most > kLift + kSlack) != 0 ||
                        (DT::code != NS_DTYPE_F16 && uneven);  // whose scores are made here alone
      if (__builtin_expect(anew, 0)) {
        const float by = DT::code != NS_DTYPE_F16 && uneven ? far[16 * n + (lane & 15)] : 1.f;
        most = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[n][j][r] = __builtin_fmaf(ks[j][r], s[n][j][r] * by, kb[j][r] * qs[n]);
            most = fmaxf(most, seen(j, r) ? x[n][j][r] : -INFINITY);
          }
        }
        const float m_new = fmaxf(m[n], group4_max_swap(most));
        const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m[n] - m_new);
        l[n] *= alpha;
        b[n] *= alpha;
        mid[n] *= alpha;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[n][i] *= alpha;
        m[n] = m_new;
        ref[n] = kLift - m_new;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[n][j][r] += ref[n];
      }
    }
    floatx4 vs[2], vb[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int at = 32 + 16 * j + 4 * g;
      const floatx4 a = *reinterpret_cast<const floatx4*>(params.of[at]);
      const floatx4 b = *reinterpret_cast<const floatx4*>(params.of[at + 2]);
      vs[j] = floatx4{a[0], a[2], b[0], b[2]} * inv_sigma;
      vb[j] = floatx4{a[1], a[3], b[1], b[3]};
    }
    half8 pv[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      auto seen = [&](int j, int r) { return !MASK || tok + 16 * j + 4 * g + r <= limit[n]; };
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // A masked place may hold anything: neither its score nor its row enters.
          const float p = seen(j, r) ? fast_exp2(x[n][j][r]) : 0.f;
          l[n] += p;
          b[n] = __builtin_fmaf(p, seen(j, r) ? vb[j][r] : 0.f, b[n]);
          pv[n][4 * j + r] = static_cast<_Float16>(p * (seen(j, r) ? vs[j][r] : 0.f));
        }
      }
    }
    v.read_codes(slot + Slot<D>::v, lane * (D / 8));
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const half8 eights = __builtin_bit_cast(half8, u32x4{0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u});
      mid[n] = mfma16x16x32(F16{}, eights, pv[n], mid[n]);
    }
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {
        const half8 a = v_operand(v.w[0][w], v.w[1][w], odd ? 0x00F000F0u : 0x000F000Fu);
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n][2 * w + odd] = mfma16x16x32(F16{}, a, pv[n], acc[n][2 * w + odd]);
      }
    }
  }

  // Unnormalised output dim (D / 4) g + (D / 16) r + i of column n.
  __device__ __forceinline__ float value(int n, int r, int i, float b_sum) const {
    const float code = (i & 1) ? acc[n][i][r] * 0.0625f : acc[n][i][r];
    // Two factors: sigma * kCodeUnit may pass float32's range where neither product does.
    return __builtin_fmaf((code - mid[n][r]) * kCodeUnit, sigma, b_sum);
  }
};

// Brings the steps first, first + stride, ... of one (sequence, KV head) into LDS.
template <class DT, int D>
struct Feed {
  const Kv4AttnParams& p;
  int s, kvh, lane, first, stride, steps, tile_last;
  Window win;

  // Tiles past tile_last are never looked up.
  __device__ __forceinline__ void fill(int i) {
    const int tpb = p.block_size >> 4;
    int tile = (first + (i + (lane >> 1)) * stride) / 16 + (lane & 1);
    tile = tile < tile_last ? tile : tile_last;
    const int at = tile / tpb, in = tile - at * tpb;
    const int64_t id = load_index(p.bt, static_cast<int64_t>(s) * p.bt_stride + at, p.bt64);
    const bool bad = id < 0 || id >= p.num_blocks;
    const int64_t off = bad ? 0 : (id * p.num_kv_heads + kvh) * p.record + in * (8 * D);
    const char* nan_page = reinterpret_cast<const char*>(DT::code == NS_DTYPE_F16 ? &kNanF16 : &kNanBF16);
    const uint64_t k = reinterpret_cast<uintptr_t>(bad ? nan_page : p.k_cache) + off;
    const uint64_t v = reinterpret_cast<uintptr_t>(bad ? reinterpret_cast<const char*>(&kZeros) : p.v_cache) + off;
    win.k_lo = static_cast<uint32_t>(k);
    win.k_hi = static_cast<uint32_t>(k >> 32);
    win.v_lo = static_cast<uint32_t>(v);
    win.v_hi = static_cast<uint32_t>(v >> 32);
    win.par = bad ? 0 : p.block_size * (D / 2) + in * (64 - 8 * D);
  }
  // Fills a slot with step i; behind the last step with the last one again, so
  // that the count of loads in flight stays what the waits expect.  Steps are
  // asked for in order.
  __device__ __forceinline__ void issue(int i, char* slot) {
    if (i < steps) {
      if ((i & 31) == 0) fill(i);
    } else {
      i = steps - 1;
    }
    const int col = lane & 15, g = lane >> 4;
    const int from = 2 * (i & 31);
    const char* k0 = lane_pointer(win.k_lo, win.k_hi, from);
    const char* k1 = lane_pointer(win.k_lo, win.k_hi, from + 1);
    const char* v0 = lane_pointer(win.v_lo, win.v_hi, from);
    const char* v1 = lane_pointer(win.v_lo, win.v_hi, from + 1);
    const int par0 = lane_value(win.par, from), par1 = lane_value(win.par, from + 1);
    if constexpr (D == 128) {
      // Every lane brings the 16 bytes that it reads: tokens of K lie 64 bytes apart.
      const uint32_t k_off = col * 64 + g * 16, v_off = lane * 16;
      dma_lds16_off(k0, k_off, slot);
      dma_lds16_off(k1, k_off, slot + 1024);
      dma_lds16_off(v0, v_off, slot + Slot<D>::v);
      dma_lds16_off(v1, v_off, slot + Slot<D>::v + 1024);
    } else {
      // Both tiles of 512 bytes in one operation, half a wave each.
      const uint32_t off = (lane & 31) * 16;
      dma_lds16((lane < 32 ? k0 : k1) + off, slot);
      dma_lds16((lane < 32 ? v0 : v1) + off, slot + Slot<D>::v);
    }
    // Lanes 0 .. 15 the first tile's words of K, then the second's, then V's.
    const char* kp = (lane & 16) ? k1 + par1 : k0 + par0;
    const char* vp = (lane & 16) ? v1 + par1 : v0 + par0;
    dma_lds4((lane < 32 ? kp : vp) + col * 4, slot + Slot<D>::par);
  }
};

// A wave by itself: tokens [first, end) of sequence s in steps `stride` tokens
// apart, into w.  Tokens from end on are masked; last is the wave's last token.
// ring: R slots of this wave's.
template <int R, class DT, int D>
__device__ __forceinline__ void run_keys(Wave<DT, D, 1>& w, const Kv4AttnParams& p, char* ring, Params& params, int s,
                                         int kvh, int lane, int first, int end, int stride, int last) {
  if (first >= end) return;
  static_assert((R & (R - 1)) == 0, "a power of two");
  const int g = lane >> 4;
  Feed<DT, D> feed = {p, s, kvh, lane, first, stride, (end - first + stride - 1) / stride, last >> 4, {}};
#pragma unroll 1
  for (int i = 0; i < R; ++i) feed.issue(i, ring + i * Slot<D>::bytes);
  const int limit[1] = {end - 1};
  int i = 0, tok = first;
  // The parameters of the step before have been read when these are written: a
  // wave's LDS operations are done in order.
  for (; tok + 32 <= end; tok += stride, ++i) {
    char* slot = ring + (i & (R - 1)) * Slot<D>::bytes;
    vector_wait<(R - 1) * Slot<D>::loads>();
    w.convert(slot, params, lane, 32);
    __builtin_amdgcn_wave_barrier();
    w.template step<false>(slot, params, lane, tok, g, limit);
    __builtin_amdgcn_wave_barrier();
    feed.issue(i + R, slot);
  }
  for (; tok < end; tok += stride, ++i) {
    char* slot = ring + (i & (R - 1)) * Slot<D>::bytes;
    vector_wait<(R - 1) * Slot<D>::loads>();
    w.convert(slot, params, lane, last + 1 - tok);
    __builtin_amdgcn_wave_barrier();
    w.template step<true>(slot, params, lane, tok, g, limit);
    __builtin_amdgcn_wave_barrier();
    feed.issue(i + R, slot);
  }
  vector_wait<0>();  // nothing lands in the ring behind its use
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

// One sequence's part of a launch: index of its work items, and its first cell.
struct Part {
  int seq, row, ql, len, index, cell;
};

// The work items of all sequences, count(query rows, ranges) each, in order, and
// the cells that those of more than one range take.  Every wave keeps the list for
// itself: lane l the sequences from l * per on, and the items up to and with
// theirs, so that an item costs one look at its lane's sequences (and, up to 64
// sequences, none).
template <class Count>
struct PartList {
  const Kv4AttnParams& p;
  const Ranges& rg;
  Count count;
  int tokens;              // of a range
  int per, upto, mine;
  int row, ql, len, cell;  // of the lane's first sequence

  __device__ __forceinline__ PartList(const Kv4AttnParams& params, const Ranges& ranges, int lane, Count c)
      : p(params), rg(ranges), count(c), tokens(ranges.tokens), per((params.num_seqs + 63) >> 6) {
    while (list(lane) > rg.cells) tokens *= 2;  // ends at the latest where no context is split
    upto = scan(mine, lane);
  }
  // Returns the cells of all sequences.
  __device__ __forceinline__ int list(int lane) {
    int cells = 0;
    mine = row = ql = len = cell = 0;
    for (int i = per - 1; i >= 0; --i) {
      const int s = lane * per + i;
      Rows r = {0, 0, 0};
      if (s < p.num_seqs) r = rows_of(p, s);
      row = static_cast<int>(r.row0);
      ql = static_cast<int>(r.ql);
      len = static_cast<int>(r.len);
      const int n = rg.of(len, tokens), items = s < p.num_seqs ? count(ql, n) : 0;
      mine += items;
      cells += items > 0 ? cells_of(ql, n) : 0;
      cells = cells < kManyCells ? cells : kManyCells;
    }
    if (rg.n == 1) return 0;
    const int sum = scan(cells, lane);
    cell = sum - cells;
    return lane_value(sum, 63);
  }
  static __device__ __forceinline__ int scan(int v, int lane) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int u = __shfl_up(v, off);
      v += lane >= off ? u : 0;
    }
    return v;
  }
  __device__ __forceinline__ int size() const { return lane_value(upto, 63); }
  // index < size().
  __device__ __forceinline__ Part find(int index, int lane) const {
    const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > index));
    index -= lane_value(upto, at) - lane_value(mine, at);
    int first = lane_value(cell, at);
    if (per == 1) return {at, lane_value(row, at), lane_value(ql, at), lane_value(len, at), index, first};
    for (int i = 0;; i += 64) {
      const int s = at * per + i + lane;
      const bool one = i + lane < per && s < p.num_seqs;
      Rows r = {0, 0, 0};
      if (one) r = rows_of(p, s);
      const int q = static_cast<int>(r.ql), n = static_cast<int>(r.len), ranges = rg.of(n, tokens);
      const int own = one ? count(q, ranges) : 0;
      const int sum = scan(own, lane);
      const int own_cells = own > 0 ? cells_of(q, ranges) : 0;
      const int cells = rg.n == 1 ? 0 : scan(own_cells, lane);
      const uint64_t hit = __builtin_amdgcn_ballot_w64(sum > index);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        return {at * per + i + l, lane_value(static_cast<int>(r.row0), l), lane_value(q, l), lane_value(n, l),
                index - (lane_value(sum, l) - lane_value(own, l)), first + lane_value(cells - own_cells, l)};
      }
      if (i + 64 >= per) return {0, 0, 0, 0, 0, 0};  // not reached: the lane has the item
      index -= lane_value(sum, 63);
      first += lane_value(cells, 63);
    }
  }
  // What the join has to know of a part, from one workgroup of its first item.
  __device__ __forceinline__ void tell(const Part& part) const {
    if (rg.n > 1 && part.index == 0 && threadIdx.x == 0) rg.places[part.seq] = Place{part.cell, tokens};
  }
};

// Rows of one-row sequences: a workgroup of W waves takes a range of one
// (sequence, KV head)'s keys for the group's query heads (up to 16 columns), its
// waves every W-th step of it, and merges their states through LDS.  It goes from
// range to range, `groups` apart in the list of all that there are, so a batch of
// unequal contexts costs no empty workgroups and ends evenly.
template <int D, int W, int R>
struct RowState {
  static constexpr int ring = R * Slot<D>::bytes;
  static_assert(ring >= 16 * (D + 4) * 4, "the outputs lie in the ring");
  float m[W][16], l[W][16], far[W][16];
  Params params[W];
  // A wave's ring, and behind its keys its unnormalised outputs: 16 columns,
  // whose stores the four floats keep on different banks.
  char rings[W][ring];
};

template <class DT, int D, int W, int R>
__device__ __forceinline__ void one_rows(const Kv4AttnParams& p, RowState<D, W, R>& lds, int first, int groups) {
  const Ranges& rg = p.one;
  auto so = [&](int wv, int c, int d) { return reinterpret_cast<float*>(lds.rings[wv]) + c * (D + 4) + d; };
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  auto ranges = [](int ql, int n) { return ql == 1 ? n : 0; };
  const PartList<decltype(ranges)> parts(p, rg, lane, ranges);
  const int items = parts.size() * p.num_kv_heads;  // the same for every wave
  for (int item = first; item < items; item += groups) {
    const int kvh = item % p.num_kv_heads;
    const Part found = parts.find(item / p.num_kv_heads, lane);
    if (kvh == 0) parts.tell(found);
    const int s = found.seq, len = found.len, range = found.index;
    const int64_t row0 = found.row;
    const int t0 = range * parts.tokens;
    const int t1 = rg.n > 1 && len - t0 > parts.tokens ? t0 + parts.tokens : len;

    Wave<DT, D, 1> w;
    w.init();
    const int head = kvh * p.group + (col < p.group ? col : p.group - 1);
    const char* const query[1] = {p.query + (row0 * p.num_heads + head) * (D * 2)};
    w.load_queries(query, g, p.scale, lds.far[wave], [](float big) { return big; });
    run_keys<R>(w, p, lds.rings[wave], lds.params[wave], s, kvh, lane, t0 + 32 * wave, t1, 32 * W, len - 1);
    const float l = group4_sum(w.l[0]), b = group4_sum(w.b[0]);
    if (g == 0) {
      lds.m[wave][col] = w.m[0];
      lds.l[wave][col] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int i = 0; i < D / 16; i += 4) {
        floatx4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = w.value(0, r, i + e, b);
        *reinterpret_cast<floatx4*>(so(wave, col, (D / 4) * g + (D / 16) * r + i)) = v;
      }
    }
    __syncthreads();

    // E dims of a column for each thread.
    constexpr int E = D / (4 * W);
    const int c = threadIdx.x / (4 * W), d0 = threadIdx.x % (4 * W) * E;
    if (c < p.group) {
      float m = -INFINITY;
#pragma unroll
      for (int v = 0; v < W; ++v) m = fmaxf(m, lds.m[v][c]);
      const float m_use = m == -INFINITY ? 0.f : m;
      float sum = 0.f, o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
      for (int v = 0; v < W; ++v) {
        const float f = fast_exp2(lds.m[v][c] - m_use);
        sum = __builtin_fmaf(f, lds.l[v][c], sum);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(f, *so(v, c, d0 + e), o[e]);
      }
      const int64_t h = kvh * p.group + c;
      const int n = rg.of(len, parts.tokens);
      if (n > 1) {
        const int64_t at = static_cast<int64_t>(found.cell) * p.num_heads + h * n + range;
        if (d0 == 0) {
          rg.maxima[at] = m;
          rg.sums[at] = sum;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) rg.outputs[at * D + d0 + e] = o[e];
      } else {
        const float inv = sum > 0.f ? 1.f / sum : sum;  // no key: zero; a NaN stays one
        uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (row0 * p.num_heads + h) * D + d0;
#pragma unroll
        for (int e = 0; e < E; e += 2)
          *reinterpret_cast<uint32_t*>(dst + e) =
              Half<DT>::from_f32(o[e] * inv) | (Half<DT>::from_f32(o[e + 1] * inv) << 16);
      }
    }
    __syncthreads();  // the next range's states go where these are read
  }
}

// A batch of one-row sequences.  Four waves: three workgroups on a compute unit
// (with four the 128 registers left for a wave spill), so up to 53 KiB of LDS
// each.  Eight where the ranges leave compute units idle.
constexpr int kDecodeGroups = 3;
template <int D>
constexpr int kDecodeRing = D == 64 ? 4 : 2;
template <class DT, int D, int W>
__global__ __launch_bounds__(64 * W, W == 4 ? kDecodeGroups : 2) void kv4_decode_kernel(Kv4AttnParams p) {
  __shared__ __align__(16) RowState<D, W, kDecodeRing<D>> lds;
  one_rows<DT>(p, lds, blockIdx.x, gridDim.x);
}

constexpr int kColumnBuffers = 2;  // of chunks; three or four are no faster

// Rows of longer queries: four waves of 16 NT flattened (query row, head) columns
// each of one (sequence, KV head), side by side over a range of its keys.  They
// walk the keys in chunks of W steps of 32 tokens, each of the W waves bringing
// and converting one step of the next chunk while all work on this one.  W = 8:
// four more waves take the second half of each chunk's steps for the same
// columns, and the two states are joined through LDS at the end.
template <int D, int NT, int W>
struct ColumnState {
  static constexpr int cells = NT * (D / 4 + 2);  // floats a lane hands over where W = 8
  struct alignas(16) Buffer {
    char slots[W][Slot<D>::bytes];
    Params params[W];
  };
  float far[W][16 * NT];
  union {
    Buffer buffers[kColumnBuffers];
    float states[W == 8 ? 4 : 1][cells * 64];
  };
};

template <int NT>
__device__ __forceinline__ int column_blocks(const Kv4AttnParams& p, int ql) {
  return (ql * p.group + 64 * NT - 1) / (64 * NT);
}
template <class DT, bool LOOP, int D, int NT, int W>
__device__ __forceinline__ void column_block(const Kv4AttnParams& p, ColumnState<D, NT, W>& lds, const Part& found,
                                             int tokens, int kvh) {
  const Ranges& rg = p.more;
  auto& buffers = lds.buffers;
  int thread = threadIdx.x;
  if (LOOP) asm volatile("" : "+v"(thread));  // nothing made of it is kept from one block to the next
  const int lane = thread & 63;
  const int wave = __builtin_amdgcn_readfirstlane(thread >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int s = found.seq, ql = found.ql, len = found.len;
  const int64_t row0 = found.row;
  const int cols = ql * p.group;
  // The last columns, which see the most keys, first.
  const int blocks = column_blocks<NT>(p, ql), ranges = rg.of(len, tokens);
  const int block = found.index / ranges, range = found.index - block * ranges;
  const int block_base = (blocks - 1 - block) * (64 * NT);
  auto last_of = [&](int end_col) { return len - ql + ((end_col < cols ? end_col : cols) - 1) / p.group; };
  const int t0 = range * tokens;
  const int block_last = last_of(block_base + 64 * NT);  // the workgroup's last key
  if (t0 > block_last && range > 0) return;              // the merge reads ranges that hold keys
  auto end_of = [&](int last) { return rg.n > 1 && last + 1 - t0 > tokens ? t0 + tokens : last + 1; };
  const int block_end = end_of(block_last);
  const int base = block_base + (wave & 3) * (16 * NT);
  const bool idle = base >= cols;  // brings keys for the others
  const int all_see = len - ql + base / p.group;  // the first column's last key
  const int last = last_of(base + 16 * NT);
  const int end = idle ? t0 : end_of(last);

  Wave<DT, D, NT> w;
  w.init();
  int limit[NT];
  int64_t row[NT];
  int head[NT];
  const char* query[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    int f = base + 16 * n + col;
    f = f < cols ? f : cols - 1;  // a column past the last repeats it and is not stored
    const int j = f / p.group;
    row[n] = row0 + j;
    head[n] = kvh * p.group + (f - j * p.group);
    limit[n] = len - ql + j;
    query[n] = p.query + (row[n] * p.num_heads + head[n]) * (D * 2);
  }
  w.load_queries(query, g, p.scale, lds.far[wave], [&](float big) {
    uint32_t* const each = reinterpret_cast<uint32_t*>(&buffers[1].params);
    if (lane == 0) each[wave] = __float_as_uint(big);  // not negative: ordered as its bits
    __syncthreads();
    for (int i = 0; i < W; ++i) big = fmaxf(big, __uint_as_float(each[i]));
    return big;
  });

  if (t0 < block_end) {
    const int chunks = (block_end - t0 + 32 * W - 1) / (32 * W);
    const int whole = all_see + 1 < end ? all_see + 1 : end;
    const int mine = t0 + 32 * wave;
    Feed<DT, D> feed = {p, s, kvh, lane, mine, 32 * W, chunks, block_last >> 4, {}};
    constexpr int kAhead = kColumnBuffers - 1;  // chunks on their way
#pragma unroll
    for (int c = 0; c < kAhead; ++c) feed.issue(c, buffers[c].slots[wave]);
    int at = 0;
    for (int c = 0; c < chunks; ++c) {
      auto& now = buffers[at];
      vector_wait<(kAhead - 1) * Slot<D>::loads>();
      w.convert(now.slots[wave], now.params[wave], lane, block_last + 1 - (mine + c * 32 * W));
      __syncthreads();  // this chunk is there, and the one before is done with
      feed.issue(c + kAhead, buffers[at == 0 ? kAhead : at - 1].slots[wave]);
      at = at == kAhead ? 0 : at + 1;
      int i = W == 8 ? (wave >> 2) * 4 : 0;
      const int to = i + 4;
      int tok = t0 + (c * W + i) * 32;
      // Steps that every column sees whole, then the others.
      for (; i < to && tok + 32 <= whole; ++i, tok += 32)
        w.template step<false>(now.slots[i], now.params[i], lane, tok, g, limit);
      for (; i < to && tok < end; ++i, tok += 32)
        w.template step<true>(now.slots[i], now.params[i], lane, tok, g, limit);
    }
    vector_wait<0>();  // nothing lands in the buffers behind their use
  }

  // A column's outputs and sum, not yet divided.
  float x[NT][D / 4], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = group4_sum(w.l[n]);
    const float b = group4_sum(w.b[n]);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < D / 16; ++i) x[n][(D / 16) * r + i] = w.value(n, r, i, b);
  }
  if constexpr (W == 8) {
    float* const other = lds.states[W == 8 ? wave & 3 : 0] + lane;
    __syncthreads();
    if (wave >= 4) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* at = other + n * (D / 4 + 2) * 64;
        at[0] = w.m[n];
        at[64] = l[n];
#pragma unroll
        for (int i = 0; i < D / 4; ++i) at[(2 + i) * 64] = x[n][i];
      }
    }
    __syncthreads();
    if (wave >= 4) return;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float* at = other + n * (D / 4 + 2) * 64;
      const float m = fmaxf(w.m[n], at[0]);
      const float m_use = m == -INFINITY ? 0.f : m;
      const float f0 = fast_exp2(w.m[n] - m_use), f1 = fast_exp2(at[0] - m_use);
      w.m[n] = m;
      l[n] = __builtin_fmaf(f1, at[64], f0 * l[n]);
#pragma unroll
      for (int i = 0; i < D / 4; ++i) x[n][i] = __builtin_fmaf(f1, at[(2 + i) * 64], f0 * x[n][i]);
    }
  }
  if (idle) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    // A range that none of the columns of this wave sees was left out by the merge.
    if (base + 16 * n + col >= cols || (range > 0 && t0 >= end)) continue;
    const int64_t at = row[n] * p.num_heads + head[n];
    if (ranges > 1) {
      const int64_t cell =
          static_cast<int64_t>(found.cell) * p.num_heads + (at - row0 * p.num_heads) * ranges + range;
      if (g == 0) {
        rg.maxima[cell] = w.m[n];
        rg.sums[cell] = l[n];
      }
      float* dst = rg.outputs + cell * D + g * (D / 4);
#pragma unroll
      for (int i = 0; i < D / 4; i += 4)
        *reinterpret_cast<floatx4*>(dst + i) = floatx4{x[n][i], x[n][i + 1], x[n][i + 2], x[n][i + 3]};
    } else {
      const float inv = l[n] > 0.f ? 1.f / l[n] : l[n];  // no key: zero; a NaN stays one
#pragma unroll
      for (int i = 0; i < D / 4; ++i) x[n][i] *= inv;
      store_row<DT, D>(p.out + (at * D + g * (D / 4)) * 2, x[n]);
    }
  }
}

// LOOP: the workgroup goes from block to block, `groups` apart; else there are as
// many workgroups as blocks at most.  (The loop alone costs long prompts 5%: values
// that outlive a block hold registers.)
template <class DT, int D, int NT, int W, bool LOOP>
__device__ __forceinline__ void columns(const Kv4AttnParams& p, ColumnState<D, NT, W>& lds, int first, int groups) {
  const int lane = threadIdx.x & 63;
  auto blocks = [&](int ql, int n) { return ql < (p.every_row ? 1 : 2) ? 0 : column_blocks<NT>(p, ql) * n; };
  // Mostly one round: for another the list is made anew, and holds no registers meanwhile.
  int item = first;
#pragma unroll 1
  for (;;) {
    int items, tokens;  // the same for every wave
    Part found;
    {
      const PartList<decltype(blocks)> parts(p, p.more, lane, blocks);
      items = parts.size() * p.num_kv_heads;
      if (item >= items) return;
      found = parts.find(item / p.num_kv_heads, lane);
      if (item % p.num_kv_heads == 0) parts.tell(found);
      tokens = parts.tokens;
    }
    column_block<DT, LOOP>(p, lds, found, tokens, item % p.num_kv_heads);
    if (!LOOP) return;
    item += groups;
    if (item >= items) return;
    __syncthreads();  // the next block's keys go where this one's states are read
  }
}

// Both kinds of rows in one launch: the column part's workgroups first, and where
// those leave compute units idle, at the start or towards the end, workgroups of
// one-row sequences.
template <class DT, int D, int NT, int W, bool LOOP>
__global__ __launch_bounds__(64 * W, D == 64 ? (NT == 1 ? 4 : W == 4 ? 3 : 2) : 2) void kv4_columns_kernel(Kv4AttnParams p) {
  constexpr int R = W == 4 ? kDecodeRing<D> : 2;
  union Lds {
    ColumnState<D, NT, W> columns;
    RowState<D, W, R> rows;
  };
  __shared__ __align__(16) Lds lds;
  const int groups = p.column_groups;
  if (static_cast<int>(blockIdx.x) < groups) columns<DT, D, NT, W, LOOP>(p, lds.columns, blockIdx.x, groups);
  else one_rows<DT>(p, lds.rows, blockIdx.x - groups, gridDim.x - groups);
}

// Joins the ranges of a row, in order: one wave per (row, query head).  DECODE:
// row r is sequence r's only one; else it is query row r.  About
// 2 us over an empty launch, a chain of the lengths, the maxima and the outputs;
// reading ahead of the lengths, weights passed between lanes instead of read as
// scalars, made it 6.7 us (32 rows of 14 heads; 4.5 so).
template <class DT, int D, bool DECODE>
__global__ __launch_bounds__(256) void kv4_merge_kernel(Kv4AttnParams p) {
  const Ranges& rg = DECODE ? p.one : p.more;
  const int lane = threadIdx.x & 63;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = at / p.num_heads;
  if (r >= (DECODE ? p.num_seqs : p.num_tokens)) return;
  const int s = DECODE ? static_cast<int>(r) : sequence_of(p, r);
  const Place place = rg.places[s];  // of another part's sequence: not used
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
  const int ranges = rg.of(static_cast<int>(rows.len), place.tokens);
  if (ranges == 1) return;  // whole: there is its output already
  const int n = keys <= 0 ? 0 : static_cast<int>((keys + place.tokens - 1) / place.tokens);
  const int64_t head = at - r * p.num_heads;
  const int64_t cell = static_cast<int64_t>(place.first) * p.num_heads + ((row - rows.row0) * p.num_heads + head) * ranges;
  const float* pm = rg.maxima + cell;
  const float* pl = rg.sums + cell;
  const float* po = rg.outputs + cell * D;
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
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + (row * p.num_heads + head) * D + (D / 64) * lane;
  if constexpr (D == 64) {
    *dst = static_cast<uint16_t>(Half<DT>::from_f32(o[0] * inv));
  } else {
    *reinterpret_cast<uint32_t*>(dst) = Half<DT>::from_f32(o[0] * inv) | (Half<DT>::from_f32(o[1] * inv) << 16);
  }
}

constexpr int kCUs = 256;

// How a call is cut.  Host arithmetic on sizes only.
struct Cut {
  bool fast, decode, columns;   // matrix-core kernels; which of them
  bool every_row;               // the column kernel takes one-row sequences too
  int dec_split, dec_n;         // tokens per range and ranges of one-row sequences
  int64_t dec_items;            // ranges of all of them, about
  int col_split, col_n;         // the same of longer queries
  int col_waves, col_tiles;     // waves of a workgroup of the column kernel, column tiles of a wave
  int64_t col_blocks, col_most; // column blocks of all queries, expected and at most
  int dec_cells, col_cells;     // Ranges::cells
  size_t dec_bytes, col_bytes;  // what they and the sequences' places take
};

int64_t round_up(int64_t x, int to) { return (x + to - 1) / to * to; }

Cut cut_of(int num_seqs, int64_t num_tokens, int max_seq_len, int64_t context, int one_row, int decode_only,
           int num_heads, int num_kv_heads, int head_dim, int block_size) {
  Cut c = {};
  c.fast = (head_dim == 64 || head_dim == 128) && block_size % 16 == 0;
  if (!c.fast) return c;
  const int group = num_heads / num_kv_heads;
  // The column part takes one-row sequences too where the caller expects none of
  // them: expectations shape the launches and never decide what is computed.
  c.every_row = group > 16 || (!decode_only && one_row == 0);
  c.decode = !c.every_row;
  c.columns = c.every_row || !decode_only;
  const int64_t longest = max_seq_len > 0 ? max_seq_len : 1;
  const int64_t all = num_seqs * longest;
  const int64_t tokens = context > 0 && context < all ? context : all;  // of K, and of V, that a KV head reads
  // Partial results: as many cells as the expected lengths can need, which is a
  // number of ranges for the device, however many sequences and whatever the
  // longest of them.
  const size_t cell_bytes = num_heads * (head_dim + 2) * sizeof(float);
  auto bytes_of = [&](int n, int cells) { return n > 1 ? cells * cell_bytes + num_seqs * sizeof(Place) : 0; };
  auto least = [](int64_t a, int64_t b) { return static_cast<int>(a < b ? a : b > 1 ? b : 1); };
  if (c.decode) {
    // About one range for each workgroup that the device holds, but not under
    // 384 tokens: a range costs its workgroup ~7 us of its own (the search, three
    // dependent loads, the merge of the waves).  32 contexts around 1K (two KV
    // heads of 64): 128 / 256 / 384 / 512 / 768 tokens 12.0 / 10.9 / 9.9 / 10.6 /
    // 11.7 us; 64 around 4K (four of 128): 512 / 1024 / 2048 tokens 70.5 / 64.6 /
    // 64.6 us.  Contexts of up to 1024 stay whole: one of 750 takes 9.7 us, in two
    // ranges 8.6 and 3.0 for the second launch.
    const int64_t split = round_up((tokens * num_kv_heads + 4 * kCUs - 1) / (4 * kCUs), 128);
    c.dec_split = longest <= 1024 ? 1024 : split < 384 ? 384 : split < 1 << 30 ? static_cast<int>(split) : 1 << 30;
    c.dec_n = static_cast<int>((longest + c.dec_split - 1) / c.dec_split);
    // A split context has under 2 len / dec_split ranges, all of them 2 tokens / dec_split.
    c.dec_cells = least(static_cast<int64_t>(num_seqs) * c.dec_n, 8 * kCUs / num_kv_heads);
    c.dec_bytes = bytes_of(c.dec_n, c.dec_cells);
    c.dec_items = (tokens / c.dec_split + num_seqs) * num_kv_heads;
  }
  if (c.columns) {
    // Column tiles of a wave: one needs a fifth more vector operations than two
    // (a step's codes are unpacked for half as many columns) and gives twice the
    // blocks.  Waves: eight, four on either half of the keys, or four.  Vector
    // issue bounds all of them once a SIMD has two waves, so few rows want many
    // blocks of eight waves, up to one on each compute unit (two at head size 64,
    // where two fit).  Head size 64 / 128, us, one tile and two: a chunk of 512 rows
    // 12.6 / 15.3 and 16.3 / 20.3, behind 2100 tokens 27 / 40 and 27 / 48, two such
    // chunks 34 and 39 (size 64), four 40 and 44.  Two tiles, eight waves and four:
    // six chunks (342 blocks, size 64) 47 and 59, two prompts of 2048 (448 blocks,
    // size 64) 43 and 56, but (896, size 128) 103 and 84, four (896, size 64) 88 and 71.
    // Without the one-row sequences, where the caller knows them.
    const int64_t ones = c.decode && one_row > 0 && one_row < num_tokens ? one_row : 0;
    const int64_t rows = num_tokens - ones;
    auto count = [&](int tiles) { return (rows * group + 64 * tiles - 1) / (64 * tiles) * num_kv_heads; };
    const int64_t few = (head_dim == 64 ? 2 : 1) * kCUs;
    c.col_tiles = count(1) <= few ? 1 : 2;
    const int64_t blocks = count(c.col_tiles);
    c.col_waves = blocks <= few ? 8 : 4;
    // Keys are split only where the blocks leave half of the device idle, and not
    // under 256 keys or in contexts of up to 768: the partials and the launch that
    // joins them cost 5 us and more, 300 keys' worth.  Four chunks of 512 rows
    // (size 64 / 128) 45 / 78 us whole, 56 / 122 in ranges of 512 keys; ranges of
    // the longer half of such contexts alone make a second round, 62 to 76 / 87 to 104.
    const int64_t want = kCUs / blocks < 1 || longest <= 768 ? 1 : kCUs / blocks;
    const int64_t split = round_up((longest + want - 1) / want, 32);
    c.col_split = static_cast<int>(split < 256 ? 256 : split);
    c.col_n = static_cast<int>((longest + c.col_split - 1) / c.col_split);
    // A sequence's last block may hold a single column.
    c.col_blocks = rows * group / (64 * c.col_tiles) + (num_seqs - ones > 0 ? num_seqs - ones : 1);
    c.col_most = num_tokens * group / (64 * c.col_tiles) + num_seqs;
    // col_n is at most kCUs / blocks, and the rows have 64 col_tiles columns a block.
    c.col_cells = least(num_tokens * c.col_n, 64 * c.col_tiles * kCUs / num_heads);
    c.col_bytes = bytes_of(c.col_n, c.col_cells);
  }
  return c;
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

hipError_t launch(const void* fn, int64_t blocks, Kv4AttnParams& p, hipStream_t st, int threads = 256) {
  if (blocks <= 0) return hipSuccess;
  if (blocks > 0x7FFFFFFF) return hipErrorInvalidValue;
  void* args[] = {&p};
  return hipLaunchKernel(fn, dim3(static_cast<unsigned>(blocks)), dim3(static_cast<unsigned>(threads)), args, 0, st);
}

template <class DT, int D>
hipError_t launch_fast(Kv4AttnParams p, const Cut& c, char* workspace, hipStream_t st) {
  const int64_t pairs = static_cast<int64_t>(p.num_seqs) * p.num_kv_heads;
  auto ranges = [&](char* at, int cells, int n, int tokens) {
    const int64_t all = static_cast<int64_t>(cells) * p.num_heads;
    float* o = reinterpret_cast<float*>(at);
    return Ranges{n, tokens, cells, o + all * D, o + all * (D + 1), o, reinterpret_cast<Place*>(o + all * (D + 2))};
  };
  const int64_t held = static_cast<int64_t>(kCUs) * kDecodeGroups;
  int64_t row_groups = 0;
  if (c.decode) {
    p.one = ranges(workspace, c.dec_cells, c.dec_n, c.dec_split);
    const int64_t most = pairs * c.dec_n < c.dec_items ? pairs * c.dec_n : c.dec_items;
    row_groups = most < held ? most : held;
  }
  // One launch for both kinds of rows where those of one row fit the device beside;
  // else the decode kernel's workgroups of four waves are worth a launch of their own.
  // A chunk of 300 rows beside 32 / 128 / 512 contexts around 400, us: four KV heads of
  // 128 together 23 / 47 / 109, apart 26 / 40 / 78; two of 64 18 / 25 / 54 and 23 / 31 / 54.
  const bool together = c.columns && row_groups < held;
  hipError_t e = hipSuccess;
  if (c.columns) {
    p.more = ranges(workspace + align256(c.dec_bytes), c.col_cells, c.col_n, c.col_split);
    p.every_row = c.every_row ? 1 : 0;
    // Where the caller's count of one-row sequences leaves far fewer blocks than the
    // rows could make, as many workgroups as blocks are expected, and a loop.
    const int64_t each = static_cast<int64_t>(p.num_kv_heads) * c.col_n;
    const bool loop = c.col_waves == 8 || c.col_most > c.col_blocks + c.col_blocks / 2;
    const int64_t groups = (loop ? c.col_blocks : c.col_most) * each;
    if (groups > 0x3FFFFFFF) return hipErrorInvalidValue;
    p.column_groups = static_cast<int>(groups);
    const void* fn = c.col_tiles == 1   ? reinterpret_cast<const void*>(&kv4_columns_kernel<DT, D, 1, 8, true>)
                     : c.col_waves == 8 ? reinterpret_cast<const void*>(&kv4_columns_kernel<DT, D, 2, 8, true>)
                     : loop             ? reinterpret_cast<const void*>(&kv4_columns_kernel<DT, D, 2, 4, true>)
                                        : reinterpret_cast<const void*>(&kv4_columns_kernel<DT, D, 2, 4, false>);
    e = launch(fn, groups + (together ? row_groups : 0), p, st, 64 * c.col_waves);
    if (e == hipSuccess && c.col_n > 1)
      e = launch(reinterpret_cast<const void*>(&kv4_merge_kernel<DT, D, false>), (p.num_tokens * p.num_heads + 3) / 4, p, st);
  }
  if (e == hipSuccess && c.decode && !together) {
    e = row_groups <= kCUs ? launch(reinterpret_cast<const void*>(&kv4_decode_kernel<DT, D, 8>), row_groups, p, st, 512)
                           : launch(reinterpret_cast<const void*>(&kv4_decode_kernel<DT, D, 4>), row_groups, p, st);
  }
  if (e == hipSuccess && c.decode && c.dec_n > 1)
    e = launch(reinterpret_cast<const void*>(&kv4_merge_kernel<DT, D, true>),
               (static_cast<int64_t>(p.num_seqs) * p.num_heads + 3) / 4, p, st);
  return e;
}

bool misaligned(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

}  // namespace
}  // namespace ns

extern "C" size_t ns_paged_attention_int4_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                                        int block_size, int max_seq_len,
                                                        int64_t num_tokens, int is_decode_only,
                                                        int64_t context_tokens, int one_row_seqs) {
  using namespace ns;
  if (num_seqs <= 0 || num_tokens <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      max_seq_len < 0 || !kv4_shape_ok(head_dim, block_size))
    return 0;
  const Cut c = cut_of(num_seqs, num_tokens, max_seq_len, context_tokens, one_row_seqs, is_decode_only, num_heads, num_kv_heads,
                       head_dim, block_size);
  return align256(c.dec_bytes) + align256(c.col_bytes);
}

extern "C" int ns_paged_attention_int4(void* out, const void* query,
                                       const void* k_cache, const void* v_cache,
                                       const void* block_tables, int64_t block_table_stride,
                                       int64_t block_table_width, int block_tables_is_int64,
                                       const void* seq_lens, int seq_lens_is_int64,
                                       const void* query_start_loc, int query_start_loc_is_int64,
                                       int num_seqs, int64_t num_tokens, int max_seq_len, int is_decode_only,
                                       int64_t context_tokens, int one_row_seqs,
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
  if (context_tokens < 0 || one_row_seqs < -1 || one_row_seqs > num_seqs) return NS_ERR_INVALID_ARG;
  if (block_table_width <= 0 || block_table_stride < block_table_width) return NS_ERR_INVALID_ARG;
  if (misaligned(out, 16) || misaligned(query, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16) ||
      misaligned(block_tables, block_tables_is_int64 ? 8 : 4) || misaligned(seq_lens, seq_lens_is_int64 ? 8 : 4) ||
      misaligned(query_start_loc, query_start_loc_is_int64 ? 8 : 4))
    return NS_ERR_INVALID_ARG;
  // Rows, heads, columns and a context's tokens are counted in 32 bits.
  if (max_seq_len > 1 << 30) return NS_ERR_UNSUPPORTED;
  if (num_heads > 65535 || num_tokens > 0x7FFFFFFF / num_heads || num_seqs > 0x7FFFFFFF / num_heads)
    return NS_ERR_UNSUPPORTED;
  const Cut cut = cut_of(num_seqs, num_tokens, max_seq_len, context_tokens, one_row_seqs, is_decode_only, num_heads, num_kv_heads,
                         head_dim, block_size);
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
  p.one = p.more = {1, 0, 0, nullptr, nullptr, nullptr, nullptr};
  p.every_row = 0;
  p.column_groups = 0;
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
