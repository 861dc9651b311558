// Paged attention for trees of drafted tokens.
//
// A sequence's query rows are the tree's nodes: row j of a sequence with context
// length L (its rows included) and q rows sees every key before the rows,
// 0 .. L - q - 1, and key L - q + i where bit i of its mask is set.  KV head of
// query head h is h / (Hq / Hkv); softmax and sums are float32; a row without keys
// is zero, and so is one whose scores are all -inf.
#include <math.h>

#include "ns_common.h"

namespace ns {
namespace {

constexpr int kRows = 64;        // rows of a sequence that a mask can name
constexpr int kSeqs = 512;       // sequences of a launch (their schedule is held in LDS)
constexpr int kMaxHeadDim = 256;
constexpr int kMostPlainRows = (1 << 26) - 1;  // of 64 threads each: a grid has less than 2^32 in a direction

struct TreeParams {
  char* out;
  const char* query;
  const char* k_cache;
  const char* v_cache;
  const void* bt;
  int64_t bt_stride;
  const void* seq_lens;
  const void* qsl;         // query offsets; NULL: row s is sequence s
  const int64_t* mask;
  int bt64, sl64, qsl64;
  int num_seqs;            // of this launch: sequences first_seq ..
  int first_seq;
  int num_heads, num_kv_heads, group, head_dim, block_size;
  int64_t num_tokens, num_blocks;
  int64_t max_ctx;         // keys a sequence may have: max_seq_len, within the table
  float scale;
  // Matrix-core kernel.  key / block_size is mulhi(key, block_mul) >> block_shift, c / group
  // is c times by_group.
  uint32_t block_mul;
  int block_shift;
  float by_group;
  float* partials;         // two slots a workgroup
  int* counters;           // one a workgroup, zero before and after
};

struct SeqRows {
  int64_t row0, ql, len;
};

__device__ __forceinline__ SeqRows rows_of(const TreeParams& p, int s) {
  SeqRows r;
  s += p.first_seq;
  if (!p.qsl) {
    r.row0 = s;
    r.ql = 1;
  } else {
    r.row0 = load_index(p.qsl, s, p.qsl64);
    r.ql = load_index(p.qsl, s + 1, p.qsl64) - r.row0;
    // Offsets that leave the query tensor are never followed.
    if (r.row0 < 0 || r.ql < 0 || r.row0 > p.num_tokens || r.ql > p.num_tokens - r.row0) r.ql = 0;
  }
  r.len = load_index(p.seq_lens, s, p.sl64);
  r.len = r.len < 0 ? 0 : (r.len < p.max_ctx ? r.len : p.max_ctx);
  return r;
}

// The part of a row's mask that falls to the 32 keys from `key` on, with the keys
// before `base` seen and those from `len` on not: bit i stands for key + i.
__device__ __forceinline__ uint32_t seen_of(uint64_t mask, int key, int base, int len) {
  const int off = key - base;
  uint32_t w;
  if (off >= 0) {
    w = off < 64 ? static_cast<uint32_t>(mask >> off) : 0u;
  } else {
    // -off keys of the prefix come first.
    const int n = -off;
    w = n >= 32 ? ~0u : (static_cast<uint32_t>(mask) << n) | ((1u << n) - 1u);
  }
  const int left = len - key;
  return left >= 32 ? w : left <= 0 ? 0u : w & ((1u << left) - 1u);
}

// ---- any shape: one wave per (token row, query head) ------------------------
//
// One key per lane: the lane's dot product of the query (in LDS, float32) with its
// key joins the wave's running maximum and sum; then every lane adds the chunk's
// weighted values into the output dims it owns, one key at a time.  Plain, for shapes
// that no serving configuration here has: every wave reads its K and V for itself, lanes a
// row apart, and waits for each (32 requests of 8 rows around 1K keys: 2.0 to 2.5 ms by type
// and head size, one of 24 rows 144 us; the matrix-core kernel takes 18 and 11 us).
// DL: output dims per lane (head_dim <= 64 * DL).
template <class T, int DL>
__global__ __launch_bounds__(64) void tree_attention_generic_kernel(TreeParams p) {
  __shared__ float q_lds[64 * DL];
  const int lane = threadIdx.x;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y;
  const int D = p.head_dim, bs = p.block_size;
  const int kvh = h / p.group;

  // The row's sequence: the last s with query_start_loc[s] <= t.
  int s = static_cast<int>(t);
  if (p.qsl) {
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (load_index(p.qsl, mid, p.qsl64) <= t) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
  }
  const SeqRows r = rows_of(p, s);
  // A row of no sequence, or past a sequence's 64th, is left as it is.
  if (t < r.row0 || t >= r.row0 + (r.ql < kRows ? r.ql : kRows)) return;
  const int64_t base = r.len - r.ql;
  const uint64_t mask = static_cast<uint64_t>(p.mask[t]);

  const T* qrow = reinterpret_cast<const T*>(p.query) + (t * p.num_heads + h) * D;
  for (int d = lane; d < 64 * DL; d += 64) q_lds[d] = d < D ? static_cast<float>(qrow[d]) : 0.f;
  __syncthreads();

  const T* kc = reinterpret_cast<const T*>(p.k_cache);
  const T* vc = reinterpret_cast<const T*>(p.v_cache);
  const int64_t bt_row = static_cast<int64_t>(s) * p.bt_stride;
  float m = -INFINITY, l = 0.f, o[DL];
#pragma unroll
  for (int j = 0; j < DL; ++j) o[j] = 0.f;
  int bad = 0;
  for (int64_t c0 = 0; c0 < r.len; c0 += 64) {
    const int64_t key = c0 + lane;
    int64_t row = 0;  // element offset of this lane's key (its K and V rows)
    bool ok = key < r.len;
    if (ok) {
      // A block outside the cache is every row's, seen or not, as in the kernel below.
      const int64_t blk = load_index(p.bt, bt_row + key / bs, p.bt64);
      ok = blk >= 0 && blk < p.num_blocks;
      if (!ok) bad = 1;
      else row = ((blk * bs + key % bs) * p.num_kv_heads + kvh) * D;
    }
    if (ok && key >= base) {
      const int64_t i = key - base;
      ok = i < kRows && ((mask >> i) & 1);
    }
    float sc = -INFINITY;
    if (ok) {
      float acc = 0.f;
      for (int d = 0; d < D; ++d) acc = __builtin_fmaf(q_lds[d], static_cast<float>(kc[row + d]), acc);
      sc = acc * p.scale;
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
    const uint64_t some = __builtin_amdgcn_ballot_w64(ok);
    const uint32_t row_lo = static_cast<uint32_t>(row), row_hi = static_cast<uint32_t>(row >> 32);
    for (int kk = 0; kk < 64; ++kk) {
      if (!((some >> kk) & 1)) continue;  // uniform: V of a key that is not seen is not read
      const float w = __shfl(pk, kk);
      const int64_t at = static_cast<int64_t>((static_cast<uint64_t>(static_cast<uint32_t>(__shfl(row_hi, kk))) << 32) |
                                              static_cast<uint32_t>(__shfl(row_lo, kk)));
#pragma unroll
      for (int j = 0; j < DL; ++j) {
        const int d = lane + 64 * j;
        if (d < D) o[j] = __builtin_fmaf(w, static_cast<float>(vc[at + d]), o[j]);
      }
    }
  }
  bad = __builtin_amdgcn_ballot_w64(bad != 0) != 0;

  T* orow = reinterpret_cast<T*>(p.out) + (t * p.num_heads + h) * D;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // no key: zero; a NaN stays one
#pragma unroll
  for (int j = 0; j < DL; ++j) {
    const int d = lane + 64 * j;
    if (d < D) orow[d] = static_cast<T>(bad ? NAN : o[j] * inv);
  }
}

template <class T>
hipError_t launch_generic(const TreeParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.num_tokens), static_cast<unsigned>(p.num_heads));
  void* args[] = {const_cast<TreeParams*>(&p)};
  const void* fn = p.head_dim <= 64    ? reinterpret_cast<const void*>(&tree_attention_generic_kernel<T, 1>)
                   : p.head_dim <= 128 ? reinterpret_cast<const void*>(&tree_attention_generic_kernel<T, 2>)
                                       : reinterpret_cast<const void*>(&tree_attention_generic_kernel<T, 4>);
  return hipLaunchKernel(fn, grid, dim3(64), args, 0, stream);
}

// ---- head sizes 64 and 128, blocks of whole 16-token tiles --------------------
//
// A sequence's rows times the heads of one KV head are columns, 16 a tile.  A group is
// up to WC * NT tiles of columns of one (sequence, KV head); a workgroup takes a range
// of a group's keys.  Its waves are KG key groups of WC column waves: key group i
// takes the range's chunks of 32 keys i, i + KG, ..., each column wave NT of the tiles
// for all of them, so that every row of K and V is loaded once for up to 16 WC NT rows
// of the product.  K and V come by LDS-DMA into a ring of the key group's, loaded by its
// waves in equal parts (with more than one, a barrier a chunk hands them over); S^T = K
// Q^T and O^T = V^T P^T run on v_mfma_f32_16x16x32.  The result layout of the first
// product (keys 4 g + r of column lane % 16 in lane group g) is the operand layout of
// the second.  The key groups meet once, at the range's end.
//
// The probabilities enter the second product in the model's dtype, and their sum
// is taken by the same product with a tile of ones, so that a rounding acts on both.
//
// Work is cut evenly: the groups' chunks, and kGroupCost for what a group costs
// beside them, are laid end to end, and workgroup k takes the k-th equal share of
// that line, whatever it covers: parts of groups, whole ones, or both.  Cuts move to
// whole rounds of the key groups.  A group that a cut falls into is joined by the last
// of its workgroups to finish, which has its own part in registers still.  Every
// workgroup works its share out of the device's lengths for itself.
//
// What bounds it (MI355X, 16-bit types, calls of a captured graph).  One request of
// 24 rows and 750 keys: 11 us, a chain of trips (lengths 1.2, schedule 1, block ids and
// queries 2, first keys 2, loop, the join of the ranges 2 to 3).  32 requests of 8
// rows around 1K keys: 18 us for 22 MB, the same chain.  64 x 12 rows around 4K keys,
// head size 128: 169 us, K and V once at 4.3 TB/s (a copy moves 4.7).  8 x 64 rows
// around 4K keys: 60 us, 550 TFLOP/s: a step of a compute unit's loop takes 2630 cycles, of
// which the matrix cores need 1090, the vector units 1110 and the LDS reads 1020.

constexpr int kMostRanges = 32;  // of a group: what the last workgroup has to join
constexpr int kGroupCost = 16;   // in chunks
constexpr float kNoScore = -3e38f;  // a column's reference before its first score; scores below it are as -inf
constexpr float kSlack = 8.f;    // binades that a score may pass its column's reference by
constexpr int kLeastRounds = 2;  // of the key groups, in a share; groups of no more stay whole

template <int D_, int KG_, int WC_, int NT_>
struct Cfg {
  static constexpr int D = D_, KG = KG_, WC = WC_, NT = NT_;
  static constexpr int W = KG * WC;             // waves
  static constexpr int THREADS = 64 * W;
  static constexpr int COLS = 16 * NT * WC;
  static constexpr int CPR = D / 8;             // 16-byte units of a row
  static constexpr int KPI = 64 / CPR;          // rows of a tile that one load brings
  static constexpr int LPT = 16 / KPI;          // loads of a tile
  static constexpr int NK = 8 / KPI;            // loads until K's swizzle repeats
  static constexpr int TILE_B = 32 * D * 2;     // K or V of a chunk
  static constexpr int SLOT_B = 2 * TILE_B;
  static constexpr int FIT = 131072 / (KG * SLOT_B);
  static constexpr int R = WC == 1 ? 2 : FIT < 4 ? FIT : 4;  // chunks in a key group's ring
  static constexpr int LOADS = 4 * LPT / WC;    // of a chunk, by one wave
  static constexpr int NC = D / 32, NN = D / 16;
  static constexpr int RING = KG * R * SLOT_B;
  static constexpr int UNIT = 256;              // floats of 16 dims of a tile: four a lane
  static constexpr int PART = COLS * (D + 2);   // words of a slot: units, then (maximum, sum) of every column
  // The key groups meet JOIN tiles of a wave at a time, as many as fit the ring.
  static constexpr int JOIN = RING / (W * NN * UNIT * 4) < NT ? RING / (W * NN * UNIT * 4) : NT;
  static constexpr bool KEEP = NT <= 2;         // a range's units stay in registers for the join of the ranges
  static constexpr int OWN = (NT * NN + KG - 1) / KG;  // units that a wave joins the ranges of
  static_assert(R >= 2 && JOIN >= 1 && NT % JOIN == 0, "chunks in flight; a tile of every wave fits the ring");
  static_assert(JOIN == NT || JOIN * NN % KG == 0, "a wave's units of the joins are its units of all");
  static_assert(2 * kMostRanges * COLS * 4 <= RING, "the ranges' maxima and sums fit the ring");
  static_assert(kGroupCost >= KG / 2, "a group's workgroups begin within its stretch of the line");
  static_assert(kLeastRounds >= 1, "a group has one cut at most that moves to its start or end");
};

constexpr int kSc1 = 16;                  // cache-policy bit SC1 of gfx950 buffer operations: device scope
constexpr int kBufferWord3 = 0x00020000;  // raw 32-bit buffer descriptor, word 3

// Until at most N of the wave's vector memory operations are pending.
template <int N>
__device__ __forceinline__ void vector_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// The same, then a barrier; the wave's LDS operations are done.
template <int N>
__device__ __forceinline__ void vector_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// 16 bytes of each lane from base + off (base uniform) to LDS address to + 16 lane.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds16(const void* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to)
               : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ float ld_sc1(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, kSc1));
}
// Unit c of row `key` of a chunk lies at unit c ^ swizzle of its row, so that the
// operand reads spread over the banks (the transposing reads of V are served 32
// lanes at a time: eight keys of two neighbouring units).
__device__ __forceinline__ int k_swizzle(int key) { return key & 7; }
template <int D>
__device__ __forceinline__ int v_swizzle(int key) {
  return D == 64 ? ((key >> 1) & 3) << 1 : (key & 7) << 1;
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Division by a uniform y > 0 of uniform 0 <= x < 2^30: by the reciprocal in float32, which
// with quotients below 2^20 is one off at most, and put right.  (The kernel's first share of
// a line can pass that, and is put right there.)
struct Divisor {
  int y;
  float r;
  __device__ __forceinline__ explicit Divisor(int y_) : y(y_), r(__builtin_amdgcn_rcpf(static_cast<float>(y_))) {}
  __device__ __forceinline__ int of(int x) const {
    int q = uniform(static_cast<int>(static_cast<float>(x) * r));
    const int rest = x - q * y;
    q -= rest < 0;
    q += rest >= y;
    return q;
  }
};

// f over the lanes up to each, for values that f leaves as they are with a zero: shifts
// within the rows of 16 lanes, then a row's last lane to the row behind it and lane 31
// to the upper half.
template <class F>
__device__ __forceinline__ int wave_scan(int x, F f) {
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false));  // row_shr:1
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false));
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1 and 3
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2 and 3
  return x;
}

// The sequences of a launch along the line of work, from the device's lengths: where
// each starts, and its rows, in LDS.
struct Held {
  int start[kSeqs], row0[kSeqs], ql[kSeqs], len[kSeqs];
  int sums[8], most[8];
};

template <class C>
struct Line {
  Held& h;
  int num_seqs, heads, group;
  int total;
  int most;               // weight of the longest group

  __device__ __forceinline__ int weight(int len) const { return ((len + 31) >> 5) + kGroupCost; }
  __device__ __forceinline__ int groups(int ql) const {
    return ((ql < kRows ? ql : kRows) * group + C::COLS - 1) / C::COLS * heads;
  }

  __device__ __forceinline__ Line(const TreeParams& p, Held& held)
      : h(held), num_seqs(p.num_seqs), heads(p.num_kv_heads), group(p.group) {
    // Up to 64 sequences every wave lists for itself, one a lane: each writes what
    // the others write, and reads it back without waiting for them.
    constexpr int PER = kSeqs / C::THREADS;
    const bool alone = num_seqs <= 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x[PER], sum = 0, m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = alone ? (i == 0 ? lane : kSeqs) : PER * static_cast<int>(threadIdx.x) + i;
      x[i] = 0;
      if (s < num_seqs) {
        const SeqRows r = rows_of(p, s);
        const int ql = static_cast<int>(r.ql), len = static_cast<int>(r.len);
        h.row0[s] = static_cast<int>(r.row0);
        h.ql[s] = ql;
        h.len[s] = len;
        const int wt = ql > 0 ? weight(len) : 0;
        m = max(m, wt);
        x[i] = groups(ql) * wt;
        sum += x[i];
      }
    }
    const int y = wave_scan(sum, [](int a, int b) { return a + b; });
    int before = y - sum;
    total = __builtin_amdgcn_readlane(y, 63);
    most = __builtin_amdgcn_readlane(wave_scan(m, [](int a, int b) { return max(a, b); }), 63);
    if (!alone) {
      if (lane == 0) {
        h.sums[w] = total;
        h.most[w] = most;
      }
      __syncthreads();
      total = 0;
      most = 0;
#pragma unroll
      for (int i = 0; i < C::W; ++i) {
        if (i < w) before += h.sums[i];
        total += h.sums[i];
        most = max(most, h.most[i]);
      }
      total = uniform(total);
      most = uniform(most);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = alone ? (i == 0 ? lane : kSeqs) : PER * static_cast<int>(threadIdx.x) + i;
      if (s < num_seqs) h.start[s] = before;
      before += x[i];
    }
    if (!alone) __syncthreads();
  }

  __device__ __forceinline__ void get(int s, int& start, int& row0, int& ql, int& len) const {
    start = uniform(h.start[s]);
    row0 = uniform(h.row0[s]);
    ql = uniform(h.ql[s]);
    len = uniform(h.len[s]);
  }

  // The sequence that place `at` of the line lies in: the last that starts there or before.
  __device__ __forceinline__ int find(int at) const {
    const int lane = threadIdx.x & 63;
    int n = -1;
    for (int s0 = 0; s0 < num_seqs; s0 += 64) {
      const int s = s0 + lane < num_seqs ? s0 + lane : 0;
      n += __popcll(__builtin_amdgcn_ballot_w64(s0 + lane < num_seqs && h.start[s] <= at));
    }
    return n;
  }
};

template <class DT, class C>
__global__ __launch_bounds__((C::THREADS), 1) void tree_attention_kernel(TreeParams p) {
  using T = typename DT::T;
  using V8 = typename DT::vec8;
  constexpr int D = C::D, KG = C::KG, WC = C::WC, NT = C::NT, W = C::W, COLS = C::COLS;
  constexpr int NC = C::NC, NN = C::NN, LPT = C::LPT, KPI = C::KPI, CPR = C::CPR, NK = C::NK, R = C::R;
  __shared__ __attribute__((aligned(1024))) char smem[C::RING];
  __shared__ Held held;
  __shared__ float maxima[KG][COLS], sums[KG][COLS];
  __shared__ int bads[W];
  __shared__ int last;

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c16 = lane & 15;
  const int w = uniform(tid >> 6);
  const int kg = w / WC, cw = w % WC;
  const int G = p.group, Hkv = p.num_kv_heads;

  const Line<C> line(p, held);
  // Shares: one a workgroup, but none too small, and no group in more than kMostRanges of them.
  const int grid = static_cast<int>(gridDim.x);
  int share = Divisor(grid).of(line.total + grid - 1);
  if (static_cast<uint32_t>(share) * grid < static_cast<uint32_t>(line.total)) ++share;
  const int least = line.most / (kMostRanges - 2) + 1;
  share = share > least ? share : least;
  share = share > kLeastRounds * KG ? share : kLeastRounds * KG;
  // Neighbouring shares, which read the same keys where a sequence has several
  // groups of columns, go to one XCD (workgroups go to the eight in turn).
  const Divisor by_share(share);
  const int shares = by_share.of(line.total + share - 1);
  const int per_xcd = (shares + 7) >> 3;
  const int k = static_cast<int>(blockIdx.x & 7) * per_xcd + static_cast<int>(blockIdx.x >> 3);
  if (static_cast<int>(blockIdx.x >> 3) >= per_xcd || k >= shares) return;

  // Log2 units per score unit; never zero, so that -inf, a key that is not seen, stays it.
  const float scale = __uint_as_float(__builtin_amdgcn_readfirstlane(
      __float_as_uint(fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1.1754944e-38f))));
  const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;  // a negative scale turns the query around, exactly
  const uint32_t ring = lds_addr(smem) + kg * (R * C::SLOT_B);
  const uint32_t stride = static_cast<uint32_t>(Hkv) * D * 2;  // bytes between a block's token rows

  // A lane's part of a load: its unit of its row, where it lies in memory.
  uint32_t koff[NK], voff[NK];
#pragma unroll
  for (int u = 0; u < NK; ++u) {
    const int key = u * KPI + lane / CPR, unit = lane % CPR;
    koff[u] = (lane / CPR) * stride + ((unit ^ k_swizzle(key)) << 4);
    voff[u] = (lane / CPR) * stride + ((unit ^ v_swizzle<D>(key)) << 4);
    if (WC > 1) koff[u] = cw & 1 ? voff[u] : koff[u];  // a column wave loads of K or of V
  }
  // Operand reads within a chunk.  K: key 16 h + c16, unit 4 c + g.  V^T: keys
  // 16 h + 4 g + e of dims 16 n + c16 (ds_read_b64_tr_b16 gives lane i of a 16-lane
  // group, as element e, element i & 3 of the 8 bytes of lane (i >> 2) + 4 e).
  uint32_t kread[NC], vread;
#pragma unroll
  for (int c = 0; c < NC; ++c) kread[c] = c16 * (D * 2) + (((4 * c + g) ^ k_swizzle(c16)) << 4);
  const int vkey = 4 * g + (c16 >> 2);
  vread = vkey * (D * 2) + ((((c16 & 3) >> 1) ^ v_swizzle<D>(vkey)) << 4) + (c16 & 1) * 8;

  constexpr int kHalf = KG / 2;
  const int place = k * share;
  int s = line.find(place);
  int start, row0, ql, len;
  line.get(s, start, row0, ql, len);
  int gi = Divisor(line.weight(len)).of(place - start);
  for (;; ++gi) {
    while (gi >= line.groups(ql)) {
      if (++s >= p.num_seqs) return;
      line.get(s, start, row0, ql, len);
      gi = 0;
    }
    // The group's place on the line, the workgroups a .. b that it falls to, and
    // the chunks c0 .. c1 of this one.
    const int n = (len + 31) >> 5;
    const int gs = start + gi * line.weight(len);
    const int a = by_share.of(gs + kHalf - 1);
    if (a > k) return;
    const int e = (n + KG - 1) / KG * KG - kHalf - 1;
    int b = n > kLeastRounds * KG ? by_share.of(gs + e) : a;
    b = b > a ? b : a;
    if (k > b) continue;
    auto cut = [&](int kk) { return (kk * share - gs + kHalf) / KG * KG; };
    const int c0 = k == a ? 0 : cut(k), c1 = k == b ? n : cut(k + 1);
    const int base = len - ql;
    const int cols = (ql < kRows ? ql : kRows) * G, cbs = (cols + COLS - 1) / COLS;
    const int kvh = Divisor(cbs).of(gi), cb = gi - kvh * cbs;
    const int col0 = cb * COLS + cw * (16 * NT);  // this wave's first column
    const int t1 = 32 * c1 < len ? 32 * c1 : len;
    const int whole = base < t1 ? base : t1;   // keys below are seen by every column
    const int steps = (c1 - c0 + KG - 1) / KG;  // of the workgroup
    const int mine = c1 - c0 > kg ? (c1 - c0 - kg + KG - 1) / KG : 0;

    // Where tile l & 1 of this wave's step l / 2 of a window of 32 steps lies, in lane
    // l: its block, then bytes from the start of a cache.
    int bad = 0;
    uint32_t at_lo = 0, at_hi = 0;
    auto key_of = [&](int step) {
      int of = lane;
      asm volatile("" : "+v"(of));
      const int key = 32 * (c0 + kg + KG * (step + (of >> 1))) + 16 * (of & 1);
      return key < t1 ? key : (t1 - 1) & ~15;  // a tile past the range repeats the last
    };
    auto entry_of = [&](int key) {
      return static_cast<int>(__umulhi(static_cast<uint32_t>(key), p.block_mul) >> p.block_shift);
    };
    auto block_of = [&](int key) {
      return load_index(p.bt, static_cast<int64_t>(p.first_seq + s) * p.bt_stride + entry_of(key), p.bt64);
    };
    auto set_window = [&](int key, int64_t blk) {
      if (blk < 0 || blk >= p.num_blocks) {
        bad = 1;
        blk = 0;
      }
      const int in = key - entry_of(key) * p.block_size;
      const uint64_t at = ((static_cast<uint64_t>(blk) * p.block_size + in) * Hkv + kvh) * (D * 2);
      at_lo = static_cast<uint32_t>(at);
      at_hi = static_cast<uint32_t>(at >> 32);
    };
    const int first_key = mine > 0 ? key_of(0) : 0;
    const int64_t first_block = mine > 0 ? block_of(first_key) : 0;

    // Column c is query head c % G of row c / G (c < 2^16: the quotient's error in
    // float32 is far below half of 1 / G).
    auto row_in = [&](int c) { return static_cast<int>((static_cast<float>(c) + 0.5f) * p.by_group); };
    // The columns' query rows (a column past the last repeats it), on their way
    // together with the block ids.
    auto row_of = [&](int i, int& head) {
      int c = c16;
      asm volatile("" : "+v"(c));  // worked out where it is needed, not held in registers over the loop
      c += col0 + 16 * i;
      c = c < cols ? c : cols - 1;
      const int j = row_in(c);
      head = kvh * G + c - j * G;
      return static_cast<int64_t>(row0) + j;
    };
    V8 q[NT][NC];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      int head;
      const int64_t row = row_of(i, head);
      const char* qr = p.query + ((row * p.num_heads + head) * D + 8 * g) * 2;
#pragma unroll
      for (int c = 0; c < NC; ++c) q[i][c] = load16<DT>(qr + 64 * c);
    }
    if (mine > 0) set_window(first_key, first_block);
    float m[NT];  // a column's reference, log2 units
    floatx4 acc[NT][NN], l[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        u32x4 x = __builtin_bit_cast(u32x4, q[i][c]);
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x[e2] ^= flip;
        lds_ready(x);  // here, so that the loop's first product waits for no load of its own
        q[i][c] = __builtin_bit_cast(V8, x);
      }
      m[i] = kNoScore;
      l[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NN; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    auto issue = [&](int step) {
      if ((step & 31) == 0 && step > 0) {
        const int key = key_of(step);
        set_window(key, block_of(key));
      }
      const uint32_t to = ring + (static_cast<uint32_t>(step) % R) * C::SLOT_B;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (WC == 4 && h != cw >> 1) continue;
        const int from = 2 * (step & 31) + h;
        const uint64_t at =
            (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at_hi), from))) << 32) |
            static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at_lo), from));
        if (WC == 1) {
          const char* kp = p.k_cache + at;
          const char* vp = p.v_cache + at;
#pragma unroll
          for (int u = 0; u < LPT; ++u) {
            load_lds16(kp + u * KPI * stride, koff[u % NK], to + (h * LPT + u) * 1024);
            load_lds16(vp + u * KPI * stride, voff[u % NK], to + C::TILE_B + (h * LPT + u) * 1024);
          }
        } else {
          const char* from_cache = (cw & 1 ? p.v_cache : p.k_cache) + at;
          const uint32_t part = to + (cw & 1) * C::TILE_B + h * LPT * 1024;
#pragma unroll
          for (int u = 0; u < LPT; ++u) load_lds16(from_cache + u * KPI * stride, koff[u % NK], part + u * 1024);
        }
      }
    };

    V8 ones;
#pragma unroll
    for (int e2 = 0; e2 < 8; ++e2) ones[e2] = static_cast<T>(1.f);
    constexpr int AHEAD = WC == 1 ? R : R - 1;  // chunks issued before the first is waited for
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < mine) issue(i);
    const int count = WC == 1 ? mine : steps;
    const bool idle = WC > 1 && col0 >= cols;  // no columns: this wave loads for the others
    // Chunk `step` has come (to all of the key group's waves, and none reads the one before it).
    auto advance = [&](int step) {
      const int younger = mine - 1 - step;
      if (WC == 1) {
        if (younger >= 1) vector_wait<C::LOADS>();
        else vector_wait<0>();
      } else {
        if (R > 3 && younger >= 2) vector_barrier<2 * C::LOADS>();
        else if (R > 2 && younger >= 1) vector_barrier<C::LOADS>();
        else vector_barrier<0>();
        if (step + R - 1 < mine) issue(step + R - 1);
      }
    };
    u32x4 kraw[2][NC];
    auto read_keys = [&](int step) {
      const uint32_t ka = ring + (static_cast<uint32_t>(step) % R) * C::SLOT_B;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        kraw[0][c] = ds_read_b128_at<0>(ka + kread[c]);
        kraw[1][c] = ds_read_b128_at<16 * D * 2>(ka + kread[c]);
      }
    };
    int step = 0;
    const int work = idle ? 0 : count;  // a key group without a chunk in the last step sees none of its keys
    if (count > 0) advance(0);
    if (work > 0) read_keys(0);
    // The inner loop holds the common chunk and nothing that changes the accumulators
    // in another way (a branch that did would cost a second set of their registers):
    // it is left at a chunk that moves a reference, whose scores are then taken again.
    // K of the next chunk is read beside the products of V, V beside the softmax.
    uint32_t odd = 0;  // bit i: the chunk of step count - 1 - i is added one key at a time
    while (step < work) {
      float top[NT];
      bool past = false;
      for (; step < work; ++step) {
        const int tb = 32 * (c0 + kg + KG * step);
        u32x2 vraw[NN][2];
        const uint32_t va = ring + (static_cast<uint32_t>(step) % R) * C::SLOT_B + C::TILE_B + vread;
        lds_wait_all();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < NC; ++c) lds_ready(kraw[h][c]);
        // Products that follow one another add to different sums.
        floatx4 sacc[NT][2];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              sacc[i][h] = mfma16x16x32(DT{}, __builtin_bit_cast(V8, kraw[h][c]), q[i][c],
                                        c == 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : sacc[i][h]);
        __builtin_amdgcn_sched_barrier(0);
        // Unit 2 j of a row: the swizzle touches bits above the lowest, and so is an exclusive or of the address.
#pragma unroll
        for (int j = 0; j < NN; ++j) {
          const uint32_t at = va ^ (j << 5);
          vraw[j][0] = ds_read_tr16_b64_at<0>(at);
          vraw[j][1] = ds_read_tr16_b64_at<16 * D * 2>(at);
        }
        const bool tail = tb + 32 > whole;  // some keys are not seen by every column
        if (tail) {
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            int head;
            const uint32_t seen = seen_of(static_cast<uint64_t>(p.mask[row_of(i, head)]), tb, base, t1) >> (4 * g);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int r = 0; r < 4; ++r) sacc[i][h][r] = (seen >> (16 * h + r)) & 1 ? sacc[i][h][r] : -INFINITY;
          }
        }
        // A column's reference follows its maximum only when a score passes it by kSlack
        // binades, which is seen without a trip between lanes.
        past = false;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          top[i] = sacc[i][0][0];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) top[i] = fmaxf(top[i], sacc[i][h][r]);
          past |= top[i] * scale > m[i] + kSlack;
        }
        past = __builtin_amdgcn_ballot_w64(past) != 0;
        lds_wait_all();
#pragma unroll
        for (int j = 0; j < NN; ++j) {
          lds_ready(vraw[j][0]);
          lds_ready(vraw[j][1]);
        }
        if (__builtin_expect(past, 0)) break;
        if (tail) {
          // V of a key past the range is taken as zero.  A chunk with an element of V that
          // is not finite is left for later (add_keys), so that it reaches only the rows
          // that see it.
          const int left = t1 - tb;
          int wild = 0;
#pragma unroll
          for (int j = 0; j < NN; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e2 = 0; e2 < 2; ++e2) {
                const int key = 16 * h + 4 * g + 2 * e2;
                uint32_t x = vraw[j][h][e2];
                x = key + 1 < left ? x : key < left ? x & 0xFFFFu : 0u;
                vraw[j][h][e2] = x;
                constexpr uint32_t inf = DT::code == NS_DTYPE_F16 ? 0x7C00u : 0x7F80u;
                wild |= (x & inf) == inf || (x & (inf << 16)) == inf << 16;
              }
          if (__builtin_amdgcn_ballot_w64(wild != 0) != 0 && count - 1 - step < 32) {
            odd |= 1u << (count - 1 - step);
#pragma unroll
            for (int j = 0; j < NN; ++j) vraw[j][0] = vraw[j][1] = u32x2{0u, 0u};
          }
        }
        // The chunk is in registers: the next but one takes its place.
        if (WC == 1 && step + R < mine) issue(step + R);
        if (step + 1 < work) {
          advance(step + 1);
          read_keys(step + 1);
        }
        V8 pt[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              pt[i][4 * h + r] = static_cast<T>(fast_exp2(__builtin_fmaf(sacc[i][h][r], scale, -m[i])));
        // Two waves share a SIMD: the one whose products are due goes before the other's softmax.
        if (WC > 1) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < NT; ++i) l[i] = mfma16x16x32(DT{}, ones, pt[i], l[i]);
#pragma unroll
        for (int j = 0; j < NN; ++j) {
          const V8 v = __builtin_bit_cast(V8, u32x4{vraw[j][0][0], vraw[j][0][1], vraw[j][1][0], vraw[j][1][1]});
#pragma unroll
          for (int i = 0; i < NT; ++i) acc[i][j] = mfma16x16x32(DT{}, v, pt[i], acc[i][j]);
        }
        if (WC > 1) __builtin_amdgcn_s_setprio(0);
      }
      if (past) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const float x = group4_max_swap(top[i]);
          const float next_m = x == -INFINITY ? m[i] : fmaxf(m[i], x * scale);
          const float alpha = fast_exp2(m[i] - next_m);
          m[i] = next_m;
          l[i] *= alpha;
#pragma unroll
          for (int j = 0; j < NN; ++j) acc[i][j] *= alpha;
        }
      }
    }

    if (WC > 1)
      while (++step < count) advance(step);  // idle: all chunks but the first

    // What follows a range's chunks works its places out anew from here, or they would
    // be held in registers over the loop.
    int tid2 = tid, w2 = w;
    asm volatile("" : "+v"(tid2), "+s"(w2));
    const int lane2 = tid2 & 63, g2 = lane2 >> 4, c2 = lane2 & 15, kg2 = w2 / WC, cw2 = w2 % WC;

    // Adds the rows of V of a chunk to this lane's outputs of column c2 of tile i, at `to`
    // (a unit's floats apart), for the keys that the column sees; their weights, which
    // the sum has, are worked out again.
    auto add_keys = [&](int i, int tb, float reference, float factor, float* to) {
      int head;
      const int64_t row = row_of(i, head);
      const uint32_t seen = seen_of(static_cast<uint64_t>(p.mask[row]), tb, base, t1);
      const T* qr = reinterpret_cast<const T*>(p.query) + (row * p.num_heads + head) * D + g2 * (D / 4);
      for (int key = tb; key < tb + 32 && key < t1; ++key) {
        const int64_t blk = block_of(key);
        if (blk < 0 || blk >= p.num_blocks) break;  // the outputs are NaN
        const int64_t at = ((blk * p.block_size + key - entry_of(key) * p.block_size) * Hkv + kvh) * D;
        const T* kr = reinterpret_cast<const T*>(p.k_cache) + at + g2 * (D / 4);
        const T* vr = reinterpret_cast<const T*>(p.v_cache) + at + 4 * g2;
        float x = 0.f;
        for (int d = 0; d < D / 4; ++d) x = __builtin_fmaf(static_cast<float>(qr[d]), static_cast<float>(kr[d]), x);
        x = group4_sum(x) * (p.scale < 0.f ? -scale : scale);
        x = static_cast<float>(static_cast<T>(fast_exp2(x - reference))) * factor;
        if ((seen >> (key - tb)) & 1) {
          for (int j = 0; j < NN; ++j)
            for (int e2 = 0; e2 < 4; ++e2) {
              float& o = to[j * C::UNIT + e2];
              o = __builtin_fmaf(x, static_cast<float>(vr[16 * j + e2]), o);
            }
        }
      }
    };

    // The key groups' states meet in LDS.  The ring is free when every wave is here.
    if (g2 == 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        maxima[kg2][(cw2 * NT + i) * 16 + c2] = m[i];
        sums[kg2][(cw2 * NT + i) * 16 + c2] = l[i][0];
      }
    }
    {
      const int wave_bad = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
      if (lane2 == 0) bads[w2] = wave_bad;
    }
    __syncthreads();
    int bad_any = 0;
#pragma unroll
    for (int ww = 0; ww < W; ++ww) bad_any |= bads[ww];
    const bool split = b > a;
    // A workgroup has at most one cut group that it begins (its last: slot 2 k + 1)
    // and one that it does not (its first: slot 2 k).
    auto part_of = [&](int kk) { return (kk == a ? 1 : 2 * (kk - a)) * C::PART; };
    const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
        p.partials + static_cast<int64_t>(2) * a * C::PART, static_cast<short>(0),
        split ? 2 * (b - a + 1) * C::PART * 4 : 0, kBufferWord3);
    T* out = reinterpret_cast<T*>(p.out);
    // Dims 16 j + 4 g .. + 3 of the columns of tile i of this wave.
    auto write = [&](int i, int j, floatx4 o, float inv) {
      const int c = col0 + 16 * i + c2;
      if (c >= cols) return;
      const int r0 = row_in(c);
      const int64_t at = ((static_cast<int64_t>(row0) + r0) * p.num_heads + kvh * G + c - r0 * G) * D + 16 * j + 4 * g2;
      typename DT::vec4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = static_cast<T>(o[r] * inv);
      *reinterpret_cast<u32x2*>(out + at) = __builtin_bit_cast(u32x2, v);
    };
    auto inverse = [&](float sum) { return sum > 0.f || sum != sum ? 1.f / sum : 0.f; };  // no key: zero; a NaN stays one
    float* buf = reinterpret_cast<float*>(smem);
    float join_top[NT], join_sum[NT];
    floatx4 own[C::OWN] = {};  // this range's units, for the join of the ranges
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int col = (cw2 * NT + i) * 16 + c2;
      join_top[i] = kNoScore;
#pragma unroll
      for (int kk = 0; kk < KG; ++kk) join_top[i] = fmaxf(join_top[i], maxima[kk][col]);
      join_sum[i] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KG; ++kk)
        join_sum[i] = __builtin_fmaf(sums[kk][col], fast_exp2(maxima[kk][col] - join_top[i]), join_sum[i]);
      if (bad_any) join_sum[i] = NAN;
      if (split && kg2 == 0 && g2 == 0)
        __builtin_amdgcn_raw_buffer_store_b64(
            u32x2{__builtin_bit_cast(uint32_t, join_top[i]), __builtin_bit_cast(uint32_t, join_sum[i])}, pr,
            4 * (part_of(k) + COLS * D + 2 * col), 0, kSc1);
    }
#pragma unroll
    for (int n0 = 0; n0 < NT; n0 += C::JOIN) {
      if (n0 > 0) __syncthreads();
      float* mine_o = buf + w2 * (C::JOIN * NN * C::UNIT) + 4 * lane2;
#pragma unroll
      for (int i = n0; i < n0 + C::JOIN; ++i) {
        const float f = fast_exp2(m[i] - join_top[i]);
#pragma unroll
        for (int j = 0; j < NN; ++j)
          *reinterpret_cast<floatx4*>(mine_o + ((i - n0) * NN + j) * C::UNIT) = acc[i][j] * f;
        if (__builtin_expect(odd != 0, 0))
          for (int left = static_cast<int>(odd); left != 0; left &= left - 1)
            add_keys(i, 32 * (c0 + kg2 + KG * (count - 1 - __builtin_ctz(left))), m[i], f,
                     mine_o + (i - n0) * NN * C::UNIT);
      }
      __syncthreads();
      // Unit u KG + kg of the tiles is this wave's to add up.
#pragma unroll
      for (int u = 0; u < (C::JOIN * NN + KG - 1) / KG; ++u) {
        const int unit = u * KG + kg2;
        if (unit < C::JOIN * NN) {
          floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kk = 0; kk < KG; ++kk)
            o += *reinterpret_cast<const floatx4*>(buf + ((kk * WC + cw2) * (C::JOIN * NN) + unit) * C::UNIT + 4 * lane2);
          const int i = unit / NN, j = unit % NN;  // of the JOIN tiles
          float sum = join_sum[n0];
#pragma unroll
          for (int ii = 1; ii < C::JOIN; ++ii) sum = i == ii ? join_sum[n0 + ii] : sum;
          if (C::KEEP) own[n0 * NN / KG + u] = o;
          if (!split)
            write(n0 + i, j, o, inverse(sum));
          else
            __builtin_amdgcn_raw_buffer_store_b128(
                __builtin_bit_cast(u32x4, o), pr,
                4 * (part_of(k) + ((cw2 * NT + n0) * NN + unit) * C::UNIT + 4 * lane2), 0, kSc1);
        }
      }
    }
    if (!split) {
      __syncthreads();  // the ring and the maxima are the next group's
      continue;
    }

    // The last of the group's workgroups to arrive joins its ranges, in their order.
    // A partial is acknowledged (device scope) before its arrival is counted.
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    if (tid2 == 0)
      last = __hip_atomic_fetch_add(&p.counters[a], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b - a;
    __syncthreads();
    if (last) {
      const int ranges = b - a + 1;
      // AT_ONCE ranges' loads are in flight together, the first beside the work on the weights.
      constexpr int AT_ONCE = NT > 2 ? 1 : C::OWN >= 8 ? 2 : 16 / C::OWN;
      floatx4 first[AT_ONCE][C::OWN];
      auto load_parts = [&](int r0, floatx4 (&part)[AT_ONCE][C::OWN]) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          if (r0 + j < ranges && !(C::KEEP && r0 + j == k - a)) {
#pragma unroll
            for (int u = 0; u < C::OWN; ++u) {
              const int unit = u * KG + kg2 < NT * NN ? u * KG + kg2 : 0;
              const int from = 4 * (part_of(a + r0 + j) + (cw2 * NT * NN + unit) * C::UNIT + 4 * lane2);
              part[j][u] = floatx4{ld_sc1(pr, from), ld_sc1(pr, from + 4), ld_sc1(pr, from + 8), ld_sc1(pr, from + 12)};
            }
          } else if (C::KEEP) {
#pragma unroll
            for (int u = 0; u < C::OWN; ++u) part[j][u] = own[u];
          }
        }
      };
      // Every range's maximum and sum of every column, then its weight, in LDS.
      for (int x = tid2; x < ranges * COLS; x += C::THREADS) {
        const int from = 4 * (part_of(a + x / COLS) + COLS * D + 2 * (x % COLS));
        buf[x] = ld_sc1(pr, from);
        buf[kMostRanges * COLS + x] = ld_sc1(pr, from + 4);
      }
      load_parts(0, first);
      __syncthreads();
      if (tid2 < COLS) {
        float top = kNoScore, sum = 0.f;
        for (int r = 0; r < ranges; ++r) top = fmaxf(top, buf[r * COLS + tid2]);
        for (int r = 0; r < ranges; ++r) {
          const float f = fast_exp2(buf[r * COLS + tid2] - top);
          buf[r * COLS + tid2] = f;
          sum = __builtin_fmaf(buf[kMostRanges * COLS + r * COLS + tid2], f, sum);
        }
        maxima[0][tid2] = inverse(sum);
      }
      __syncthreads();
      floatx4 o[C::OWN];
#pragma unroll
      for (int u = 0; u < C::OWN; ++u) o[u] = floatx4{0.f, 0.f, 0.f, 0.f};
      auto add_parts = [&](int r0, const floatx4 (&part)[AT_ONCE][C::OWN]) {
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          if (r0 + j < ranges) {
#pragma unroll
            for (int u = 0; u < C::OWN; ++u) {
              const float f = buf[(r0 + j) * COLS + (cw2 * NT + (u * KG + kg2) / NN % NT) * 16 + c2];
#pragma unroll
              for (int r = 0; r < 4; ++r) o[u][r] = __builtin_fmaf(part[j][u][r], f, o[u][r]);
            }
          }
        }
      };
      add_parts(0, first);
      for (int r0 = AT_ONCE; r0 < ranges; r0 += AT_ONCE) {
        floatx4 part[AT_ONCE][C::OWN];
        load_parts(r0, part);
        add_parts(r0, part);
      }
#pragma unroll
      for (int u = 0; u < C::OWN; ++u) {
        const int unit = u * KG + kg2;
        if (unit < NT * NN) write(unit / NN, unit % NN, o[u], maxima[0][(cw2 * NT + unit / NN) * 16 + c2]);
      }
      if (tid2 == 0) __hip_atomic_store(&p.counters[a], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------

bool takes_tiles(int head_dim, int block_size, int group, int dtype) {
  return (dtype == NS_DTYPE_F16 || dtype == NS_DTYPE_BF16) && (head_dim == 64 || head_dim == 128) &&
         block_size % 16 == 0 && group <= 1024;
}

int device_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
    return 256;
  return n;
}

// Workgroups that the device holds at once, in whole rounds of the XCDs.
int places() { return (device_cus() + 7) / 8 * 8; }

// Column tiles that a kernel's blocks should hold at least: those of the widest sequence
// over the number of its blocks.  Wide blocks load K and V for more columns at once, narrow
// ones leave more groups to work on at the same time: as wide as leaves a quarter of the
// device's workgroups a group.  The kernels come in a few widths, so that a sequence's last
// block may hold fewer columns than the others (28 tiles in blocks of 8: 8, 8, 8 and 4).
int tiles_of(int num_seqs, int num_kv_heads, int max_rows, int group, int head_dim) {
  const int64_t rows = max_rows < 1 ? 1 : max_rows < kRows ? max_rows : kRows;
  const int64_t tiles = (rows * group + 15) / 16;
  int64_t blocks = 0;
  for (int most = head_dim == 64 ? 16 : 8; most >= 2; most /= 2) {
    blocks = (tiles + most - 1) / most;
    if (num_seqs * blocks * num_kv_heads * 4 >= places()) break;
  }
  return static_cast<int>((tiles + blocks - 1) / blocks);
}

// The kernels, by head size and tiles: key groups, column waves and tiles of a wave.
template <int D, class F>
auto with_shape(int tiles, F&& f) {
  if constexpr (D == 64) {
    if (tiles <= 1) return f(Cfg<64, 8, 1, 1>{});
    if (tiles <= 2) return f(Cfg<64, 8, 1, 2>{});
    if (tiles <= 4) return f(Cfg<64, 4, 2, 2>{});
    if (tiles <= 8) return f(Cfg<64, 2, 4, 2>{});
    return f(Cfg<64, 2, 4, 4>{});
  } else {
    if (tiles <= 1) return f(Cfg<128, 4, 1, 1>{});
    if (tiles <= 2) return f(Cfg<128, 4, 1, 2>{});
    if (tiles <= 4) return f(Cfg<128, 4, 2, 2>{});
    return f(Cfg<128, 2, 4, 2>{});
  }
}

size_t workspace_bytes_of(int head_dim, int tiles) {
  auto words = [](auto c) { return static_cast<size_t>(decltype(c)::PART); };
  return static_cast<size_t>(2) * places() * 4 * (head_dim == 64 ? with_shape<64>(tiles, words) : with_shape<128>(tiles, words));
}

template <class DT, int D>
hipError_t launch_tiles(const TreeParams& p, int tiles, hipStream_t stream) {
  return with_shape<D>(tiles, [&](auto c) {
    using C = decltype(c);
    // A launch's line of work is counted in 32 bits: as many sequences as it is sure to hold.
    const int64_t groups = (static_cast<int64_t>(kRows) * p.group + C::COLS - 1) / C::COLS * p.num_kv_heads;
    const int64_t line = groups * (p.max_ctx / 32 + 1 + kGroupCost);
    const int64_t fits = (int64_t{1} << 30) / line;
    if (fits < 1) return hipErrorNotSupported;
    const int most = static_cast<int>(fits < kSeqs ? fits : kSeqs);
    TreeParams part = p;
    void* args[] = {&part};
    for (int s = 0; s < p.num_seqs; s += most) {
      part.first_seq = s;
      part.num_seqs = p.num_seqs - s < most ? p.num_seqs - s : most;
      const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&tree_attention_kernel<DT, C>),
                                           dim3(static_cast<unsigned>(places())), dim3(C::THREADS), args, 0, stream);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  });
}

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

bool sizes_ok(int num_seqs, int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size) {
  return num_seqs >= 0 && num_tokens >= 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 &&
         head_dim > 0 && block_size > 0;
}

}  // namespace
}  // namespace ns

extern "C" int ns_paged_attention_tree_counters(void) { return ns::places(); }

extern "C" size_t ns_paged_attention_tree_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                                         int block_size, int max_query_len, int64_t num_tokens,
                                                         int dtype) {
  using namespace ns;
  if (!sizes_ok(num_seqs, num_tokens, num_heads, num_kv_heads, head_dim, block_size) || num_seqs == 0 ||
      num_tokens == 0 || !takes_tiles(head_dim, block_size, num_heads / num_kv_heads, dtype))
    return 0;
  return workspace_bytes_of(head_dim, tiles_of(num_seqs, num_kv_heads, max_query_len, num_heads / num_kv_heads, head_dim));
}

extern "C" int ns_paged_attention_tree(void* out, const void* query,
                                       const void* k_cache, const void* v_cache,
                                       const void* block_tables, int64_t block_table_stride,
                                       int64_t block_table_width, int block_tables_is_int64,
                                       const void* seq_lens, int seq_lens_is_int64,
                                       const void* query_start_loc, int query_start_loc_is_int64,
                                       const int64_t* tree_mask,
                                       int num_seqs, int64_t num_tokens, int max_query_len, int max_seq_len,
                                       int num_heads, int num_kv_heads, int head_dim,
                                       int block_size, int64_t num_blocks,
                                       float scale, int dtype,
                                       int* counters, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ns;
  if (!sizes_ok(num_seqs, num_tokens, num_heads, num_kv_heads, head_dim, block_size) || num_blocks <= 0 ||
      max_query_len < 0 || max_seq_len < 0 || !(fabsf(scale) < INFINITY))
    return NS_ERR_INVALID_ARG;
  if (dtype != NS_DTYPE_F32 && dtype != NS_DTYPE_F16 && dtype != NS_DTYPE_BF16) return NS_ERR_UNSUPPORTED;
  if (head_dim > kMaxHeadDim || max_query_len > kRows) return NS_ERR_UNSUPPORTED;
  if (num_seqs == 0 || num_tokens == 0) return NS_OK;
  if (!out || !query || !k_cache || !v_cache || !block_tables || !seq_lens || !tree_mask) return NS_ERR_INVALID_ARG;
  if (!query_start_loc && num_tokens != num_seqs) return NS_ERR_INVALID_ARG;
  if (block_table_width <= 0 || block_table_stride < block_table_width) return NS_ERR_INVALID_ARG;
  const int group = num_heads / num_kv_heads;
  const bool tiles = takes_tiles(head_dim, block_size, group, dtype);
  const size_t align = tiles ? 16 : dtype == NS_DTYPE_F32 ? 4 : 2;
  if (misaligned(out, align) || misaligned(query, align) || misaligned(k_cache, align) || misaligned(v_cache, align) ||
      misaligned(block_tables, block_tables_is_int64 ? 8 : 4) || misaligned(seq_lens, seq_lens_is_int64 ? 8 : 4) ||
      misaligned(query_start_loc, query_start_loc_is_int64 ? 8 : 4) || misaligned(tree_mask, 8))
    return NS_ERR_INVALID_ARG;
  // Rows, columns, items and a context's tokens are counted in 32 bits.
  if (max_seq_len > 1 << 30 || num_heads > 65535 || num_tokens > 0x3FFFFFFF / num_heads ||
      num_seqs > 0x3FFFFFFF / num_heads || static_cast<int64_t>(num_kv_heads) * head_dim * 2 * 16 > 0x7FFFFFFF)
    return NS_ERR_UNSUPPORTED;
  if (!tiles && num_tokens > kMostPlainRows) return NS_ERR_UNSUPPORTED;
  TreeParams p;
  p.out = static_cast<char*>(out);
  p.query = static_cast<const char*>(query);
  p.k_cache = static_cast<const char*>(k_cache);
  p.v_cache = static_cast<const char*>(v_cache);
  p.bt = block_tables;
  p.bt_stride = block_table_stride;
  p.seq_lens = seq_lens;
  p.qsl = query_start_loc;
  p.mask = tree_mask;
  p.bt64 = block_tables_is_int64;
  p.sl64 = seq_lens_is_int64;
  p.qsl64 = query_start_loc_is_int64;
  p.num_seqs = num_seqs;
  p.first_seq = 0;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = group;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_tokens = num_tokens;
  p.num_blocks = num_blocks;
  const int64_t held = block_table_width > (int64_t{1} << 30) ? max_seq_len : block_table_width * block_size;
  p.max_ctx = max_seq_len < held ? max_seq_len : held;
  p.scale = scale;
  // For keys below 2^31 and 2^(l - 1) < block_size <= 2^l: 2^(31 + l) / block_size, rounded up.
  int l = 1;
  while ((int64_t{1} << l) < block_size) ++l;
  p.block_mul = static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + block_size - 1) / block_size);
  p.block_shift = l - 1;
  p.by_group = 1.f / static_cast<float>(group);
  p.partials = static_cast<float*>(workspace);
  p.counters = counters;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e;
  if (!tiles) {
    e = dtype == NS_DTYPE_F32   ? launch_generic<float>(p, st)
        : dtype == NS_DTYPE_F16 ? launch_generic<_Float16>(p, st)
                                : launch_generic<__bf16>(p, st);
  } else {
    const int nt = tiles_of(num_seqs, num_kv_heads, max_query_len, group, head_dim);
    if (!counters || misaligned(counters, 4) || !workspace || misaligned(workspace, 16) ||
        workspace_bytes < workspace_bytes_of(head_dim, nt))
      return NS_ERR_WORKSPACE;
    e = dtype == NS_DTYPE_F16 ? (head_dim == 64 ? launch_tiles<F16, 64>(p, nt, st) : launch_tiles<F16, 128>(p, nt, st))
                              : (head_dim == 64 ? launch_tiles<BF16, 64>(p, nt, st) : launch_tiles<BF16, 128>(p, nt, st));
  }
  return e == hipSuccess ? NS_OK : e == hipErrorNotSupported ? NS_ERR_UNSUPPORTED : NS_ERR_HIP;
}
