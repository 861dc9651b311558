// Paged attention for trees of drafted tokens.
//
// A sequence's query rows are the tree's nodes: row j of a sequence with context
// length L (its rows included) and q rows sees every key before the rows,
// 0 .. L - q - 1, and key L - q + i where bit i of its mask is set.  KV head of
// query head h is h / (Hq / Hkv); softmax and sums are float32; a row without keys
// is zero.
#include <math.h>

#include "ns_common.h"

namespace ns {
namespace {

constexpr int kRows = 64;        // rows of a sequence that a mask can name
constexpr int kSeqs = 512;       // sequences of a launch (their schedule is held in LDS)
constexpr int kMaxHeadDim = 256;

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
  // Matrix-core kernel.
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
// weighted values into the output dims it owns, one key at a time.  Plain: the
// serving shapes run the matrix-core kernel.
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
  if (t < r.row0 || t >= r.row0 + r.ql) return;  // a row of no sequence is left as it is
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
    if (ok && key >= base) {
      const int64_t i = key - base;
      ok = i < kRows && ((mask >> i) & 1);
    }
    if (ok) {
      const int64_t blk = load_index(p.bt, bt_row + key / bs, p.bt64);
      if (blk < 0 || blk >= p.num_blocks) {
        bad = 1;
        ok = false;
      } else {
        row = ((blk * bs + key % bs) * p.num_kv_heads + kvh) * D;
      }
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
// A sequence's rows times the heads of one KV head are columns, 16 a tile.  A group
// is up to NT tiles of columns of one (sequence, KV head); a workgroup takes a range
// of a group's keys, and a wave the range's chunks of 32 keys w, w + 4, ... for all of
// the group's columns, so that every row of K and V is loaded once for up to 16 NT
// rows of the product, and the waves meet once, at the range's end.  K and V come by
// LDS-DMA into a ring of each wave's own, S^T = K Q^T and O^T = V^T P^T on
// v_mfma_f32_16x16x32.  The result layout of the first product (keys 4 g + r of
// column lane % 16 in lane group g) is the operand layout of the second.
//
// The probabilities enter the second product in the model's dtype, and their sum
// is taken by the same product with a tile of ones, so that a rounding acts on both.
//
// Work is cut evenly: the groups' chunks, and kGroupCost for what a group costs
// beside them, are laid end to end, and workgroup k takes the k-th equal share of
// that line, whatever it covers: parts of groups, whole ones, or both.  Cuts move to
// whole rounds of the four waves.  A group that a cut falls into is joined by the last
// of its workgroups to finish.  Every workgroup works its share out of the device's
// lengths for itself.

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kMostRanges = 32;  // of a group: what the last workgroup has to join
constexpr int kGroupCost = 4;    // in chunks
constexpr int kLeastShare = 8;   // chunks

template <int D, int NT>
struct Cfg {
  static constexpr int COLS = 16 * NT;
  static constexpr int CPR = D / 8;             // 16-byte units of a row
  static constexpr int KPI = 64 / CPR;          // rows of a tile that one load brings
  static constexpr int LPT = 16 / KPI;          // loads of a tile
  static constexpr int NK = 8 / KPI;            // loads until K's swizzle repeats
  static constexpr int TILE_B = 32 * D * 2;     // K or V of a chunk
  static constexpr int SLOT_B = 2 * TILE_B;
  static constexpr int R = 2;                   // chunks in the ring
  static constexpr int PER_CHUNK = 4 * LPT;     // loads of a chunk
  static constexpr int NC = D / 32, NN = D / 16;
  static constexpr int RING = kWaves * R * SLOT_B;
  static constexpr int PART = COLS * (D + 2);   // words of a slot: outputs, then (maximum, sum) of every column
  // The waves meet a group of column tiles at a time, as many as fit the ring.
  static constexpr int JOIN = RING / (kWaves * 16 * D * 4) < NT ? RING / (kWaves * 16 * D * 4) : NT;
  static constexpr int OWN = COLS * (D / 4) / kThreads;  // float4 of the output per thread
  static_assert(JOIN >= 1, "a column tile of every wave fits the ring");
  static_assert(2 * kMostRanges * COLS * 4 <= RING, "the ranges' maxima and sums fit the ring");
};

constexpr int kSc1 = 16;                  // cache-policy bit SC1 of gfx950 buffer operations: device scope
constexpr int kBufferWord3 = 0x00020000;  // raw 32-bit buffer descriptor, word 3

template <int N>
__device__ __forceinline__ void vector_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
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

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ int64_t lane_value64(int64_t x, int lane) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ int64_t shuffle_up64(int64_t x, int by) {
  const uint32_t lo = static_cast<uint32_t>(__shfl_up(static_cast<int>(x), by));
  const uint32_t hi = static_cast<uint32_t>(__shfl_up(static_cast<int>(x >> 32), by));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
// x / y for x >= 0, y > 0: the quotient in float32, put right.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  int64_t q = static_cast<int64_t>(static_cast<float>(x) / static_cast<float>(y));
  while (q * y > x) --q;
  while ((q + 1) * y <= x) ++q;
  return q;
}

// The sequences of a launch along the line of work, from the device's lengths.  Up to
// 64 of them live in the lanes of every wave; more are held in LDS.
struct Held {
  int64_t start[kSeqs];
  int row0[kSeqs], ql[kSeqs], len[kSeqs];
  int64_t sums[kWaves];
  int most[kWaves];
};

template <int COLS>
struct Line {
  int64_t start;          // this lane's sequence (num_seqs <= 64)
  int row0, ql, len;
  Held* held;             // otherwise
  int num_seqs, heads, group;
  int64_t total;
  int most;               // weight of the longest group

  __device__ __forceinline__ int weight(int len_) const { return ((len_ + 31) >> 5) + kGroupCost; }
  __device__ __forceinline__ int groups(int ql_) const { return (ql_ * group + COLS - 1) / COLS * heads; }

  __device__ __forceinline__ void scan(int64_t x, int m, int lane, int64_t& before, int64_t& all, int& longest) {
    int64_t y = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t z = shuffle_up64(y, off);
      if (lane >= off) y += z;
      m = max(m, __shfl_xor(m, off));
    }
    before = y - x;
    all = lane_value64(y, 63);
    longest = __builtin_amdgcn_readfirstlane(m);
  }

  __device__ __forceinline__ void make(const TreeParams& p, Held& h) {
    const int lane = threadIdx.x & 63;
    held = &h;
    num_seqs = p.num_seqs;
    heads = p.num_kv_heads;
    group = p.group;
    row0 = ql = len = 0;
    if (num_seqs <= 64) {
      int64_t x = 0;
      int m = 0;
      if (lane < num_seqs) {
        const SeqRows r = rows_of(p, lane);
        row0 = static_cast<int>(r.row0);
        ql = static_cast<int>(r.ql);
        len = static_cast<int>(r.len);
        m = ql > 0 ? weight(len) : 0;
        x = static_cast<int64_t>(groups(ql)) * m;
      }
      scan(x, m, lane, start, total, most);
      return;
    }
    constexpr int PER = kSeqs / kThreads;
    const int w = threadIdx.x >> 6;
    int64_t x[PER], sum = 0;
    int m = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = PER * static_cast<int>(threadIdx.x) + i;
      x[i] = 0;
      if (s < num_seqs) {
        const SeqRows r = rows_of(p, s);
        h.row0[s] = static_cast<int>(r.row0);
        h.ql[s] = static_cast<int>(r.ql);
        h.len[s] = static_cast<int>(r.len);
        const int wt = r.ql > 0 ? weight(static_cast<int>(r.len)) : 0;
        m = max(m, wt);
        x[i] = static_cast<int64_t>(groups(static_cast<int>(r.ql))) * wt;
        sum += x[i];
      }
    }
    int64_t before, all;
    scan(sum, m, lane, before, all, most);
    if (lane == 0) {
      h.sums[w] = all;
      h.most[w] = most;
    }
    __syncthreads();
    total = 0;
    most = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < w) before += h.sums[i];
      total += h.sums[i];
      most = max(most, h.most[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = PER * static_cast<int>(threadIdx.x) + i;
      if (s < num_seqs) h.start[s] = before;
      before += x[i];
    }
    __syncthreads();
    total = uniform64(total);
    most = __builtin_amdgcn_readfirstlane(most);
  }

  __device__ __forceinline__ void get(int s, int64_t& start_, int& row0_, int& ql_, int& len_) const {
    if (num_seqs <= 64) {
      start_ = lane_value64(start, s);
      row0_ = __builtin_amdgcn_readlane(row0, s);
      ql_ = __builtin_amdgcn_readlane(ql, s);
      len_ = __builtin_amdgcn_readlane(len, s);
    } else {
      start_ = uniform64(held->start[s]);
      row0_ = __builtin_amdgcn_readfirstlane(held->row0[s]);
      ql_ = __builtin_amdgcn_readfirstlane(held->ql[s]);
      len_ = __builtin_amdgcn_readfirstlane(held->len[s]);
    }
  }

  // The sequence that place `at` of the line lies in: the last that starts there or before.
  __device__ __forceinline__ int find(int64_t at) const {
    const int lane = threadIdx.x & 63;
    if (num_seqs <= 64) return 63 - __builtin_clzll(__builtin_amdgcn_ballot_w64(lane < num_seqs && start <= at));
    int n = -1;
    for (int s0 = 0; s0 < num_seqs; s0 += 64)
      n += __popcll(__builtin_amdgcn_ballot_w64(s0 + lane < num_seqs && held->start[s0 + lane < num_seqs ? s0 + lane : 0] <= at));
    return n;
  }
};

template <class DT, int D, int NT>
__global__ __launch_bounds__(kThreads, D == 64 ? 2 : 1) void tree_attention_kernel(TreeParams p) {
  using C = Cfg<D, NT>;
  using T = typename DT::T;
  using V8 = typename DT::vec8;
  constexpr int NC = C::NC, NN = C::NN, LPT = C::LPT, KPI = C::KPI, CPR = C::CPR, NK = C::NK;
  __shared__ __attribute__((aligned(1024))) char smem[C::RING];
  __shared__ Held held;
  __shared__ float maxima[kWaves][C::COLS], sums[kWaves][C::COLS];
  __shared__ int bads[kWaves];
  __shared__ int last;

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c16 = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = p.group, Hkv = p.num_kv_heads;

  Line<C::COLS> line;
  line.make(p, held);
  // Shares: one a workgroup, but none too small, and no group in more than kMostRanges of them.
  const int grid = static_cast<int>(gridDim.x);
  int64_t share = quotient(line.total + grid - 1, grid);
  const int least = line.most / (kMostRanges - 2) + 1;
  share = share > least ? share : least;
  share = share > kLeastShare ? share : kLeastShare;
  // Neighbouring shares, which read the same keys where a sequence has several
  // groups of columns, go to one XCD (workgroups go to the eight in turn).
  const int shares = static_cast<int>(quotient(line.total + share - 1, share));
  const int per_xcd = (shares + 7) >> 3;
  const int k = static_cast<int>(blockIdx.x & 7) * per_xcd + static_cast<int>(blockIdx.x >> 3);
  if (static_cast<int>(blockIdx.x >> 3) >= per_xcd || k >= shares) return;

  const float scale = fabsf(p.scale) * 1.4426950408889634f;
  const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;  // a negative scale turns the query around, exactly
  char* ring = smem + w * (C::R * C::SLOT_B);
  const uint32_t stride = static_cast<uint32_t>(Hkv) * D * 2;  // bytes between a block's token rows

  // A lane's part of a load: its unit of its row, where it lies in memory.
  uint32_t koff[NK], voff[NK];
#pragma unroll
  for (int u = 0; u < NK; ++u) {
    const int key = u * KPI + lane / CPR, unit = lane % CPR;
    koff[u] = (lane / CPR) * stride + ((unit ^ k_swizzle(key)) << 4);
    voff[u] = (lane / CPR) * stride + ((unit ^ v_swizzle<D>(key)) << 4);
  }
  // Operand reads within a chunk.  K: key 16 h + c16, unit 4 c + g.  V^T: keys
  // 16 h + 4 g + e of dims 16 n + c16 (ds_read_b64_tr_b16 gives lane i of a 16-lane
  // group, as element e, element i & 3 of the 8 bytes of lane (i >> 2) + 4 e).
  uint32_t kread[NC], vread;
#pragma unroll
  for (int c = 0; c < NC; ++c) kread[c] = c16 * (D * 2) + (((4 * c + g) ^ k_swizzle(c16)) << 4);
  const int vkey = 4 * g + (c16 >> 2);
  vread = vkey * (D * 2) + ((((c16 & 3) >> 1) ^ v_swizzle<D>(vkey)) << 4) + (c16 & 1) * 8;

  int s = line.find(k * share);
  int64_t start;
  int row0, ql, len;
  line.get(s, start, row0, ql, len);
  int64_t gi = quotient(k * share - start, line.weight(len));
  for (;; ++gi) {
    while (gi >= line.groups(ql)) {
      if (++s >= p.num_seqs) return;
      line.get(s, start, row0, ql, len);
      gi = 0;
    }
    // The group's place on the line, the workgroups a .. b that it falls to, and
    // the chunks c0 .. c1 of this one.
    const int n = (len + 31) >> 5;
    const int64_t gs = start + gi * line.weight(len);
    const int a = static_cast<int>(quotient(gs + 1, share));
    if (a > k) return;
    const int e = (n + 3) / 4 * 4 - 3;
    int b = e > 0 ? static_cast<int>(quotient(gs + e, share)) : a;
    b = b > a ? b : a;
    if (k > b) continue;
    auto cut = [&](int kk) { return static_cast<int>(kk * share - gs + 2) >> 2 << 2; };
    const int c0 = k == a ? 0 : cut(k), c1 = k == b ? n : cut(k + 1);
    const int base = len - ql;
    const int cols = ql * G, cbs = (cols + C::COLS - 1) / C::COLS;
    const int kvh = static_cast<int>(gi) / cbs, cb = static_cast<int>(gi) % cbs;
    const int t1 = 32 * c1 < len ? 32 * c1 : len;
    const int mine = c1 - c0 > w ? (c1 - c0 - w + kWaves - 1) / kWaves : 0;

    // The columns' query rows and masks.
    V8 q[NT][NC];
    uint64_t mask[NT];
    int bad = 0;
    float m[NT];
    floatx4 acc[NT][NN], l[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      int c = cb * C::COLS + 16 * n + c16;
      c = c < cols ? c : cols - 1;
      const int64_t row = row0 + c / G;
      const char* qr = p.query + ((row * p.num_heads + kvh * G + c % G) * D + 8 * g) * 2;
      mask[n] = static_cast<uint64_t>(p.mask[row]);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        u32x4 x = *reinterpret_cast<const u32x4*>(qr + 64 * i);
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) x[e2] ^= flip;
        q[n][i] = __builtin_bit_cast(V8, x);
      }
      m[n] = -INFINITY;
      l[n] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NN; ++i) acc[n][i] = floatx4{0.f, 0.f, 0.f, 0.f};
    }

    // Lane l: where tile l & 1 of this wave's step l / 2 of a window of 32 steps
    // lies, as bytes from the start of a cache.
    uint32_t at_lo = 0, at_hi = 0;
    auto window = [&](int step) {
      const int64_t bt_row = static_cast<int64_t>(p.first_seq + s) * p.bt_stride;
      int key = 32 * (c0 + w + kWaves * (step + (lane >> 1))) + 16 * (lane & 1);
      key = key < t1 ? key : (t1 - 1) & ~15;  // a tile past the range repeats the last
      int64_t blk = load_index(p.bt, bt_row + key / p.block_size, p.bt64);
      if (blk < 0 || blk >= p.num_blocks) {
        bad = 1;
        blk = 0;
      }
      const uint64_t at = ((static_cast<uint64_t>(blk) * p.block_size + key % p.block_size) * Hkv + kvh) * (D * 2);
      at_lo = static_cast<uint32_t>(at);
      at_hi = static_cast<uint32_t>(at >> 32);
    };
    auto issue = [&](int step) {
      if ((step & 31) == 0) window(step);
      char* to = ring + (step % C::R) * C::SLOT_B;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int from = 2 * (step & 31) + h;
        const uint64_t at =
            (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at_hi), from))) << 32) |
            static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at_lo), from));
        const char* kp = p.k_cache + at;
        const char* vp = p.v_cache + at;
#pragma unroll
        for (int u = 0; u < LPT; ++u) {
          dma_lds16_off(kp + u * KPI * stride, koff[u % NK], to + (h * LPT + u) * 1024);
          dma_lds16_off(vp + u * KPI * stride, voff[u % NK], to + C::TILE_B + (h * LPT + u) * 1024);
        }
      }
    };

    auto step_of = [&](int step) {
      const int tb = 32 * (c0 + w + kWaves * step);
      const char* kt = ring + (step % C::R) * C::SLOT_B;
      const char* vt = kt + C::TILE_B;
      u32x4 kraw[2][NC];
      u32x2 vraw[NN][2];
      const uint32_t ka = lds_addr(kt), va = lds_addr(vt) + vread;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        kraw[0][c] = ds_read_b128_at<0>(ka + kread[c]);
        kraw[1][c] = ds_read_b128_at<16 * D * 2>(ka + kread[c]);
      }
      // Unit 2 n of a row: the swizzle touches bits above the lowest, and so is an exclusive or of the address.
#pragma unroll
      for (int n = 0; n < NN; ++n) {
        const uint32_t a = va ^ (n << 5);
        vraw[n][0] = ds_read_tr16_b64_at<0>(a);
        vraw[n][1] = ds_read_tr16_b64_at<16 * D * 2>(a);
      }
      lds_wait_all();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < NC; ++c) lds_ready(kraw[h][c]);
#pragma unroll
      for (int n = 0; n < NN; ++n) {
        lds_ready(vraw[n][0]);
        lds_ready(vraw[n][1]);
      }
      const bool tail = tb + 32 > base || tb + 32 > len;
      // Keys that not every column sees: V of a key past the end is taken as zero, and
      // a chunk with an element of V that is not finite is added one key at a time, so
      // that it reaches only the rows that see it.
      bool odd = false;
      if (tail) {
        const int left = len - tb;
        int wild = 0;
#pragma unroll
        for (int n = 0; n < NN; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = 16 * h + 4 * g + 2 * e;
              uint32_t x = vraw[n][h][e];
              x = key + 1 < left ? x : key < left ? x & 0xFFFFu : 0u;
              vraw[n][h][e] = x;
              constexpr uint32_t top = DT::code == NS_DTYPE_F16 ? 0x7C00u : 0x7F80u;
              wild |= (x & top) == top || (x & (top << 16)) == top << 16;
            }
        odd = __builtin_amdgcn_ballot_w64(wild != 0) != 0;
      }
      // The chunk is in registers (odd ones are read again): the next but one takes its place.
      const int next = step + C::R;
      if (!odd && next < mine) issue(next);
      V8 ones;
#pragma unroll
      for (int e = 0; e < 8; ++e) ones[e] = static_cast<T>(1.f);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        floatx4 sacc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sacc[h] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < NC; ++c) sacc[h] = mfma16x16x32(DT{}, __builtin_bit_cast(V8, kraw[h][c]), q[n][c], sacc[h]);
        }
        uint32_t seen = ~0u;
        if (tail) {
          seen = seen_of(mask[n], tb, base, len) >> (4 * g);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) sacc[h][r] = (seen >> (16 * h + r)) & 1 ? sacc[h][r] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, sacc[h][r]);
        top = group4_max_swap(top);
        top = top == -INFINITY ? top : top * scale;
        if (__builtin_amdgcn_ballot_w64(top > m[n]) != 0) {
          const float next_m = fmaxf(m[n], top);
          const float alpha = next_m == -INFINITY ? 1.f : fast_exp2(m[n] - next_m);
          m[n] = next_m;
          l[n] *= alpha;
#pragma unroll
          for (int i = 0; i < NN; ++i) acc[n][i] *= alpha;
        }
        const float ref = m[n] == -INFINITY ? 0.f : m[n];
        float pr[2][4];
        V8 pt;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = fast_exp2(__builtin_fmaf(sacc[h][r], scale, -ref));
            if (tail) x = (seen >> (16 * h + r)) & 1 ? x : 0.f;
            pr[h][r] = x;
            pt[4 * h + r] = static_cast<T>(x);
          }
        l[n] = mfma16x16x32(DT{}, ones, pt, l[n]);
        if (!odd) {
#pragma unroll
          for (int i = 0; i < NN; ++i) {
            const V8 v = __builtin_bit_cast(V8, u32x4{vraw[i][0][0], vraw[i][0][1], vraw[i][1][0], vraw[i][1][1]});
            acc[n][i] = mfma16x16x32(DT{}, v, pt, acc[n][i]);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              for (int gk = 0; gk < 4; ++gk) {
                const int key = 16 * h + 4 * gk + r;
                const float x = __shfl(static_cast<float>(static_cast<T>(pr[h][r])), 16 * gk + c16);
                const int sees = __shfl(static_cast<int>((seen >> (16 * h + r)) & 1), 16 * gk + c16);
                if (sees) {
#pragma unroll
                  for (int i = 0; i < NN; ++i) {
                    const int unit = 2 * i + (g >> 1);
                    const typename DT::vec4 v = *reinterpret_cast<const typename DT::vec4*>(
                        vt + key * (D * 2) + ((unit ^ v_swizzle<D>(key)) << 4) + (g & 1) * 8);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                      acc[n][i][e] = __builtin_fmaf(x, static_cast<float>(v[e]), acc[n][i][e]);
                  }
                }
              }
        }
      }
      if (odd) {
        lds_wait_all();
        if (next < mine) issue(next);
      }
    };

    if (mine > 0) issue(0);
    if (mine > 1) issue(1);
    for (int step = 0; step < mine; ++step) {
      if (step + 1 < mine) vector_wait<C::PER_CHUNK>();
      else vector_wait<0>();
      step_of(step);
    }

    // The waves' states meet in LDS, JOIN column tiles at a time.  The ring is free
    // when every wave is here.
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        maxima[w][16 * i + c16] = m[i];
        sums[w][16 * i + c16] = l[i][0];
      }
    }
    {
      const int wave_bad = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
      if (lane == 0) bads[w] = wave_bad;
    }
    const bool split = b > a;
    // A workgroup has at most one cut group that it begins (its last: slot 2 k + 1)
    // and one that it does not (its first: slot 2 k).
    auto slot_of = [&](int kk) { return kk == a ? 2 * kk + 1 : 2 * kk; };
    const __amdgpu_buffer_rsrc_t pr = __builtin_amdgcn_make_buffer_rsrc(
        p.partials + static_cast<int64_t>(2) * a * C::PART, static_cast<short>(0),
        split ? 2 * (b - a + 1) * C::PART * 4 : 0, kBufferWord3);
    auto part_of = [&](int kk) { return (slot_of(kk) - 2 * a) * C::PART; };
    T* out = reinterpret_cast<T*>(p.out);
    auto write = [&](int col, int f, floatx4 o, float inv) {
      const int c = cb * C::COLS + col;
      const int64_t at = ((static_cast<int64_t>(row0) + c / G) * p.num_heads + kvh * G + c % G) * D + 4 * f;
      typename DT::vec4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = static_cast<T>(o[r] * inv);
      *reinterpret_cast<u32x2*>(out + at) = __builtin_bit_cast(u32x2, v);
    };
    auto inverse = [&](float sum) { return sum > 0.f || sum != sum ? 1.f / sum : 0.f; };  // no key: zero; a NaN stays one
    const int here = cols - cb * C::COLS < C::COLS ? cols - cb * C::COLS : C::COLS;  // columns of the group
#pragma unroll
    for (int n0 = 0; n0 < NT; n0 += C::JOIN) {
      __syncthreads();
      float* mine_o = reinterpret_cast<float*>(smem) + w * (C::JOIN * 16 * D);
#pragma unroll
      for (int i = n0; i < n0 + C::JOIN && i < NT; ++i)
#pragma unroll
        for (int j = 0; j < NN; ++j)
          *reinterpret_cast<floatx4*>(mine_o + (16 * (i - n0) + c16) * D + 4 * ((4 * j + g) ^ c16)) = acc[i][j];
      __syncthreads();
      int bad_any = 0;
#pragma unroll
      for (int ww = 0; ww < kWaves; ++ww) bad_any |= bads[ww];
      for (int x = tid; x < C::JOIN * 16 * (D / 4); x += kThreads) {
        const int col = 16 * n0 + x / (D / 4), f = x % (D / 4);
        if (col >= here) break;
        float mw[kWaves], lw[kWaves], top = -INFINITY;
        floatx4 ow[kWaves];
#pragma unroll
        for (int ww = 0; ww < kWaves; ++ww) {
          mw[ww] = maxima[ww][col];
          lw[ww] = sums[ww][col];
          ow[ww] = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(smem) +
                                                     ww * (C::JOIN * 16 * D) + (col - 16 * n0) * D + 4 * (f ^ (col & 15)));
          top = fmaxf(top, mw[ww]);
        }
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ww = 0; ww < kWaves; ++ww) {
          const float f2 = fast_exp2(mw[ww] - ref);
          sum = __builtin_fmaf(lw[ww], f2, sum);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = __builtin_fmaf(ow[ww][r], f2, o[r]);
        }
        if (bad_any) {
          sum = NAN;
          o = floatx4{NAN, NAN, NAN, NAN};
        }
        if (!split) {
          write(col, f, o, inverse(sum));
        } else {
          const int to = 4 * (part_of(k) + col * D + 4 * f);
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), pr, to, 0, kSc1);
          if (f == 0)
            __builtin_amdgcn_raw_buffer_store_b64(
                u32x2{__builtin_bit_cast(uint32_t, top), __builtin_bit_cast(uint32_t, sum)}, pr,
                4 * (part_of(k) + C::COLS * D + 2 * col), 0, kSc1);
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
    if (tid == 0)
      last = __hip_atomic_fetch_add(&p.counters[a], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b - a;
    __syncthreads();
    if (last) {
      const int ranges = b - a + 1;
      // Every range's maximum and sum of every column, then its weight, in LDS.
      float* ml = reinterpret_cast<float*>(smem);
      for (int x = tid; x < ranges * C::COLS; x += kThreads) {
        const int r = x / C::COLS, col = x % C::COLS;
        if (col < here) {
          const int from = 4 * (part_of(a + r) + C::COLS * D + 2 * col);
          ml[x] = ld_sc1(pr, from);
          ml[kMostRanges * C::COLS + x] = ld_sc1(pr, from + 4);
        }
      }
      __syncthreads();
      if (tid < here) {
        float top = -INFINITY, sum = 0.f;
        for (int r = 0; r < ranges; ++r) top = fmaxf(top, ml[r * C::COLS + tid]);
        const float ref = top == -INFINITY ? 0.f : top;
        for (int r = 0; r < ranges; ++r) {
          const float f2 = fast_exp2(ml[r * C::COLS + tid] - ref);
          ml[r * C::COLS + tid] = f2;
          sum = __builtin_fmaf(ml[kMostRanges * C::COLS + r * C::COLS + tid], f2, sum);
        }
        maxima[0][tid] = inverse(sum);
      }
      __syncthreads();
      floatx4 o[C::OWN];
#pragma unroll
      for (int i = 0; i < C::OWN; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
      constexpr int AT_ONCE = 16 / C::OWN;  // ranges whose loads are in flight together
      for (int r0 = 0; r0 < ranges; r0 += AT_ONCE) {
        floatx4 part[AT_ONCE][C::OWN];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          const int r = r0 + j < ranges ? r0 + j : ranges - 1;
#pragma unroll
          for (int i = 0; i < C::OWN; ++i) {
            const int from = 4 * (part_of(a + r) + 4 * (tid + i * kThreads));
            part[j][i] = floatx4{ld_sc1(pr, from), ld_sc1(pr, from + 4), ld_sc1(pr, from + 8), ld_sc1(pr, from + 12)};
          }
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          if (r0 + j < ranges) {
#pragma unroll
            for (int i = 0; i < C::OWN; ++i) {
              const int col = (tid + i * kThreads) / (D / 4);
              if (col < here) {
                const float f2 = ml[(r0 + j) * C::COLS + col];
#pragma unroll
                for (int r = 0; r < 4; ++r) o[i][r] = __builtin_fmaf(part[j][i][r], f2, o[i][r]);
              }
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < C::OWN; ++i) {
        const int x = tid + i * kThreads, col = x / (D / 4);
        if (col < here) write(col, x % (D / 4), o[i], maxima[0][col]);
      }
      if (tid == 0) __hip_atomic_store(&p.counters[a], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
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

// Column tiles of an item for sequences of up to max_rows rows: those of the widest
// sequence, in equal blocks of at most four.
int tiles_of(int max_rows, int group) {
  const int64_t rows = max_rows < 1 ? 1 : max_rows < kRows ? max_rows : kRows;
  const int64_t tiles = (rows * group + 15) / 16;
  const int64_t blocks = (tiles + 3) / 4;
  return static_cast<int>((tiles + blocks - 1) / blocks);
}

// Workgroups that the device holds at once, in whole rounds of the XCDs.
int places_of(int head_dim) { return (device_cus() + 7) / 8 * 8 * (head_dim == 64 ? 2 : 1); }

size_t slot_bytes(int head_dim, int nt) { return static_cast<size_t>(16) * nt * (head_dim + 2) * 4; }

template <class DT, int D>
hipError_t launch_tiles(const TreeParams& p, int nt, hipStream_t stream) {
  const void* fn = nt == 1   ? reinterpret_cast<const void*>(&tree_attention_kernel<DT, D, 1>)
                   : nt == 2 ? reinterpret_cast<const void*>(&tree_attention_kernel<DT, D, 2>)
                   : nt == 3 ? reinterpret_cast<const void*>(&tree_attention_kernel<DT, D, 3>)
                             : reinterpret_cast<const void*>(&tree_attention_kernel<DT, D, 4>);
  TreeParams part = p;
  void* args[] = {&part};
  for (int s = 0; s < p.num_seqs; s += kSeqs) {
    part.first_seq = s;
    part.num_seqs = p.num_seqs - s < kSeqs ? p.num_seqs - s : kSeqs;
    const hipError_t e = hipLaunchKernel(fn, dim3(static_cast<unsigned>(places_of(D))), dim3(kThreads), args, 0, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

bool sizes_ok(int num_seqs, int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size) {
  return num_seqs >= 0 && num_tokens >= 0 && num_heads > 0 && num_kv_heads > 0 && num_heads % num_kv_heads == 0 &&
         head_dim > 0 && block_size > 0;
}

}  // namespace
}  // namespace ns

extern "C" int ns_paged_attention_tree_counters(void) { return ns::places_of(64); }

extern "C" size_t ns_paged_attention_tree_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                                         int block_size, int max_query_len, int64_t num_tokens,
                                                         int dtype) {
  using namespace ns;
  if (!sizes_ok(num_seqs, num_tokens, num_heads, num_kv_heads, head_dim, block_size) || num_seqs == 0 ||
      num_tokens == 0 || !takes_tiles(head_dim, block_size, num_heads / num_kv_heads, dtype))
    return 0;
  return static_cast<size_t>(2) * places_of(head_dim) *
         slot_bytes(head_dim, tiles_of(max_query_len, num_heads / num_kv_heads));
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
  p.partials = static_cast<float*>(workspace);
  p.counters = counters;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  hipError_t e;
  if (!tiles) {
    e = dtype == NS_DTYPE_F32   ? launch_generic<float>(p, st)
        : dtype == NS_DTYPE_F16 ? launch_generic<_Float16>(p, st)
                                : launch_generic<__bf16>(p, st);
  } else {
    const int nt = tiles_of(max_query_len, group);
    if (!counters || misaligned(counters, 4) || !workspace || misaligned(workspace, 16) ||
        workspace_bytes < static_cast<size_t>(2) * places_of(head_dim) * slot_bytes(head_dim, nt))
      return NS_ERR_WORKSPACE;
    e = dtype == NS_DTYPE_F16 ? (head_dim == 64 ? launch_tiles<F16, 64>(p, nt, st) : launch_tiles<F16, 128>(p, nt, st))
                              : (head_dim == 64 ? launch_tiles<BF16, 64>(p, nt, st) : launch_tiles<BF16, 128>(p, nt, st));
  }
  return e == hipSuccess ? NS_OK : NS_ERR_HIP;
}
