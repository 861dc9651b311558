// sample_rows: one token per row of logits by temperature, top-k, top-p and
// min-p from a given uniform number.
//
// With z the row as float32, z_max its largest and w_i = exp((z_i - z_max) / T),
// order the tokens by z descending, then index ascending.  Every filter keeps a
// prefix of that order: the first k; those with w >= min_p; those with the sum
// of w before them below top_p times the sum over the first k (the first
// always).  The token is the first whose running sum exceeds u times the sum of
// the shortest of these prefixes.
//
// No sort of the row, which is cut into slices:
//   1. every slice's largest element, smallest finite one, and the largest of each
//      group of threads;
//   2. every slice's histogram over z_max - z in 1024 steps, counts and sums of
//      w, and its part of the min-p prefix.  Where k groups of threads had their
//      largest in the first bins, the first k elements lie there too, and only
//      those bins' elements are counted, and listed;
//   3. one workgroup per row adds the slices' histograms and scans them.  Every
//      prefix's end, and the token, then lie in known bins: the end of the first k
//      in one, those that follow from its weight in one or two, since that weight
//      is known to within a bin;
//   4. the elements of these bins are collected, from the list of the second
//      stage or from all slices;
//   5. one workgroup per row sorts them, sums their weights and decides.
// Where the bins hold more than the list takes (nearly equal logits, temperatures
// far from 1), the last workgroup finds each end by itself: it cuts the bin by
// 256-way histograms of the elements' keys, each a pass over the row, until what
// is left can be sorted.
//
// A token is decided by comparing sums, so the sums have to be the same however
// they are formed: w is computed in float64 and held as an integer, w times
// 2^44 at 150K tokens (2^62 over the next power of two above the row's length,
// so that a row's sum fits 63 bits).  Integer sums do not depend on the order of
// additions; the rounding, 2^-45 of the largest weight, moves a border by less
// than 1e-9 of the row's sum even where all 150K roundings agree.
//
// Bound: for a few rows the five launches (one row of 152K float16: 4.5, 8, 7,
// 3.5 and 5.5 us); for many the three passes over the logits, of which the second
// evaluates a float64 exponential (about 40 operations) for every element of the
// rows without a top-k.  256 rows of 152K float32, three quarters with a top-k of
// 20 to 400: 31 (5.1 TB/s), 42, 8.9, 19 and 16 us; with every element counted and
// collected from the slices 31, 58, 8.5, 35 and 16.
#include <math.h>

#include <type_traits>

#include "row_keys.h"

namespace ns {
namespace {

constexpr int kSliceThreads = 256;     // of the stages that read slices
constexpr int kRowThreads = 1024;      // of the stages with one workgroup per row
constexpr int kBins = 1024;            // one per thread of the third stage
constexpr float kReach = 36.f;         // the bins span this much of (z_max - z) / T, or the row
constexpr int kList = 4096;            // collected elements of a row
constexpr int kSort = 1024;            // elements that the long way sorts at once
constexpr int kSub = 256;              // sub-bins of its histograms
constexpr int kMostSlices = 16;        // of a row

// What the third stage decides about a row.
struct Plan {
  uint32_t lo[3], hi[3];  // ranges of bins to collect, disjoint; empty where lo > hi
  uint32_t mode;          // one of the below
};
constexpr uint32_t kDone = 0, kCollect = 1, kLong = 2, kListed = 3;

struct SampleParams {
  int64_t* out;
  const char* x;
  int64_t row_bytes;
  int64_t n;
  const float* u;
  const float* temperature;
  const void* top_k;       // or null
  int top_k64;
  const float* top_p;      // or null
  const float* min_p;      // or null
  int slices;
  int64_t slice_elems;     // a multiple of 8
  int64_t collect_elems;   // the same of the fourth stage's slices
  int shift;               // weights are w * 2^shift
  double zero_below;       // ln w below which a weight rounds to 0
  uint64_t* keys;          // [rows, slices]: the largest element's
  uint32_t* least;         // [rows, slices]: the smallest finite element's order
  uint32_t* parts;         // [rows, slices, kSliceThreads / part_lanes]: the largest order of a group of threads
  int part_lanes;          // threads of a group: 1, 2 or 4
  uint64_t* hist_w;        // [rows, slices, kBins]
  uint32_t* hist_c;
  int* last_bin;           // [rows]: the bins behind it were not counted, nor written
  uint64_t* min_w;         // [rows, slices]
  uint32_t* min_c;
  uint64_t* cum_w;         // [rows, kBins + 1]: weight and count before each bin
  uint32_t* cum_c;
  Plan* plan;              // [rows]
  uint64_t* kept_w;        // [rows]: the min-p prefix
  uint32_t* kept_c;
  uint32_t* list_n;        // [rows]
  uint32_t* cand_n;        // [rows]: elements in the first bins, where these alone were counted; or 0
  uint64_t* cands;         // [rows, list_cap]: their keys
  uint64_t* list;          // [rows, list_cap]: collected keys
  int list_cap;
};

// f(value, index) for the elements [s0, s1) of a row, over the workgroup.  SOME:
// elements below `least` may be left out, and are where a whole wave's vector has
// no other: a test and a branch for every element would cost as much as the rest.
template <int DT, int THREADS, bool SOME = false, class F>
__device__ __forceinline__ void each_element(const char* row, int64_t s0, int64_t s1, F f, float least = 0.f) {
  constexpr int ESZ = DT == NS_DTYPE_F32 ? 4 : 2;
  constexpr int VEC = 16 / ESZ;
  // Elements up to the first 16-byte boundary, whole vectors, the rest.
  const int64_t off = static_cast<int64_t>((reinterpret_cast<uintptr_t>(row) + s0 * ESZ) & 15) / ESZ;
  int64_t v0 = s0 + (off ? VEC - off : 0);
  v0 = v0 < s1 ? v0 : s1;
  const int64_t vecs = (s1 - v0) / VEC;
  const int tid = threadIdx.x;
  const u32x4* v = reinterpret_cast<const u32x4*>(row + v0 * ESZ);
  int64_t j = tid;
  auto vector = [&](const u32x4& w, int64_t at) {
    if (SOME) {
      float most = vec_elem_f32<DT>(w, 0);
#pragma unroll
      for (int e = 1; e < VEC; ++e) most = fmaxf(most, vec_elem_f32<DT>(w, e));
      if (!(most >= least)) return;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) f(vec_elem_f32<DT>(w, e), static_cast<uint32_t>(v0 + at * VEC + e));
  };
  // Four loads in flight.
  for (; j + 3 * THREADS < vecs; j += 4 * THREADS) {
    u32x4 w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = v[j + q * THREADS];
#pragma unroll
    for (int q = 0; q < 4; ++q) vector(w[q], j + q * THREADS);
  }
  for (; j < vecs; j += THREADS) vector(v[j], j);
  const int64_t head = v0 - s0, t0 = v0 + vecs * VEC;
  if (tid < head + (s1 - t0)) {
    const int64_t i = tid < head ? s0 + tid : t0 + (tid - head);
    f(elem_f32<DT>(row, i), static_cast<uint32_t>(i));
  }
}

// A row's constants.
struct Row {
  float top;         // z_max
  float bin_scale;   // bins per unit of z
  double inv_t;
  double zero_below;
  int shift;
};

// Taylor coefficients 1 / 2! .. 1 / 12!, held in scalar registers: as literals
// each would take two moves in front of its multiply-add.
struct Series {
  double c[11];
  __device__ __forceinline__ void load() {
    constexpr double k[11] = {1.0 / 2,     1.0 / 6,      1.0 / 24,      1.0 / 120,      1.0 / 720,      1.0 / 5040,
                              1.0 / 40320, 1.0 / 362880, 1.0 / 3628800, 1.0 / 39916800, 1.0 / 479001600};
#pragma unroll
    for (int i = 0; i < 11; ++i) {
      c[i] = k[i];
      asm volatile("" : "+s"(c[i]));
    }
  }
};

// exp((z - z_max) / T) * 2^shift as an integer.  exp(a) = 2^n exp(r) with
// n = rint(a / ln 2), r = a - n ln 2 in [-0.347, 0.347], and exp(r) by its
// Taylor series to r^12 / 12! (the rest is below 2^-52).  No branches, so that
// the steps of several elements interleave.
__device__ __forceinline__ uint64_t weight_of(const Row& r, const Series& t, float z) {
#pragma clang fp contract(off)
  const double a = (static_cast<double>(z) - static_cast<double>(r.top)) * r.inv_t;
  const double n = __builtin_rint(a * 1.4426950408889634);
  const double x = __builtin_fma(n, -0.6931471805599453, a);
  double e = t.c[10];
#pragma unroll
  for (int i = 9; i >= 0; --i) e = __builtin_fma(e, x, t.c[i]);
  e = __builtin_fma(e, x, 1.0);
  e = __builtin_fma(e, x, 1.0);
  // Below 2^52 a sum with 2^52 holds the rounded integer in its mantissa.
  const double v = __builtin_ldexp(e, static_cast<int>(n) + r.shift) + 4503599627370496.0;
  const uint64_t w = __builtin_bit_cast(uint64_t, v) & 0xFFFFFFFFFFFFFull;
  // Far below, and for a z of -inf whatever the temperature: nothing.
  return a > r.zero_below ? w : 0;
}

// Monotone in z: a larger z never has a larger bin.
__device__ __forceinline__ int bin_of(const Row& r, float z) {
  const float b = (r.top - z) * r.bin_scale;
  return b < kBins - 1 ? static_cast<int>(b) : kBins - 1;
}

// The key of the row's largest element and the order of its smallest finite one
// from its slices', by each wave for itself.
struct Ends {
  uint64_t top;
  uint32_t least;
};
__device__ __forceinline__ Ends row_ends(const SampleParams& p, int64_t row) {
  const int lane = threadIdx.x & 63;
  Ends e = {0, kNanOrder};
  if (lane < p.slices) {  // 16 at most
    e.top = p.keys[row * p.slices + lane];
    e.least = p.least[row * p.slices + lane];
  }
  e.top = lane_of(row_best(e.top, max_u64), 0);
  e.least = lane_of(row_best(e.least, min_u32), 0);
  return e;
}

__device__ __forceinline__ int64_t index_of(uint64_t key) {
  return static_cast<int64_t>(0xFFFFFFFFu - static_cast<uint32_t>(key));
}

// Whether the row takes its largest element: no temperature, a NaN, or a largest
// element that is not finite.
__device__ __forceinline__ bool takes_largest(uint64_t key, float temperature) {
  const uint32_t ord = static_cast<uint32_t>(key >> 32);
  return !(temperature > 0.f) || ord == kNanOrder || !(fabsf(value_of(ord)) < INFINITY);
}

__device__ __forceinline__ Row row_of(const SampleParams& p, const Ends& e, float temperature) {
  Row r;
  r.top = value_of(static_cast<uint32_t>(e.top >> 32));
  r.inv_t = 1.0 / static_cast<double>(temperature);
  const float span = fminf(kReach * temperature, r.top - value_of(e.least));
  r.bin_scale = span > 0.f ? (kBins - 1) / span : 0.f;
  r.zero_below = p.zero_below;
  r.shift = p.shift;
  return r;
}

// An element's place in the row's order, ascending: the order of its value
// complemented, then its index.
__device__ __forceinline__ uint64_t place_of(float z, uint32_t i) {
  return (static_cast<uint64_t>(~order_of(z)) << 32) | i;
}

// A row's top-k, or 0 where it cuts nothing off.
__device__ __forceinline__ int64_t top_k_of(const SampleParams& p, int64_t r) {
  const int64_t k = p.top_k ? load_index(p.top_k, r, p.top_k64) : 0;
  return k > 0 && k < p.n ? k : 0;
}

// f(value, index) for the workgroup's slice of row blockIdx.y.
template <int DT, bool SOME = false, class F>
__device__ __forceinline__ void each_of_slice(const SampleParams& p, int64_t elems, F f, float least = 0.f) {
  const int64_t s0 = static_cast<int64_t>(blockIdx.x) * elems;
  const int64_t s1 = s0 + elems < p.n ? s0 + elems : p.n;
  each_element<DT, kSliceThreads, SOME>(p.x + static_cast<int64_t>(blockIdx.y) * p.row_bytes, s0, s1, f, least);
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads) void sample_ends_kernel(SampleParams p) {
  __shared__ uint64_t wk[kSliceThreads / 64];
  __shared__ uint32_t wl[kSliceThreads / 64];
  uint64_t best = 0;
  uint32_t least = kNanOrder;
  each_of_slice<DT>(p, p.slice_elems, [&](float v, uint32_t i) {
    const uint64_t k = key_of(v, i);
    best = max_u64(best, k);
    const uint32_t ord = static_cast<uint32_t>(k >> 32);
    least = ord < least && v > -INFINITY ? ord : least;
  });
  if (p.top_k) {
    uint32_t part = static_cast<uint32_t>(best >> 32);
    for (int off = 1; off < p.part_lanes; off <<= 1) {
      const uint32_t v = __shfl_xor(part, off);
      part = v > part ? v : part;
    }
    const int64_t at = static_cast<int64_t>(blockIdx.y) * p.slices + blockIdx.x;
    if (threadIdx.x % p.part_lanes == 0)
      p.parts[(at * kSliceThreads + threadIdx.x) / p.part_lanes] = part;
  }
  best = wave_max(best);
  least = wave_best(least, min_u32);
  if ((threadIdx.x & 63) == 0) {
    wk[threadIdx.x >> 6] = best;
    wl[threadIdx.x >> 6] = least;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSliceThreads / 64; ++w) {
      best = max_u64(best, wk[w]);
      least = wl[w] < least ? wl[w] : least;
    }
    const int64_t at = static_cast<int64_t>(blockIdx.y) * p.slices + blockIdx.x;
    p.keys[at] = best;
    p.least[at] = least;
    if (blockIdx.x == 0) p.list_n[blockIdx.y] = p.cand_n[blockIdx.y] = 0;
  }
}

// Keys on their way to a row's list: a workgroup's first kLocal go out together.
constexpr uint32_t kLocal = 1024;
struct Outbox {
  uint64_t keys[kLocal];
  uint32_t n, base;

  // Whether the key is among those.
  __device__ __forceinline__ bool add(uint64_t key, uint64_t* list, uint32_t* list_n, uint32_t cap) {
    const uint32_t at = atomicAdd(&n, 1u);
    if (at < kLocal) {
      keys[at] = key;
      return true;
    }
    const uint32_t to = atomicAdd(list_n, 1u);
    if (to < cap) list[to] = key;
    return false;
  }
  // By the whole workgroup.
  __device__ __forceinline__ void send(uint64_t* list, uint32_t* list_n, uint32_t cap) {
    __syncthreads();
    const uint32_t here = n < kLocal ? n : kLocal;
    if (threadIdx.x == 0 && here > 0) base = atomicAdd(list_n, here);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < here; i += kSliceThreads)
      if (base + i < cap) list[base + i] = keys[i];
  }
};

// Groups of threads of a row.
__device__ __forceinline__ int groups_of(const SampleParams& p) {
  return p.slices * kSliceThreads / p.part_lanes;  // 1024 at most
}

// A bin such that the first k elements lie in it and the bins before it: k groups
// of threads had their largest there.  The last bin where there are not so many
// groups.  count: kBins zeros, and zeros again afterwards.
__device__ __forceinline__ int last_bin_for(const SampleParams& p, const Row& row, int64_t k,
                                            const uint32_t (&part)[4], uint32_t* count) {
  __shared__ uint32_t upto[kSliceThreads / 64];
  __shared__ int found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int groups = groups_of(p);
  if (k == 0 || k > groups) return kBins - 1;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i * kSliceThreads + tid < groups) atomicAdd(&count[bin_of(row, value_of(part[i]))], 1u);
  __syncthreads();
  static_assert(kBins == 4 * kSliceThreads, "four bins for each thread");
  u32x4& mine = reinterpret_cast<u32x4*>(count)[tid];
  const u32x4 c = mine;
  mine = u32x4{0, 0, 0, 0};
  const uint32_t all = c[0] + c[1] + c[2] + c[3];
  uint32_t sum = all;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t v = __shfl_up(sum, off);
    sum += lane >= off ? v : 0;
  }
  if (lane == 63) upto[wave] = sum;
  __syncthreads();
  for (int i = 0; i < wave; ++i) sum += upto[i];
  uint32_t before = sum - all;
  if (before < k && sum >= k) {
    int b = 0;
    while (before + c[b] < k) before += c[b++];
    found = 4 * tid + b;
  }
  __syncthreads();
  return found;
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads, 4) void sample_hist_kernel(SampleParams p) {
  // The last bin, which may hold most of a row, has a place for every lane:
  // atomics on one address wait for each other.
  __shared__ uint64_t hw[kBins + 64];
  __shared__ __align__(16) uint32_t hc[kBins + 64];
  __shared__ Outbox box;
  __shared__ uint64_t mw;
  __shared__ uint32_t mc;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.y;
  // Everything that is read besides the row, at once.
  const int64_t k = top_k_of(p, r);
  const float t = p.temperature[r];
  const float mp = p.min_p ? p.min_p[r] : 0.f;
  uint32_t part[4] = {0, 0, 0, 0};
  if (p.top_k) {
    const int groups = groups_of(p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i * kSliceThreads + tid < groups) part[i] = p.parts[r * groups + i * kSliceThreads + tid];
  }
  const Ends ends = row_ends(p, r);
  if (takes_largest(ends.top, t)) return;
  for (int b = tid; b < kBins + 64; b += kSliceThreads) {
    hw[b] = 0;
    hc[b] = 0;
  }
  if (tid == 0) {
    mw = 0;
    mc = 0;
    box.n = 0;
  }
  __syncthreads();
  const Row row = row_of(p, ends, t);
  Series series;
  series.load();
  const int last = kBins - 1 + (tid & 63);
  // Elements behind the first k decide nothing and are left out, where a bin that
  // they cannot lie in is known: most of a row then needs no exponential, and the
  // others can be listed at once.
  const int most = last_bin_for(p, row, k, part, hc);
  auto count = [&](int b, uint64_t w) {
    b = b == kBins - 1 ? last : b;
    atomicAdd(&hc[b], 1u);
    atomicAdd(reinterpret_cast<unsigned long long*>(&hw[b]), static_cast<unsigned long long>(w));
  };
  // The prefix of w >= min_p, as integers.
  const uint64_t enough =
      mp > 0.f && mp < 4.f ? static_cast<uint64_t>(ceil(static_cast<double>(mp) * __builtin_ldexp(1.0, p.shift))) : ~0ull;
  uint32_t min_c = 0;
  uint64_t min_w = 0;
  auto count_min = [&](uint64_t w) {
    min_c += w >= enough ? 1 : 0;
    min_w += w >= enough ? w : 0;
  };
  if (most < kBins - 1) {
    uint64_t* const cands = p.cands + r * p.list_cap;
    auto weigh = [&](float z) {
      const uint64_t w = weight_of(row, series, z);
      count_min(w);
      count(bin_of(row, z), w);
    };
    // Nothing below this lies in the bins up to `most` (a bin's width, and a
    // rounding of the result, to be sure).
    const double edge = static_cast<double>(row.top) - (most + 2) / static_cast<double>(row.bin_scale);
    const float least = static_cast<float>(edge) - fabsf(static_cast<float>(edge)) * 2.4e-7f;
    each_of_slice<DT, true>(
        p, p.slice_elems,
        [&](float z, uint32_t i) {
          if (bin_of(row, z) > most) return;
          if (!box.add(place_of(z, i), cands, &p.cand_n[r], p.list_cap)) weigh(z);
        },
        least);
    __syncthreads();
    const uint32_t here = box.n < kLocal ? box.n : kLocal;
    for (uint32_t i = tid; i < here; i += kSliceThreads) weigh(value_of(~static_cast<uint32_t>(box.keys[i] >> 32)));
    box.send(cands, &p.cand_n[r], p.list_cap);
  } else if (mp > 0.f) {
    each_of_slice<DT>(p, p.slice_elems, [&](float z, uint32_t) {
      const uint64_t w = weight_of(row, series, z);
      count_min(w);
      count(bin_of(row, z), w);
    });
  } else {
    each_of_slice<DT>(p, p.slice_elems, [&](float z, uint32_t) { count(bin_of(row, z), weight_of(row, series, z)); });
  }
  if (mp > 0.f) {
    atomicAdd(&mc, min_c);
    atomicAdd(reinterpret_cast<unsigned long long*>(&mw), static_cast<unsigned long long>(min_w));
  }
  __syncthreads();
  if (tid > 0 && tid < 64) {
    atomicAdd(&hc[kBins - 1], hc[last]);
    atomicAdd(reinterpret_cast<unsigned long long*>(&hw[kBins - 1]), static_cast<unsigned long long>(hw[last]));
  }
  __syncthreads();
  const int64_t at = r * p.slices + blockIdx.x;
  for (int b = tid; b <= most; b += kSliceThreads) {
    p.hist_w[at * kBins + b] = hw[b];
    p.hist_c[at * kBins + b] = hc[b];
  }
  if (tid == 0) {
    if (blockIdx.x == 0) p.last_bin[r] = most;
    p.min_c[at] = mc;
    p.min_w[at] = mw;
  }
}

// Inclusive scan of one (count, weight) per thread of a row's workgroup.
struct ScanScratch {
  uint64_t w[kRowThreads / 64];
  uint32_t c[kRowThreads / 64];
};
__device__ __forceinline__ void scan(ScanScratch& s, uint32_t& c, uint64_t& w) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t pc = __shfl_up(c, off);
    const uint64_t pw = __shfl_up(w, off);
    if (lane >= off) {
      c += pc;
      w += pw;
    }
  }
  if (lane == 63) {
    s.c[wave] = c;
    s.w[wave] = w;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 64 - 1; ++i) {
    c += i < wave ? s.c[i] : 0;
    w += i < wave ? s.w[i] : 0;
  }
  __syncthreads();
}

// The first i in [0, n) with cum[i] >= goal; cum ascends, cum[n - 1] >= goal and
// n <= 4096.  A wave looks at 64 places at a time: two reads deep, where a
// bisection of 4096 would be twelve.
template <class T>
__device__ __forceinline__ int first_reaching(const T* cum, int n, uint64_t goal) {
  const int lane = threadIdx.x & 63;
  const int step = (n + 63) >> 6;
  int at = (lane + 1) * step - 1;
  at = at < n ? at : n - 1;
  uint64_t hit = __builtin_amdgcn_ballot_w64(cum[at] >= goal);
  const int from = hit ? __builtin_ctzll(hit) * step : n - 1;
  at = from + lane < n ? from + lane : n - 1;
  hit = __builtin_amdgcn_ballot_w64(lane < step && cum[at] >= goal);
  at = from + (hit ? __builtin_ctzll(hit) : 0);
  return at < n ? at : n - 1;
}

// A prefix of the row's order.
struct Prefix {
  uint32_t count;
  uint64_t weight;
};

// The weight that a top-p prefix has to reach: a token stays while the sum
// before it is below top_p times the sum, so up to the first whose running sum
// is not.
__device__ __forceinline__ uint64_t top_p_goal(float top_p, uint64_t weight) {
  const double bound = ceil(static_cast<double>(top_p) * static_cast<double>(weight));
  return bound >= 1.0 ? static_cast<uint64_t>(bound) : 1;
}
// The running sum that the token has to reach.
__device__ __forceinline__ uint64_t draw_goal(float u, uint64_t weight) {
  const double target = (u > 0.f ? static_cast<double>(u) : 0.0) * static_cast<double>(weight);
  const uint64_t goal = target < static_cast<double>(weight) ? static_cast<uint64_t>(target) + 1 : weight;
  return goal < weight ? goal : weight;
}
// A row's top-p, or 1.
__device__ __forceinline__ float top_p_of(const SampleParams& p, int64_t r) {
  const float v = p.top_p ? p.top_p[r] : 1.f;
  return v < 1.f ? v : 1.f;
}

__global__ __launch_bounds__(kRowThreads) void sample_plan_kernel(SampleParams p) {
  __shared__ uint64_t cum_w[kBins + 1];
  __shared__ uint32_t cum_c[kBins + 1];
  __shared__ ScanScratch scratch;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  static_assert(kBins == kRowThreads, "one bin per thread");
  // Everything that is read, at once: each of these is a round trip past this
  // XCD's cache.  (A greedy row has no histograms; its sums go nowhere.)
  uint32_t c = 0;
  uint64_t w = 0;
  auto add = [&](auto most) {
#pragma unroll
    for (int i = 0; i < most; ++i) {
      // No branch, so that no read waits for another.
      const int64_t at = (r * p.slices + (i < p.slices ? i : p.slices - 1)) * kBins + tid;
      const uint32_t ci = p.hist_c[at];
      const uint64_t wi = p.hist_w[at];
      c += i < p.slices ? ci : 0;
      w += i < p.slices ? wi : 0;
    }
  };
  if (p.slices <= 4) add(std::integral_constant<int, 4>());
  else add(std::integral_constant<int, kMostSlices>());
  const float u = p.u[r], temperature = p.temperature[r], tp = top_p_of(p, r);
  const int64_t k = top_k_of(p, r);
  const bool has_min = p.min_p && p.min_p[r] > 0.f;
  const uint32_t listed = p.cand_n[r];
  const int last_bin = p.last_bin[r];
  const Ends ends = row_ends(p, r);
  if (takes_largest(ends.top, temperature)) {
    if (tid == 0) {
      p.out[r] = index_of(ends.top);
      p.plan[r].mode = kDone;
    }
    return;
  }
  if (tid > last_bin) {
    c = 0;
    w = 0;
  }
  scan(scratch, c, w);
  cum_c[tid + 1] = c;
  cum_w[tid + 1] = w;
  if (tid == 0) {
    cum_c[0] = 0;
    cum_w[0] = 0;
  }
  p.cum_c[r * (kBins + 1) + tid + 1] = c;
  p.cum_w[r * (kBins + 1) + tid + 1] = w;
  __syncthreads();
  if (tid >= 64) return;  // the rest is one thread's work, which a wave does alike

  Prefix least = {0, 0};
  if (has_min) {
    for (int i = tid; i < p.slices; i += 64) {
      least.count += p.min_c[r * p.slices + i];
      least.weight += p.min_w[r * p.slices + i];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      least.count += __shfl_xor(least.count, off);
      least.weight += __shfl_xor(least.weight, off);
    }
  } else {
    least = Prefix{static_cast<uint32_t>(p.n), cum_w[kBins]};
  }
  // Bounds of the kept prefix's weight, and with them the bins that ends can lie in.
  const uint64_t one = 1ull << p.shift;  // the largest element's weight
  const uint64_t all = cum_w[kBins];
  auto bin_w = [&](uint64_t goal) { return first_reaching(cum_w + 1, kBins, goal < all ? goal : all); };
  uint64_t lo_w = all, hi_w = all;
  int lo[3] = {1, 1, 1}, hi[3] = {0, 0, 0};
  if (k > 0) {
    const int b = first_reaching(cum_c + 1, kBins, static_cast<uint64_t>(k));
    hi_w = lo_w = cum_w[b + 1];
    if (cum_c[b + 1] != static_cast<uint64_t>(k)) {
      lo[0] = hi[0] = b;
      lo_w = cum_w[b] > one ? cum_w[b] : one;
    }
  }
  if (tp < 1.f) {
    lo[1] = bin_w(top_p_goal(tp, lo_w));
    hi[1] = bin_w(top_p_goal(tp, hi_w));
    const uint64_t from = cum_w[lo[1]] > one ? cum_w[lo[1]] : one;
    lo_w = from < lo_w ? from : lo_w;
    hi_w = cum_w[hi[1] + 1] < hi_w ? cum_w[hi[1] + 1] : hi_w;
  }
  lo_w = least.weight < lo_w ? least.weight : lo_w;
  hi_w = least.weight < hi_w ? least.weight : hi_w;
  if (least.count > 0) {
    lo[2] = bin_w(draw_goal(u, lo_w));
    hi[2] = bin_w(draw_goal(u, hi_w));
  }
  // Overlapping ranges become one.
  auto join = [&](int a, int b) {
    if (lo[a] > hi[a] || lo[b] > hi[b] || lo[a] > hi[b] || lo[b] > hi[a]) return;
    lo[a] = lo[a] < lo[b] ? lo[a] : lo[b];
    hi[a] = hi[a] > hi[b] ? hi[a] : hi[b];
    lo[b] = 1;
    hi[b] = 0;
  };
  join(0, 1);
  join(0, 2);
  join(1, 2);
  join(0, 1);
  uint32_t count = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) count += lo[i] <= hi[i] ? cum_c[hi[i] + 1] - cum_c[lo[i]] : 0;
  if (tid == 0) {
    Plan plan;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      plan.lo[i] = lo[i];
      plan.hi[i] = hi[i];
    }
    const uint32_t cap = p.list_cap;
    plan.mode = listed > 0 && listed <= cap ? kListed : count <= cap ? kCollect : kLong;
    if (least.count == 0) {  // min_p above 1: the largest alone
      plan.mode = kDone;
      p.out[r] = index_of(ends.top);
    }
    p.plan[r] = plan;
    p.kept_c[r] = least.count;
    p.kept_w[r] = least.weight;
    p.cum_c[r * (kBins + 1)] = 0;
    p.cum_w[r * (kBins + 1)] = 0;
  }
}

template <int DT>
__global__ __launch_bounds__(kSliceThreads) void sample_collect_kernel(SampleParams p) {
  __shared__ Outbox box;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.y;
  const Plan plan = p.plan[r];
  if (plan.mode != kCollect && (plan.mode != kListed || blockIdx.x > 0)) return;
  const Row row = row_of(p, row_ends(p, r), p.temperature[r]);
  if (tid == 0) box.n = 0;
  __syncthreads();
  uint64_t* list = p.list + r * p.list_cap;
  auto collect = [&](float z, uint32_t i) {
    const uint32_t b = bin_of(row, z);
    bool in = false;
#pragma unroll
    for (int q = 0; q < 3; ++q) in = in || (b >= plan.lo[q] && b <= plan.hi[q]);
    if (in) box.add(place_of(z, i), list, &p.list_n[r], p.list_cap);
  };
  if (plan.mode == kListed) {
    const uint32_t n = p.cand_n[r];
    for (uint32_t i = tid; i < n; i += kSliceThreads) {
      const uint64_t place = p.cands[r * p.list_cap + i];
      collect(value_of(~static_cast<uint32_t>(place >> 32)), static_cast<uint32_t>(place));
    }
  } else {
    each_of_slice<DT>(p, p.collect_elems, collect);
  }
  box.send(list, &p.list_n[r], p.list_cap);
}

// Sorts E elements per thread (element e of thread t is number t * E + e),
// ascending, by a bitonic network over the first `size` (a power of two, a
// multiple of E; the others stay apart).  Partners within a thread are compared
// in place, within a wave by a lane exchange, further ones through `swap`; only
// the latter need the workgroup to wait.
template <int E>
__device__ __forceinline__ void sort_registers(uint64_t (&v)[E], uint64_t* swap, uint32_t size) {
  const uint32_t tid = threadIdx.x;
  // Waves without any of the elements only wait with the others.
  const bool here = __builtin_amdgcn_readfirstlane(tid) * E < size;
  for (uint32_t k = 2; k <= size; k <<= 1) {
    for (uint32_t j = k >> 1; j > 0; j >>= 1) {
      if (j < E) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
          for (int bit = 1; bit < E; bit <<= 1) {
            if (j == static_cast<uint32_t>(bit) && (e & bit) == 0) {
              const bool up = ((tid * E + e) & k) == 0;
              const uint64_t x = v[e], y = v[e + bit];
              if ((x > y) == up) {
                v[e] = y;
                v[e + bit] = x;
              }
            }
          }
        }
        continue;
      }
      const uint32_t lanes = j / E;
      uint64_t other[E];
      if (lanes < 64) {
        if (!here) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) other[e] = __shfl_xor(v[e], static_cast<int>(lanes));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) swap[e * kRowThreads + tid] = v[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) other[e] = swap[e * kRowThreads + (tid ^ lanes)];
        __syncthreads();
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool up = ((tid * E + e) & k) == 0, lower = (tid & lanes) == 0;
        v[e] = (up == lower) == (other[e] < v[e]) ? other[e] : v[e];
      }
    }
  }
}

// The last stage's workgroup.
struct Pick {
  uint64_t cum_w[kBins + 1];
  uint32_t cum_c[kBins + 1];
  uint64_t list[kList];
  uint64_t run[kList];       // running weights of the sorted list (before: the sort's exchange)
  ScanScratch scratch;
  uint64_t sub_w[kSub];      // the long way's
  uint32_t sub_c[kSub];
  uint64_t lo, hi;
  uint32_t n;
  int found;
};

// Where a prefix ends: its elements, their weight, and the last one's index.
struct End {
  uint32_t count;
  uint64_t weight;
  uint32_t index;
};

// The shortest prefix with at least `goal` elements (BY_COUNT) or weight, from the
// collected and sorted elements; its end lies in a collected bin, or (BY_COUNT) at
// the end of one.
template <bool BY_COUNT>
__device__ __forceinline__ End end_in_list(const Pick& s, const Plan& plan, uint64_t goal) {
  const int bin = BY_COUNT ? first_reaching(s.cum_c + 1, kBins, goal) : first_reaching(s.cum_w + 1, kBins, goal);
  End e;
  e.index = 0;
  if (BY_COUNT && s.cum_c[bin + 1] == goal) {
    e.count = static_cast<uint32_t>(goal);
    e.weight = s.cum_w[bin + 1];
    return e;
  }
  int from = 0;  // collected elements of the bins before
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    const int lo = plan.lo[q], upto = static_cast<int>(plan.hi[q]) + 1 < bin ? plan.hi[q] + 1 : bin;
    if (lo < upto && plan.lo[q] <= plan.hi[q]) from += s.cum_c[upto] - s.cum_c[lo];
  }
  const int n = s.cum_c[bin + 1] - s.cum_c[bin];
  const uint64_t before = from > 0 ? s.run[from - 1] : 0;
  const int at = BY_COUNT ? static_cast<int>(goal - s.cum_c[bin]) - 1
                          : first_reaching(s.run + from, n, goal - s.cum_w[bin] + before);
  e.count = s.cum_c[bin] + at + 1;
  e.weight = s.cum_w[bin] + s.run[from + at] - before;
  e.index = static_cast<uint32_t>(s.list[from + at]);
  return e;
}

// The shortest prefix of the row's order with at least `goal` elements
// (by_count) or weight; the row has that much, and goal > 0.
template <int DT>
__device__ __forceinline__ End end_by_passes(const SampleParams& p, Pick& s, const Row& row, const Series& series,
                                             const char* x, bool by_count, uint64_t goal) {
  const int tid = threadIdx.x;
  if (tid == 0) s.found = kBins - 1;
  __syncthreads();
  {
    const uint64_t before = by_count ? s.cum_c[tid] : s.cum_w[tid];
    const uint64_t upto = by_count ? s.cum_c[tid + 1] : s.cum_w[tid + 1];
    if (before < goal && goal <= upto) s.found = tid;
  }
  __syncthreads();
  const int bin = s.found;
  uint32_t base_c = s.cum_c[bin], n = s.cum_c[bin + 1] - base_c;
  uint64_t base_w = s.cum_w[bin];
  uint64_t lo = 0, hi = ~0ull;  // the keys looked at; with `bin` until they are known
  bool by_bin = true;
  __syncthreads();
  if (n > kSort) {
    if (tid == 0) {
      s.lo = ~0ull;
      s.hi = 0;
    }
    __syncthreads();
    uint64_t a = ~0ull, b = 0;
    each_element<DT, kRowThreads>(x, 0, p.n, [&](float z, uint32_t i) {
      if (bin_of(row, z) != bin) return;
      const uint64_t k = place_of(z, i);
      a = k < a ? k : a;
      b = max_u64(b, k);
    });
    atomicMin(reinterpret_cast<unsigned long long*>(&s.lo), static_cast<unsigned long long>(a));
    atomicMax(reinterpret_cast<unsigned long long*>(&s.hi), static_cast<unsigned long long>(b));
    __syncthreads();
    lo = s.lo;
    hi = s.hi;
    by_bin = false;
    while (n > kSort) {
      const int bits = 64 - __builtin_clzll((hi - lo) | 1);
      const int cut = bits > 8 ? bits - 8 : 0;  // keys differ, so more than kSort of them span over 8 bits
      __syncthreads();
      if (tid < kSub) {
        s.sub_c[tid] = 0;
        s.sub_w[tid] = 0;
      }
      if (tid == 0) {  // the search below always finds its sub-bin; were it not to, the loop would end
        s.found = 0;
        s.n = 0;
        s.lo = base_w;
        s.hi = base_c;
      }
      __syncthreads();
      each_element<DT, kRowThreads>(x, 0, p.n, [&](float z, uint32_t i) {
        const uint64_t k = place_of(z, i);
        if (k < lo || k > hi) return;
        const int b = static_cast<int>((k - lo) >> cut);
        atomicAdd(&s.sub_c[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.sub_w[b]),
                  static_cast<unsigned long long>(weight_of(row, series, z)));
      });
      __syncthreads();
      uint32_t c = tid < kSub ? s.sub_c[tid] : 0;
      uint64_t w = tid < kSub ? s.sub_w[tid] : 0;
      const uint32_t own_c = c;
      const uint64_t own_w = w;
      scan(s.scratch, c, w);
      const uint64_t upto = by_count ? base_c + c : base_w + w, mine = by_count ? own_c : own_w;
      if (tid < kSub && upto - mine < goal && goal <= upto) {
        s.found = tid;
        s.n = own_c;
        s.lo = base_w + (w - own_w);
        s.hi = base_c + (c - own_c);
      }
      __syncthreads();
      n = s.n;
      base_w = s.lo;
      base_c = static_cast<uint32_t>(s.hi);
      lo += static_cast<uint64_t>(s.found) << cut;
      const uint64_t span = (1ull << cut) - 1;  // lo + span may pass 2^64
      hi = hi - lo > span ? lo + span : hi;
      __syncthreads();
    }
  }
  // Collect, sort (a bitonic network over the next power of two), sum.
  if (tid == 0) {
    s.n = 0;
    s.found = 0;
    s.lo = base_w;
    s.hi = 0;
  }
  uint32_t size = 1;
  while (size < n) size <<= 1;
  s.list[tid] = ~0ull;
  __syncthreads();
  each_element<DT, kRowThreads>(x, 0, p.n, [&](float z, uint32_t i) {
    if (by_bin && bin_of(row, z) != bin) return;
    const uint64_t k = place_of(z, i);
    if (k < lo || k > hi) return;
    const uint32_t at = atomicAdd(&s.n, 1u);
    if (at < kSort) s.list[at] = k;
  });
  __syncthreads();
  uint64_t place[1] = {s.list[tid]};
  __syncthreads();
  sort_registers(place, s.run, size);
  const uint64_t key = tid < static_cast<int>(n) ? place[0] : 0;
  uint32_t c = tid < static_cast<int>(n) ? 1 : 0;
  uint64_t w = c ? weight_of(row, series, value_of(~static_cast<uint32_t>(key >> 32))) : 0;
  const uint64_t own_w = w;
  scan(s.scratch, c, w);
  if (tid < static_cast<int>(n)) {
    const uint64_t upto = by_count ? base_c + c : base_w + w, mine = by_count ? 1 : own_w;
    if (upto - mine < goal && goal <= upto) {
      s.found = tid;
      s.lo = base_w + w;
      s.hi = key;
    }
  }
  __syncthreads();
  End e;
  e.count = base_c + s.found + 1;
  e.weight = s.lo;
  e.index = static_cast<uint32_t>(s.hi);
  __syncthreads();
  return e;
}

// list's n keys into s.list, ascending, and the running sums of their weights
// into s.run.  early: the thread's one of the first kRowThreads.
template <int E>
__device__ __forceinline__ void sort_and_sum(Pick& s, const Row& row, const Series& series, const uint64_t* list,
                                             uint64_t early, uint32_t n) {
  const uint32_t first = threadIdx.x * E;
  uint64_t v[E], sum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    // Which thread starts with which key does not matter.
    const uint32_t i = e * kRowThreads + threadIdx.x;
    v[e] = i >= n ? ~0ull : e == 0 ? early : list[i];
  }
  uint32_t size = E;
  while (size < n) size <<= 1;
  if (E > 1) size = E * kRowThreads;  // the keys start in all threads
  sort_registers(v, s.run, size);
  uint64_t w = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (first + e < n) w += weight_of(row, series, value_of(~static_cast<uint32_t>(v[e] >> 32)));
    sum[e] = w;
  }
  uint32_t none = 0;
  const uint64_t mine = w;
  scan(s.scratch, none, w);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (first + e < n) {
      s.list[first + e] = v[e];
      s.run[first + e] = w - mine + sum[e];
    }
  }
}

template <int DT>
__global__ __launch_bounds__(kRowThreads) void sample_pick_kernel(SampleParams p) {
  __shared__ Pick s;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  // Everything that is read, at once, the first collected keys among it.
  const Plan plan = p.plan[r];
  const uint32_t cc = p.cum_c[r * (kBins + 1) + tid + 1];
  const uint64_t cw = p.cum_w[r * (kBins + 1) + tid + 1];
  const uint64_t* list = p.list + r * p.list_cap;
  const uint64_t early = tid < p.list_cap ? list[tid] : 0;
  const uint32_t listed = p.list_n[r];
  const float u = p.u[r], temperature = p.temperature[r], tp = top_p_of(p, r);
  const int64_t k = top_k_of(p, r);
  const Prefix least = {p.kept_c[r], p.kept_w[r]};  // the min-p prefix
  const Ends ends = row_ends(p, r);
  if (plan.mode == kDone) return;
  const Row row = row_of(p, ends, temperature);
  Series series;
  series.load();
  s.cum_c[tid + 1] = cc;
  s.cum_w[tid + 1] = cw;
  if (tid == 0) {
    s.cum_c[0] = 0;
    s.cum_w[0] = 0;
  }
  if (plan.mode == kLong) {
    __syncthreads();
    const char* x = p.x + r * p.row_bytes;
    Prefix first = {static_cast<uint32_t>(p.n), s.cum_w[kBins]};
    Prefix kept = least.count < first.count ? least : first;
    // One inlined copy for the three ends: calls would give the kernel a stack,
    // which costs every launch of it 11 us.
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {
      if ((step == 0 && k == 0) || (step == 1 && !(tp < 1.f))) continue;
      const uint64_t goal = step == 0   ? static_cast<uint64_t>(k)
                            : step == 1 ? top_p_goal(tp, first.weight)
                                        : draw_goal(u, kept.weight);
      const End e = end_by_passes<DT>(p, s, row, series, x, step == 0, goal);
      if (step == 0) first = Prefix{e.count, e.weight};
      if (step < 2 && e.count < kept.count) kept = Prefix{e.count, e.weight};
      if (step == 2 && tid == 0) p.out[r] = e.index;
    }
    return;
  }

  // The collected elements: sorted, and their weights' running sums.
  const uint32_t n = listed < static_cast<uint32_t>(p.list_cap) ? listed : p.list_cap;
  if (n <= kRowThreads) sort_and_sum<1>(s, row, series, list, early, n);
  else if (n <= 2 * kRowThreads) sort_and_sum<2>(s, row, series, list, early, n);
  else sort_and_sum<4>(s, row, series, list, early, n);
  __syncthreads();
  if (tid >= 64) return;
  Prefix kept = least;
  Prefix first = {static_cast<uint32_t>(p.n), s.cum_w[kBins]};
  if (k > 0) {
    const End e = end_in_list<true>(s, plan, static_cast<uint64_t>(k));
    first = Prefix{e.count, e.weight};
  }
  if (first.count < kept.count) kept = first;
  if (tp < 1.f) {
    const End e = end_in_list<false>(s, plan, top_p_goal(tp, first.weight));
    if (e.count < kept.count) kept = Prefix{e.count, e.weight};
  }
  const End e = end_in_list<false>(s, plan, draw_goal(u, kept.weight));
  if (tid == 0) p.out[r] = e.index;
}

// How the rows are cut, and where the workspace's parts lie (byte offsets).
struct Layout {
  int slices, collect_slices, list_cap;
  int64_t slice_elems, collect_elems;
  int part_lanes;
  size_t keys, hist_w, min_w, cum_w, kept_w, list, cands, least, parts, hist_c, min_c, cum_c, kept_c,
      list_n, cand_n, last_bin, plan, total;
};

Layout layout_of(int64_t M, int64_t N) {
  Layout l;
  // About four workgroups for each compute unit, up to 16 slices of at least 2048
  // elements; eight for many rows, whose work is unequal (rows with and without a
  // top-k; 512 rows of 152K 172 us, 198 with four, 1024 314 and 412, but 256 and 128
  // rows 4 and 6 us more).  The fourth stage, where most rows are done with, takes
  // more still (256 rows: 28, 21, 19 us with 4, 8, 16 slices).
  auto cut = [&](int64_t groups, int& slices, int64_t& elems) {
    int64_t n = groups / M < 1 ? 1 : groups / M;
    n = n > kMostSlices ? kMostSlices : n;
    const int64_t most = (N + 2047) / 2048;
    n = n > most ? most : n;
    elems = ((N + n - 1) / n + 7) / 8 * 8;
    slices = static_cast<int>((N + elems - 1) / elems);
  };
  cut(M > 256 ? 2048 : 1024, l.slices, l.slice_elems);
  cut(4096, l.collect_slices, l.collect_elems);
  l.list_cap = N < kList ? static_cast<int>(N) : kList;
  size_t at = 0;
  const size_t m = static_cast<size_t>(M), cells = m * l.slices;
  auto take = [&](size_t n) {
    const size_t here = at;
    at += n;
    return here;
  };
  l.keys = take(cells * 8);
  l.hist_w = take(cells * kBins * 8);
  l.min_w = take(cells * 8);
  l.cum_w = take(m * (kBins + 1) * 8);
  l.kept_w = take(m * 8);
  l.list = take(m * l.list_cap * 8);
  l.cands = take(m * l.list_cap * 8);
  l.least = take(cells * 4);
  // Up to 1024 groups of a row.
  l.part_lanes = l.slices > 8 ? 4 : l.slices > 4 ? 2 : 1;
  l.parts = take(cells * (kSliceThreads / l.part_lanes) * 4);
  l.hist_c = take(cells * kBins * 4);
  l.min_c = take(cells * 4);
  l.cum_c = take(m * (kBins + 1) * 4);
  l.kept_c = take(m * 4);
  l.list_n = take(m * 4);
  l.cand_n = take(m * 4);
  l.last_bin = take(m * 4);
  l.plan = take(m * sizeof(Plan));
  l.total = at;
  return l;
}

bool misaligned(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

template <int DT>
hipError_t launch(SampleParams& p, int64_t M, int collect_slices, hipStream_t st) {
  void* args[] = {&p};
  const unsigned m = static_cast<unsigned>(M);
  const void* by_slice[] = {reinterpret_cast<const void*>(&sample_ends_kernel<DT>),
                            reinterpret_cast<const void*>(&sample_hist_kernel<DT>), nullptr,
                            reinterpret_cast<const void*>(&sample_collect_kernel<DT>), nullptr};
  const void* by_row[] = {nullptr, nullptr, reinterpret_cast<const void*>(&sample_plan_kernel), nullptr,
                          reinterpret_cast<const void*>(&sample_pick_kernel<DT>)};
  for (int i = 0; i < 5; ++i) {
    const dim3 slices(static_cast<unsigned>(i == 3 ? collect_slices : p.slices), m);
    const hipError_t e = by_slice[i] ? hipLaunchKernel(by_slice[i], slices, dim3(kSliceThreads), args, 0, st)
                                     : hipLaunchKernel(by_row[i], dim3(m), dim3(kRowThreads), args, 0, st);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace
}  // namespace ns

extern "C" size_t ns_sample_rows_workspace_size(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0 || M > 65535 || N > 0x7FFFFFFF) return 0;
  return ns::layout_of(M, N).total;
}

extern "C" int ns_sample_rows(int64_t* out, const void* x, int64_t x_stride_row, int64_t M, int64_t N, int dtype,
                              const float* uniform, const float* temperature,
                              const void* top_k, int top_k_is_int64, const float* top_p, const float* min_p,
                              void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ns;
  const int esz = dtype_size(dtype);
  if (esz == 0) return NS_ERR_UNSUPPORTED;
  if (M < 0 || N <= 0 || x_stride_row < N || M > 65535 || N > 0x7FFFFFFF) return NS_ERR_INVALID_ARG;
  if (M == 0) return NS_OK;
  if (!out || !x || !uniform || !temperature) return NS_ERR_INVALID_ARG;
  if (misaligned(out, 8) || misaligned(x, esz) || misaligned(uniform, 4) || misaligned(temperature, 4) ||
      misaligned(top_k, top_k_is_int64 ? 8 : 4) || misaligned(top_p, 4) || misaligned(min_p, 4))
    return NS_ERR_INVALID_ARG;
  const Layout l = layout_of(M, N);
  if (!workspace || workspace_bytes < l.total || misaligned(workspace, 8)) return NS_ERR_WORKSPACE;
  SampleParams p;
  char* ws = static_cast<char*>(workspace);
  p.out = out;
  p.x = static_cast<const char*>(x);
  p.row_bytes = x_stride_row * esz;
  p.n = N;
  p.u = uniform;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_k64 = top_k_is_int64 ? 1 : 0;
  p.top_p = top_p;
  p.min_p = min_p;
  auto u64 = [&](size_t at) { return reinterpret_cast<uint64_t*>(ws + at); };
  auto u32 = [&](size_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
  p.slices = l.slices;
  p.slice_elems = l.slice_elems;
  p.collect_elems = l.collect_elems;
  p.list_cap = l.list_cap;
  p.keys = u64(l.keys);
  p.hist_w = u64(l.hist_w);
  p.min_w = u64(l.min_w);
  p.cum_w = u64(l.cum_w);
  p.kept_w = u64(l.kept_w);
  p.list = u64(l.list);
  p.cands = u64(l.cands);
  p.least = u32(l.least);
  p.parts = u32(l.parts);
  p.part_lanes = l.part_lanes;
  p.hist_c = u32(l.hist_c);
  p.min_c = u32(l.min_c);
  p.cum_c = u32(l.cum_c);
  p.kept_c = u32(l.kept_c);
  p.list_n = u32(l.list_n);
  p.cand_n = u32(l.cand_n);
  p.last_bin = reinterpret_cast<int*>(ws + l.last_bin);
  p.plan = reinterpret_cast<Plan*>(ws + l.plan);
  int log = 0;
  while ((1ll << log) < N) ++log;
  p.shift = 62 - log < 51 ? 62 - log : 51;
  p.zero_below = -(p.shift + 1) * 0.6931471805599453;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const hipError_t e = dtype == NS_DTYPE_F32   ? launch<NS_DTYPE_F32>(p, M, l.collect_slices, st)
                       : dtype == NS_DTYPE_F16 ? launch<NS_DTYPE_F16>(p, M, l.collect_slices, st)
                                               : launch<NS_DTYPE_BF16>(p, M, l.collect_slices, st);
  return e == hipSuccess ? NS_OK : NS_ERR_HIP;
}
