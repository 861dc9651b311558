// The two ends of a decode step that verifies drafted tokens: its addresses, made
// on the device from the requests' lengths, and the commit of the accepted rows.
//
// Both are bound by latency (a launch and two or three dependent trips to memory):
// the first moves a few hundred bytes a request, the second the accepted rows of
// every layer.  On MI355X: addresses 3.4 us for one request, 4.5 for 32 of 8 rows, 9.1
// for 1024 (their prefixes summed by every workgroup); commits 4.2 us for one request
// and 24 layers, 4.5 for 32, 15 for 128 of 32 rows and 28 layers of 1 KB rows.
#include "ns_common.h"

namespace ns {
namespace {

constexpr int kThreads = 256;
constexpr int kTreeRows = 64;  // rows of a request that form a tree

// ---- step inputs ----------------------------------------------------------------
//
// Workgroup (i, y) works on request i: it sums the query lengths before it (every
// workgroup for itself: a scan in a launch of its own would cost more than the
// reads), and its threads take the request's columns and rows.  What a step appends
// to a table is taken from the list of new blocks by every reader, so that no
// workgroup waits for another's write.  The last i takes the rows behind the last
// request.

struct StepParams {
  void* tables;
  int64_t table_rows, width, table_stride;
  const void* rows;
  const void* computed;
  const void* query_lens;
  const void* new_blocks;  // NULL: no request has new ones
  const void* new_start;
  const void* held;
  const void* parents;     // NULL: no trees
  int64_t* qsl;
  int64_t* seq_lens;
  int64_t* positions;
  int64_t* slots;
  int64_t* mask;
  void* block_tables;
  int64_t num_seqs, num_tokens, num_new, max_blocks;
  int block_size, tables64, index64;
};

__device__ __forceinline__ int64_t clamp_to(int64_t x, int64_t most) { return x < 0 ? 0 : x < most ? x : most; }

__global__ __launch_bounds__(kThreads) void step_inputs_kernel(StepParams p) {
  __shared__ int64_t sums[kThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t i = blockIdx.x;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * kThreads + tid;
  const int64_t step = static_cast<int64_t>(gridDim.y) * kThreads;
  constexpr int64_t kMost = int64_t{1} << 30;  // of a length: positions fit 32 bits

  int64_t start = 0;
  for (int64_t k = tid; k < i; k += kThreads) start += clamp_to(load_index(p.query_lens, k, p.index64), kMost);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) start += __shfl_xor(start, off);
  if (lane == 0) sums[tid >> 6] = start;
  __syncthreads();
  start = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) start += sums[w];

  if (i == p.num_seqs) {
    if (first == 0) p.qsl[i] = start;
    for (int64_t t = start + first; t < p.num_tokens; t += step) {
      p.positions[t] = 0;
      p.slots[t] = -1;
      if (p.parents) p.mask[t] = 0;
    }
    return;
  }

  const int64_t computed = clamp_to(load_index(p.computed, i, p.index64), kMost);
  const int64_t q = clamp_to(load_index(p.query_lens, i, p.index64), kMost);
  const int64_t row = load_index(p.rows, i, p.index64);
  const bool has_table = row >= 0 && row < p.table_rows;
  const int64_t table = has_table ? row * p.table_stride : 0;
  int64_t held = 0, n0 = 0, fresh = 0;  // the new blocks: columns held .. held + fresh
  if (p.new_blocks) {
    held = load_index(p.held, i, p.index64);
    n0 = clamp_to(load_index(p.new_start, i, p.index64), p.num_new);
    fresh = clamp_to(load_index(p.new_start, i + 1, p.index64), p.num_new) - n0;
    if (held < 0 || held >= p.width || fresh < 0 || !has_table) fresh = 0;
  }
  auto block = [&](int64_t col) -> int64_t {
    if (!has_table || col >= p.width) return -1;
    const int64_t k = col - held;
    if (k >= 0 && k < fresh) return load_index(p.new_blocks, n0 + k, p.index64);
    return load_index(p.tables, table + col, p.tables64);
  };
  auto put = [&](void* to, int64_t at, int64_t v) {
    if (p.tables64) static_cast<int64_t*>(to)[at] = v;
    else static_cast<int32_t*>(to)[at] = static_cast<int32_t>(v);
  };

  const int64_t len = computed + q;
  if (first == 0) {
    p.qsl[i] = start;
    p.seq_lens[i] = len;
  }
  const uint32_t bs = static_cast<uint32_t>(p.block_size);
  const int64_t used = (static_cast<uint32_t>(len) + bs - 1) / bs;
  for (int64_t c = first; c < p.max_blocks; c += step) put(p.block_tables, i * p.max_blocks + c, c < used ? block(c) : 0);
  for (int64_t j = first; j < q && start + j < p.num_tokens; j += step) {
    const uint32_t at = static_cast<uint32_t>(computed + j);
    const int64_t b = block(at / bs);
    p.slots[start + j] = b < 0 ? -1 : b * bs + at % bs;
    if (!p.parents || j >= kTreeRows) {
      p.positions[start + j] = at;
      if (p.parents) p.mask[start + j] = 0;
    }
  }
  for (int64_t k = first; k < fresh && held + k < p.width; k += step)
    put(p.tables, table + held + k, load_index(p.new_blocks, n0 + k, p.index64));

  // The tree: lane j is row j.  Every round doubles the ancestors that a row has.
  if (p.parents && blockIdx.y == 0 && tid < 64) {
    const bool there = lane < q && start + lane < p.num_tokens;
    int up = there ? static_cast<int>(clamp_to(load_index(p.parents, start + lane, p.index64) + 1, kTreeRows)) - 1 : -1;
    if (up >= lane) up = -1;  // only an earlier row can be a parent
    uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
#pragma unroll
    for (int r = 0; r < 6; ++r) {
      const int from = up < 0 ? lane : up;
      lo |= static_cast<uint32_t>(__shfl(static_cast<int>(lo), from));
      hi |= static_cast<uint32_t>(__shfl(static_cast<int>(hi), from));
      const int next = __shfl(up, from);
      up = up < 0 ? -1 : next;
    }
    if (there) {
      p.mask[start + lane] = static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
      p.positions[start + lane] = computed + __popc(lo) + __popc(hi) - 1;
    }
  }
}

// ---- commit ---------------------------------------------------------------------
//
// Every wave walks its request's tree for itself: lane j holds row j, a step of the
// walk is one ballot over the children of the current row that hold its choice, and
// lane d ends with the path's row d.  The threads then own units of the accepted
// rows of the caches: a path's rows lie at or behind their new places, in order, so
// that a thread that goes along the path never overwrites what it has still to read.

constexpr int kCaches = 128;              // of a launch, at most
constexpr int kGridY = 65535;             // workgroups of a launch along y
constexpr int kMostSeqs = (1 << 24) - 1;  // along x: a grid has less than 2^32 threads in a direction

struct CommitParams {
  const void* chosen;
  const void* ids;
  const void* parents;
  const void* qsl;
  const void* slots;
  int64_t* counts;
  int64_t* tokens;
  int64_t num_tokens, num_slots;
  int64_t row_bytes;
  int max_rows, units, num_caches;  // units of a row
  int index64, qsl64, slots64;
  char* caches[kCaches];
};

__device__ __forceinline__ int64_t lane_value64(int64_t x, int lane) {
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), lane));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}
__device__ __forceinline__ int64_t shuffle64(int64_t x, int lane) {
  const uint32_t lo = static_cast<uint32_t>(__shfl(static_cast<int>(x), lane));
  const uint32_t hi = static_cast<uint32_t>(__shfl(static_cast<int>(x >> 32), lane));
  return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
}

template <class U>
__global__ __launch_bounds__(kThreads) void commit_drafts_kernel(CommitParams p) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t i = blockIdx.x;
  const int64_t row0 = load_index(p.qsl, i, p.qsl64);
  int64_t rows = load_index(p.qsl, i + 1, p.qsl64) - row0;
  // Offsets that leave the batch are never followed.
  if (row0 < 0 || rows < 0 || row0 > p.num_tokens || rows > p.num_tokens - row0) rows = 0;
  const int q = static_cast<int>(rows < p.max_rows ? rows : p.max_rows);

  const bool there = lane < q;
  const int64_t t = row0 + lane;
  const int64_t chosen = there ? load_index(p.chosen, t, p.index64) : -1;
  const int64_t id = there ? load_index(p.ids, t, p.index64) : -1;
  const int64_t up64 = there ? load_index(p.parents, t, p.index64) : -1;
  const int64_t slot = there ? load_index(p.slots, t, p.slots64) : -1;
  const int up = up64 >= 0 && up64 < lane ? static_cast<int>(up64) : -1;

  int path = 0, count = q > 0 ? 1 : 0, at = 0;
  while (count > 0 && count < q) {
    const uint64_t next = __builtin_amdgcn_ballot_w64(up == at && id == lane_value64(chosen, at));
    if (next == 0) break;
    at = __builtin_ctzll(next);
    if (lane == count) path = at;
    ++count;
  }
  const int64_t token = shuffle64(chosen, path);
  const int64_t from = shuffle64(slot, path);
  if (blockIdx.y == 0 && tid < 64) {
    if (lane < p.max_rows) p.tokens[i * p.max_rows + lane] = lane < count ? token : -1;
    if (lane == 0) p.counts[i] = count;
  }

  const int x = static_cast<int>(blockIdx.y) * kThreads + tid;
  if (x >= p.num_caches * p.units) return;
  char* cache = p.caches[x / p.units] + static_cast<int64_t>(x % p.units) * sizeof(U);
  for (int d0 = 1; d0 < count; d0 += 8) {
    U held[8];
    bool move[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = d0 + k < count ? d0 + k : 0;
      const int64_t a = lane_value64(from, d), b = lane_value64(slot, d);
      move[k] = d > 0 && a != b && a >= 0 && a < p.num_slots && b >= 0 && b < p.num_slots;
      if (move[k]) held[k] = *reinterpret_cast<const U*>(cache + a * p.row_bytes);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int d = d0 + k < count ? d0 + k : 0;
      if (move[k]) *reinterpret_cast<U*>(cache + lane_value64(slot, d) * p.row_bytes) = held[k];
    }
  }
}

template <class U>
hipError_t launch_commit(CommitParams& p, int64_t num_seqs, hipStream_t stream) {
  const int64_t units = static_cast<int64_t>(p.num_caches) * p.units;
  const unsigned y = static_cast<unsigned>(units > 0 ? (units + kThreads - 1) / kThreads : 1);
  void* args[] = {&p};
  return hipLaunchKernel(reinterpret_cast<const void*>(&commit_drafts_kernel<U>), dim3(static_cast<unsigned>(num_seqs), y),
                         dim3(kThreads), args, 0, stream);
}

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

}  // namespace
}  // namespace ns

extern "C" int ns_step_inputs(void* tables, int64_t table_rows, int64_t table_width, int64_t table_stride,
                              int tables_is_int64,
                              const void* rows, const void* computed, const void* query_lens,
                              const void* new_blocks, const void* new_start, const void* held, int64_t num_new,
                              const void* parents, int index_is_int64,
                              int64_t num_seqs, int64_t num_tokens, int block_size, int64_t max_blocks,
                              int64_t* query_start_loc, int64_t* seq_lens, int64_t* positions,
                              int64_t* slot_mapping, void* block_tables, int64_t* tree_mask, void* stream) {
  using namespace ns;
  if (num_seqs < 0 || num_tokens < 0 || block_size <= 0 || max_blocks < 0 || table_rows < 0 || table_width < 0 ||
      num_new < 0)
    return NS_ERR_INVALID_ARG;
  if (num_seqs > 65535 || num_tokens > 1 << 30 || max_blocks > 1 << 30 || block_size > 1 << 30)
    return NS_ERR_UNSUPPORTED;
  if (!query_start_loc || (num_tokens > 0 && (!positions || !slot_mapping || (parents && !tree_mask))))
    return NS_ERR_INVALID_ARG;
  if (num_seqs > 0 && (!rows || !computed || !query_lens || !seq_lens || (max_blocks > 0 && !block_tables)))
    return NS_ERR_INVALID_ARG;
  if (table_rows > 0 && table_width > 0 && (!tables || table_stride < table_width)) return NS_ERR_INVALID_ARG;
  if (num_new > 0 && (!new_blocks || !new_start || !held)) return NS_ERR_INVALID_ARG;
  const size_t index = index_is_int64 ? 8 : 4, entry = tables_is_int64 ? 8 : 4;
  if (misaligned(tables, entry) || misaligned(block_tables, entry) || misaligned(rows, index) ||
      misaligned(computed, index) || misaligned(query_lens, index) || misaligned(new_blocks, index) ||
      misaligned(new_start, index) || misaligned(held, index) || misaligned(parents, index) ||
      misaligned(query_start_loc, 8) || misaligned(seq_lens, 8) || misaligned(positions, 8) ||
      misaligned(slot_mapping, 8) || misaligned(tree_mask, 8))
    return NS_ERR_INVALID_ARG;
  StepParams p;
  p.tables = tables;
  p.table_rows = table_rows;
  p.width = table_width;
  p.table_stride = table_stride;
  p.rows = rows;
  p.computed = computed;
  p.query_lens = query_lens;
  p.new_blocks = num_new > 0 ? new_blocks : nullptr;
  p.new_start = new_start;
  p.held = held;
  p.parents = num_tokens > 0 ? parents : nullptr;
  p.qsl = query_start_loc;
  p.seq_lens = seq_lens;
  p.positions = positions;
  p.slots = slot_mapping;
  p.mask = tree_mask;
  p.block_tables = block_tables;
  p.num_seqs = num_seqs;
  p.num_tokens = num_tokens;
  p.num_new = num_new;
  p.max_blocks = max_blocks;
  p.block_size = block_size;
  p.tables64 = tables_is_int64;
  p.index64 = index_is_int64;
  // One request may have every row: workgroups of a request as for that, a few thousand in all.
  const int64_t most = num_tokens > max_blocks ? num_tokens : max_blocks;
  int64_t y = (most + kThreads - 1) / kThreads;
  const int64_t room = 1024 / (num_seqs + 1);
  y = y < room ? y : room;
  y = y < 1 ? 1 : y;
  void* args[] = {&p};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(&step_inputs_kernel),
                                       dim3(static_cast<unsigned>(num_seqs + 1), static_cast<unsigned>(y)),
                                       dim3(kThreads), args, 0, static_cast<hipStream_t>(stream));
  return e == hipSuccess ? NS_OK : NS_ERR_HIP;
}

extern "C" int ns_commit_drafts(int64_t* counts, int64_t* tokens,
                                const void* chosen, const void* input_ids, const void* parents, int index_is_int64,
                                const void* query_start_loc, int query_start_loc_is_int64,
                                const void* slot_mapping, int slot_mapping_is_int64,
                                int64_t num_seqs, int64_t num_tokens, int max_rows,
                                void* const* caches, int num_caches, int64_t num_slots, int64_t row_bytes,
                                void* stream) {
  using namespace ns;
  if (num_seqs < 0 || num_tokens < 0 || max_rows < 0 || num_caches < 0 || num_slots < 0 || row_bytes < 0)
    return NS_ERR_INVALID_ARG;
  if (max_rows > kTreeRows || num_seqs > kMostSeqs || row_bytes > 1 << 20 || num_slots > int64_t{1} << 40)
    return NS_ERR_UNSUPPORTED;
  if (num_seqs == 0) return NS_OK;
  if (!counts || (max_rows > 0 && !tokens) || !query_start_loc) return NS_ERR_INVALID_ARG;
  if (num_tokens > 0 && (!chosen || !input_ids || !parents || !slot_mapping)) return NS_ERR_INVALID_ARG;
  if (num_caches > 0 && (!caches || row_bytes == 0)) return NS_ERR_INVALID_ARG;
  const size_t index = index_is_int64 ? 8 : 4;
  if (misaligned(counts, 8) || misaligned(tokens, 8) || misaligned(chosen, index) || misaligned(input_ids, index) ||
      misaligned(parents, index) || misaligned(query_start_loc, query_start_loc_is_int64 ? 8 : 4) ||
      misaligned(slot_mapping, slot_mapping_is_int64 ? 8 : 4))
    return NS_ERR_INVALID_ARG;
  // A row of two caches in one place would be moved twice, the second time perhaps from
  // where the first move has written already.
  uintptr_t all = static_cast<uintptr_t>(row_bytes);
  const uint64_t bytes = static_cast<uint64_t>(num_slots) * static_cast<uint64_t>(row_bytes);
  uint64_t low = ~uint64_t{0}, high = 0;  // the caches so far lie in between
  for (int c = 0; c < num_caches; ++c) {
    const uint64_t at = reinterpret_cast<uintptr_t>(caches[c]);
    if (!at) return NS_ERR_INVALID_ARG;
    for (int b = 0; b < c && at < high && at + bytes > low; ++b) {
      const uint64_t before = reinterpret_cast<uintptr_t>(caches[b]);
      if ((at < before ? before - at : at - before) < bytes) return NS_ERR_INVALID_ARG;
    }
    low = at < low ? at : low;
    high = at + bytes > high ? at + bytes : high;
    all |= at;
  }
  CommitParams p;
  p.chosen = chosen;
  p.ids = input_ids;
  p.parents = parents;
  p.qsl = query_start_loc;
  p.slots = slot_mapping;
  p.counts = counts;
  p.tokens = tokens;
  p.num_tokens = num_tokens;
  p.num_slots = num_slots;
  p.row_bytes = row_bytes;
  p.max_rows = max_rows;
  p.index64 = index_is_int64;
  p.qsl64 = query_start_loc_is_int64;
  p.slots64 = slot_mapping_is_int64;
  const int unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
  p.units = static_cast<int>(row_bytes / unit);
  // As many caches a launch as its grid holds: 15 or more, of rows of 2^20 units.
  const int fits = p.units > 0 ? kGridY * kThreads / p.units : kCaches;
  const int most = fits < kCaches ? fits : kCaches;
  for (int c0 = 0; c0 == 0 || c0 < num_caches; c0 += most) {
    p.num_caches = num_caches - c0 < most ? num_caches - c0 : most;
    for (int c = 0; c < kCaches; ++c) p.caches[c] = c < p.num_caches ? static_cast<char*>(caches[c0 + c]) : nullptr;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = unit == 16  ? launch_commit<u32x4>(p, num_seqs, st)
                         : unit == 4 ? launch_commit<uint32_t>(p, num_seqs, st)
                         : unit == 2 ? launch_commit<uint16_t>(p, num_seqs, st)
                                     : launch_commit<uint8_t>(p, num_seqs, st);
    if (e != hipSuccess) return NS_ERR_HIP;
  }
  return NS_OK;
}
