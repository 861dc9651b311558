// Order keys of logits, shared by the greedy (argmax.hip) and the stochastic
// (sample.hip) token selection.
//
// torch.argmax's rules -- the first index among equal maxima, the first NaN if
// the row holds one -- are folded into one 64-bit key per candidate:
//     key = order(value) << 32 | (2^32 - 1 - index)
// where order() maps floats to unsigned integers in value order (+0 and -0
// equal, every NaN above +inf), so the largest key is the answer.
#pragma once

#include "ns_convert.h"

namespace ns {

constexpr uint32_t kNanOrder = 0xFFFFFFFFu;

__device__ __forceinline__ uint32_t order_of(float v) {
  uint32_t u = __float_as_uint(v);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return kNanOrder;
  if (u == 0x80000000u) u = 0u;        // -0 == +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
// The value of an order (not NaN's).
__device__ __forceinline__ float value_of(uint32_t ord) {
  return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7FFFFFFFu) : ~ord);
}

__device__ __forceinline__ uint64_t key_of(float v, uint32_t idx) {
  return (static_cast<uint64_t>(order_of(v)) << 32) | static_cast<uint64_t>(0xFFFFFFFFu - idx);
}

__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// Another lane of the same 16 by a data-parallel move, which costs a register
// move where a shuffle is a trip through LDS.
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false));
}
template <int CTRL>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  return (static_cast<uint64_t>(moved<CTRL>(static_cast<uint32_t>(v >> 32))) << 32) |
         moved<CTRL>(static_cast<uint32_t>(v));
}
// The 16 lanes' best, on each of them: neighbours, pairs, fours and eights
// exchange (the two mirrors meet lanes that hold the same by then).
template <class T, class Best>
__device__ __forceinline__ T row_best(T v, Best best) {
  v = best(v, moved<0xB1>(v));   // lane ^ 1
  v = best(v, moved<0x4E>(v));   // lane ^ 2
  v = best(v, moved<0x141>(v));  // 7 - lane, of eight
  return best(v, moved<0x140>(v));  // 15 - lane
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  return (static_cast<uint64_t>(lane_of(static_cast<uint32_t>(v >> 32), lane)) << 32) |
         lane_of(static_cast<uint32_t>(v), lane);
}
template <class T, class Best>
__device__ __forceinline__ T wave_best(T v, Best best) {
  v = row_best(v, best);
  return best(best(lane_of(v, 0), lane_of(v, 16)), best(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ uint32_t min_u32(uint32_t a, uint32_t b) { return a < b ? a : b; }
__device__ __forceinline__ uint64_t wave_max(uint64_t k) { return wave_best(k, max_u64); }

template <int DT>
__device__ __forceinline__ float elem_f32(const char* row, int64_t i) {
  if constexpr (DT == NS_DTYPE_F32) return reinterpret_cast<const float*>(row)[i];
  const uint16_t h = reinterpret_cast<const uint16_t*>(row)[i];
  if constexpr (DT == NS_DTYPE_F16) return static_cast<float>(__builtin_bit_cast(_Float16, h));
  return __uint_as_float(static_cast<uint32_t>(h) << 16);
}

// Element e of a 16-byte vector of row elements.
template <int DT>
__device__ __forceinline__ float vec_elem_f32(const u32x4& w, int e) {
  if constexpr (DT == NS_DTYPE_F32) return __uint_as_float(w[e]);
  const uint16_t h = static_cast<uint16_t>((w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
  return DT == NS_DTYPE_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, h))
                            : __uint_as_float(static_cast<uint32_t>(h) << 16);
}

}  // namespace ns
