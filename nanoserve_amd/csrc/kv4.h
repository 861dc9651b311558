// The paged KV cache held in 4 bits: its record layout, shared by the writer
// (kv4_cache.hip) and the attention that reads it (kv4_attention.hip).
//
// K and V of a layer are one byte tensor each, [num_blocks, num_kv_heads,
// block_size, head_dim / 2 + 4].  The record of a (block, head) is
//   block_size * head_dim / 2 bytes of codes, then
//   block_size 32-bit words, one per token: scale << 16 | offset, both in the
//   model's dtype; a value is scale * code + offset.
// K's codes lie token after token, dims 2i and 2i + 1 in the low and high
// nibble of byte i.  V's lie in groups of four tokens: the byte of dims 2i and
// 2i + 1 of token t is byte 4 i + pos(t % 4) of group t / 4, pos = 0, 2, 1, 3.
//
// Both orders are what the matrix cores want.  A 16-token tile of either is
// head_dim * 8 contiguous bytes.  A lane's bytes of K are consecutive dims of
// one token (the contraction of q.k), its bytes of V four tokens of a few dims
// (the contraction of p.v), and in both a mask of every fourth nibble leaves
// two codes in the two halves of a register: x & 0x000F000F and
// (x >> 8) & 0x000F000F hold the codes, x & 0x00F000F0 and its shift 16 times
// the codes.  As half-precision bits such a half is the subnormal number
// code * 2^-24 (or code * 2^-20), exact, so the matrix cores take the codes
// with no conversion at all; the powers of two leave with the scale.
#pragma once

#include "ns_common.h"

namespace ns {

// Bytes of one (block, head) record.
__host__ __device__ __forceinline__ int64_t kv4_record_bytes(int block_size, int head_dim) {
  return static_cast<int64_t>(block_size) * (head_dim / 2 + 4);
}

// What both entry points ask of a cache.
inline bool kv4_shape_ok(int head_dim, int block_size) {
  return head_dim > 0 && head_dim % 8 == 0 && head_dim <= 256 && block_size > 0 && block_size % 4 == 0;
}

// Byte of token slot t (in its block) within a group of four tokens of V.
__device__ __forceinline__ int kv4_v_pos(int t) { return ((t & 1) << 1) | ((t >> 1) & 1); }

// Conversions of the model dtypes.  from_f32 rounds to nearest even.
template <class DT>
struct Half;
template <>
struct Half<F16> {
  static __device__ __forceinline__ float to_f32(uint32_t b) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(b)));
  }
  static __device__ __forceinline__ uint32_t from_f32(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
  }
  static constexpr uint32_t nan = 0x7E00u;
};
template <>
struct Half<BF16> {
  static __device__ __forceinline__ float to_f32(uint32_t b) { return __uint_as_float(b << 16); }
  static __device__ __forceinline__ uint32_t from_f32(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  }
  static constexpr uint32_t nan = 0x7FC0u;
};

// Scale and offset of a parameter word.
template <class DT>
__device__ __forceinline__ float kv4_scale(uint32_t w) {
  if constexpr (DT::code == NS_DTYPE_BF16) return __uint_as_float(w & 0xFFFF0000u);
  return Half<DT>::to_f32(w >> 16);
}
template <class DT>
__device__ __forceinline__ float kv4_offset(uint32_t w) {
  return Half<DT>::to_f32(w & 0xFFFFu);
}

}  // namespace ns
