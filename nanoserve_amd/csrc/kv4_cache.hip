// The 4-bit paged cache's writer, with and without the rotary embedding, and
// its reader by slot (record layout: kv4.h).
//
// A row x of head_dim values becomes
//   offset = R(min x),  scale = R((max x - min x) * (1 / 15)),
//   code   = clamp(rint((x - offset) / scale), 0, 15)      (0 where scale is 0)
// with R the rounding to the model's dtype and everything else in float32 (the
// factor 1 / 15 too, which moves the scale by a float32 step at most, where R drops
// 13 or 16 of those bits), so a stored value is within half a scale of the row's, plus the roundings of
// scale and offset.  The rotary embedding in front of it is evaluated in
// float32 from the model-dtype cos and sin and not rounded before the codes
// are taken; the rotated query is rounded once.  A row that holds a NaN or an
// infinity, or whose scale or offset leaves the dtype's range, is stored as
// code 0, scale 0, offset NaN: whatever reads it gets NaN, and nothing else does.
//
// Bound: launches and memory (with rotary, 32 tokens of 14 + 4 heads of 64 4.0 us,
// 2048 of 28 + 8 heads of 128 10.3: 37 MB at 3.6 TB/s).  A row is read once and leaves a quarter of its
// bytes behind; the only reduction is the row's minimum and maximum, over the
// lanes that hold it (head_dim / 8 of them, so 8 rows of 64 in a wave).  A
// lane holds four values of the row's first half and the four that
// rotate_half couples with them.
#include "kv4.h"

// Every product and sum is rounded by itself: a value next to the border of two
// codes is stored as the formula above has it, however a compiler would fuse them.
#pragma clang fp contract(off)

namespace ns {
namespace {

struct Kv4WriteParams {
  char* q_out;             // [T, Hq, D] contiguous (may alias q)
  const char* q;
  const char* key;
  const char* value;
  const char* cos;
  const char* sin;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, cs_st;  // element strides
  char* k_cache;
  char* v_cache;
  const void* slots;
  int slots64;
  int num_heads, num_kv_heads, head_dim, block_size;
  int64_t num_slots, record;
  int64_t nq, nk;          // groups of query rows (0 without rotary), key rows (value rows = nk)
  int groups;              // of a token's query rows
  int lane_shift;          // a row has 1 << lane_shift lanes, head_dim / 8 of them with values
  int vec;                 // rows start on 8-byte boundaries
};

// Four consecutive 16-bit values as float32.
template <class DT>
__device__ __forceinline__ void load4(const char* p, int vec, float (&x)[4]) {
  uint32_t w0, w1;
  if (vec) {
    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
    w0 = w[0];
    w1 = w[1];
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    w0 = h[0] | (static_cast<uint32_t>(h[1]) << 16);
    w1 = h[2] | (static_cast<uint32_t>(h[3]) << 16);
  }
  x[0] = Half<DT>::to_f32(w0 & 0xFFFFu);
  x[1] = Half<DT>::to_f32(w0 >> 16);
  x[2] = Half<DT>::to_f32(w1 & 0xFFFFu);
  x[3] = Half<DT>::to_f32(w1 >> 16);
}

template <class DT>
__device__ __forceinline__ void store4(char* p, int vec, const float (&x)[4]) {
  const uint32_t w0 = Half<DT>::from_f32(x[0]) | (Half<DT>::from_f32(x[1]) << 16);
  const uint32_t w1 = Half<DT>::from_f32(x[2]) | (Half<DT>::from_f32(x[3]) << 16);
  if (vec) {
    *reinterpret_cast<u32x2*>(p) = u32x2{w0, w1};
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
    h[0] = static_cast<uint16_t>(w0);
    h[1] = static_cast<uint16_t>(w0 >> 16);
    h[2] = static_cast<uint16_t>(w1);
    h[3] = static_cast<uint16_t>(w1 >> 16);
  }
}

// QROWS query rows of a token share one read of its cos and sin: a row is 16 bytes
// a lane in and out, the tables 32.
template <class DT, int QROWS>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4WriteParams p) {
  const int lanes = 1 << p.lane_shift;
  const int c = threadIdx.x & (lanes - 1);
  int64_t r = static_cast<int64_t>(blockIdx.x) * (256 >> p.lane_shift) + (threadIdx.x >> p.lane_shift);
  if (r >= p.nq + 2 * p.nk) return;  // whole rows leave together: the shuffles below stay within one
  const int kind = r < p.nq ? 0 : r < p.nq + p.nk ? 1 : 2;
  r -= kind == 0 ? 0 : kind == 1 ? p.nq : p.nq + p.nk;
  const int heads = kind == 0 ? p.groups : p.num_kv_heads;
  const int64_t t = r / heads;
  const int h = static_cast<int>(r - t * heads);
  const int half = p.head_dim / 2;
  const bool has = 8 * c < p.head_dim;

  int64_t slot = 0;
  if (kind != 0) {
    slot = load_index(p.slots, t, p.slots64);
    if (slot < 0 || slot >= p.num_slots) return;  // padding / invalid slot: never written
  }
  const int e0 = 4 * c;
  float c1[4], c2[4], s1[4], s2[4];
  if (has && kind != 2 && p.cos) {
    const char* cs = p.cos + t * p.cs_st * 2;
    const char* sn = p.sin + t * p.cs_st * 2;
    load4<DT>(cs + e0 * 2, p.vec, c1);
    load4<DT>(cs + (half + e0) * 2, p.vec, c2);
    load4<DT>(sn + e0 * 2, p.vec, s1);
    load4<DT>(sn + (half + e0) * 2, p.vec, s2);
  }
  auto rotate = [&](float (&lo)[4], float (&hi)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x1 = lo[e], x2 = hi[e];
      lo[e] = x1 * c1[e] - x2 * s1[e];
      hi[e] = x2 * c2[e] + x1 * s2[e];
    }
  };
  if (kind == 0) {
    if (!has) return;
    const int h0 = h * QROWS;
    float lo[QROWS][4], hi[QROWS][4];
#pragma unroll
    for (int j = 0; j < QROWS; ++j) {
      // Past the last head the last one again, so that all are read at once.
      const int hj = h0 + j < p.num_heads ? h0 + j : p.num_heads - 1;
      const char* src = p.q + (t * p.q_st + hj * p.q_sh) * 2;
      load4<DT>(src + e0 * 2, p.vec, lo[j]);
      load4<DT>(src + (half + e0) * 2, p.vec, hi[j]);
    }
#pragma unroll
    for (int j = 0; j < QROWS; ++j) {
      if (h0 + j >= p.num_heads) break;
      rotate(lo[j], hi[j]);
      char* d = p.q_out + (t * p.num_heads + h0 + j) * static_cast<int64_t>(p.head_dim) * 2;
      store4<DT>(d + e0 * 2, p.vec, lo[j]);
      store4<DT>(d + (half + e0) * 2, p.vec, hi[j]);
    }
    return;
  }
  const char* src = kind == 1 ? p.key + (t * p.k_st + h * p.k_sh) * 2 : p.value + (t * p.v_st + h * p.v_sh) * 2;
  float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
  if (has) {
    load4<DT>(src + e0 * 2, p.vec, lo);
    load4<DT>(src + (half + e0) * 2, p.vec, hi);
    if (kind == 1 && p.cos) rotate(lo, hi);
  }

  // The row's minimum and maximum; a lane with a NaN or an infinity makes the maximum infinite.
  float mn = INFINITY, mx = -INFINITY;
  if (has) {
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      mn = fminf(mn, fminf(lo[e], hi[e]));
      mx = fmaxf(mx, fmaxf(lo[e], hi[e]));
      fine = fine && fabsf(lo[e]) < INFINITY && fabsf(hi[e]) < INFINITY;
    }
    if (!fine) mx = INFINITY;
  }
  for (int off = lanes >> 1; off > 0; off >>= 1) {
    mn = fminf(mn, __shfl_xor(mn, off));
    mx = fmaxf(mx, __shfl_xor(mx, off));
  }
  float step = (mx - mn) * (1.f / 15.f);
  asm("" : "+v"(step));  // rounded to float32 first: the compiler would round the product to float16 at once
  uint32_t sb = Half<DT>::from_f32(step), ob = Half<DT>::from_f32(mn);
  float s = Half<DT>::to_f32(sb);
  const float b = Half<DT>::to_f32(ob);
  if (!(s < INFINITY) || !(fabsf(b) < INFINITY)) {
    sb = 0;
    ob = Half<DT>::nan;
    s = 0.f;
  }
  auto code = [&](float x) -> uint32_t {
    return s > 0.f ? static_cast<uint32_t>(fminf(fmaxf(rintf((x - b) / s), 0.f), 15.f)) : 0u;
  };
  uint32_t w1 = 0, w2 = 0;  // four codes each
  if (has) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w1 |= code(lo[e]) << (4 * e);
      w2 |= code(hi[e]) << (4 * e);
    }
  }
  const int64_t blk = slot / p.block_size;
  const int tk = static_cast<int>(slot - blk * p.block_size);
  char* rec = (kind == 1 ? p.k_cache : p.v_cache) + (blk * p.num_kv_heads + h) * p.record;
  if (has) {
    if (kind == 1) {
      char* d = rec + tk * half;
      *reinterpret_cast<uint16_t*>(d + 2 * c) = static_cast<uint16_t>(w1);
      *reinterpret_cast<uint16_t*>(d + half / 2 + 2 * c) = static_cast<uint16_t>(w2);
    } else {
      char* d = rec + (tk >> 2) * (4 * half) + kv4_v_pos(tk);
      d[4 * (2 * c)] = static_cast<char>(w1);
      d[4 * (2 * c + 1)] = static_cast<char>(w1 >> 8);
      d[4 * (half / 2 + 2 * c)] = static_cast<char>(w2);
      d[4 * (half / 2 + 2 * c + 1)] = static_cast<char>(w2 >> 8);
    }
  }
  if (c == 0) *reinterpret_cast<uint32_t*>(rec + p.block_size * half + 4 * tk) = (sb << 16) | ob;
}

struct Kv4GatherParams {
  char* k_out;
  char* v_out;
  const char* k_cache;
  const char* v_cache;
  const void* slots;
  int slots64;
  int num_kv_heads, head_dim, block_size;
  int64_t num_slots, record, rows;  // rows = tokens * kv heads
};

// One thread per eight values of a row; rows of slots outside the cache are zero.
template <class DT>
__global__ __launch_bounds__(256) void kv4_gather_kernel(Kv4GatherParams p) {
  const int chunks = p.head_dim / 8;
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t per = p.rows * chunks;
  if (i >= 2 * per) return;
  const bool is_v = i >= per;
  i -= is_v ? per : 0;
  const int64_t r = i / chunks;
  const int c = static_cast<int>(i - r * chunks);
  const int64_t t = r / p.num_kv_heads;
  const int h = static_cast<int>(r - t * p.num_kv_heads);
  const int64_t slot = load_index(p.slots, t, p.slots64);
  u32x4 out = {0u, 0u, 0u, 0u};
  if (slot >= 0 && slot < p.num_slots) {
    const int64_t blk = slot / p.block_size;
    const int tk = static_cast<int>(slot - blk * p.block_size);
    const int half = p.head_dim / 2;
    const char* rec = (is_v ? p.v_cache : p.k_cache) + (blk * p.num_kv_heads + h) * p.record;
    const uint32_t par = *reinterpret_cast<const uint32_t*>(rec + p.block_size * half + 4 * tk);
    uint32_t w = 0;  // codes of dims 8c .. 8c + 7
    if (is_v) {
      const uint8_t* d = reinterpret_cast<const uint8_t*>(rec) + (tk >> 2) * (4 * half) + 16 * c + kv4_v_pos(tk);
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= static_cast<uint32_t>(d[4 * e]) << (8 * e);
    } else {
      w = *reinterpret_cast<const uint32_t*>(rec + tk * half + 4 * c);
    }
    const float s = kv4_scale<DT>(par), b = kv4_offset<DT>(par);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      out[e >> 1] |= Half<DT>::from_f32(s * static_cast<float>((w >> (4 * e)) & 15u) + b) << (16 * (e & 1));
  }
  *reinterpret_cast<u32x4*>((is_v ? p.v_out : p.k_out) + i * 16) = out;
}

int launch_write(Kv4WriteParams& p, int dtype, hipStream_t stream) {
  int shift = 0;
  while ((8 << shift) < p.head_dim) ++shift;
  p.lane_shift = shift;
  const int64_t per = 256 >> shift;
  auto blocks_of = [&] { return (p.nq + 2 * p.nk + per - 1) / per; };
  // Four query rows a thread where there are more than four workgroups for each
  // compute unit without: 2048 tokens of 28 heads of 128 10.3 us, 12.3 singly; 32 of 14
  // of 64 4.4 and 4.1.
  const bool four = blocks_of() > 4 * 256 && p.nq > 0;
  if (four) {
    const int64_t tokens = p.nq / p.groups;
    p.groups = (p.num_heads + 3) / 4;
    p.nq = tokens * p.groups;
  }
  const int64_t blocks = blocks_of();
  if (blocks > 0x7FFFFFFF) return NS_ERR_INVALID_ARG;
  void* args[] = {&p};
  const void* fn = dtype == NS_DTYPE_F16 ? (four ? reinterpret_cast<const void*>(&kv4_write_kernel<F16, 4>)
                                                 : reinterpret_cast<const void*>(&kv4_write_kernel<F16, 1>))
                                         : (four ? reinterpret_cast<const void*>(&kv4_write_kernel<BF16, 4>)
                                                 : reinterpret_cast<const void*>(&kv4_write_kernel<BF16, 1>));
  const hipError_t e = hipLaunchKernel(fn, dim3(static_cast<unsigned>(blocks)), dim3(256), args, 0, stream);
  return e == hipSuccess ? NS_OK : NS_ERR_HIP;
}

bool misaligned(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

// Checks shared by the two writers; fills what they share.
int fill_write(Kv4WriteParams& p, const void* key, int64_t k_st, int64_t k_sh, const void* value, int64_t v_st,
               int64_t v_sh, void* k_cache, void* v_cache, const void* slots, int slots64, int64_t T, int Hkv, int D,
               int block_size, int64_t num_blocks, int dtype) {
  if (dtype != NS_DTYPE_F16 && dtype != NS_DTYPE_BF16) return NS_ERR_UNSUPPORTED;
  if (T < 0 || Hkv <= 0 || D <= 0 || block_size <= 0 || num_blocks <= 0) return NS_ERR_INVALID_ARG;
  if (!kv4_shape_ok(D, block_size)) return NS_ERR_UNSUPPORTED;
  if (T == 0) return NS_OK;
  if (!key || !value || !k_cache || !v_cache || !slots) return NS_ERR_INVALID_ARG;
  if (misaligned(k_cache, 16) || misaligned(v_cache, 16) || misaligned(key, 2) || misaligned(value, 2) ||
      misaligned(slots, slots64 ? 8 : 4))
    return NS_ERR_INVALID_ARG;
  p.key = static_cast<const char*>(key);
  p.value = static_cast<const char*>(value);
  p.k_st = k_st;
  p.k_sh = k_sh;
  p.v_st = v_st;
  p.v_sh = v_sh;
  p.k_cache = static_cast<char*>(k_cache);
  p.v_cache = static_cast<char*>(v_cache);
  p.slots = slots;
  p.slots64 = slots64 ? 1 : 0;
  p.num_kv_heads = Hkv;
  p.head_dim = D;
  p.block_size = block_size;
  p.num_slots = num_blocks * block_size;
  p.record = kv4_record_bytes(block_size, D);
  p.nk = T * Hkv;
  p.vec = !misaligned(key, 8) && !misaligned(value, 8) && k_st % 4 == 0 && k_sh % 4 == 0 && v_st % 4 == 0 &&
          v_sh % 4 == 0;
  return NS_OK;
}

}  // namespace
}  // namespace ns

extern "C" int ns_reshape_and_cache_int4(const void* key, const void* value,
                                         int64_t key_stride_token, int64_t key_stride_head,
                                         int64_t value_stride_token, int64_t value_stride_head,
                                         void* k_cache, void* v_cache,
                                         const void* slot_mapping, int slot_mapping_is_int64,
                                         int64_t num_tokens, int num_kv_heads, int head_dim,
                                         int block_size, int64_t num_blocks, int dtype, void* stream) {
  using namespace ns;
  Kv4WriteParams p = {};
  const int rc = fill_write(p, key, key_stride_token, key_stride_head, value, value_stride_token, value_stride_head,
                            k_cache, v_cache, slot_mapping, slot_mapping_is_int64, num_tokens, num_kv_heads, head_dim,
                            block_size, num_blocks, dtype);
  if (rc != NS_OK || num_tokens == 0) return rc;
  return launch_write(p, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int ns_rope_reshape_and_cache_int4(void* q_out, const void* query,
                                              int64_t q_stride_token, int64_t q_stride_head,
                                              const void* key, int64_t key_stride_token, int64_t key_stride_head,
                                              const void* value, int64_t value_stride_token, int64_t value_stride_head,
                                              const void* cos, const void* sin, int64_t cos_sin_stride_token,
                                              void* k_cache, void* v_cache,
                                              const void* slot_mapping, int slot_mapping_is_int64,
                                              int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim,
                                              int block_size, int64_t num_blocks, int dtype, void* stream) {
  using namespace ns;
  if (num_heads <= 0) return NS_ERR_INVALID_ARG;
  Kv4WriteParams p = {};
  const int rc = fill_write(p, key, key_stride_token, key_stride_head, value, value_stride_token, value_stride_head,
                            k_cache, v_cache, slot_mapping, slot_mapping_is_int64, num_tokens, num_kv_heads, head_dim,
                            block_size, num_blocks, dtype);
  if (rc != NS_OK || num_tokens == 0) return rc;
  if (!q_out || !query || !cos || !sin) return NS_ERR_INVALID_ARG;
  if (misaligned(q_out, 2) || misaligned(query, 2) || misaligned(cos, 2) || misaligned(sin, 2))
    return NS_ERR_INVALID_ARG;
  p.q_out = static_cast<char*>(q_out);
  p.q = static_cast<const char*>(query);
  p.q_st = q_stride_token;
  p.q_sh = q_stride_head;
  p.cos = static_cast<const char*>(cos);
  p.sin = static_cast<const char*>(sin);
  p.cs_st = cos_sin_stride_token;
  p.num_heads = num_heads;
  p.groups = num_heads;
  p.nq = num_tokens * num_heads;
  p.vec = p.vec && !misaligned(q_out, 8) && !misaligned(query, 8) && !misaligned(cos, 8) && !misaligned(sin, 8) &&
          q_stride_token % 4 == 0 && q_stride_head % 4 == 0 && cos_sin_stride_token % 4 == 0;
  return launch_write(p, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int ns_gather_cache_int4(void* k_out, void* v_out, const void* k_cache, const void* v_cache,
                                    const void* slot_mapping, int slot_mapping_is_int64,
                                    int64_t num_tokens, int num_kv_heads, int head_dim,
                                    int block_size, int64_t num_blocks, int dtype, void* stream) {
  using namespace ns;
  if (dtype != NS_DTYPE_F16 && dtype != NS_DTYPE_BF16) return NS_ERR_UNSUPPORTED;
  if (num_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks <= 0)
    return NS_ERR_INVALID_ARG;
  if (!kv4_shape_ok(head_dim, block_size)) return NS_ERR_UNSUPPORTED;
  if (num_tokens == 0) return NS_OK;
  if (!k_out || !v_out || !k_cache || !v_cache || !slot_mapping) return NS_ERR_INVALID_ARG;
  if (misaligned(k_out, 16) || misaligned(v_out, 16) || misaligned(k_cache, 16) || misaligned(v_cache, 16) ||
      misaligned(slot_mapping, slot_mapping_is_int64 ? 8 : 4))
    return NS_ERR_INVALID_ARG;
  Kv4GatherParams p;
  p.k_out = static_cast<char*>(k_out);
  p.v_out = static_cast<char*>(v_out);
  p.k_cache = static_cast<const char*>(k_cache);
  p.v_cache = static_cast<const char*>(v_cache);
  p.slots = slot_mapping;
  p.slots64 = slot_mapping_is_int64 ? 1 : 0;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_slots = num_blocks * block_size;
  p.record = kv4_record_bytes(block_size, head_dim);
  p.rows = num_tokens * num_kv_heads;
  const int64_t blocks = (2 * p.rows * (head_dim / 8) + 255) / 256;
  if (blocks > 0x7FFFFFFF) return NS_ERR_INVALID_ARG;
  void* args[] = {&p};
  const void* fn = dtype == NS_DTYPE_F16 ? reinterpret_cast<const void*>(&kv4_gather_kernel<F16>)
                                         : reinterpret_cast<const void*>(&kv4_gather_kernel<BF16>);
  const hipError_t e = hipLaunchKernel(fn, dim3(static_cast<unsigned>(blocks)), dim3(256), args, 0,
                                       static_cast<hipStream_t>(stream));
  return e == hipSuccess ? NS_OK : NS_ERR_HIP;
}
