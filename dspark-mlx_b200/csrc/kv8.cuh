// Layout and conversions of the paged 8-bit KV cache, shared by its append and its attention.
//
// A page holds page_size tokens (a multiple of 64) of every KV head. Per page and KV head:
//   keys    page_size rows of head_dim e4m3 codes. From head_dim 128 on, the 16-byte chunk c of
//           token t's row is stored at position c ^ (t & 7), so that the eight 16-byte loads of
//           one shared-memory phase (four chunks of two neighbouring tokens) fall in distinct
//           banks when a page is copied to shared memory as it is;
//   values  page_size / 64 groups of [head_dim][64 tokens] codes: the product over tokens reads
//           16 tokens of one column with one 16-byte load;
//   scales  one fp32 power of two for the keys and one for the values, value = code * scale.
// A power of two costs an e4m3 code no precision, and makes a later growth of the scale an exact
// shift of the codes already there, except where they reach e4m3's subnormals.
#pragma once

#include "common.cuh"

namespace dsm {

constexpr int kKv8Group = 64;       // tokens per value group: page sizes are multiples of it
constexpr int kKv8MaxPage = 1024;   // tokens per page
constexpr int kKv8MaxBatch = 8192;  // sequences per call
constexpr int kKv8MaxPages = 1 << 20;  // pages per sequence: page sums of a scan block stay in 32 bits
constexpr int kKv8MinExp = -120, kKv8MaxExp = 120;  // scale exponents; 2^-e stays a normal fp32

// the stored position of 16-byte chunk c of token t's key row
template <int HD>
__device__ __forceinline__ int kv8_key_chunk(int c, int t) {
  return HD >= 128 ? (c ^ (t & 7)) : c;
}

// four e4m3 codes of w -> fp32
__device__ __forceinline__ void kv8_to_f32(uint32_t w, float (&o)[4]) {
  uint32_t lo, hi;
  e4m3x4_to_f16(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  o[0] = a.x;
  o[1] = a.y;
  o[2] = b.x;
  o[3] = b.y;
}

// four fp32 values -> e4m3 codes, nearest even (NaN -> 0x7f; callers keep |x| <= 448 or NaN)
__device__ __forceinline__ uint32_t kv8_from_f32(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n"
      " mov.b32 %0, {lo, hi};\n}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

__device__ __forceinline__ float kv8_exp2i(int e) { return __int_as_float((e + 127) << 23); }  // |e| <= 126
__device__ __forceinline__ int kv8_exponent(float pow2) { return int((__float_as_uint(pow2) >> 23) & 0xffu) - 127; }

// the least e in [kKv8MinExp, kKv8MaxExp] with amax <= 448 * 2^e = 1.75 * 2^(e + 8), amax finite
__device__ __forceinline__ int kv8_scale_exp(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = int(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return amax > 0.f ? min(max(e, kKv8MinExp), kKv8MaxExp) : kKv8MinExp;
}

__device__ __forceinline__ float kv8_warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float kv8_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// x / d == umulhi(x, kv8_per_page) for page = 64 d, d = 2 .. 16, and x < 2^28: ceil(2^32 / d) is off by less than
// 1, so the product by less than x <= 2^32 / d, a step of the quotient. 0 stands for d = 1
inline uint32_t kv8_per_page(int page) {
  const int64_t d = page / kKv8Group;
  return d == 1 ? 0u : uint32_t(((int64_t(1) << 32) + d - 1) / d);
}

inline bool kv8_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool kv8_head_dim_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }
inline bool kv8_page_ok(int page) { return page > 0 && page % kKv8Group == 0 && page <= kKv8MaxPage; }

}  // namespace dsm
