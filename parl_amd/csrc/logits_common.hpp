// logits_common.hpp — rows of logits in float32, bfloat16 or float16: loads, and the order of values.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace parlhip {

int* device_error_flag();  // scan_kernels.hip

struct bf16_t { uint16_t bits; };
struct f16_t { _Float16 v; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((uint32_t)x.bits << 16); }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)x.v; }

// one rounding, to nearest even
__device__ __forceinline__ void from_f32(float x, float& o) { o = x; }
__device__ __forceinline__ void from_f32(float x, f16_t& o) { o.v = (_Float16)x; }
__device__ __forceinline__ void from_f32(float x, bf16_t& o) {
  const __bf16 h = (__bf16)x;
  o.bits = __builtin_bit_cast(uint16_t, h);
}

// 16 bytes from / to an address that is only aligned to the element: a row of an odd length starts anywhere.  Global
// memory takes such an access whole (the target runs in unaligned-access mode), so no row needs an aligned head.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2), may_alias));
typedef u32x4 u32x4_at4 __attribute__((aligned(4), may_alias));
template <typename T>
struct Vec16 {
  static constexpr int n = 16 / sizeof(T);
  u32x4 raw;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(T) == 4) raw = *reinterpret_cast<const u32x4_at4*>(p);
    else raw = *reinterpret_cast<const u32x4_at2*>(p);
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4_at4*>(p) = raw;
    else *reinterpret_cast<u32x4_at2*>(p) = raw;
  }
  __device__ __forceinline__ float get(int i) const;   // i: a constant after unrolling
  __device__ __forceinline__ void unpack(float (&f)[n]) const {
#pragma unroll
    for (int i = 0; i < n; ++i) f[i] = get(i);
  }
  __device__ __forceinline__ void pack(const float (&f)[n]);
};
template <> __device__ __forceinline__ float Vec16<float>::get(int i) const { return __uint_as_float(raw[i]); }
template <> __device__ __forceinline__ float Vec16<bf16_t>::get(int i) const {
  const uint32_t w = raw[i >> 1];
  return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
}
template <> __device__ __forceinline__ float Vec16<f16_t>::get(int i) const {
  const uint32_t w = raw[i >> 1];
  const uint16_t h = (uint16_t)((i & 1) ? (w >> 16) : w);
  return (float)__builtin_bit_cast(_Float16, h);
}
template <> __device__ __forceinline__ void Vec16<float>::pack(const float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i] = __float_as_uint(f[i]);
}
template <> __device__ __forceinline__ void Vec16<bf16_t>::pack(const float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bf16_t lo, hi;
    from_f32(f[2 * i], lo);
    from_f32(f[2 * i + 1], hi);
    raw[i] = (uint32_t)lo.bits | ((uint32_t)hi.bits << 16);
  }
}
template <> __device__ __forceinline__ void Vec16<f16_t>::pack(const float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f16_t lo, hi;
    from_f32(f[2 * i], lo);
    from_f32(f[2 * i + 1], hi);
    raw[i] = (uint32_t)__builtin_bit_cast(uint16_t, lo.v) | ((uint32_t)__builtin_bit_cast(uint16_t, hi.v) << 16);
  }
}

__device__ __forceinline__ float wave_max_f32(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
  return x;
}

}  // namespace parlhip
