// Rows of 8-bit integer codes (device side), shared by what makes them and the
// product that reads them.
#pragma once

#include "kvcache.h"

namespace vnx {

// Eight values of dtype TS at p (on their own size only) to fp32.
template <typename TS>
__device__ __forceinline__ void q8_ld8(const TS* p, float (&v)[8]) {
  if constexpr (sizeof(TS) == 4) {
    f32x4 a, b;
    __builtin_memcpy(&a, p, 16);
    __builtin_memcpy(&b, p + 4, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  } else {
    u32x4 a;
    __builtin_memcpy(&a, p, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(TS, _Float16)) {
        const uint32_t w = a[i];
        const f16x2 h = __builtin_bit_cast(f16x2, w);
        v[2 * i] = (float)h[0];
        v[2 * i + 1] = (float)h[1];
      } else {
        v[2 * i] = __uint_as_float(a[i] << 16);
        v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
      }
    }
  }
}

template <typename TS>
__device__ __forceinline__ float q8_ld1(const TS* p) {
  if constexpr (__is_same(TS, uint16_t)) return __uint_as_float((uint32_t)*p << 16);
  else return (float)*p;
}

// x rounded to TS (nearest even) and back.
template <typename TS>
__device__ __forceinline__ float q8_round(float x) {
  if constexpr (__is_same(TS, float)) return x;
  else if constexpr (__is_same(TS, _Float16)) return (float)(_Float16)x;
  else return (float)(__bf16)x;
}

template <typename TS>
__device__ __forceinline__ void q8_st1(TS* p, float x) {
  if constexpr (__is_same(TS, uint16_t)) *p = __builtin_bit_cast(uint16_t, (__bf16)x);
  else *p = (TS)x;
}

// Eight fp32 values rounded to TS at p (on its own size only).
template <typename TS>
__device__ __forceinline__ void q8_st8(TS* p, const float (&v)[8]) {
  if constexpr (sizeof(TS) == 4) {
    const f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
    __builtin_memcpy(p, &a, 16);
    __builtin_memcpy(p + 4, &b, 16);
  } else {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(TS, _Float16))
        o[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
      else o[i] = kv_pk_bf16(v[2 * i], v[2 * i + 1]);
    }
    __builtin_memcpy(p, &o, 16);
  }
}

// Calls f(TS{}) for a dtype code: float, uint16_t (bf16 bits) or _Float16.
template <typename F>
int q8_by_type(int dtype, F&& f) {
  if (dtype == VNX_F32) return f(float{});
  if (dtype == VNX_BF16) return f(uint16_t{});
  return f(_Float16{});
}

inline bool q8_float(int dtype) { return dtype == VNX_F32 || dtype == VNX_BF16 || dtype == VNX_F16; }

}  // namespace vnx
