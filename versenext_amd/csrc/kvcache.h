// Codes of the 8-bit KV cache (device side), shared by its writer, its reader
// and the attention over it.
#pragma once

#include "vnx_internal.h"

namespace vnx {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

enum { KV_I8 = 0, KV_E4M3 = 1, KV_BF16 = 2 };

inline bool aligned_to(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Two fp32 values to a bf16 pair, nearest even (v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t kv_pk_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// The four codes of a word as fp32 (exact).
template <int KT>
__device__ __forceinline__ void kv_f32x4(uint32_t w, float* f) {
  if constexpr (KT == KV_I8) {
    f[0] = (float)(int8_t)w;
    f[1] = (float)(int8_t)(w >> 8);
    f[2] = (float)(int8_t)(w >> 16);
    f[3] = (float)(int8_t)(w >> 24);
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
  }
}

}  // namespace vnx
