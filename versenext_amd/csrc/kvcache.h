// Codes of the 8-bit KV cache (device side), shared by its writer, its reader
// and the attention over it.
#pragma once

#include <initializer_list>

#include "vnx_internal.h"

namespace vnx {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

enum { KV_I8 = 0, KV_E4M3 = 1, KV_BF16 = 2 };

inline bool aligned_to(const void* p, unsigned n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Rows of `extent` at sum i_k stride_k, i_k < size_k.
struct Rows {
  int64_t stride[3], size[3], extent;
  int n = 0;  // dims of more than one row, by stride

  Rows(int64_t extent_, const int64_t* st, std::initializer_list<int64_t> sz) : extent(extent_) {
    for (int64_t z : sz) {
      if (z > 1) {
        int i = n++;
        for (; i > 0 && stride[i - 1] > *st; --i) stride[i] = stride[i - 1], size[i] = size[i - 1];
        stride[i] = *st, size[i] = z;
      }
      ++st;
    }
  }
  // Every dim steps over the whole of the smaller ones: no two rows meet.
  // (Layouts that interleave without nesting are not looked for.)
  bool apart() const {
    __int128 span = extent;
    for (int i = 0; i < n; ++i) {
      if (stride[i] < span) return false;
      span += (__int128)stride[i] * (size[i] - 1);
    }
    return true;
  }
  // Whether rows of these and of the same rows `delta` further on meet (apart() holds).
  bool meet(__int128 delta, int i) const {
    if (i == 0) return delta > -(__int128)extent && delta < extent;
    const __int128 s = stride[i - 1], q = delta >= 0 ? delta / s : -((-delta + s - 1) / s);  // floor
    for (__int128 k = q; k <= q + 1; ++k)
      if (k > -(__int128)size[i - 1] && k < size[i - 1] && meet(delta - k * s, i - 1)) return true;
    return false;
  }
  bool meet(const void* a, const void* b, int bytes) const {
    // the distance in elements; a part of one counts as the next (rows start on elements)
    const __int128 d = (__int128)reinterpret_cast<uintptr_t>(b) - (__int128)reinterpret_cast<uintptr_t>(a);
    return meet(d / bytes, n) || (d % bytes && meet(d / bytes + (d > 0 ? 1 : -1), n));
  }
};

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
