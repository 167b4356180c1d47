// Rows of 8-bit integer codes on gfx950: vnx_q8_quantize, vnx_q8_rmsnorm and
// vnx_q8_dequantize.
//
// A row t of K values is held as K codes and one fp32 scale:
//   a = max|t|,  code = rint(t * RN(127 / a)),  scale = RN(a / 127)
// and stands for code * scale.  Of an RMS norm, t = s * w and the norm's factor
// f = 1 / sqrt(mean(s^2) + eps) is the same for the whole row: it divides out of
// the codes and goes into the scale alone.  So the maximum and the sum of squares
// are one reduction, and the codes of a row are the same however its squares
// are summed.
//
// A row is read once: T threads hold it as fp32 (NV x 8 values each) from the
// load to the store.  The last vector of a row that 8 does not divide starts at
// K - 8 and so repeats values of the one before it: they are left out of the
// sum, and stored twice alike.
//
// HBM bounds it, or a few rows the launch.  us and TB/s of bytes in and out, from
// a graph: quantize 4,096 x 8,200 fp32 28.7 (5.8), 4,096 x 10,944 bf16 22.6 (6.0),
// 1 x 10,944 2.2; norm with a bf16 residual 4,096 x 10,944 bf16 47.7 (6.6; partly
// the last-level cache's), 2,048 x 4,096 fp32 15.5 (5.9).  A large copy: 5.1 TB/s.
#include <climits>

#include "q8.h"

namespace vnx {
namespace {

constexpr float kQ8Tiny = 7.8886090522101181e-31f;  // 2^-100: 127 / a stays finite above it
constexpr float kQ8Up = 0x1p100f;

struct Q8RowParams {
  const void* x;
  const void* res;
  const float* w;
  void* sum;
  int8_t* codes;
  float* scale;
  int64_t ldx, ldr, lds, ldc, M;
  int K;
  float eps;
};

// The row's scale and the factor of its codes (0: codes of 0) from the bits of
// max|t| (NaN above infinity above every number) and, of a norm, the sum of s^2
// (tiny: of (2^100 s)^2).
template <bool NORM>
__device__ __forceinline__ float q8_scale(uint32_t am, float ss, bool tiny, const Q8RowParams& p, float* r) {
  const float a = __uint_as_float(am);
  *r = 0.0f;
  if (am >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  if (a < kQ8Tiny) return 0.0f;
  *r = 127.0f / a;
  const float s = a / 127.0f;
  if constexpr (!NORM) return s;
  // a sum of squares past fp32's range: no scale rather than one of 0
  if (!(ss < __builtin_inff())) return __uint_as_float(0x7FC00000u);
  if (tiny) {
    const float root = sqrtf(ss / (float)p.K + p.eps * kQ8Up * kQ8Up);
    return s < 1.0f ? s * kQ8Up / root : s / root * kQ8Up;  // (s may be far from the rows' size: weights)
  }
  return s / sqrtf(ss / (float)p.K + p.eps);
}

// Whether a row's mean square and eps lie where fp32 loses the squares' bits, or
// the squares: they are then summed again, of values 2^100 as large (exact; below
// 2^-110 times K the new sum stays below 2^121).  Above, a square's rounding to a
// multiple of 2^-149 is 2^-40 of the mean.  The same in all threads of a row.
// Kernels of their own (EPS0) for an eps below 2^-110, the only ones that can
// meet such a row: the branch costs registers (4,096 x 16,000 bf16 85 -> 93 us).
__device__ __forceinline__ bool q8_tiny(float am, float ss, const Q8RowParams& p) {
  return am >= kQ8Tiny && ss / (float)p.K + p.eps < 0x1p-110f;
}

// Eight codes of v * r, |v * r| <= 127: adding 1.5 * 2^23 rounds to a whole
// number (nearest even) whose low byte is the code.
__device__ __forceinline__ uint2 q8_codes(const float (&v)[8], float r) {
  uint32_t u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = __float_as_uint(v[i] * r + 12582912.0f);
  auto word = [&](int b) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[b + 3], u[b + 2], 0x0C0C0400u),
                                 __builtin_amdgcn_perm(u[b + 1], u[b], 0x0C0C0400u), 0x05040100u);
  };
  return make_uint2(word(0), word(4));
}

__device__ __forceinline__ float max_bits(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
}

// T threads a row (a wave, or a workgroup), NV vectors of 8 values a thread:
// 8 <= K <= 8 T NV.  TR void: no residual.
template <typename TX, typename TR, bool NORM, bool EPS0, int T, int NV>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_q8_rows(Q8RowParams p) {
  constexpr int RPW = T < 256 ? 256 / T : 1;
  constexpr bool RES = !__is_void(TR);
  const int t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / T;
  if (row >= p.M) return;  // whole waves; a workgroup of one row never
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx;
  float s[NV][8], w[NV][8];
  int at[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) at[v] = min((v * T + t) * 8, p.K - 8);
#pragma unroll
  for (int v = 0; v < NV; ++v) q8_ld8(x + at[v], s[v]);
  if constexpr (RES) {
    const TR* r = static_cast<const TR*>(p.res) + row * p.ldr;
    float y[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) q8_ld8(r + at[v], y[v]);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[v][i] = q8_round<TX>(s[v][i] + y[v][i]);
  }
  if constexpr (NORM)
#pragma unroll
    for (int v = 0; v < NV; ++v) q8_ld8(p.w + at[v], w[v]);
  float am = 0.0f, ss = 0.0f;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int skip = (v * T + t) * 8 - at[v];   // values of another vector (8 and more: all)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float u = s[v][i];
      if constexpr (NORM) {
        ss += i >= skip ? u * u : 0.0f;
        u *= w[v][i];
        w[v][i] = u;
      }
      am = max_bits(am, __uint_as_float(__float_as_uint(u) & 0x7FFFFFFFu));
    }
  }
  am = wave_reduce(am, max_bits);
  if constexpr (NORM) ss = wave_reduce(ss, [](float a, float b) { return a + b; });
  __shared__ float la[T / 64], ls[T / 64];
  if constexpr (T > 64) {
    if ((t & 63) == 0) {
      la[t >> 6] = am;
      ls[t >> 6] = ss;
    }
    __syncthreads();
    am = la[0], ss = ls[0];
#pragma unroll
    for (int i = 1; i < T / 64; ++i) {
      am = max_bits(am, la[i]);
      ss += ls[i];
    }
  }
  bool tiny = false;
  if constexpr (EPS0) {
    tiny = q8_tiny(am, ss, p);
    if (tiny) {
      ss = 0.0f;
#pragma unroll 1
      for (int i = t; i < p.K; i += T) {
        float u = q8_ld1(x + i);
        if constexpr (RES) u = q8_round<TX>(u + q8_ld1(static_cast<const TR*>(p.res) + row * p.ldr + i));
        u *= kQ8Up;
        ss += u * u;
      }
      ss = wave_reduce(ss, [](float a, float b) { return a + b; });
      if constexpr (T > 64) {
        __syncthreads();
        if ((t & 63) == 0) ls[t >> 6] = ss;
        __syncthreads();
        ss = ls[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) ss += ls[i];
      }
    }
  }
  // (stores from here on: every load of the row is done, so the sum may be
  // written over x or the residual)
  float r;
  const float sc = q8_scale<NORM>(__float_as_uint(am), ss, tiny, p, &r);
  if (t == 0) p.scale[row] = sc;
  int8_t* codes = p.codes + row * p.ldc;
  TX* sum = static_cast<TX*>(p.sum) + row * p.lds;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if ((v * T + t) * 8 >= p.K) continue;
    uint2 c = make_uint2(0, 0);
    if (r != 0.0f) c = NORM ? q8_codes(w[v], r) : q8_codes(s[v], r);
    __builtin_memcpy(codes + at[v], &c, 8);
    if (NORM && p.sum) q8_st8(sum + at[v], s[v]);
  }
}

// Rows of any length (fewer than 8 values, or more than a workgroup holds): one
// workgroup a row, which reads it twice, a value a load.  That load bounds it: norm
// of 2,048 x 40,000 bf16 with a residual 325 us, 1.8 TB/s (32,000 by k_q8_rows 102).
template <typename TX, typename TR, bool NORM, bool EPS0>
__global__ __launch_bounds__(256) void k_q8_rows_any(Q8RowParams p) {
  constexpr bool RES = !__is_void(TR);
  const int t = threadIdx.x;
  const int64_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(p.x) + row * p.ldx;
  TX* sum = p.sum ? static_cast<TX*>(p.sum) + row * p.lds : nullptr;
  auto at = [&](int i) {
    float u = q8_ld1(x + i);
    if constexpr (RES) {
      const TR* r = static_cast<const TR*>(p.res) + row * p.ldr;
      u = q8_round<TX>(u + q8_ld1(r + i));
    }
    return u;
  };
  float am = 0.0f, ss = 0.0f;
  for (int64_t i = t; i < p.K; i += 256) {
    float u = at((int)i);
    if constexpr (NORM) {
      if (sum) q8_st1(sum + i, u);  // (this thread's own value: read before, and not again)
      ss += u * u;
      u *= p.w[i];
    }
    am = max_bits(am, __uint_as_float(__float_as_uint(u) & 0x7FFFFFFFu));
  }
  am = wave_reduce(am, max_bits);
  if constexpr (NORM) ss = wave_reduce(ss, [](float a, float b) { return a + b; });
  __shared__ float la[4], ls[4];
  if ((t & 63) == 0) {
    la[t >> 6] = am;
    ls[t >> 6] = ss;
  }
  __syncthreads();
  am = max_bits(max_bits(la[0], la[1]), max_bits(la[2], la[3]));
  ss = ls[0] + ls[1] + ls[2] + ls[3];
  bool tiny = false;
  if constexpr (EPS0) {
    tiny = q8_tiny(am, ss, p);
    if (tiny) {
      ss = 0.0f;
      for (int64_t i = t; i < p.K; i += 256) {
        const float u = (sum ? q8_ld1(sum + i) : at((int)i)) * kQ8Up;  // (the sum: this thread's own store)
        ss += u * u;
      }
      ss = wave_reduce(ss, [](float a, float b) { return a + b; });
      __syncthreads();
      if ((t & 63) == 0) ls[t >> 6] = ss;
      __syncthreads();
      ss = ls[0] + ls[1] + ls[2] + ls[3];
    }
  }
  float r;
  const float sc = q8_scale<NORM>(__float_as_uint(am), ss, tiny, p, &r);
  if (t == 0) p.scale[row] = sc;
  for (int64_t i = t; i < p.K; i += 256) {
    float u = NORM && sum ? q8_ld1(sum + i) : at((int)i);
    if constexpr (NORM) u *= p.w[i];
    p.codes[row * p.ldc + i] = r != 0.0f ? (int8_t)__float_as_uint(u * r + 12582912.0f) : (int8_t)0;
  }
}

template <typename TX, typename TR, bool NORM, bool EPS0 = false>
int q8_rows(const Q8RowParams& p, hipStream_t st) {
  if constexpr (NORM && !EPS0)
    if (p.eps < 0x1p-110f) return q8_rows<TX, TR, true, true>(p, st);
  // A wave a row up to 2,048 values (no barrier, and a token's row is short),
  // then a workgroup of 4 to 16 waves, with no more values a thread than it needs:
  // registers and idle lanes are bytes not in flight (4,096 rows of 8,200 fp32
  // by 16 waves of 32 values: quantize 36.2 us, norm 107; by 8 of 24, 28.7 and 70.3).
  auto go = [&](auto tc, auto nc) -> int {
    constexpr int T = decltype(tc)::value, NV = decltype(nc)::value, NT = T < 256 ? 256 : T;
    const int64_t wgs = (p.M + NT / T - 1) / (NT / T);
    if (!launch_fits(wgs, NT)) return VNX_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((k_q8_rows<TX, TR, NORM, EPS0, T, NV>), dim3((unsigned)wgs), dim3(NT), 0, st, p);
    VNX_LAUNCH_CHECK();
    return VNX_OK;
  };
  if (p.K >= 8) {
    if (p.K <= 512) return go(IntC<64>{}, IntC<1>{});
    if (p.K <= 1024) return go(IntC<64>{}, IntC<2>{});
    if (p.K <= 2048) return go(IntC<64>{}, IntC<4>{});
    if (p.K <= 4096) return go(IntC<256>{}, IntC<2>{});
    if (p.K <= 8192) return go(IntC<256>{}, IntC<4>{});
    if (p.K <= 12288) return go(IntC<512>{}, IntC<3>{});
    if (p.K <= 16384) return go(IntC<1024>{}, IntC<2>{});
    if (p.K <= 32768) return go(IntC<1024>{}, IntC<4>{});
  }
  if (!launch_fits(p.M, 256)) return VNX_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((k_q8_rows_any<TX, TR, NORM, EPS0>), dim3((unsigned)p.M), dim3(256), 0, st, p);
  VNX_LAUNCH_CHECK();
  return VNX_OK;
}

struct Q8ValParams {
  const int8_t* codes;
  const float* scale;
  void* out;
  int64_t ldc, ldo, M;
  int K, chunks;   // chunks of 8 L values a row
};

// Eight values a thread, L threads a chunk of a row.
template <typename TO, int L>
__global__ __launch_bounds__(256) void k_q8_values(Q8ValParams p) {
  const int64_t unit = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const int64_t row = unit / p.chunks;
  const int e0 = ((int)(unit - row * p.chunks) * L + (int)(threadIdx.x % L)) * 8;
  if (row >= p.M || e0 >= p.K) return;
  const int8_t* c = p.codes + row * p.ldc;
  TO* o = static_cast<TO*>(p.out) + row * p.ldo;
  const float s = p.scale[row];
  if (e0 + 8 > p.K) {
    for (int i = e0; i < p.K; ++i) q8_st1(o + i, (float)c[i] * s);
    return;
  }
  uint2 w;
  __builtin_memcpy(&w, c + e0, 8);
  float v[8];
  kv_f32x4<KV_I8>(w.x, v);
  kv_f32x4<KV_I8>(w.y, v + 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= s;
  q8_st8(o + e0, v);
}

// M rows of K elements, from p on: whether two of them share a byte.
bool spans_meet(const void* a, int64_t lda, int ea, const void* b, int64_t ldb, int eb, int64_t M, int64_t K) {
  const __int128 a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  const __int128 a1 = a0 + ((__int128)(M - 1) * lda + K) * ea, b1 = b0 + ((__int128)(M - 1) * ldb + K) * eb;
  return a0 < b1 && b0 < a1;
}

// Whether writing rows at `out` spoils rows at `in` that are still to be read:
// they meet, and are not the very same rows.
bool spoils(const void* out, int64_t ldo, int eo, const void* in, int64_t ldi, int ei, int64_t M, int64_t K) {
  if (!spans_meet(out, ldo, eo, in, ldi, ei, M, K)) return false;
  if (eo != ei || ldo != ldi) return true;
  if (out == in) return false;
  return Rows(K, &ldo, {M}).meet(out, in, eo);
}

// Whether one of M rows of K elements from p on shares a byte with the n bytes at s.
bool rows_meet(const void* p, int64_t ld, int e, int64_t M, int64_t K, const void* s, __int128 n) {
  const __int128 at = (__int128)reinterpret_cast<uintptr_t>(s) - (__int128)reinterpret_cast<uintptr_t>(p);
  const __int128 row = (__int128)K * e, pitch = (__int128)ld * e;
  const __int128 m = at < row ? 0 : (at - row) / pitch + 1;  // the first row that ends behind s
  return m < M && m * pitch < at + n;
}

}  // namespace
}  // namespace vnx

using namespace vnx;

extern "C" {

int vnx_q8_quantize(const void* x, int dtype, int64_t ldx, int64_t M, int64_t K, int8_t* codes, int64_t ldc,
                    float* scale, void* stream) {
  if (M < 0 || K < 1 || ldx < K || ldc < K) return VNX_ERR_INVALID_ARG;
  if (!q8_float(dtype) || K >= INT_MAX - 65536) return VNX_ERR_UNSUPPORTED;
  if (M == 0) return VNX_OK;
  const int e = elem_size(dtype);
  if (!x || !codes || !scale || !aligned_to(x, e) || !aligned_to(scale, 4)) return VNX_ERR_INVALID_ARG;
  const __int128 ns = (__int128)M * 4;
  if (spans_meet(codes, ldc, 1, x, ldx, e, M, K) || rows_meet(x, ldx, e, M, K, scale, ns) ||
      rows_meet(codes, ldc, 1, M, K, scale, ns))
    return VNX_ERR_INVALID_ARG;
  Q8RowParams p{};
  p.x = x; p.ldx = ldx; p.codes = codes; p.ldc = ldc; p.scale = scale; p.M = M; p.K = (int)K;
  return q8_by_type(dtype, [&](auto tx) {
    return q8_rows<decltype(tx), void, false>(p, static_cast<hipStream_t>(stream));
  });
}

int vnx_q8_rmsnorm(const void* x, int dtype, int64_t ldx, const void* res, int res_dtype, int64_t ldr, const float* w,
                   float eps, int64_t M, int64_t K, void* sum, int64_t lds, int8_t* codes, int64_t ldc, float* scale,
                   void* stream) {
  if (M < 0 || K < 1 || ldx < K || ldc < K || !(eps >= 0.0f) || eps > 3.4e38f) return VNX_ERR_INVALID_ARG;
  if ((res && ldr < K) || (sum && lds < K)) return VNX_ERR_INVALID_ARG;
  if (!q8_float(dtype) || (res && !q8_float(res_dtype)) || K >= INT_MAX - 65536) return VNX_ERR_UNSUPPORTED;
  if (M == 0) return VNX_OK;
  const int e = elem_size(dtype), er = elem_size(res_dtype);
  if (!x || !w || !codes || !scale || !aligned_to(x, e) || !aligned_to(w, 4) || !aligned_to(scale, 4) ||
      (res && !aligned_to(res, er)) || (sum && !aligned_to(sum, e)))
    return VNX_ERR_INVALID_ARG;
  if (spans_meet(codes, ldc, 1, x, ldx, e, M, K) || (res && spans_meet(codes, ldc, 1, res, ldr, er, M, K)) ||
      (sum && (spans_meet(codes, ldc, 1, sum, lds, e, M, K) || spoils(sum, lds, e, x, ldx, e, M, K) ||
               (res && spoils(sum, lds, e, res, ldr, er, M, K)))))
    return VNX_ERR_INVALID_ARG;
  // the weight is read by every row's workgroup, whichever others have ended
  const __int128 ns = (__int128)M * 4, nw = (__int128)K * 4;
  if (rows_meet(codes, ldc, 1, M, K, w, nw) || (sum && rows_meet(sum, lds, e, M, K, w, nw)) ||
      rows_meet(w, K, 4, 1, K, scale, ns) || rows_meet(x, ldx, e, M, K, scale, ns) ||
      (res && rows_meet(res, ldr, er, M, K, scale, ns)) || (sum && rows_meet(sum, lds, e, M, K, scale, ns)) ||
      rows_meet(codes, ldc, 1, M, K, scale, ns))
    return VNX_ERR_INVALID_ARG;
  Q8RowParams p{};
  p.x = x; p.ldx = ldx; p.res = res; p.ldr = ldr; p.w = w; p.eps = eps; p.sum = sum; p.lds = lds;
  p.codes = codes; p.ldc = ldc; p.scale = scale; p.M = M; p.K = (int)K;
  const auto st = static_cast<hipStream_t>(stream);
  return q8_by_type(dtype, [&](auto tx) -> int {
    using TX = decltype(tx);
    if (!res) return q8_rows<TX, void, true>(p, st);
    return q8_by_type(res_dtype, [&](auto tr) { return q8_rows<TX, decltype(tr), true>(p, st); });
  });
}

int vnx_q8_dequantize(const int8_t* codes, int64_t ldc, const float* scale, int64_t M, int64_t K, void* out,
                      int out_dtype, int64_t ldo, void* stream) {
  if (M < 0 || K < 1 || ldc < K || ldo < K) return VNX_ERR_INVALID_ARG;
  if (!q8_float(out_dtype) || K >= INT_MAX - 65536) return VNX_ERR_UNSUPPORTED;
  if (M == 0) return VNX_OK;
  const int e = elem_size(out_dtype);
  if (!codes || !scale || !out || !aligned_to(out, e) || !aligned_to(scale, 4)) return VNX_ERR_INVALID_ARG;
  if (spans_meet(codes, ldc, 1, out, ldo, e, M, K) || rows_meet(out, ldo, e, M, K, scale, (__int128)M * 4))
    return VNX_ERR_INVALID_ARG;
  Q8ValParams p{codes, scale, out, ldc, ldo, M, (int)K, 1};
  auto go = [&](auto to, auto lc) -> int {
    constexpr int L = decltype(lc)::value;
    p.chunks = (int)((K + 8 * L - 1) / (8 * L));
    if (M > INT64_MAX / p.chunks) return VNX_ERR_UNSUPPORTED;
    const int64_t wgs = (M * p.chunks + 256 / L - 1) / (256 / L);
    if (!launch_fits(wgs, 256)) return VNX_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((k_q8_values<decltype(to), L>), dim3((unsigned)wgs), dim3(256), 0,
                       static_cast<hipStream_t>(stream), p);
    VNX_LAUNCH_CHECK();
    return VNX_OK;
  };
  return q8_by_type(out_dtype, [&](auto to) {
    if (K <= 256) return go(to, IntC<32>{});
    if (K <= 1024) return go(to, IntC<128>{});
    return go(to, IntC<256>{});
  });
}

}  // extern "C"
