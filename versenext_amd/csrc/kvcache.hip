// The KV cache in 8 bits on gfx950: vnx_kv_write and vnx_kv_read.
//
// A cache row (one token of one KV head) is d codes and one fp32 scale:
//   int8   scale = RN(amax / 127),  code = rint(x * RN(127 / amax))
//   e4m3   scale = RN(amax / 448),  code = e4m3(x * RN(448 / amax))
// and stands for code * scale; bf16 caches hold the values and no scale.  One
// scale per row and head keeps a row's write independent of every other row
// and lets the attention apply it to a whole column of scores.
//
// vnx_kv_write, one pass over the q | k | v rows of a projection: the
// per-head RMSNorm of q and k, the rotation (x * cos + rotate_half(x) * sin,
// TriSparseAttention._apply_rope,
// packages/verse_nex/verse_nex/tri_sparse_attn.py:182-221), q to the attention
// layout, k and v quantised into the cache at rows lens[b] + i.  A head is
// d / 16 lanes; a lane holds 8 values of the lower half and the 8 of the upper
// half that rotate with them, so the rotation needs no exchange and the norm
// and the maximum one reduction over the head's lanes.
// vnx_kv_read: codes * scale of a range of rows.
// Both are bound by HBM where the rows are many (on the GPU: 16,384 tokens x 48
// heads of 128 with norms, int8, 71 us for 371 MB, 5.2 TB/s; 131,072 rows x 8
// heads of 128 from e4m3, 151 us, 5.4 TB/s; a large copy runs at 5.3) and by the
// launch elsewhere (one token: 2.8 us and 2.9).
#include <climits>

#include "kvcache.h"

namespace vnx {
namespace {

constexpr float kKvTiny = 7.8886090522101181e-31f;  // 2^-100: top / amax stays finite above it

struct KvWriteParams {
  const void* qkv;
  int64_t ldq;
  const int32_t* lens;
  const float* cos;      // NULL: no rotation
  const float* sin;
  const float* qn;       // NULL: no norm
  const float* kn;
  uint16_t* q;
  char* kc;
  char* vc;
  float* ks;
  float* vs;
  int64_t c_sb, c_sh, c_sr;  // elements
  int64_t s_sb, s_sh;
  int64_t cap;               // rows below cap (and the tables') are written
  uint32_t tokens;           // B * n
  int chunks, per;           // waves a token, head groups a wave
  int n, H, Hkv;
  float eps;
};

template <typename T>
__device__ __forceinline__ void kv_ld8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  } else {
    // 16-bit rows are read once (past the caches 71.1 us, else 77.1 for 16,384
    // tokens x 48 heads of 128; fp32 rows come through the loads of the tables
    // and norms, which are read again)
    const u32x4 a = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, _Float16)) {
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

__device__ __forceinline__ u32x4 kv_bf16x8(const float (&v)[8]) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = kv_pk_bf16(v[2 * i], v[2 * i + 1]);
  return o;
}

// Eight codes of values already multiplied by top / amax.
template <int KT>
__device__ __forceinline__ uint2 kv_codes(const float (&v)[8], float r) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = v[4 * h + i] * r;
    if constexpr (KT == KV_I8) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        t |= ((uint32_t)(int)__builtin_rintf(fminf(fmaxf(y[i], -127.0f), 127.0f)) & 0xFFu) << (8 * i);
      w[h] = t;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = fminf(fmaxf(y[i], -448.0f), 448.0f);
      int t = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      t = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], t, true);
      w[h] = (uint32_t)t;
    }
  }
  return make_uint2(w[0], w[1]);
}

// L = d / 16 lanes a head, a wave 64 / L heads of one token at a time, `per`
// times: the tables' row is loaded once for all of them, the next heads' values
// under the current ones' arithmetic.
template <typename TS, int KT, int L>
__global__ __launch_bounds__(256) void k_kv_write(KvWriteParams p) {
  constexpr int D = 16 * L, HD = D / 2, G = 64 / L;
  const int lane = threadIdx.x % L, gi = threadIdx.x % 64 / L;
  const uint32_t unit = (uint32_t)__builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const uint32_t tok = unit / (uint32_t)p.chunks;
  if (tok >= p.tokens) return;
  const int b = (int)(tok / (uint32_t)p.n), i = (int)(tok - (uint32_t)b * (uint32_t)p.n);
  const int64_t pos = (int64_t)p.lens[b] + i;
  const bool in = pos >= 0 && pos < p.cap;
  const int HT = p.H + 2 * p.Hkv, HQK = p.H + p.Hkv;
  const int h0 = (int)(unit - tok * (uint32_t)p.chunks) * p.per * G + gi;
  const int h1 = min(HT, h0 - gi + p.per * G);
  const TS* src = static_cast<const TS*>(p.qkv) + (int64_t)tok * p.ldq + lane * 8;
  float nlo[8], nhi[8];
  auto fetch = [&](int head) {
    if (head < h1) {
      kv_ld8(src + (int64_t)head * D, nlo);
      kv_ld8(src + (int64_t)head * D + HD, nhi);
    }
  };
  fetch(h0);
  const bool turn = p.cos && in && h0 - gi < HQK;
  float cl[8], ch[8], sl[8], sh[8];
  if (turn) {
    const float* c = p.cos + pos * D + lane * 8;
    const float* s = p.sin + pos * D + lane * 8;
    kv_ld8(c, cl);
    kv_ld8(c + HD, ch);
    kv_ld8(s, sl);
    kv_ld8(s + HD, sh);
  }
  for (int head = h0; head < h1; head += G) {
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { lo[e] = nlo[e]; hi[e] = nhi[e]; }
    fetch(head + G);
    const bool is_q = head < p.H, is_v = head >= HQK;
    if (!in && !is_q) continue;  // (a head's lanes go together: the reductions below stay inside one)
    if (!is_v) {
      const float* nw = is_q ? p.qn : p.kn;
      if (nw) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], ss));
#pragma unroll
        for (int off = L / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off, L);
        const float r = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
        float wl[8], wh[8];
        kv_ld8(nw + lane * 8, wl);
        kv_ld8(nw + HD + lane * 8, wh);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          lo[e] = lo[e] * r * wl[e];
          hi[e] = hi[e] * r * wh[e];
        }
      }
      if (turn) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = lo[e], y = hi[e];
          lo[e] = x * cl[e] - y * sl[e];
          hi[e] = y * ch[e] + x * sh[e];
        }
      }
    }
    if (is_q) {
      uint16_t* o = p.q + (((int64_t)b * p.H + head) * p.n + i) * D + lane * 8;
      u32x4 x = kv_bf16x8(lo), y = kv_bf16x8(hi);
      if (!in) x = y = u32x4{0, 0, 0, 0};  // a position outside the cache: zeros
      *reinterpret_cast<u32x4*>(o) = x;
      *reinterpret_cast<u32x4*>(o + HD) = y;
      continue;
    }
    const int kvh = head - p.H - (is_v ? p.Hkv : 0);
    char* cache = is_v ? p.vc : p.kc;
    const int64_t off = (int64_t)b * p.c_sb + (int64_t)kvh * p.c_sh + pos * p.c_sr + lane * 8;
    if constexpr (KT == KV_BF16) {
      uint16_t* o = reinterpret_cast<uint16_t*>(cache) + off;
      *reinterpret_cast<u32x4*>(o) = kv_bf16x8(lo);
      *reinterpret_cast<u32x4*>(o + HD) = kv_bf16x8(hi);
    } else {
      // the maximum of the magnitudes' bit patterns: NaN above infinity above
      // every number, so one test finds a row that has either
      uint32_t am = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        am = max(am, __float_as_uint(lo[e]) & 0x7FFFFFFFu);
        am = max(am, __float_as_uint(hi[e]) & 0x7FFFFFFFu);
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) am = max(am, (uint32_t)__shfl_xor((int)am, o, L));
      constexpr float top = KT == KV_I8 ? 127.0f : 448.0f;
      const float amax = __uint_as_float(am);
      float r = 0.0f, s = am >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : 0.0f;
      if (am < 0x7F800000u && amax >= kKvTiny) {
        r = top / amax;
        s = amax / top;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] = hi[e] = 0.0f;  // not x * 0: -0, or NaN
      }
      *reinterpret_cast<uint2*>(cache + off) = kv_codes<KT>(lo, r);
      *reinterpret_cast<uint2*>(cache + off + HD) = kv_codes<KT>(hi, r);
      if (lane == 0) (is_v ? p.vs : p.ks)[(int64_t)b * p.s_sb + (int64_t)kvh * p.s_sh + pos] = s;
    }
  }
}

struct KvReadParams {
  const char* c[2];        // k, v codes
  const float* s[2];
  void* o[2];
  const int32_t* start;    // NULL: 0
  int64_t c_sb, c_sh, c_sr, s_sb, s_sh, cap;
  int64_t o_sb, o_sh, o_sr;
  int rows, Hkv, BH;
};

// Eight values a thread (8 bytes of codes in, 16 or 32 out), L = d / 8 threads a row.
template <typename TO, int KT, int L>
__global__ __launch_bounds__(256) void k_kv_read(KvReadParams p) {
  const int which = blockIdx.z;
  const int lane = threadIdx.x % L;
  const int64_t i = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  if (i >= p.rows) return;
  for (int bh = blockIdx.y; bh < p.BH; bh += gridDim.y) {
    const int b = bh / p.Hkv, h = bh - b * p.Hkv;
    const int64_t row = i + (p.start ? p.start[b] : 0);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (row >= 0 && row < p.cap) {
      const int64_t off = b * p.c_sb + h * p.c_sh + row * p.c_sr + lane * 8;
      if constexpr (KT == KV_BF16) {
        kv_ld8(reinterpret_cast<const __hip_bfloat16*>(p.c[which]) + off, v);
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p.c[which] + off);
        const float s = p.s[which][b * p.s_sb + h * p.s_sh + row];
        float f[8];
        kv_f32x4<KT>(w.x, f);
        kv_f32x4<KT>(w.y, f + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = f[e] * s;
      }
    }
    TO* o = static_cast<TO*>(p.o[which]) + b * p.o_sb + h * p.o_sh + i * p.o_sr + lane * 8;
    if constexpr (sizeof(TO) == 4) {
      *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else if constexpr (__is_same(TO, _Float16)) {
      u32x4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) t[e] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[2 * e], (_Float16)v[2 * e + 1]});
      *reinterpret_cast<u32x4*>(o) = t;
    } else {
      *reinterpret_cast<u32x4*>(o) = kv_bf16x8(v);
    }
  }
}

// Calls f(IntC<L>{}) for a power of two L in [LO, HI].
template <int LO, int HI, typename F>
int by_lanes(int l, F&& f) {
  if constexpr (LO > HI) {
    return VNX_ERR_UNSUPPORTED;
  } else {
    return l == LO ? f(IntC<LO>{}) : by_lanes<LO * 2, HI>(l, f);
  }
}

inline bool strides16(const int64_t* s, int64_t bytes) {
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] * bytes % 16) return false;
  return true;
}

template <typename TS, int KT>
int kv_write_launch(KvWriteParams p, int d, hipStream_t st) {
  return by_lanes<1, 16>(d / 16, [&](auto l) {
    constexpr int L = decltype(l)::value;
    // a wave a head group while that leaves the chip room (16 waves a CU), else a
    // token's all (us, 16,384 tokens x 48 heads of 128 with norms: 82.7 / 71.1)
    const int groups = (p.H + 2 * p.Hkv + 64 / L - 1) / (64 / L);
    p.per = (int64_t)p.tokens * groups <= 16 * (int64_t)device_cus() ? 1 : groups;
    p.chunks = (groups + p.per - 1) / p.per;
    const int64_t grid = ((int64_t)p.tokens * p.chunks + 3) / 4;
    if (!launch_fits(grid, 256)) return (int)VNX_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((k_kv_write<TS, KT, L>), dim3((unsigned)grid), dim3(256), 0, st, p);
    VNX_LAUNCH_CHECK();
    return (int)VNX_OK;
  });
}

template <typename TS>
int kv_write_cache(const KvWriteParams& p, int cache_dtype, int d, hipStream_t st) {
  if (cache_dtype == VNX_I8) return kv_write_launch<TS, KV_I8>(p, d, st);
  if (cache_dtype == VNX_E4M3) return kv_write_launch<TS, KV_E4M3>(p, d, st);
  return kv_write_launch<TS, KV_BF16>(p, d, st);
}

inline bool head_ok(int d) { return d >= 16 && d <= 256 && (d & (d - 1)) == 0; }

}  // namespace
}  // namespace vnx

using namespace vnx;

extern "C" {

int vnx_kv_write(const vnx_kv_write_args* a, void* stream) {
  if (!a) return VNX_ERR_INVALID_ARG;
  if (a->B < 0 || a->n < 1 || a->H < 1 || a->Hkv < 1 || a->d < 1 || a->cap < 1) return VNX_ERR_INVALID_ARG;
  if (a->dtype != VNX_F32 && a->dtype != VNX_BF16 && a->dtype != VNX_F16) return VNX_ERR_UNSUPPORTED;
  const bool q8 = a->cache_dtype == VNX_I8 || a->cache_dtype == VNX_E4M3;
  if (!q8 && a->cache_dtype != VNX_BF16) return VNX_ERR_UNSUPPORTED;
  if (!head_ok(a->d)) return VNX_ERR_UNSUPPORTED;
  if (a->B == 0) return VNX_OK;
  if (!a->qkv || !a->lens || !a->q_out || !a->k_cache || !a->v_cache) return VNX_ERR_INVALID_ARG;
  if (q8 && (!a->k_scale || !a->v_scale)) return VNX_ERR_INVALID_ARG;
  if (!a->cos_table != !a->sin_table || (a->cos_table && a->table_rows < 1)) return VNX_ERR_INVALID_ARG;
  if ((a->q_norm || a->k_norm) && !(a->eps >= 0.0f)) return VNX_ERR_INVALID_ARG;
  const int64_t HT = (int64_t)a->H + 2 * (int64_t)a->Hkv;
  if (a->ldq < HT * a->d || a->cache_strides[2] < a->d || a->scale_strides[0] < 0 || a->scale_strides[1] < 0)
    return VNX_ERR_INVALID_ARG;
  if (HT > INT_MAX || a->B > INT_MAX / a->n || a->B * a->n > (INT_MAX - 256) / HT) return VNX_ERR_UNSUPPORTED;
  // 16-byte loads and stores
  if (!aligned16(a->qkv) || a->ldq * elem_size(a->dtype) % 16 || !aligned16(a->q_out) || !aligned16(a->k_cache) ||
      !aligned16(a->v_cache) || !aligned16(a->cos_table) || !aligned16(a->sin_table) || !aligned16(a->q_norm) ||
      !aligned16(a->k_norm) || !strides16(a->cache_strides, q8 ? 1 : 2) || !aligned_to(a->lens, 4) ||
      !aligned_to(a->k_scale, 4) || !aligned_to(a->v_scale, 4))
    return VNX_ERR_UNSUPPORTED;
  // rows written must not lie on one another
  const Rows rows(a->d, a->cache_strides, {a->B, a->Hkv, a->cap}), scales(a->cap, a->scale_strides, {a->B, a->Hkv});
  if (!rows.apart() || rows.meet(a->k_cache, a->v_cache, q8 ? 1 : 2) ||
      (q8 && (!scales.apart() || scales.meet(a->k_scale, a->v_scale, 4))))
    return VNX_ERR_INVALID_ARG;
  KvWriteParams p{};
  p.qkv = a->qkv; p.ldq = a->ldq; p.lens = a->lens;
  p.cos = a->cos_table; p.sin = a->sin_table; p.qn = a->q_norm; p.kn = a->k_norm;
  p.q = static_cast<uint16_t*>(a->q_out);
  p.kc = static_cast<char*>(a->k_cache); p.vc = static_cast<char*>(a->v_cache);
  p.ks = a->k_scale; p.vs = a->v_scale;
  p.c_sb = a->cache_strides[0]; p.c_sh = a->cache_strides[1]; p.c_sr = a->cache_strides[2];
  p.s_sb = a->scale_strides[0]; p.s_sh = a->scale_strides[1];
  p.cap = a->cos_table && a->table_rows < a->cap ? a->table_rows : a->cap;
  p.tokens = (uint32_t)(a->B * a->n);
  p.n = a->n; p.H = a->H; p.Hkv = a->Hkv; p.eps = a->eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (a->dtype == VNX_F32) return kv_write_cache<float>(p, a->cache_dtype, a->d, st);
  if (a->dtype == VNX_F16) return kv_write_cache<_Float16>(p, a->cache_dtype, a->d, st);
  return kv_write_cache<__hip_bfloat16>(p, a->cache_dtype, a->d, st);
}

int vnx_kv_read(const vnx_kv_read_args* a, void* stream) {
  if (!a) return VNX_ERR_INVALID_ARG;
  if (a->B < 0 || a->rows < 0 || a->Hkv < 1 || a->d < 1 || a->cap < 1) return VNX_ERR_INVALID_ARG;
  if (a->out_dtype != VNX_F32 && a->out_dtype != VNX_BF16 && a->out_dtype != VNX_F16) return VNX_ERR_UNSUPPORTED;
  const bool q8 = a->cache_dtype == VNX_I8 || a->cache_dtype == VNX_E4M3;
  if (!q8 && a->cache_dtype != VNX_BF16) return VNX_ERR_UNSUPPORTED;
  if (!head_ok(a->d)) return VNX_ERR_UNSUPPORTED;
  if (a->B == 0 || a->rows == 0) return VNX_OK;
  if (!a->k_cache || !a->v_cache || !a->k_out || !a->v_out) return VNX_ERR_INVALID_ARG;
  if (q8 && (!a->k_scale || !a->v_scale)) return VNX_ERR_INVALID_ARG;
  if (a->cache_strides[2] < a->d || a->out_strides[2] < a->d || a->scale_strides[0] < 0 || a->scale_strides[1] < 0)
    return VNX_ERR_INVALID_ARG;
  if (a->B > INT_MAX / a->Hkv) return VNX_ERR_UNSUPPORTED;
  if (!aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->k_out) || !aligned16(a->v_out) ||
      !strides16(a->cache_strides, q8 ? 1 : 2) || !strides16(a->out_strides, elem_size(a->out_dtype)) ||
      !aligned_to(a->start, 4) || !aligned_to(a->k_scale, 4) || !aligned_to(a->v_scale, 4))
    return VNX_ERR_UNSUPPORTED;
  const Rows out(a->d, a->out_strides, {a->B, a->Hkv, a->rows});
  if (!out.apart() || out.meet(a->k_out, a->v_out, elem_size(a->out_dtype))) return VNX_ERR_INVALID_ARG;
  KvReadParams p{};
  p.c[0] = static_cast<const char*>(a->k_cache); p.c[1] = static_cast<const char*>(a->v_cache);
  p.s[0] = a->k_scale; p.s[1] = a->v_scale;
  p.o[0] = a->k_out; p.o[1] = a->v_out;
  p.start = a->start;
  p.c_sb = a->cache_strides[0]; p.c_sh = a->cache_strides[1]; p.c_sr = a->cache_strides[2];
  p.s_sb = a->scale_strides[0]; p.s_sh = a->scale_strides[1]; p.cap = a->cap;
  p.o_sb = a->out_strides[0]; p.o_sh = a->out_strides[1]; p.o_sr = a->out_strides[2];
  p.rows = a->rows; p.Hkv = a->Hkv; p.BH = (int)(a->B * a->Hkv);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto to, auto kt) {
    using TO = decltype(to);
    constexpr int KT = decltype(kt)::value;
    return by_lanes<2, 32>(a->d / 8, [&](auto l) {
      constexpr int L = decltype(l)::value;
      const int64_t gx = ((int64_t)p.rows + 256 / L - 1) / (256 / L);
      if (!launch_fits(gx, 256)) return (int)VNX_ERR_UNSUPPORTED;
      hipLaunchKernelGGL((k_kv_read<TO, KT, L>), dim3((unsigned)gx, (unsigned)(p.BH < 65535 ? p.BH : 65535), 2), dim3(256), 0,
                         st, p);
      VNX_LAUNCH_CHECK();
      return (int)VNX_OK;
    });
  };
  auto by_out = [&](auto kt) {
    if (a->out_dtype == VNX_F32) return go(float{}, kt);
    if (a->out_dtype == VNX_F16) return go(_Float16{}, kt);
    return go(__hip_bfloat16{}, kt);
  };
  if (a->cache_dtype == VNX_I8) return by_out(IntC<KV_I8>{});
  return q8 ? by_out(IntC<KV_E4M3>{}) : by_out(IntC<KV_BF16>{});
}

}  // extern "C"
