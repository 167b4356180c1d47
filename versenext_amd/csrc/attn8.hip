// Attention of the new rows of every sequence over its 8-bit KV cache
// (vnx_tree_attn_q8) on gfx950: a token tree, a chain of any length, one token.
//
//   S_ij = scale * sk_j * (q_i . kc_j),  P = softmax over the keys i sees,
//   O_i = sum_j P_ij sv_j vc_j           (kc, vc codes; sk, sv their scales)
//   out_i = g0 * O_i + g1 * (the same over the second segment, bf16 rows)
//   (g0, g1 = gates[0], gates[1]; no gates: g0 = 1)
//
// A code is exact in bf16 and in fp16 (8 significant bits), so the products run
// on v_mfma_f32_16x16x32_bf16 (the scores, with the bf16 queries) and _f16 (the
// values) with the codes as operands and the scales applied to scores and
// probabilities, one multiply each.
//
// A wave owns 16 CT query columns of one KV head (column c is node c / rep of
// query head kvh * rep + c % rep, so heads that share K and V share every
// loaded row) and walks keys 32 at a time.  No row passes through LDS: each
// operand is loaded in the order in which the matrix core wants it.
//   S^T[key][col]    A = K: a lane holds D / 4 consecutive bytes of key lane % 16
//                    (the order of d inside a product is free, q is loaded
//                    the same way);
//   O^T[dim][col]    A = V^T: a lane holds D / 16 consecutive bytes of each of
//                    8 keys, row m of dim tile t standing for dim m D/16 + t.
//                    The 8 keys are those of its own 8 scores, so P goes from
//                    the score registers into the B operand as it is.
// A step's rows are loaded into registers under the previous step's math.
// Statistics and sums are fp32; P * sv is rounded once to fp16 (2^-11 of each
// term), or goes in two bf16 parts where the scales lie far apart (q8_steps).
// The running maximum of a column moves only when a score passes it by 2^8:
// until then P stays below 2^8, and the step needs no exchange between lanes
// and no rescaling.
//
// Long caches with few rows are bound by HBM (8 x 5 rows over 16,000 keys, heads
// of 128: 46.8 us for 269 MB, 5.7 TB/s, and 4.8 for the join), prompts by the
// vector ALU's issue rate beside the products (2,048 rows over 8,192: 110-112 us,
// 0.7 PFLOP/s of the 1.17 of a large bf16 product), small steps by launch,
// prologue and merge (32 x 7 rows over 617: 7.9 us).
#include <climits>

#include "kvcache.h"

namespace vnx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kQ8MaxN = 64;      // nodes of a tree: bits of an ancestor word
constexpr int kQ8Split = 32;     // key splits of a launch at most
constexpr float kQ8Jump = 8.0f;  // log2 of what P may grow to before the maximum moves

struct Q8Words {
  uint64_t w[kQ8MaxN];
};

struct Q8Params {
  const uint16_t* q;
  const char* kc;
  const char* vc;
  const float* ks;
  const float* vs;
  const int32_t* lens;
  const uint64_t* anc;     // per-row words on the device (tree == 2)
  const char* k2;          // bf16 rows of the second segment
  const char* v2;
  const float* gates;
  void* out;
  float* part_o;           // [(unit * slots + slot) * 16 CT + col][D]
  float2* part_ml;
  int64_t q_sb, q_sh, q_sr;
  int64_t c_sb, c_sh, c_sr;
  int64_t s_sb, s_sh;
  int64_t o_sb, o_sh, o_sr;
  int64_t s2_sb, s2_sh, s2_sr;  // bytes
  int64_t anc_sb;
  int B, H, Hkv, rep, N, cols, Tp, T2, window;
  int tree;                // 0 chain, 1 words by value, 2 words on the device
  int groups, splits, slots;
  int f16;                 // output type: fp16, else bf16
  float c;                 // scale * log2(e)
};

__device__ __forceinline__ float q8_ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Maximum / sum over the four lanes lane % 16 + {0, 16, 32, 48}: v_permlane
// swaps pair the halves without LDS.
__device__ __forceinline__ float q8_max4(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float q8_sum4(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// v_max3_f32: a NaN is passed over (fmaxf would quiet every operand first).
__device__ __forceinline__ float q8_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ __forceinline__ float q8_absmax3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ __forceinline__ float q8_absmin3(float a, float b, float c) {
  float r;
  asm("v_min3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Where a wave's keys lie.
struct Q8Src {
  const char* k;
  const char* v;
  const float* ks;
  const float* vs;
  uint32_t sr;   // row pitch in bytes
  int rows;      // rows that may be read
};

// A buffer of the `left` rows (at most 32) from p on: what lies behind them
// reads as zeros, dword by dword, so a step needs no test of its last rows and
// a step behind the end (left <= 0) moves no data.
template <int BYTES>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t q8_buffer(const void* p, uint32_t pitch, int left) {
  const int n = min(left, 32);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, n > 0 ? (n - 1) * (int)pitch + BYTES : 0, 0x00027000);
}

// fp32 to an fp16 pair, nearest even.
__device__ __forceinline__ uint32_t q8_pk_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}

// The scales of this lane's 8 keys.
__device__ __forceinline__ void q8_scales(const float* s, int k0, int left, int g, f32x4 (&o)[2]) {
  const auto rs = q8_buffer<4>(s + k0, 4, left);
#pragma unroll
  for (int t = 0; t < 2; ++t)
    o[t] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * g, 64 * t, 0));
}

// The loaded rows of one step of 32 keys from k0 on, `left` of them to be read.
// AUX 2: past the caches (rows that nobody reads again).
template <int D, int KT, int AUX>
struct Q8Keys {
  static constexpr int E = KT == KV_BF16 ? 2 : 1;
  static constexpr int W = D / 64 * E;  // 16-byte loads a key tile
  u32x4 k[2][W];
  f32x4 sk[2];

  __device__ __forceinline__ void load(const Q8Src& s, int k0, int left, int lane) {
    const int m = lane & 15, g = lane >> 4;
    const auto rs = q8_buffer<D * E>(s.k + (int64_t)k0 * s.sr, s.sr, left);
    const int o = m * (int)s.sr + g * (D / 4 * E);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < W; ++i)
        k[t][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
            rs, o + 16 * i, 16 * t * (int)s.sr, AUX));
    if constexpr (KT != KV_BF16) q8_scales(s.ks, k0, left, g, sk);
  }

  // Operands of key tile t.
  __device__ __forceinline__ void frag(int t, bf16x8 (&f)[D / 32]) const {
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      u32x4 w;
      if constexpr (KT == KV_BF16) {
        w = k[t][s];
      } else {
        const u32x4 c = k[t][s / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = c[2 * (s % 2) + h];
          if constexpr (KT == KV_E4M3) {
            w[2 * h] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false));
            w[2 * h + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true));
          } else {
            float y[4];
            kv_f32x4<KV_I8>(x, y);
            w[2 * h] = kv_pk_bf16(y[0], y[1]);
            w[2 * h + 1] = kv_pk_bf16(y[2], y[3]);
          }
        }
      }
      f[s] = __builtin_bit_cast(bf16x8, w);
    }
  }
};

template <int D, int KT, int AUX>
struct Q8Vals {
  static constexpr int E = KT == KV_BF16 ? 2 : 1;
  static constexpr int W = D / 64 * E;  // words of a key's values a lane
  uint32_t v[8][W];
  f32x4 sv[2];

  __device__ __forceinline__ void load(const Q8Src& s, int k0, int left, int lane) {
    const int m = lane & 15, g = lane >> 4;
    const auto rs = q8_buffer<D * E>(s.v + (int64_t)k0 * s.sr, s.sr, left);
    const int o = 4 * g * (int)s.sr + m * (D / 16 * E);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int so = ((j < 4 ? 0 : 16) + (j & 3)) * (int)s.sr;
      if constexpr (W == 1) {
        v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, o, so, AUX);
      } else if constexpr (W == 2) {
        const auto w = __builtin_amdgcn_raw_buffer_load_b64(rs, o, so, AUX);
        v[j][0] = w[0]; v[j][1] = w[1];
      } else {
        const auto w = __builtin_amdgcn_raw_buffer_load_b128(rs, o, so, AUX);
        v[j][0] = w[0]; v[j][1] = w[1]; v[j][2] = w[2]; v[j][3] = w[3];
      }
    }
    if constexpr (KT != KV_BF16) q8_scales(s.vs, k0, left, g, sv);
  }

  // Operands of dim tiles 4 x .. (codes; 2 x .. of bf16 rows) from word x: the
  // 8 keys of this lane, bf16 pairs, or fp16 pairs of codes.
  template <bool BF16>
  __device__ __forceinline__ void frag(u32x4 (&f)[D / 16]) const {
#pragma unroll
    for (int x = 0; x < W; ++x) {
      if constexpr (KT == KV_BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[2 * x][j] = __builtin_amdgcn_perm(v[2 * j + 1][x], v[2 * j][x], 0x05040100u);
          f[2 * x + 1][j] = __builtin_amdgcn_perm(v[2 * j + 1][x], v[2 * j][x], 0x07060302u);
        }
      } else if constexpr (KT == KV_E4M3) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t c[2][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w = v[2 * j + h][x];
            if constexpr (BF16) {
              c[h][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
              c[h][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
            } else {
              c[h][0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
              c[h][1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
            }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            f[4 * x + 2 * h][j] = __builtin_amdgcn_perm(c[1][h], c[0][h], 0x05040100u);
            f[4 * x + 2 * h + 1][j] = __builtin_amdgcn_perm(c[1][h], c[0][h], 0x07060302u);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float a[4], b[4];
          kv_f32x4<KV_I8>(v[2 * j][x], a);
          kv_f32x4<KV_I8>(v[2 * j + 1][x], b);
#pragma unroll
          for (int i = 0; i < 4; ++i)  // (exact: the rounding mode does not matter)
            f[4 * x + i][j] = BF16 ? kv_pk_bf16(a[i], b[i])
                                   : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a[i], b[i]));
        }
      }
    }
  }
};

// What the columns of a wave see.  Keys [full_lo, full_hi) are seen by every
// column; elsewhere column ct of node[ct] sees key j when
//   Q8_CHAIN  j <= tp + node and j > tp + node - window;
//   Q8_TREE   j < tp + N, j > its position - window, and from tp on its word has
//             the bit (words read where they are needed: few steps do);
//   Q8_ALL    j < rows (the second segment).
enum { Q8_CHAIN = 0, Q8_TREE = 1, Q8_ALL = 2 };
template <int CT>
struct Q8Mask {
  int node[CT];
  int tp, window, rows, full_lo, full_hi;
  const uint64_t* words;
};

// Bit e set: key k0 + 16 (e / 4) + g4 + e % 4 is hidden from the column.
template <int KIND>
__device__ __forceinline__ uint32_t q8_hidden(int tp, int window, int rows, const uint64_t* words, int node, int k0,
                                              int g4) {
  int lo, hi;
  uint64_t w = 0;
  if constexpr (KIND == Q8_ALL) {
    lo = 0;
    hi = rows;
  } else if constexpr (KIND == Q8_CHAIN) {
    lo = tp + node - window + 1;
    hi = tp + node + 1;
  } else {
    w = words[node];
    lo = tp + __popcll(w) - window;
    hi = rows;
  }
  uint32_t hide = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int key = k0 + 16 * (e / 4) + g4 + e % 4;
    uint32_t no = (uint32_t)(key < lo) | (uint32_t)(key >= hi);
    if constexpr (KIND == Q8_TREE) {
      const int j = key - tp;  // (>= 64 only from hi on)
      no |= (uint32_t)(j >= 0) & ~(uint32_t)(w >> (j & 63));
    }
    hide |= (no & 1u) << e;
  }
  return hide;
}

template <int CT, int D>
struct Q8State {
  f32x4 acc[CT][D / 16];
  float m[CT];    // the columns' maxima, the same in the four lanes of a column; 0 before the first key
  float lim[CT];  // what a score may pass m by: -inf before the first key, then kQ8Jump
  float l[CT];    // this lane's share of the sums
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      m[ct] = 0.0f;
      lim[ct] = kNegInf;
      l[ct] = 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) acc[ct][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }
  __device__ __forceinline__ void scale(float f) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int d = 0; d < D / 16; ++d) acc[ct][d] *= f;
  }
};

// Eight fp32 values in two bf16 parts (2^-17 of each value).
__device__ __forceinline__ void q8_split(const float (&p)[8], u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t h = kv_pk_bf16(p[2 * e], p[2 * e + 1]);
    hi[e] = h;
    lo[e] = kv_pk_bf16(p[2 * e] - __uint_as_float(h << 16), p[2 * e + 1] - __uint_as_float(h & 0xFFFF0000u));
  }
}

// Walks steps s0, s0 + ds, .. < s1 of 32 keys from key `first` on: online
// softmax into st, acc in units of R.
//   not WIDE  codes only: P sv / R in fp16, 2^-11 of a term.  R is a power of two
//             that puts the largest scale so far in [2^6, 2^7) R: P <= 2^8 stays
//             in range, and fp16's smallest step costs a term 2^-25 R at most.  R
//             moves with every loaded row, seen or not, and a row's scale may lie
//             far below it, so the walk gives up (true) at a step with a scale
//             outside [2^-6, 2^7) R, to be walked again WIDE.
//   WIDE      P sv / R (bf16 rows: P) in two bf16 parts: 2^-17 of a term, in
//             fp32's range (R at most 2^40, moved by scales of 2^80 R and more): no
//             row that a column does not see costs it a bit.
template <int D, int KT, int CT, int KIND, int AUX, bool WIDE>
__device__ __forceinline__ bool q8_steps(const Q8Src& src, int first, int s0, int ds, int s1, const Q8Mask<CT>& mk,
                                        float c, const bf16x8 (&qf)[CT][D / 32], Q8State<CT, D>& st, float& R, int lane) {
  if (s0 >= s1) return false;
  const int g4 = (lane >> 4) * 4;
  Q8Keys<D, KT, AUX> keys;
  Q8Vals<D, KT, AUX> vals;
  auto left = [&](int s) { return s < s1 ? src.rows - (first + 32 * s) : 0; };
  int end = uni(s1);
  float iR = 1.0f / R;  // (infinite before the first row)
  // the rows in the order in which the loop waits for them (in another order its
  // waits for a step's keys are waits for its values too: 8 x 5 rows over 16,000
  // 58.9 us instead of 50.6)
  keys.load(src, first + 32 * s0, left(s0), lane);
  __builtin_amdgcn_sched_barrier(0);
  vals.load(src, first + 32 * s0, left(s0), lane);
  __builtin_amdgcn_sched_barrier(0);
  for (int s = s0; s < end; s += ds) {
    const int k0 = first + 32 * s;
    float x[CT][8];  // scores relative to the maxima, in the exp2 domain
    {
      bf16x8 kf[2][D / 32];
      keys.frag(0, kf[0]);
      keys.frag(1, kf[1]);
      float fk[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) fk[e] = KT == KV_BF16 ? c : keys.sk[e / 4][e % 4] * c;
      keys.load(src, k0 + 32 * ds, left(s + ds), lane);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < D / 32; ++i) a = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[t][i], qf[ct][i], a, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[ct][4 * t + i] = fmaf(a[i], fk[4 * t + i], -st.m[ct]);
        }
    }
    u32x4 vf[D / 16];
    float sv[8];
    {
      vals.template frag<WIDE>(vf);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) asm volatile("" : "+v"(vf[d]));  // converted here: the rows' registers are free
      if constexpr (KT != KV_BF16) {
        // The scales' range: in the common step by two instructions a pair, which
        // see infinities and zeros too; where that finds something, exactly.
        constexpr float kTop = WIDE ? 0x1p80f : 0x1p7f;
        float top = 0.0f, low = 0x1p127f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) top = q8_absmax3(top, vals.sv[e / 4][e % 4], vals.sv[e / 4][e % 4 + 1]);
        if constexpr (!WIDE) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) low = q8_absmin3(low, vals.sv[e / 4][e % 4], vals.sv[e / 4][e % 4 + 1]);
        }
        // (bitwise: branches between lanes here cost a copy of acc a step)
        if (__any((bool)((uint32_t)!(top < R * kTop) | (uint32_t)(!WIDE && low < R * 0x1p-6f)))) {
          uint32_t least = 0xFFFFFFFFu;  // twice the bits less 2: the sign gone, zero the largest
          top = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = fabsf(vals.sv[e / 4][e % 4]);
            top = fmaxf(top, a < __builtin_inff() ? a : 0.0f);
            least = min(least, (__float_as_uint(a) << 1) - 2);
          }
          auto out = [&] {
            const uint32_t low2 = (__float_as_uint(R) << 1) - 2 - (6u << 24);
            return (bool)((uint32_t)!(top < R * kTop) | (uint32_t)(!WIDE && least < low2));
          };
          if (__any(out())) {
            // the largest scale's exponent alone, times 2^-6, in [2^-110, 2^40]
            const int ex = min(max(uni((int)(__float_as_uint(q8_max4(top)) >> 23)) - 6, 17), 167);
            const float r = fmaxf(R, __uint_as_float((uint32_t)ex << 23));
            iR = __uint_as_float(0x7F000000u - __float_as_uint(r));  // 1 / r
            st.scale(R * iR);
            R = r;
            if (!WIDE && __any(out())) end = s;  // (the last step: what it adds is not used)
          }
        }
        asm volatile("" : "+s"(end));  // (one way out of the loop, at its end: no copies of acc)
#pragma unroll
        for (int e = 0; e < 8; ++e) sv[e] = vals.sv[e / 4][e % 4] * iR;
      }
      vals.load(src, k0 + 32 * ds, left(s + ds), lane);
    }
    if (k0 < mk.full_lo || k0 + 32 > mk.full_hi) {
      // some column does not see some key.  A scale that is not finite must
      // reach the columns that see its key alone: through the score, not sv
      uint32_t bad = 0;
      if constexpr (KT != KV_BF16) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool b = !(fabsf(sv[e]) < __builtin_inff());
          bad |= (uint32_t)b << e;
          sv[e] = b ? 0.0f : sv[e];
        }
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const uint32_t hide = q8_hidden<KIND>(mk.tp, mk.window, mk.rows, mk.words, mk.node[ct], k0, g4);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[ct][e] = hide >> e & 1 ? kNegInf : bad >> e & 1 ? __builtin_nanf("") : x[ct][e];
      }
    }
    {
      float top[CT];
      bool any = false;
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        top[ct] = q8_max3(q8_max3(x[ct][0], x[ct][1], x[ct][2]), q8_max3(x[ct][3], x[ct][4], x[ct][5]),
                          fmaxf(x[ct][6], x[ct][7]));
        any |= top[ct] > st.lim[ct];
      }
      if (__any(any)) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const bool none = st.lim[ct] == kNegInf;
          const float t = q8_max4(top[ct]);
          const float up = t > (none ? kNegInf : 0.0f) ? t : 0.0f;
          const float al = none ? 0.0f : q8_ex2(-up);
          st.m[ct] += up;
          if (t > kNegInf) st.lim[ct] = kQ8Jump;
          st.l[ct] *= al;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[ct][e] -= up;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) st.acc[ct][d] *= al;
        }
      }
    }
    auto weigh = [&](int ct, float (&p)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = q8_ex2(x[ct][e]);
        st.l[ct] += p[e];
        if constexpr (KT != KV_BF16) p[e] *= sv[e];
      }
    };
    if constexpr (WIDE) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        if constexpr (KT != KV_BF16) __builtin_amdgcn_sched_barrier(0);  // (a rare path: registers before overlap)
        float p[8];
        weigh(ct, p);
        u32x4 hi, lo;
        q8_split(p, hi, lo);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          const bf16x8 v = __builtin_bit_cast(bf16x8, vf[d]);
          st.acc[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, hi), st.acc[ct][d], 0, 0, 0);
          st.acc[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, lo), st.acc[ct][d], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float p[8];
        weigh(ct, p);
        const u32x4 w = {q8_pk_f16(p[0], p[1]), q8_pk_f16(p[2], p[3]), q8_pk_f16(p[4], p[5]), q8_pk_f16(p[6], p[7])};
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
          st.acc[ct][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, vf[d]),
                                                                __builtin_bit_cast(f16x8, w), st.acc[ct][d], 0, 0, 0);
      }
    }
  }
  return end != s1;
}

// The walk from a cleared state; acc absolute afterwards.
template <int D, int KT, int CT, int KIND, int AUX = 0>
__device__ __forceinline__ void q8_walk(const Q8Src& src, int first, int s0, int ds, int s1, const Q8Mask<CT>& mk,
                                        float c, const bf16x8 (&qf)[CT][D / 32], Q8State<CT, D>& st, int lane) {
  st.clear();
  if constexpr (KT == KV_BF16) {
    float R = 1.0f;
    q8_steps<D, KT, CT, KIND, AUX, true>(src, first, s0, ds, s1, mk, c, qf, st, R, lane);
  } else {
    float R = 0.0f;
    if (q8_steps<D, KT, CT, KIND, AUX, false>(src, first, s0, ds, s1, mk, c, qf, st, R, lane)) {
      st.clear();
      q8_steps<D, KT, CT, KIND, AUX, true>(src, first, s0, ds, s1, mk, c, qf, st, R, lane);
    }
    st.scale(R);
  }
}

// A column's node and query head.
__device__ __forceinline__ void q8_col(const Q8Params& p, int col, int& node, int& h) {
  node = col / p.rep;
  h = col - node * p.rep;
}

template <int D, int CT>
struct Q8Tile {
  int b, kvh, col0, tp;
  bf16x8 qf[CT][D / 32];
  Q8Mask<CT> mask;
  Q8Src src;
  int first, steps;   // steps of 32 keys from key first on
  Q8Src src2;

  // E: bytes of the cache's elements
  __device__ __forceinline__ void init(const Q8Params& p, const Q8Words& tw, int bh, int c0, int lane) {
    const int m = lane & 15, g = lane >> 4;
    b = bh / p.Hkv;
    kvh = bh - b * p.Hkv;
    col0 = c0;
    tp = uni(min(max(p.lens[b], 0), p.Tp));
    const int n0 = c0 / p.rep, n1 = min((c0 + 16 * CT - 1) / p.rep, p.N - 1);
    const int W = p.window > 0 ? p.window : INT_MAX / 2;  // (sums with positions stay in range)
    const int rows = tp + p.N;
    mask.tp = tp;
    mask.rows = rows;
    mask.window = W;
    mask.words = p.tree == 2 ? p.anc + b * p.anc_sb : tw.w;
    int lo_min, hi_max;
    if (p.tree) {
      lo_min = p.window > 0 ? max(0, tp - 1 - W + 1) : 0;             // an empty word sits at tp - 1
      mask.full_lo = p.window > 0 ? max(0, tp + p.N - 1 - W + 1) : 0;  // depth N - 1 at most
      hi_max = rows;
      mask.full_hi = tp;
    } else {
      lo_min = p.window > 0 ? max(0, tp + n0 - W + 1) : 0;
      mask.full_lo = p.window > 0 ? max(0, tp + n1 - W + 1) : 0;
      hi_max = tp + n1 + 1;
      mask.full_hi = tp + n0 + 1;
    }
    first = lo_min & ~15;
    steps = (hi_max - first + 31) / 32;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int col = min(c0 + 16 * ct + m, p.cols - 1);
      int node, h;
      q8_col(p, col, node, h);
      const uint16_t* q = p.q + b * p.q_sb + (int64_t)(kvh * p.rep + h) * p.q_sh + (int64_t)node * p.q_sr;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        qf[ct][i] = *reinterpret_cast<const bf16x8*>(q + D / 4 * g + 8 * i);
      mask.node[ct] = node;
    }
    const int64_t kv = b * p.c_sb + kvh * p.c_sh, ss = b * p.s_sb + kvh * p.s_sh;
    src.k = p.kc + kv;
    src.v = p.vc + kv;
    src.ks = p.ks + ss;
    src.vs = p.vs + ss;
    src.sr = (uint32_t)p.c_sr;
    src.rows = rows;
    const int64_t s2 = b * p.s2_sb + kvh * p.s2_sh;
    src2.k = p.k2 + s2;
    src2.v = p.v2 + s2;
    src2.ks = src2.vs = nullptr;
    src2.sr = (uint32_t)p.s2_sr;
    src2.rows = p.T2;
  }

  __device__ __forceinline__ Q8Mask<CT> mask2(int T2) const {
    Q8Mask<CT> k;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) k.node[ct] = 0;
    k.tp = k.window = k.full_lo = 0;
    k.rows = k.full_hi = T2;
    k.words = nullptr;
    return k;
  }
};

template <int NW>
__device__ __forceinline__ void q8_store(const Q8Params& p, int64_t off, const float* v) {
  uint32_t w[NW / 2];
#pragma unroll
  for (int i = 0; i < NW / 2; ++i) {
    if (p.f16) w[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
    else w[i] = kv_pk_bf16(v[2 * i], v[2 * i + 1]);
  }
  uint16_t* o = static_cast<uint16_t*>(p.out) + off;
  if constexpr (NW == 4) {
    *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < NW / 8; ++i)
      *reinterpret_cast<u32x4*>(o + 8 * i) = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
  }
}

__device__ __forceinline__ int64_t q8_out_off(const Q8Params& p, int b, int kvh, int col) {
  int node, h;
  q8_col(p, col, node, h);
  return b * p.o_sb + (int64_t)(kvh * p.rep + h) * p.o_sh + (int64_t)node * p.o_sr;
}

// A workgroup is CW column tiles (16 CT columns each) by KW waves that share a
// tile's keys, 32 at a time in turn; `splits` workgroups share them further.
//   KW = 1          many tiles (prompts): no exchange between waves;
//   KW = 2, 4, 8    the waves' (acc, m, l) meet in LDS, 16 columns at a time.
// With one split the result is written, else the split's partial (relative to
// its own maxima).  The second segment: for KW <= 2 it is walked first, its
// weighted result kept in LDS meanwhile (KW = 1: by the lane, else by the
// thread that adds it again); for KW >= 4 (few steps a wave) a wave of its own
// walks it beside the others, in the last split.  (us, 32 x 7 rows over 617,
// 128 global rows: 8.2 with that wave at KW = 4, 13.2 walked first at KW = 2; the
// same KW both ways on an earlier build 7.8 and 10.1.  4 x 512 rows: 17.0 walked first at
// KW = 2, 23.9 with the wave at KW = 4, 4 tiles.)
// Waves a SIMD has registers for.
constexpr int q8_occ(int d, int ct) { return d == 64 && ct <= 2 ? 5 - ct : 2; }

template <int D, int KT, int CT, int KIND, bool SEG2, int KW, int CW, int AUX = 0>
__global__ __launch_bounds__((KW * CW + (SEG2 && KW >= 4)) * 64,
                                 KIND == Q8_TREE && CT == 2 ? 2 : q8_occ(D, CT)) void k_attn8(Q8Params p, Q8Words tw) {
  constexpr bool WAVE2 = SEG2 && KW >= 4, LDS2 = SEG2 && KW < 4;
  constexpr int NW = KW * CW + WAVE2, COLS = 16 * CT;
  constexpr int PD = D + 4;                         // row pitch in LDS
  constexpr int TPC = KW == 2 ? 8 : 16;             // threads a column in the merge
  constexpr int DP = D / TPC;                       // their dims
  __shared__ __attribute__((aligned(16))) float s_o[KW > 1 ? NW * 16 * PD : 4];
  __shared__ __attribute__((aligned(16))) float s_2[LDS2 ? CW * COLS * D : 4];
  __shared__ float s_m[KW > 1 ? NW : 1][COLS], s_l[KW > 1 ? NW : 1][COLS];
  const int lane = threadIdx.x & 63, w = uni(threadIdx.x >> 6);
  const bool extra = WAVE2 && w == KW;
  const int kw = w % KW, cw = extra ? 0 : w / KW;
  const int BH = p.B * p.Hkv;
  // later tiles see the most keys and start first; a head's workgroups share an XCD where BH % 8 == 0
  const int bh = blockIdx.x % BH, rest = blockIdx.x / BH;
  const int grp = p.groups - 1 - rest % p.groups, split = rest / p.groups;
  Q8Tile<D, CT> t;
  t.init(p, tw, bh, min((grp * CW + cw) * COLS, (p.cols - 1) / COLS * COLS), lane);  // (a tile past the last: the last again)
  Q8State<CT, D> st;
  // where this thread stands in the merge
  const int mc = threadIdx.x / TPC, dd = threadIdx.x % TPC * DP;   // column (of 16 CW), first dim
  const int mcw = mc / 16, cc = mc % 16;
  const bool merges = mc < 16 * CW;
  const int gcol = (grp * CW + mcw) * COLS + cc;                   // + 16 ct: the column
  const int64_t unit = (int64_t)bh * p.groups + grp;

  // Calls f(ct, values of DP dims, maximum, sum) for this thread's columns.
  auto merge = [&](auto&& f) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float l = q8_sum4(st.l[ct]);
      if (lane < 16) {
        s_m[w][16 * ct + lane] = st.lim[ct] == kNegInf ? kNegInf : st.m[ct];
        s_l[w][16 * ct + lane] = l;
      }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float* o = s_o + (w * 16 + (lane & 15)) * PD + (lane >> 4) * (D / 4);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < D / 16; d += 4)
          *reinterpret_cast<f32x4*>(o + i * (D / 16) + d) =
              f32x4{st.acc[ct][d][i], st.acc[ct][d + 1][i], st.acc[ct][d + 2][i], st.acc[ct][d + 3][i]};
      __syncthreads();
      if (merges) {
        float mx = kNegInf;
#pragma unroll
        for (int i = 0; i < KW; ++i) mx = fmaxf(mx, s_m[mcw * KW + i][16 * ct + cc]);
        float sum = 0.0f, v[DP] = {};
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const float mi = s_m[mcw * KW + i][16 * ct + cc];
          const float e = mi == kNegInf ? 0.0f : q8_ex2(mi - mx);
          sum += s_l[mcw * KW + i][16 * ct + cc] * e;
          const float* r = s_o + ((mcw * KW + i) * 16 + cc) * PD + dd;
#pragma unroll
          for (int d = 0; d < DP; ++d) v[d] = fmaf(r[d], e, v[d]);
        }
        f(ct, v, mx, sum);
      }
      __syncthreads();  // s_o (s_m, s_l) may be written again
    }
  };

  const float g0 = SEG2 || p.gates ? p.gates[0] : 1.0f;
  const float g1 = SEG2 ? p.gates[1] : 0.0f;
  if constexpr (LDS2) {
    q8_walk<D, KV_BF16, CT, Q8_ALL>(t.src2, 0, kw, KW, (p.T2 + 31) / 32, t.mask2(p.T2), p.c, t.qf, st, lane);
    if constexpr (KW > 1) {
      merge([&](int ct, float (&v)[DP], float mx, float sum) {
#pragma unroll
        for (int d = 0; d < DP; ++d) s_2[(mcw * COLS + 16 * ct + cc) * D + dd + d] = v[d] * (g1 / sum);
      });
    } else {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const float inv = g1 / q8_sum4(st.l[ct]);
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
          *reinterpret_cast<f32x4*>(s_2 + (((w * CT + ct) * (D / 16) + d) * 64 + lane) * 4) = st.acc[ct][d] * inv;
      }
    }
  }
  st.clear();  // (for a wave that walks nothing)
  const bool second = WAVE2 && split == p.splits - 1;
  if (!extra) {
    const int per = (t.steps + p.splits - 1) / p.splits;
    q8_walk<D, KT, CT, KIND, AUX>(t.src, t.first, split * per + kw, KW, min(t.steps, (split + 1) * per), t.mask, p.c, t.qf,
                             st, lane);
  } else if (second) {
    q8_walk<D, KV_BF16, CT, Q8_ALL>(t.src2, 0, 0, 1, (p.T2 + 31) / 32, t.mask2(p.T2), p.c, t.qf, st, lane);
  }
  if constexpr (KW > 1) {
    merge([&](int ct, float (&v)[DP], float mx, float sum) {
      const int col = gcol + 16 * ct;
      if (col >= p.cols) return;
      const float* o2 = s_o + (KW * 16 + cc) * PD + dd;  // (WAVE2)
      if (p.splits > 1) {
        const int64_t r = (unit * p.slots + split) * COLS + 16 * ct + cc;  // (CW = 1)
#pragma unroll
        for (int d = 0; d < DP; d += 4)
          *reinterpret_cast<f32x4*>(p.part_o + r * D + dd + d) = f32x4{v[d], v[d + 1], v[d + 2], v[d + 3]};
        if (dd == 0) p.part_ml[r] = make_float2(mx, sum);
        if (second) {
#pragma unroll
          for (int d = 0; d < DP; d += 4)
            *reinterpret_cast<f32x4*>(p.part_o + (r + COLS) * D + dd + d) = *reinterpret_cast<const f32x4*>(o2 + d);
          if (dd == 0) p.part_ml[r + COLS] = make_float2(s_m[KW][16 * ct + cc], s_l[KW][16 * ct + cc]);
        }
        return;
      }
      const float inv = sum == 0.0f ? 0.0f : g0 / sum;
      float inv2 = 0.0f;
      if constexpr (WAVE2) inv2 = g1 / s_l[KW][16 * ct + cc];
#pragma unroll
      for (int d = 0; d < DP; ++d) {
        v[d] *= inv;
        if constexpr (LDS2) v[d] += s_2[(mcw * COLS + 16 * ct + cc) * D + dd + d];
        if constexpr (WAVE2) v[d] = fmaf(o2[d], inv2, v[d]);
      }
      q8_store<DP>(p, q8_out_off(p, t.b, t.kvh, col) + dd, v);
    });
  } else {
    const int c0 = (grp * CW + cw) * COLS;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const float sum = q8_sum4(st.l[ct]);
      const float inv = sum == 0.0f ? 0.0f : g0 / sum;
      float v[D / 4];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        f32x4 o = st.acc[ct][d] * inv;
        if constexpr (SEG2) o += *reinterpret_cast<const f32x4*>(s_2 + (((w * CT + ct) * (D / 16) + d) * 64 + lane) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i * (D / 16) + d] = o[i];
      }
      const int col = c0 + 16 * ct + (lane & 15);
      if (col < p.cols) q8_store<D / 4>(p, q8_out_off(p, t.b, t.kvh, col) + (lane >> 4) * (D / 4), v);
    }
  }
}

// Joins the splits' partials, a wave a column: lane s takes split s's weight,
// then D / 4 lanes (four dims each) walk the splits 256 / D at a time.
template <int D>
__global__ __launch_bounds__(256) void k_attn8_join(Q8Params p, int ct16) {
  constexpr int L = D / 4, G = 64 / L;
  const int lane = threadIdx.x & 63;
  const int64_t cell = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // unit * ct16 + column of the group (CW = 1)
  const int64_t unit = cell / ct16;
  if (unit >= (int64_t)p.B * p.Hkv * p.groups) return;
  const int cc = (int)(cell - unit * ct16);
  const int bh = (int)(unit / p.groups), grp = (int)(unit - (int64_t)bh * p.groups);
  const int col = grp * ct16 + cc;
  if (col >= p.cols) return;
  const int64_t r0 = unit * p.slots * ct16 + cc;
  float2 ml = make_float2(kNegInf, 0.0f);
  if (lane < p.splits) ml = p.part_ml[r0 + (int64_t)lane * ct16];
  float mx = ml.x;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  const float e = ml.x == kNegInf ? 0.0f : q8_ex2(ml.x - mx);
  float sum = ml.y * e;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  const int g = lane / L, dd = lane % L * 4;
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = g; s < p.splits; s += G) {
    const float w = __shfl(e, s, 64);
    const f32x4 o = *reinterpret_cast<const f32x4*>(p.part_o + (r0 + (int64_t)s * ct16) * D + dd);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaf(o[i], w, v[i]);
  }
#pragma unroll
  for (int o = L; o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += __shfl_xor(v[i], o, 64);
  if (g) return;
  const float g0 = p.gates ? p.gates[0] : 1.0f;
  v *= sum == 0.0f ? 0.0f : g0 / sum;
  if (p.T2 > 0) {
    const int64_t r = r0 + (int64_t)p.splits * ct16;
    const float inv = p.gates[1] / p.part_ml[r].y;
    const f32x4 o = *reinterpret_cast<const f32x4*>(p.part_o + r * D + dd);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaf(o[i], inv, v[i]);
  }
  const int b = bh / p.Hkv, kvh = bh - b * p.Hkv;
  const float t[4] = {v[0], v[1], v[2], v[3]};
  q8_store<4>(p, q8_out_off(p, b, kvh, col) + dd, t);
}

// The launch shape: column tiles of 16 a wave, waves that share a tile's keys,
// column groups, key splits.
struct Q8Plan {
  int ct, kw, groups, splits;
};

// Waves that share a workgroup's columns, per keys wave.
constexpr int q8_cw(int kw) { return kw == 1 ? 4 : kw == 2 ? 2 : 1; }

// Estimated us of a launch shape, for comparing shapes.  A step of a wave costs
// the conversion of its rows and its columns' softmax: kCol a column tile in a
// lone wave; per SIMD half of it, a wave issuing one instruction in 8 cycles and
// a SIMD one in 4 (measured), and there the conversions count (in column
// tiles, kConv).  Rows read by several column groups cost memory time again.  A
// second launch joins splits.  The constants are fitted to 1,700 timings of 70
// shapes (1-64 sequences, 1-1,500 new rows, 1-16,000 keys, both head sizes); of 67
// others it picks the fastest launch shape within 2% on average and 21% at
// worst.  The constants stand for nothing but that fit (mem's 10.2 TB/s is no rate
// of the memory), and the kernel has gained a test a step since; what is measured
// on it, us: 16 trees of 40 nodes over 2,048 rows ct 3 x 8 waves 18.9, ct 3 x 4 20.5,
// ct 1 x 4 21.5, ct 2 x 8 25.8; 4 prompts of 512 ct 2 x 2 waves 17.0, ct 4 x 2 21.2, ct 4 x 4
// 23.9; 8 x 5 rows over 16,000, heads of 128, ct 2 x 4 splits 50.1, no split 130,
// ct 1 x 4 splits 72.9; 2,048 rows over 8,192 ct 4 x 4 waves 111.4, ct 3 x 4 132, ct 4 x 1 287.
float q8_cost(int BH, int d2, bool i8, float last, float mean, float mem, int T2, int cus, int ct, int kw, int S,
              int groups) {
  constexpr float kMerge = 0.813f, kLone = 1.66f, kJoin = 1.09f, kPart = 5.9e-3f, kStep = 0.078f, kCol = 0.252f,
                  kSeg2 = 1.32f, kEight = 3.7f, kRound = 7.0f, kAgain = 2.07f;
  const float kConv = i8 ? 3.35f : 2.26f;
  const int cw = q8_cw(kw);
  const float cols = ct * (1.0f + 0.3f * (d2 - 1));
  const int occ = q8_occ(64 * d2, ct);
  const int waves = kw * cw + (T2 > 0 && kw >= 4);
  const int per = occ * 4 / waves > 1 ? occ * 4 / waves : 1;      // workgroups a CU
  const float wgs = (float)BH * groups * S, rounds = wgs / ((float)cus * per);
  float nl = __builtin_ceilf(__builtin_ceilf(last / 32) / (kw * S));  // steps of the longest wave, of the mean one
  float nm = mean / 32 > kw * S ? mean / 32 / (kw * S) : 1.0f;
  if (T2 > 0 && kw < 4) {
    const float e = __builtin_ceilf((float)T2 / 32 / kw);
    nl += e;
    nm += e;
  }
  const float simd = (wgs / cus < per ? wgs / cus : per) * kw * cw / 4;  // waves a SIMD at a time
  const float lone = kCol * (0.284f * d2 + cols), all = nm * 0.25f * (kConv * d2 + cols) * simd / 2;
  float t;
  if (rounds <= 1.0f) {
    t = nl * kStep + (nl * lone > all ? nl * lone : all);
  } else {
    t = (nm * kStep + (nm * lone > all ? nm * lone : all)) * (rounds < 2.5f ? __builtin_ceilf(rounds) : rounds + 0.3f);
    t += kRound * (__builtin_ceilf(rounds) - 1);
  }
  t += (kw > 1 ? kMerge * ct * d2 : kLone) * (simd > 2.0f ? simd / 2 : 1.0f) * (rounds > 1.0f ? rounds : 1.0f);
  t += (kw == 8 ? kEight : 0.0f) + (T2 > 0 && kw < 4 ? kSeg2 : 0.0f);
  const float m = mem * (1.0f + kAgain * (groups * cw < 4 ? groups * cw - 1 : 3));
  t = t > m ? t : m;
  return S > 1 ? t + kJoin + kPart * BH * groups * ct * S * d2 : t;
}

Q8Plan q8_plan(const vnx_attn_q8_args* a) {
  const int rep = a->H / a->Hkv, BH = a->B * a->Hkv, d2 = a->d / 64;
  const int tiles = (int)(((int64_t)rep * a->N + 15) / 16);
  const bool tree = a->anc || a->anc_host;
  const float W = a->window > 0 ? (float)a->window : 1e9f, keys = (float)a->Tp + a->N;
  const int cus = device_cus();
  // memory time of the rows once, us (the rate is the fit's)
  const float mem = BH * (keys < W + a->N ? keys : W + a->N) * 2 * (a->d + 4) / 10.2e6f;
  Q8Plan best{1, 4, tiles, 1};
  float least = 1e30f;
  for (int ct = 1; ct <= 4 / d2; ++ct) {
    if (a->force_tiles ? ct != a->force_tiles : ct > tiles) continue;
    const float span = (float)(16 * ct / rep + 2 < a->N ? 16 * ct / rep + 2 : a->N);  // rows of a tile
    const float end = tree ? (float)a->N : span;
    const float last = keys < W + end ? keys : W + end;
    const float mid = tree ? keys : (float)a->Tp + (a->N + span) / 2;
    const float mean = mid < W + end ? mid : W + end;
    for (int kw = tree ? 4 : 1; kw <= (a->T2 > 0 ? 4 : 8); kw *= 2) {
      if (a->force_waves && kw != a->force_waves) continue;
      const int groups = (tiles + ct * q8_cw(kw) - 1) / (ct * q8_cw(kw));
      for (int S = 1; S <= (kw < 4 ? 1 : kQ8Split); S *= 2) {
        if (a->force_splits ? S != a->force_splits : S > 1 && ((int64_t)BH * groups * S > 6 * cus || last < 32 * S))
          continue;
        const float t = q8_cost(BH, d2, a->kv_dtype == VNX_I8, last, mean, mem, a->T2, cus, ct, kw, S, groups);
        if (t < least) {
          least = t;
          best = {ct, kw, groups, S};
        }
      }
    }
  }
  return best;
}

size_t q8_ws_bytes(const vnx_attn_q8_args* a, const Q8Plan& pl, Q8Params* p, void* ws) {
  if (pl.splits == 1) return 0;
  const int slots = pl.splits + (a->T2 > 0);
  const size_t rows = (size_t)a->B * a->Hkv * pl.groups * slots * 16 * pl.ct;
  Carve c(ws);
  float* o = c.take<float>(rows * a->d);
  float2* ml = c.take<float2>(rows);
  if (p) {
    p->part_o = o;
    p->part_ml = ml;
    p->slots = slots;
  }
  return c.bytes();
}

// Everything that needs no pointer.
int q8_check_sizes(const vnx_attn_q8_args* a) {
  if (a->B < 0 || a->H < 1 || a->Hkv < 1 || a->H % a->Hkv || a->N < 1 || a->Tp < 0 || a->T2 < 0 || a->window < 0)
    return VNX_ERR_INVALID_ARG;
  if (a->d != 64 && a->d != 128) return VNX_ERR_UNSUPPORTED;
  if (a->kv_dtype != VNX_I8 && a->kv_dtype != VNX_E4M3) return VNX_ERR_UNSUPPORTED;
  if (a->out_dtype != VNX_BF16 && a->out_dtype != VNX_F16) return VNX_ERR_UNSUPPORTED;
  if ((int64_t)a->Tp + a->N > a->cap) return VNX_ERR_INVALID_ARG;
  const bool tree = a->anc || a->anc_host;
  if (tree && (a->N > kQ8MaxN || (a->window > 0 && a->window < a->N))) return VNX_ERR_UNSUPPORTED;
  // launch shapes that there are
  const int ft = a->force_tiles, fw = a->force_waves, fs = a->force_splits;
  if (ft < 0 || ft > 256 / a->d || (fw && fw != 1 && fw != 2 && fw != 4 && fw != 8) || (fw && fw < 4 && tree) ||
      (fw > 4 && a->T2 > 0) || fs < 0 || fs > kQ8Split || (fs & (fs - 1)) || (fs > 1 && fw && fw < 4))
    return VNX_ERR_UNSUPPORTED;
  // 32-bit row, column and workgroup numbers
  if (a->cap > INT_MAX - 64 || (int64_t)a->Tp + a->N > INT_MAX - 64 || a->T2 > INT_MAX - 64 ||
      (int64_t)a->H / a->Hkv * a->N > INT_MAX / 2 ||
      (__int128)a->B * a->Hkv * (((int64_t)a->H / a->Hkv * a->N + 15) / 16) * kQ8Split > INT_MAX)
    return VNX_ERR_UNSUPPORTED;
  return VNX_OK;
}

inline bool q8_strides(const int64_t* s, int n, int64_t unit) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % unit) return false;
  return true;
}

template <int D, int KT, int CT, int KIND, bool SEG2>
void q8_launch(const Q8Params& p, const Q8Words& tw, const Q8Plan& pl, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * p.Hkv * pl.groups * pl.splits));
  if constexpr (KIND == Q8_CHAIN) {  // (a tree's walk is no shorter in its first column groups: 4 waves and more)
    if (pl.kw == 1) {
      hipLaunchKernelGGL((k_attn8<D, KT, CT, KIND, SEG2, 1, 4>), grid, dim3(256), 0, st, p, tw);
      return;
    }
    if (pl.kw == 2) {
      hipLaunchKernelGGL((k_attn8<D, KT, CT, KIND, SEG2, 2, 2>), grid, dim3(256), 0, st, p, tw);
      return;
    }
  }
  auto go = [&](auto aux) {
    constexpr int AUX = decltype(aux)::value;
    if constexpr (!SEG2) {  // (a ninth wave would leave 168 registers a lane)
      if (pl.kw == 8) {
        hipLaunchKernelGGL((k_attn8<D, KT, CT, KIND, SEG2, 8, 1, AUX>), grid, dim3(512), 0, st, p, tw);
        return;
      }
    }
    hipLaunchKernelGGL((k_attn8<D, KT, CT, KIND, SEG2, 4, 1, AUX>), grid, dim3(256 + 64 * SEG2), 0, st, p, tw);
  };
  // Rows that one column group reads go past the caches from 192 MiB on, where
  // the next layer's rows push them out before they are read again.  us past /
  // cached (before q8_steps tested the scales), 5 rows a sequence, heads of 128, two caches read in turn: 125 MiB
  // 32.3 / 29.7, 156 51.1 / 49.1, 188 49.1 / 49.0, 219 49.8 / 51.3, 250 51.8 /
  // 56.1, 500 (heads of 64) 93.1 / 101.7.  A single cache read again at once
  // keeps more: 250 MiB 51.4 / 48.2.  Rows that several groups read lose (16
  // trees over 2,048: 19.7 / 17.5).
  const int64_t rows = p.window > 0 && p.window < p.Tp ? p.window : p.Tp;
  if constexpr (CT <= 2) {
    if (pl.groups == 1 && (int64_t)p.B * p.Hkv * rows * 2 * D >= (192 << 20)) return go(IntC<2>{});
  }
  go(IntC<0>{});
}

template <int D, int KT, int KIND, bool SEG2>
int q8_by_ct(const Q8Params& p, const Q8Words& tw, const Q8Plan& pl, hipStream_t st) {
  if (pl.ct == 1) q8_launch<D, KT, 1, KIND, SEG2>(p, tw, pl, st);
  else if (pl.ct == 2) q8_launch<D, KT, 2, KIND, SEG2>(p, tw, pl, st);
  if constexpr (D == 64) {
    if (pl.ct == 3) q8_launch<D, KT, 3, KIND, SEG2>(p, tw, pl, st);
    else if (pl.ct == 4) q8_launch<D, KT, 4, KIND, SEG2>(p, tw, pl, st);
  }
  VNX_LAUNCH_CHECK();
  if (pl.splits > 1) {
    hipLaunchKernelGGL((k_attn8_join<D>), dim3((unsigned)(p.B * p.Hkv * p.groups * 4 * pl.ct)), dim3(256), 0, st, p,
                       16 * pl.ct);
    VNX_LAUNCH_CHECK();
  }
  return VNX_OK;
}

}  // namespace
}  // namespace vnx

using namespace vnx;

extern "C" {

size_t vnx_tree_attn_q8_workspace(const vnx_attn_q8_args* a) {
  if (!a || q8_check_sizes(a) != VNX_OK || a->B == 0) return 256;
  const size_t n = q8_ws_bytes(a, q8_plan(a), nullptr, nullptr);
  return n < 256 ? 256 : n;
}

int vnx_tree_attn_q8(const vnx_attn_q8_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!a) return VNX_ERR_INVALID_ARG;
  const int bad = q8_check_sizes(a);
  if (bad != VNX_OK) return bad;
  if (a->B == 0) return VNX_OK;
  if (!a->q || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->lens || !a->out)
    return VNX_ERR_INVALID_ARG;
  if (!(a->scale > 0.0f) || !__builtin_isfinite(a->scale) || a->anc_batch_stride < 0) return VNX_ERR_INVALID_ARG;
  if (a->cache_strides[2] < a->d || !q8_strides(a->scale_strides, 2, 1)) return VNX_ERR_INVALID_ARG;
  if (a->T2 > 0 && (!a->k_seg2 || !a->v_seg2 || !a->gates)) return VNX_ERR_INVALID_ARG;
  // 16-byte loads; a step's row offsets in 32 bits
  if (!q8_strides(a->q_strides, 3, 8) || !q8_strides(a->cache_strides, 3, 16) || !q8_strides(a->out_strides, 3, 8) ||
      (a->T2 > 0 && !q8_strides(a->seg2_strides, 3, 8)) || a->cache_strides[2] >= (1 << 25) ||
      (a->T2 > 0 && a->seg2_strides[2] >= (1 << 24)))
    return VNX_ERR_UNSUPPORTED;
  if (!aligned16(a->q) || !aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->out) ||
      (a->T2 > 0 && (!aligned16(a->k_seg2) || !aligned16(a->v_seg2))) || !aligned_to(a->gates, 4) ||
      !aligned_to(a->k_scale, 4) || !aligned_to(a->v_scale, 4) || !aligned_to(a->lens, 4) || !aligned_to(a->anc, 8))
    return VNX_ERR_UNSUPPORTED;
  if (!Rows(a->d, a->out_strides, {a->B, a->H, a->N}).apart()) return VNX_ERR_INVALID_ARG;  // rows on one another
  const Q8Plan pl = q8_plan(a);
  const int64_t units = (int64_t)a->B * a->Hkv * pl.groups;
  if (!launch_fits(units * pl.splits, 64 * (pl.kw * q8_cw(pl.kw) + (a->T2 > 0 && pl.kw >= 4))) ||
      (pl.splits > 1 && !launch_fits(units * 4 * pl.ct, 256)))
    return VNX_ERR_UNSUPPORTED;
  Q8Params p{};
  p.slots = 1;
  const size_t need = q8_ws_bytes(a, pl, &p, workspace);
  if (need && (!workspace || workspace_bytes < need)) return VNX_ERR_WORKSPACE;
  p.q = static_cast<const uint16_t*>(a->q);
  p.kc = static_cast<const char*>(a->k_cache); p.vc = static_cast<const char*>(a->v_cache);
  p.ks = a->k_scale; p.vs = a->v_scale;
  p.lens = a->lens;
  p.out = a->out;
  p.q_sb = a->q_strides[0]; p.q_sh = a->q_strides[1]; p.q_sr = a->q_strides[2];
  p.c_sb = a->cache_strides[0]; p.c_sh = a->cache_strides[1]; p.c_sr = a->cache_strides[2];
  p.s_sb = a->scale_strides[0]; p.s_sh = a->scale_strides[1];
  p.o_sb = a->out_strides[0]; p.o_sh = a->out_strides[1]; p.o_sr = a->out_strides[2];
  p.B = a->B; p.H = a->H; p.Hkv = a->Hkv; p.rep = a->H / a->Hkv; p.N = a->N; p.cols = p.rep * a->N;
  p.Tp = a->Tp; p.T2 = a->T2; p.window = a->window;
  if (a->T2 > 0) {
    p.k2 = static_cast<const char*>(a->k_seg2); p.v2 = static_cast<const char*>(a->v_seg2);
    p.s2_sb = 2 * a->seg2_strides[0]; p.s2_sh = 2 * a->seg2_strides[1]; p.s2_sr = 2 * a->seg2_strides[2];
  }
  p.gates = a->gates;
  Q8Words tw{};
  if (a->anc) {
    p.tree = 2;
    p.anc = a->anc;
    p.anc_sb = a->anc_batch_stride;
  } else if (a->anc_host) {
    p.tree = 1;
    for (int i = 0; i < a->N; ++i) tw.w[i] = a->anc_host[i];
  }
  p.groups = pl.groups; p.splits = pl.splits;
  p.f16 = a->out_dtype == VNX_F16;
  p.c = (float)((double)a->scale * 1.4426950408889634);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto go = [&](auto d, auto kt) {
    constexpr int D = decltype(d)::value, KT = decltype(kt)::value;
    if (p.tree) return p.T2 > 0 ? q8_by_ct<D, KT, Q8_TREE, true>(p, tw, pl, st) : q8_by_ct<D, KT, Q8_TREE, false>(p, tw, pl, st);
    return p.T2 > 0 ? q8_by_ct<D, KT, Q8_CHAIN, true>(p, tw, pl, st) : q8_by_ct<D, KT, Q8_CHAIN, false>(p, tw, pl, st);
  };
  if (a->d == 64) return a->kv_dtype == VNX_I8 ? go(IntC<64>{}, IntC<KV_I8>{}) : go(IntC<64>{}, IntC<KV_E4M3>{});
  return a->kv_dtype == VNX_I8 ? go(IntC<128>{}, IntC<KV_I8>{}) : go(IntC<128>{}, IntC<KV_E4M3>{});
}

}  // extern "C"
