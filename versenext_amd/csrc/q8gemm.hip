// Products of 8-bit integer rows on gfx950 (vnx_q8_linear): x (M, K) codes with a
// scale a row times W (N, K) codes with a scale a row,
//   acc[m, n] = sum_k x[m, k] * W[n, k]          (exact in int32: K <= 131,071)
//   y[m, n] = acc * x_scale[m] * w_scale[n] (+ bias[n]) (+ residual[m, n])
// or, of gate rows and up rows, silu(gate) * up.  The sums are whole numbers, so
// how K is split never changes a result.
#include <algorithm>
#include <climits>
#include <utility>

#include "q8.h"

namespace vnx {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kQ8Chunk = 128;   // bytes of k a chunk: a cache line of a row
constexpr int kQ8Xcds = 8;
constexpr int64_t kQ8MaxK = 131071;  // K * 2^14 < 2^31

struct Q8LinParams {
  const int8_t* x;
  const int8_t* w;
  const float* xs;
  const float* ws;
  const float* bias;
  const void* res;
  void* y;
  int64_t ldx, ldw, ldr, ldy;
  int M, N, K;
  int cols;        // columns of y: N, or N / 2
  int mt, nt;      // tiles
  int res_dtype, y_dtype;
  int y_vec;       // rows of y lie on 16 bytes
  int per;         // slabs a split of k has (sums alone)
};

// Up to eight columns n.. of row m: y = v (already scaled, with bias or SwiGLU
// done) + residual, rounded once.
__device__ __forceinline__ void q8_out8(const Q8LinParams& p, int m, int n, float (&v)[8]) {
  if (n + 8 <= p.cols) {
    if (p.res) {
      float r[8];
      const int64_t o = (int64_t)m * p.ldr + n;
      if (p.res_dtype == VNX_F32) q8_ld8(static_cast<const float*>(p.res) + o, r);
      else if (p.res_dtype == VNX_BF16) q8_ld8(static_cast<const uint16_t*>(p.res) + o, r);
      else q8_ld8(static_cast<const _Float16*>(p.res) + o, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += r[i];
    }
    const int64_t o = (int64_t)m * p.ldy + n;
    if (p.y_dtype == VNX_F32) q8_st8(static_cast<float*>(p.y) + o, v);
    else if (p.y_dtype == VNX_BF16) q8_st8(static_cast<uint16_t*>(p.y) + o, v);
    else q8_st8(static_cast<_Float16*>(p.y) + o, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (n + i >= p.cols) break;
    if (p.res) {
      const int64_t o = (int64_t)m * p.ldr + n + i;
      v[i] += p.res_dtype == VNX_F32    ? q8_ld1(static_cast<const float*>(p.res) + o)
              : p.res_dtype == VNX_BF16 ? q8_ld1(static_cast<const uint16_t*>(p.res) + o)
                                        : q8_ld1(static_cast<const _Float16*>(p.res) + o);
    }
    const int64_t o = (int64_t)m * p.ldy + n + i;
    if (p.y_dtype == VNX_F32) q8_st1(static_cast<float*>(p.y) + o, v[i]);
    else if (p.y_dtype == VNX_BF16) q8_st1(static_cast<uint16_t*>(p.y) + o, v[i]);
    else q8_st1(static_cast<_Float16*>(p.y) + o, v[i]);
  }
}

// silu(g) * u.  __expf is off by about |g| 2^-24 relative; for g far below zero
// it is infinite and the quotient -0.
__device__ __forceinline__ float q8_swiglu(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

// Eight sums of row m, W rows r .. r + 7 (those at or past `rows` are anything),
// scaled, with the bias.
__device__ __forceinline__ void q8_scale8(const Q8LinParams& p, float xs, int r, int rows, const int (&a)[8],
                                          float (&v)[8]) {
  float s[8];
  if (r + 8 <= rows) {
    q8_ld8(p.ws + r, s);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = p.ws[min(r + i, rows - 1)];
  }
  float b[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = p.bias[min(r + i, rows - 1)];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fmaf((float)a[i] * xs, s[i], b[i]);
}

__device__ __forceinline__ i32x4 q8_mma(u32x4 a, u32x4 b, i32x4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// k_q8_direct: few rows of y.  A workgroup owns 16 rows of x and 16 of W; its KW
// waves take chunks of 128 bytes of k in turn, operands straight from memory to
// the matrix cores, and their sums meet in LDS.  The order of k inside a product
// is free as long as both operands have the same, so a lane loads two 16-byte
// pieces side by side of its row (lane (r, g): row r, bytes 32 g .. + 32), whole
// lines over the wave.
//
// Memory's latency bounds it, then the copies of x and W that every workgroup reads
// for itself.  us, from a graph (32 x 32 tiles): 1 x 2,048 x 1,024 2.5 (2.7), 1 x
// 1,024 x 4,096 4.1 (5.1), 64 x 1,024 x 2,752 4.0 (5.2), 32 x 4,096 x 1,024 3.8
// (2.8).  Eight or sixteen waves, or loads of the next chunks ahead, took longer.
// ---------------------------------------------------------------------------
template <int KW>
__global__ __launch_bounds__(64 * KW) void k_q8_direct(Q8LinParams p) {
  constexpr int PITCH = 20;                          // of a row of sums
  __shared__ __attribute__((aligned(16))) int red[KW * 16 * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, kw = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  // the row tiles that share W rows follow each other on one XCD
  const int xcd = blockIdx.x % kQ8Xcds, at = blockIdx.x / kQ8Xcds;
  const int m0 = at % p.mt * 16, n0 = (at / p.mt * kQ8Xcds + xcd) * 16;
  if (n0 >= p.N) return;                             // uniform over the workgroup
  const int8_t* xp = p.x + (int64_t)min(m0 + r, p.M - 1) * p.ldx + g * 32;
  const int8_t* wp = p.w + (int64_t)min(n0 + r, p.N - 1) * p.ldw + g * 32;
  i32x4 acc = {0, 0, 0, 0};
  struct Set { u32x4 x[2], w[2]; };
  const int nf = p.K / kQ8Chunk, mine = nf > kw ? (nf - kw + KW - 1) / KW : 0;  // whole chunks, and this wave's
  auto load = [&](int i, Set& q) {                   // this wave's chunk i
    const int64_t k = (int64_t)(kw + i * KW) * kQ8Chunk;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      q.w[s] = *reinterpret_cast<const u32x4*>(wp + k + s * 16);
      q.x[s] = *reinterpret_cast<const u32x4*>(xp + k + s * 16);
    }
  };
  auto mma = [&](const Set& q) {
#pragma unroll
    for (int s = 0; s < 2; ++s) acc = q8_mma(q.x[s], q.w[s], acc);
  };
  // two chunks under way, none of them loaded twice (a short row has no time for that)
  if (mine == 1) {                                   // uniform, as the others
    Set a;
    load(0, a);
    mma(a);
  } else if (mine > 1) {
    Set a, b;
    load(0, a);
    load(1, b);
    int i = 0;
    for (; i + 3 < mine; i += 2) {
      mma(a);
      load(i + 2, a);
      mma(b);
      load(i + 3, b);
    }
    mma(a);
    if (i + 2 < mine) load(i + 2, a);
    mma(b);
    if (i + 2 < mine) mma(a);
  }
  if (p.K % kQ8Chunk && kw == nf % KW) {
    // The last chunk's pieces: those past the row's end come from its start, and
    // every byte of x at or past K counts as 0 (of W there may be anything).
    Set q;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int64_t k = (int64_t)nf * kQ8Chunk + s * 16;
      const int left = p.K - (int)k - g * 32;        // bytes of this piece inside the row
      const int64_t o = left > 0 ? k : -g * 32;
      q.w[s] = *reinterpret_cast<const u32x4*>(wp + o);
      u32x4 v = *reinterpret_cast<const u32x4*>(xp + o);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = left - 4 * e;                  // bytes of this word inside the row
        v[e] = n >= 4 ? v[e] : n <= 0 ? 0u : v[e] & ((1u << (8 * n)) - 1u);
      }
      q.x[s] = v;
    }
    mma(q);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[(kw * 16 + 4 * g + e) * PITCH + r] = acc[e];
  __syncthreads();
  if (tid >= 32) return;
  const int row = tid >> 1, m = m0 + row, n = n0 + (tid & 1) * 8;
  if (m >= p.M || n >= p.N) return;
  int a[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < KW; ++k) {
    const int* src = red + (k * 16 + row) * PITCH + (tid & 1) * 8;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(src), hi = *reinterpret_cast<const i32x4*>(src + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] += lo[i]; a[4 + i] += hi[i]; }
  }
  float v[8];
  q8_scale8(p, p.xs[m], n, p.N, a, v);
  q8_out8(p, m, n, v);
}

template <int KW>
int q8_direct(Q8LinParams p, hipStream_t st) {
  p.mt = (p.M + 15) / 16;
  p.nt = (p.N + 15) / 16;
  const int64_t wgs = (int64_t)p.mt * ((p.nt + kQ8Xcds - 1) / kQ8Xcds * kQ8Xcds);
  if (wgs >= INT_MAX || !launch_fits(wgs, 64 * KW)) return VNX_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((k_q8_direct<KW>), dim3((unsigned)wgs), dim3(64 * KW), 0, st, p);
  VNX_LAUNCH_CHECK();
  return VNX_OK;
}

// ---------------------------------------------------------------------------
// k_q8_tile: BM x BN tiles of y, WM x WN waves, slabs of KS parts of 64 bytes of k
// in a ring of NS buffers in LDS, a tile a workgroup.
//
// The slabs come by direct copies from memory to LDS (1 KB an instruction: 16
// rows of 64 bytes, lane l's 16 bytes at 16 l), so the tile's layout is made by
// which piece of its row a lane asks for: piece c of row R lies at c ^ (-R / 4 %
// 4), and the sixteen lanes that LDS serves together, four runs of four rows,
// read sixteen different 16-byte columns of its 256.  A wave holds two sets of
// operands: it reads slab g + 1 while the products of slab g run, and slab g + NS
// comes into the buffer that slab g has left, so one barrier a slab does.
//
// W is the products' first operand: lane (r, g) then holds four columns of y of
// row r.
//
// What bounds it, by shape:
//   256 x 256, eight waves   the chip's power: 8,192^3 takes 442-458 us (2,400-2,490
//                            TOP/s) at about 1.55 GHz with the matrix cores busy two
//                            thirds of the time, 326 with codes of zero; copies gone
//                            348, LDS reads gone 381, stores gone 408.  Products of
//                            32 x 32 x 32: 474; four waves of 128 x 128: 566.
//   128^2, 64 x 128, 64^2    copies into a CU's LDS, about 70 GB/s of them, and the
//                            last round of workgroups.
//   32 x 32                  the chain of a slab: wait, barrier, LDS read, product (0.2
//                            us per 256 bytes of k, 0.13 per 128, so slabs are long;
//                            of 512 they gain 6% at a k of 4,096 and lose half at
//                            1,024; eight buffers instead of four gain nothing).
// One workgroup a CU that fetches its next tile's slabs during the results: 1-6%
// slower at every size.
//
// TY int: the sums alone, of the p.per slabs of k that are blockIdx.y's, into the
// 32-bit matrix [split][row][column] of whole tiles at p.y.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Lane l's 16 bytes at base + off to LDS at `to` + 16 l (counted by vmcnt).
__device__ __forceinline__ void copy_to_lds(uint32_t to, uint32_t off, const int8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(to), "v"(off), "s"(base)
               : "memory", "m0");
}

// Lane l's value at p to LDS at `to` + 4 l.
__device__ __forceinline__ void copy_to_lds(uint32_t to, const float* p) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(to), "v"(p) : "memory", "m0");
}

// Waits until at most N of this wave's copies are under way.
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "i"(N) : "memory");
}

// Every wave's LDS reads and writes so far are done, and every wave is here.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), in a form that the compiler counts with
  asm volatile("s_barrier" : : : "memory");
}

template <typename F, int... J>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, J...>) {
  (f(IntC<J>{}), ...);
}

// Four values rounded to TY at p (on its own size only).
template <typename TY>
__device__ __forceinline__ void q8_st4(TY* p, const float (&v)[4]) {
  if constexpr (sizeof(TY) == 4) {
    const f32x4 a = {v[0], v[1], v[2], v[3]};
    __builtin_memcpy(p, &a, 16);
  } else {
    u32x2 o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (__is_same(TY, _Float16))
        o[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
      else o[i] = kv_pk_bf16(v[2 * i], v[2 * i + 1]);
    }
    __builtin_memcpy(p, &o, 8);
  }
}

// v += the residual's four values from element o on.
__device__ __forceinline__ void q8_add4(const Q8LinParams& p, int64_t o, float (&v)[4]) {
  if (p.res_dtype == VNX_F32) {  // uniform
    f32x4 a;
    __builtin_memcpy(&a, static_cast<const float*>(p.res) + o, 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += a[i];
  } else {
    u32x2 a;
    __builtin_memcpy(&a, static_cast<const uint16_t*>(p.res) + o, 8);
    const bool bf = p.res_dtype == VNX_BF16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = a[i / 2];
      const float x = __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16), y = (float)__builtin_bit_cast(f16x2, w)[i & 1];
      v[i] += bf ? x : y;
    }
  }
}

__device__ __forceinline__ float q8_res1(const Q8LinParams& p, int64_t o) {
  return p.res_dtype == VNX_F32    ? q8_ld1(static_cast<const float*>(p.res) + o)
         : p.res_dtype == VNX_BF16 ? q8_ld1(static_cast<const uint16_t*>(p.res) + o)
                                   : q8_ld1(static_cast<const _Float16*>(p.res) + o);
}

template <typename TY, bool RES, bool SW, int BM, int BN, int WM, int WN, int KS, int NS, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_q8_tile(Q8LinParams p) {
  constexpr int NW = WM * WN, RT = BM / WM / 16, CT = BN / WN / 16;
  constexpr int SLAB = 64 * KS, PART = (BM + BN) * 64, STAGE = KS * PART, OC = SW ? BN / 2 : BN;
  constexpr int PW = (BM + BN) / 16 / NW, CW = PW * KS;  // a wave's copies of a part, and of a slab
  static_assert((BM + BN) / 16 % NW == 0 && (NS - 1) * CW < 64 && NS % 2 == 0 && (!SW || CT % 2 == 0), "");
  __shared__ __attribute__((aligned(256))) char smem[NS * STAGE];
  constexpr int SM = (BM + 63) / 64 * 64, SN = (BN + 63) / 64 * 64;
  __shared__ __attribute__((aligned(256))) float scales[SM + 2 * SN];  // of x, of W, the bias
  // results: tiles of a row (CTO, ST in a strip), values in 16 bytes, lanes a row, pitch
  constexpr int CTO = SW ? CT / 2 : CT, VE = 16 / sizeof(TY), ST = CTO < 8 / (int)sizeof(TY) ? CTO : 8 / (int)sizeof(TY);
  constexpr int LR = ST * 16 / VE, SP = ST * 16 * (int)sizeof(TY) + 16;
  static_assert(CTO % ST == 0, "");
  static_assert(NW * 16 * SP <= NS * STAGE, "");     // (the ring is free by then)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN, r = lane & 15, g4 = lane >> 4;
  // Each XCD takes a run of tiles, in blocks of eight rows of tiles: the tiles
  // that run at once on it share rows of x and of W in its L2.
  int m0, o0;                                        // first row and column of y
  {
    const int total = p.mt * p.nt, run = (total + kQ8Xcds - 1) / kQ8Xcds, at = blockIdx.x / kQ8Xcds;
    const int i = blockIdx.x % kQ8Xcds * run + at;
    if (at >= run || i >= total) return;             // uniform over the workgroup
    const int blk = i / (8 * p.nt), in = i - blk * 8 * p.nt, h = min(8, p.mt - blk * 8), ni = in / h;
    m0 = (blk * 8 + in - ni * h) * BM;
    o0 = ni * OC;
  }
  constexpr bool SUMS = __is_same(TY, int);
  const int k0 = SUMS ? (int)blockIdx.y * p.per * SLAB : 0, K = SUMS ? min(p.K - k0, p.per * SLAB) : p.K;
  const int nsl = (K + 2 * SLAB - 1) / (2 * SLAB) * 2;  // an even number: the last may be all zeros
  const uint32_t lds0 = lds_addr(smem);

  // this wave's copies of a part: rows 16 (wave PW + q) + lane / 4 of [x tile; W tile]
  const int piece = (lane & 3) ^ (-(lane >> 4) & 3); // of the row's four in a part
  uint32_t off[PW];
  const int8_t* base[PW];                            // uniform
#pragma unroll
  for (int q = 0; q < PW; ++q) {
    const int r0 = (wave * PW + q) * 16;
    if (r0 < BM) {
      base[q] = p.x + (int64_t)m0 * p.ldx + k0;
      off[q] = (uint32_t)min(r0 + (lane >> 2), p.M - 1 - m0) * (uint32_t)p.ldx + piece * 16;
    } else {
      const int w0 = r0 - BM, up = SW ? w0 / 16 & 1 : 0, row = SW ? w0 / 32 * 16 : w0;
      base[q] = p.w + (int64_t)(up ? p.cols + o0 : o0) * p.ldw + k0;
      off[q] = (uint32_t)min(row + (lane >> 2), p.cols - 1 - o0) * (uint32_t)p.ldw + piece * 16;
    }
  }
  // copy j of slab c (a piece past the row's end: its first instead)
  auto copy = [&](int c, int j) {
    const int part = j / PW, q = j % PW, k = c * SLAB + part * 64;
    const uint32_t back = k + piece * 16 < K ? 0u : piece * 16u;
    const uint32_t to = lds0 + c % NS * STAGE + part * PART + (wave * PW + q) * 1024;
    copy_to_lds(__builtin_amdgcn_readfirstlane(to), off[q] - back, base[q] + (k < K ? k : 0));
  };
  // bytes of x at or past K count as 0, in the pieces of slab c that this lane copied
  auto clear = [&](int c) {
#pragma unroll
    for (int j = 0; j < CW; ++j) {
      const int part = j / PW, q = j % PW, in = K - c * SLAB - part * 64 - piece * 16;
      if ((wave * PW + q) * 16 >= BM || in >= 16) continue;
      u32x4* d = reinterpret_cast<u32x4*>(smem + c % NS * STAGE + part * PART + (wave * PW + q) * 1024 + lane * 16);
      u32x4 v = *d;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = in - 4 * e;
        v[e] = n >= 4 ? v[e] : n <= 0 ? 0u : v[e] & ((1u << (8 * n)) - 1u);
      }
      *d = v;
    }
  };

  // ---- operands and products ----
  i32x4 acc[RT][CT];
  const int col = (g4 ^ (-(r >> 2) & 3)) * 16;
  const int xo = (wm * RT * 16 + r) * 64 + col, wo = (BM + wn * CT * 16 + r) * 64 + col;
  struct Set { u32x4 x[KS][RT], w[KS][CT]; };
  constexpr int OPS = KS * (RT + CT), PROD = KS * RT * CT;
  auto read1 = [&](const char* b, int j, Set& q) {
    const int part = j / (RT + CT), i = j % (RT + CT);
    b += part * PART;
    if (i < CT) q.w[part][i] = *reinterpret_cast<const u32x4*>(b + wo + i * 1024);
    else q.x[part][i - CT] = *reinterpret_cast<const u32x4*>(b + xo + (i - CT) * 1024);
  };
  auto product = [&](const Set& q, int j) {
    const int part = j / (RT * CT), i = j / CT % RT, t = i & 1 ? CT - 1 - j % CT : j % CT;
    acc[i][t] = q8_mma(q.w[part][t], q.x[part][i], acc[i][t]);
  };
  // Slab c's products.  The copies of slab c + NS (COPY) and the reads of slab c + 1
  // (unless LAST) are spread over them, the reads early.  left: of the slabs behind
  // c + 1, how many are under way.
  auto step = [&](auto left, auto copies, auto last, int c, const Set& cur, Set& nxt) {
    constexpr bool COPY = decltype(copies)::value, LAST = decltype(last)::value;
    constexpr int G = PROD < 8 ? PROD : 8, PG = PROD / G, RG = (OPS + G * 3 / 4 - 1) / (G * 3 / 4);
    static_assert(PROD % G == 0, "");
    if constexpr (!LAST) {
      wait_copies<decltype(left)::value * CW>();
      if ((c + 2) * SLAB > K) clear(c + 1);     // uniform
      lds_barrier();
    }
    const char* b = smem + (c + 1) % NS * STAGE;
#pragma unroll
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int j = 0; j < PG; ++j) product(cur, g * PG + j);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (COPY)
#pragma unroll
        for (int q = g * CW / G; q < (g + 1) * CW / G; ++q) copy(c + NS, q);
      if constexpr (!LAST)
#pragma unroll
        for (int j = 0; j < RG; ++j)
          if (g * RG + j < OPS) read1(b, g * RG + j, nxt);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if constexpr (!SUMS) {
    // the scales, 64 a copy
    for (int u = wave; u < (SM + (p.bias ? 2 : 1) * SN) / 64; u += NW) {
      const int j = u * 64 + lane;
      const float* src;
      if (u * 64 < SM) {
        src = p.xs + m0 + min(j, p.M - 1 - m0);
      } else {
        const int w = j < SM + SN ? j - SM : j - SM - SN, up = SW ? w / 16 & 1 : 0, row = SW ? w / 32 * 16 + w % 16 : w;
        src = (j < SM + SN ? p.ws : p.bias) + (int64_t)up * p.cols + min(o0 + row, p.cols - 1);
      }
      copy_to_lds(lds_addr(scales) + u * 256, src);
    }
    if (!p.bias)
      for (int i = tid; i < SN; i += 64 * NW) scales[SM + SN + i] = 0.0f;
  }
#pragma unroll 1
  for (int c = 0; c < NS; ++c)                       // (of fewer slabs: the first again, not read)
#pragma unroll
    for (int j = 0; j < CW; ++j) copy(c, j);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][t][e] = 0;
  wait_copies<(NS - 1) * CW>();
  if (SLAB > K) clear(0);
  lds_barrier();
  Set a, b;
#pragma unroll
  for (int j = 0; j < OPS; ++j) read1(smem, j, a);
  constexpr auto yes = BoolC<true>{};
  constexpr auto no = BoolC<false>{};
  int c = 0;
#pragma unroll 1
  for (; c + NS < nsl; c += 2) {
    step(IntC<NS - 2>{}, yes, no, c, a, b);
    step(IntC<NS - 2>{}, yes, no, c + 1, b, a);
  }
  // the last NS slabs, or all of fewer (of which the last reads a slab for nothing)
  auto tail = [&](auto at) {
    constexpr int J = decltype(at)::value;
    if (c + J >= nsl) return;                        // uniform
    if constexpr (J % 2 == 0) step(IntC<NS - 2 - J>{}, no, no, c + J, a, b);
    else if constexpr (J + 1 < NS) step(IntC<NS - 2 - J>{}, no, no, c + J, b, a);
    else step(IntC<0>{}, no, yes, c + J, b, a);
  };
  each(tail, std::make_integer_sequence<int, NS>{});
  wait_copies<0>();
  if constexpr (SUMS) {
    const int64_t ld = (int64_t)p.nt * BN;
    int* y = static_cast<int*>(p.y) + ((int64_t)blockIdx.y * p.mt * BM + m0 + wm * RT * 16 + r) * ld + o0 + wn * CT * 16 + 4 * g4;
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int t = 0; t < CT; ++t) *reinterpret_cast<i32x4*>(y + i * 16 * ld + t * 16) = acc[i][t];
    return;
  }
  lds_barrier();                                     // every wave has its operands: the ring is free

  // Sixteen rows of up to 128 bytes at a time leave through a part of LDS of the
  // wave's own, so that each store takes whole runs of a row; past the caches,
  // which would hold the stores up (the 248,320 head at 224 rows: 105 us through
  // them, 79 past, 74 with no stores at all).
  auto leave = [&](auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    constexpr bool LATE = RES && sizeof(TY) == 4;  // the residual is added behind LDS, which holds fp32
    const float* sw = scales + SM + wn * CT * 16 + 4 * g4;  // of this lane's W rows (read again and again: registers are few)
    const int n0 = o0 + wn * CTO * 16;
    char* mine = smem + wave * 16 * SP;
    const int lr = lane / LR, lc = lane % LR * VE; // row and first column of this lane's 16 bytes
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int rl = (wm * RT + i) * 16;
      const float sx = scales[rl + r];
#pragma unroll
      for (int q = 0; q < CTO; q += ST) {
#pragma unroll
        for (int u = 0; u < ST; ++u) {
          const int t = (q + u) * (SW ? 2 : 1);
          float v[4];
          auto val = [&](int at, float (&d)[4]) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(sw + at * 16), c = *reinterpret_cast<const f32x4*>(sw + SN + at * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = fmaf((float)acc[i][at][e] * sx, w[e], c[e]);
          };
          val(t, v);
          if constexpr (SW) {
            float up[4];
            val(t + 1, up);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = q8_swiglu(v[e], up[e]);
          }
          if constexpr (RES && !LATE) {
            const int m = m0 + rl + r, n = n0 + (q + u) * 16 + 4 * g4;
            const int64_t o = (int64_t)m * p.ldr + n;
            if (!EDGE || (m < p.M && n + 4 <= p.cols)) {
              q8_add4(p, o, v);
            } else if (m < p.M) {
#pragma unroll
              for (int e = 0; e < 3; ++e)
                if (n + e < p.cols) v[e] += q8_res1(p, o + e);
            }
          }
          q8_st4(static_cast<TY*>(__builtin_assume_aligned(mine + r * SP + (u * 16 + 4 * g4) * (int)sizeof(TY), 4 * sizeof(TY))), v);
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int h = 0; h < 16; h += 64 / LR) {
          if (64 / LR > 16 && lr >= 16) break;
          const int m = m0 + rl + h + lr, n = n0 + q * 16 + lc;
          u32x4 d = *reinterpret_cast<const u32x4*>(mine + (h + lr) * SP + lane % LR * 16);
          TY* y = static_cast<TY*>(p.y) + (int64_t)m * p.ldy + n;
          if (!EDGE || (m < p.M && n + VE <= p.cols)) {
            if constexpr (LATE) {
              float v[4];
              __builtin_memcpy(v, &d, 16);
              q8_add4(p, (int64_t)m * p.ldr + n, v);
              __builtin_memcpy(&d, v, 16);
            }
            if (p.y_vec) __builtin_nontemporal_store(d, reinterpret_cast<u32x4*>(y));
            else __builtin_memcpy(y, &d, 16);
          } else if (m < p.M) {
            TY v[VE];
            __builtin_memcpy(v, &d, 16);
#pragma unroll
            for (int e = 0; e < VE - 1; ++e) {
              if (n + e >= p.cols) break;
              if constexpr (LATE) v[e] += q8_res1(p, (int64_t)m * p.ldr + n + e);
              y[e] = v[e];
            }
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      }
    }
  };
  if constexpr (!SUMS) {
    if (m0 + BM <= p.M && o0 + OC <= p.cols) leave(BoolC<false>{});
    else leave(BoolC<true>{});
  }
}

template <bool SW, int BM, int BN, int WM, int WN, int KS, int NS, int OCC>
int q8_tile(Q8LinParams p, hipStream_t st) {
  constexpr int OC = SW ? BN / 2 : BN;
  p.mt = (p.M + BM - 1) / BM;
  p.nt = (p.cols + OC - 1) / OC;
  const int64_t total = (int64_t)p.mt * p.nt;
  if (total >= INT_MAX / 2 || (int64_t)8 * p.nt >= INT_MAX) return VNX_ERR_UNSUPPORTED;
  const int64_t wgs64 = (total + kQ8Xcds - 1) / kQ8Xcds * kQ8Xcds;
  if (!launch_fits(wgs64, 64 * WM * WN)) return VNX_ERR_UNSUPPORTED;
  const unsigned wgs = (unsigned)wgs64;
  const int ey = elem_size(p.y_dtype);
  p.y_vec = aligned16(p.y) && p.ldy * ey % 16 == 0;
  return q8_by_type(p.y_dtype, [&](auto ty) -> int {
    using TY = decltype(ty);
    if constexpr (!SW) {
      if (p.res) {
        hipLaunchKernelGGL((k_q8_tile<TY, true, SW, BM, BN, WM, WN, KS, NS, OCC>), dim3(wgs), dim3(64 * WM * WN), 0, st, p);
        VNX_LAUNCH_CHECK();
        return VNX_OK;
      }
    }
    hipLaunchKernelGGL((k_q8_tile<TY, false, SW, BM, BN, WM, WN, KS, NS, OCC>), dim3(wgs), dim3(64 * WM * WN), 0, st, p);
    VNX_LAUNCH_CHECK();
    return VNX_OK;
  });
}

// ---------------------------------------------------------------------------
// Launch shapes, and the choice between them by an estimate of their time: `once`
// us a launch and, n the workgroups a CU, n times `slab` us per 64 bytes of k
// (`alone` where less than half of the CUs has one; k to whole pairs of slabs, four
// slabs at least) and `rest` us.  Fitted to 168 sizes (1 to 8,192 rows): the shape
// taken is 1.1% slower than the fastest on average, 16% at most.  us by the estimate
// / measured (M x N x K; the shape taken first):
//   2,048 x 2,048 x 1,024    128^2 8.3 / 8.7; 64 x 128 9.5 / 9.8, 64^2 10.3 / 10.6, 256^2 15.4 / 16.2
//   2,048 x 1,024 x 2,752    64 x 128 11.7 / 12.5; 64^2 13.1 / 14.2, 128^2 14.2 / 17.3
//   400 x 2,048 x 2,048      64^2 6.1 / 6.0; 64 x 128 8.4 / 8.4, 32^2 9.2 / 8.7
//   224 x 1,024 x 4,096      32^2 5.6 / 5.8; 64^2 9.2 / 9.6, direct 14.6 / 16.5
//   32 x 4,096 x 1,024       32^2 2.9 / 2.8; direct 3.8 / 3.8, 64^2 3.9 / 3.9
//   1 x 1,024 x 4,096        direct 4.6 / 4.1; 32^2 5.5 / 5.1
// ---------------------------------------------------------------------------
constexpr int kQ8Direct = 4, kQ8Split = 5, kQ8Shapes = 7;
struct Q8Shape { int shape, bm, bn, ks; double slab, alone, rest, once; };
constexpr Q8Shape kQ8Tiles[5] = {{0, 256, 256, 1, 0.795, 0.562, 4.96, 1.49},
                                 {1, 128, 128, 1, 0.295, 0.243, 1.04, 2.52},
                                 {2, 64, 128, 1, 0.207, 0.183, 0.317, 2.2},
                                 {3, 64, 64, 2, 0.124, 0.111, 0.071, 2.08},
                                 {6, 32, 32, 4, 0.055, 0.053, 0.045, 2.02}};
constexpr Q8Shape kQ8Pairs = {6, 32, 32, 4, 0.066, 0.091, 0, 2.31};  // of SwiGLU: two waves

// A split's sums joined: thread i has eight columns of a row.
template <bool SW>
__global__ __launch_bounds__(256) void k_q8_join(Q8LinParams p, const int* part, int64_t split, int64_t ld, int splits) {
  const int pieces = (p.cols + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / pieces;
  if (row >= p.M) return;
  const int m = (int)row, n = (int)(i - row * pieces) * 8;
  auto sum8 = [&](int col, int (&a)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a[e] = 0;
    const int* src = part + m * ld + col;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      i32x4 lo, hi;
      __builtin_memcpy(&lo, src + s * split, 16);
      __builtin_memcpy(&hi, src + s * split + 4, 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) { a[e] += lo[e]; a[4 + e] += hi[e]; }
    }
  };
  int a[8];
  float v[8];
  const float xs = p.xs[m];
  sum8(n, a);
  if constexpr (SW) {
    float u[8];
    q8_scale8(p, xs, n, p.cols, a, v);
    sum8(p.cols + n, a);
    q8_scale8(p, xs, p.cols + n, p.N, a, u);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = q8_swiglu(v[e], u[e]);
  } else {
    q8_scale8(p, xs, n, p.N, a, v);
  }
  q8_out8(p, m, n, v);
}

struct Q8Plan {
  int shape, per, splits;  // kQ8Split: slabs of 128 a split, splits
  size_t bytes;            // workspace
};

// The splits of k that 64 x 64 tiles in `want` of them have.
Q8Plan q8_split(const Q8LinParams& p, int want) {
  const int nsl = (p.K + 255) / 256 * 2, per = (nsl + 2 * want - 1) / (2 * want) * 2;
  const int splits = (nsl + per - 1) / per;
  const int64_t cells = (int64_t)((p.M + 63) / 64) * ((p.N + 63) / 64) * 4096;
  return {kQ8Split, per, splits, (size_t)(cells * splits * 4 + 64)};  // (the join may read 28 bytes on)
}

template <bool SW>
Q8Plan q8_plan(const Q8LinParams& p, int force) {
  const int64_t cus = device_cus();
  const double hbm = ((double)p.M * p.K + (double)p.N * p.K + (double)p.M * p.cols * elem_size(p.y_dtype)) / 5e6;
  Q8Plan best{0, 0, 0, 0};
  double least = 1e300;
  auto take = [&](double t, int shape) {
    const double us = t > hbm ? t : hbm + 0.01 * t;
    if (us < least) least = us, best.shape = shape;
  };
  for (int i = 0; i < 5; ++i) {
    const Q8Shape& s = SW && i == 4 ? kQ8Pairs : kQ8Tiles[i];
    const int oc = SW ? s.bn / 2 : s.bn, slabs = 2 * s.ks * std::max(2, (p.K + 128 * s.ks - 1) / (128 * s.ks));
    const int64_t tiles = (int64_t)((p.M + s.bm - 1) / s.bm) * ((p.cols + oc - 1) / oc);
    take(s.once + (double)((tiles + cus - 1) / cus) * (slabs * (2 * tiles <= cus ? s.alone : s.slab) + s.rest), s.shape);
  }
  if (!SW) {
    // 16 x 16 of y a workgroup; rows of x that are one and the same line cost less
    const int64_t wgs = (int64_t)((p.M + 15) / 16) * ((p.N + 15) / 16);
    take(1.98 + (double)(wgs > cus ? wgs : cus) / cus * ((p.K + 63) / 64) * (p.M <= 4 ? 0.0403 : 0.0557), kQ8Direct);
  }
  // Few tiles and a long k: a CU's 70 GB/s of copies to LDS bounds a tile, so k is
  // shared by more of them, at the price of a second launch.  32 x 256 x 16,384 14.8
  // -> 9.6 us, 16 x 1,024 x 11,008 11.6 -> 8.7; 224 x 1,024 x 4,096 would take 9.0
  // (5.8 as it is).
  const int64_t tiles = (int64_t)((p.M + 63) / 64) * ((p.N + 63) / 64);
  if (force == kQ8Split + 1) least = 1e300;
  for (int want = 2; want <= 32 && (want == 2 || tiles * want <= 2 * cus); want *= 2) {
    const Q8Plan s = q8_split(p, want);
    const int64_t wgs = tiles * s.splits;
    const double us = 4.4 + (double)((wgs + cus - 1) / cus) * (s.per * 2 * (2 * wgs <= cus ? 0.091 : 0.131) + 1.13) +
                      (double)s.bytes / 3e6;
    if (us < 0.95 * least && s.bytes < (size_t)1 << 30) least = us, best = s;
  }
  if (force && force != kQ8Split + 1) best = {force - 1, 0, 0, 0};
  return best;
}

template <bool SW>
int q8_linear(const Q8LinParams& p, int force, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Q8Plan plan = q8_plan<SW>(p, force);
  switch (plan.shape) {
    case 0: return q8_tile<SW, 256, 256, 2, 4, 1, 4, 1>(p, st);
    case 1: return q8_tile<SW, 128, 128, 2, 2, 1, 4, 2>(p, st);
    case 2: return q8_tile<SW, 64, 128, 2, 2, 1, 4, 3>(p, st);
    case 3: return q8_tile<SW, 64, 64, 2, 2, 2, 4, 2>(p, st);
    case 6: return q8_tile<SW, 32, 32, 2, SW ? 1 : 2, 4, 4, 2>(p, st);
    case kQ8Direct:
      if constexpr (!SW) return q8_direct<4>(p, st);
      return VNX_ERR_UNSUPPORTED;
  }
  if (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace)) return VNX_ERR_WORKSPACE;
  Q8LinParams q = p;
  q.cols = p.N;  // (gate and up rows are columns like any)
  q.y = workspace, q.per = plan.per;
  q.mt = (p.M + 63) / 64, q.nt = (p.N + 63) / 64;
  const int64_t tiles = ((int64_t)q.mt * q.nt + kQ8Xcds - 1) / kQ8Xcds * kQ8Xcds, rows = (int64_t)q.mt * 64;
  const int64_t joins = ((int64_t)p.M * ((p.cols + 7) / 8) + 255) / 256;
  if ((int64_t)q.mt * q.nt >= INT_MAX / 2 || (int64_t)8 * q.nt >= INT_MAX || !launch_fits(tiles * plan.splits, 256) ||
      !launch_fits(joins, 256))
    return VNX_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((k_q8_tile<int, false, false, 64, 64, 2, 2, 2, 4, 2>), dim3((unsigned)tiles, plan.splits), dim3(256), 0,
                     st, q);
  VNX_LAUNCH_CHECK();
  hipLaunchKernelGGL((k_q8_join<SW>), dim3((unsigned)joins), dim3(256), 0, st, p, static_cast<const int*>(workspace),
                     rows * q.nt * 64, (int64_t)q.nt * 64, plan.splits);
  VNX_LAUNCH_CHECK();
  return VNX_OK;
}

// The checks that need no pointer, and the sizes.
int q8_sizes(const vnx_q8_linear_args* a, Q8LinParams* p) {
  if (!a || a->M < 0 || a->N < 0 || a->K < 1 || a->ldx < a->K || a->ldw < a->K) return VNX_ERR_INVALID_ARG;
  if (a->epilogue != VNX_EPI_NONE && a->epilogue != VNX_EPI_SWIGLU) return VNX_ERR_INVALID_ARG;
  const bool sw = a->epilogue == VNX_EPI_SWIGLU;
  const int64_t cols = sw ? a->N / 2 : a->N;
  if ((sw && (a->N % 2 || a->res)) || a->ldy < cols || (a->res && a->ldr < cols)) return VNX_ERR_INVALID_ARG;
  if (!q8_float(a->y_dtype) || (a->res && !q8_float(a->res_dtype))) return VNX_ERR_UNSUPPORTED;
  // rows and columns are numbered to the end of their last tile in 32 bits
  if (a->K > kQ8MaxK || a->M >= INT_MAX - 4096 || a->N >= INT_MAX - 4096) return VNX_ERR_UNSUPPORTED;
  if (a->force_shape < 0 || a->force_shape > kQ8Shapes) return VNX_ERR_UNSUPPORTED;
  p->M = (int)a->M; p->N = (int)a->N; p->K = (int)a->K; p->cols = (int)cols;
  p->y_dtype = a->y_dtype; p->res_dtype = a->res_dtype;
  return VNX_OK;
}

// Bytes from a on that rows `ld` apart take.
bool bytes_meet(const void* a, __int128 na, const void* b, __int128 nb) {
  const __int128 a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
  return a0 < b0 + nb && b0 < a0 + na;
}

}  // namespace
}  // namespace vnx

using namespace vnx;

extern "C" {

size_t vnx_q8_linear_workspace(const vnx_q8_linear_args* a) {
  Q8LinParams p{};
  if (q8_sizes(a, &p) != VNX_OK || a->M == 0 || a->N == 0) return 256;
  const size_t n = (a->epilogue == VNX_EPI_SWIGLU ? q8_plan<true>(p, a->force_shape) : q8_plan<false>(p, a->force_shape)).bytes;
  return n > 256 ? n : 256;
}

int vnx_q8_linear(const vnx_q8_linear_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  Q8LinParams p{};
  if (const int rc = q8_sizes(a, &p)) return rc;
  const bool sw = a->epilogue == VNX_EPI_SWIGLU;
  const int64_t cols = p.cols;
  if (a->M == 0 || a->N == 0) return VNX_OK;
  if (!a->x || !a->x_scale || !a->w || !a->w_scale || !a->y) return VNX_ERR_INVALID_ARG;
  const int ey = elem_size(a->y_dtype), er = elem_size(a->res_dtype);
  if (!aligned_to(a->y, ey) || (a->res && !aligned_to(a->res, er)) || !aligned_to(a->x_scale, 4) ||
      !aligned_to(a->w_scale, 4) || (a->bias && !aligned_to(a->bias, 4)))
    return VNX_ERR_INVALID_ARG;
  if (!aligned16(a->x) || !aligned16(a->w) || a->ldx % 16 || a->ldw % 16) return VNX_ERR_UNSUPPORTED;
  if (a->ldx >= (int64_t)1 << 22 || a->ldw >= (int64_t)1 << 22) return VNX_ERR_UNSUPPORTED;
  // y on something that other workgroups still read (the residual's own place is
  // read before it is written, by the same thread)
  const __int128 ny = ((__int128)(a->M - 1) * a->ldy + cols) * ey;
  if (bytes_meet(a->y, ny, a->x, (__int128)(a->M - 1) * a->ldx + a->K) ||
      bytes_meet(a->y, ny, a->w, (__int128)(a->N - 1) * a->ldw + a->K) ||
      bytes_meet(a->y, ny, a->x_scale, 4 * a->M) || bytes_meet(a->y, ny, a->w_scale, 4 * a->N) ||
      (a->bias && bytes_meet(a->y, ny, a->bias, 4 * a->N)))
    return VNX_ERR_INVALID_ARG;
  if (a->res && !(a->res == a->y && a->ldr == a->ldy && er == ey) &&
      bytes_meet(a->y, ny, a->res, ((__int128)(a->M - 1) * a->ldr + cols) * er)) {
    if (er != ey || a->ldr != a->ldy || a->res == a->y || Rows(cols, &a->ldy, {a->M}).meet(a->y, a->res, ey))
      return VNX_ERR_INVALID_ARG;
  }
  p.x = a->x; p.w = a->w; p.xs = a->x_scale; p.ws = a->w_scale; p.bias = a->bias; p.res = a->res; p.y = a->y;
  p.ldx = a->ldx; p.ldw = a->ldw; p.ldr = a->ldr; p.ldy = a->ldy;
  const auto st = static_cast<hipStream_t>(stream);
  return sw ? q8_linear<true>(p, a->force_shape, workspace, workspace_bytes, st)
            : q8_linear<false>(p, a->force_shape, workspace, workspace_bytes, st);
}

}  // extern "C"
