// Products of 8-bit integer rows on gfx950 (vnx_q8_linear): x (M, K) codes with a
// scale a row times W (N, K) codes with a scale a row,
//   acc[m, n] = sum_k x[m, k] * W[n, k]          (exact in int32: K <= 131,071)
//   y[m, n] = acc * x_scale[m] * w_scale[n] (+ bias[n]) (+ residual[m, n])
// or, of gate rows and up rows, silu(gate) * up.  The sums are whole numbers, so
// how K is split never changes a result.
//
// k_q8_direct: operands straight from global memory to the matrix cores (the
// order of k inside a product is free as long as both operands have the same,
// so each lane loads whole pieces of its row), the K pieces of a tile shared by
// KW waves whose sums meet in LDS.
#include <climits>

#include "q8.h"

namespace vnx {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

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
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (float)a[i] * xs * s[i];
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += p.bias[min(r + i, rows - 1)];
  }
}

template <int S>
struct Mfma;
template <>
struct Mfma<16> {
  typedef i32x4 Acc;
  static constexpr int P = 2;          // 16-byte pieces of a lane's row a chunk
  __device__ __forceinline__ static Acc mma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
  // row of the tile that register e of lane group g holds
  __device__ __forceinline__ static int row(int g, int e) { return 4 * g + e; }
};
template <>
struct Mfma<32> {
  typedef i32x16 Acc;
  static constexpr int P = 4;
  __device__ __forceinline__ static Acc mma(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
  }
  __device__ __forceinline__ static int row(int g, int e) { return 8 * (e >> 2) + 4 * g + (e & 3); }
};

// A workgroup: MT x S rows of x by NW waves' NT x S rows of W each; SW: a wave's
// tiles are gate and up rows in turn.
template <int S, int MT, int NT, int KW, int NW, bool SW>
__global__ __launch_bounds__(64 * KW * NW) void k_q8_direct(Q8LinParams p) {
  using F = Mfma<S>;
  constexpr int P = F::P, ACC = S * S / 64;
  constexpr int ROWS = S * MT, WCOLS = S * NT, PITCH = WCOLS + 4;
  constexpr int OCOLS = SW ? WCOLS / 2 : WCOLS;    // columns of y a wave
  __shared__ __attribute__((aligned(16))) int red[KW * NW * ROWS * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave % KW, nw = wave / KW;
  const int r = lane % S, g = lane / S;
  // the row tiles that share W rows follow each other on one XCD
  const int xcd = blockIdx.x % kQ8Xcds, at = blockIdx.x / kQ8Xcds;
  const int mi = at % p.mt, ni = at / p.mt * kQ8Xcds + xcd;
  if (ni >= p.nt) return;  // uniform over the workgroup
  const int m0 = mi * ROWS, o0 = (ni * NW + nw) * OCOLS;   // first row and column of y
  const int8_t *xp[MT], *wp[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xp[i] = p.x + (int64_t)min(m0 + i * S + r, p.M - 1) * p.ldx + g * (16 * P);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = SW ? min(o0 + t / 2 * S + r, p.cols - 1) + (t & 1) * p.cols : min(o0 + t * S + r, p.N - 1);
    wp[t] = p.w + (int64_t)row * p.ldw + g * (16 * P);
  }
  typename F::Acc acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < ACC; ++e) acc[i][t][e] = 0;

  struct Set { u32x4 x[MT][P], w[NT][P]; };
  const int nf = p.K / kQ8Chunk;
  auto load = [&](int c, Set& q) {
    const int64_t k = (int64_t)c * kQ8Chunk;
#pragma unroll
    for (int s = 0; s < P; ++s) {
#pragma unroll
      for (int t = 0; t < NT; ++t) q.w[t][s] = *reinterpret_cast<const u32x4*>(wp[t] + k + s * 16);
#pragma unroll
      for (int i = 0; i < MT; ++i) q.x[i][s] = *reinterpret_cast<const u32x4*>(xp[i] + k + s * 16);
    }
  };
  auto mma = [&](const Set& q) {
#pragma unroll
    for (int s = 0; s < P; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][t] = F::mma(q.x[i][s], q.w[t][s], acc[i][t]);
  };
  if (kw < nf) {
    Set a, b;
    const int last = kw + (nf - 1 - kw) / KW * KW;   // this wave's last chunk
    load(kw, a);
    for (int c = kw; c < nf; c += 2 * KW) {
      load(min(c + KW, last), b);
      mma(a);
      load(min(c + 2 * KW, last), a);
      if (c + KW < nf) mma(b);                       // uniform
    }
  }
  if (p.K % kQ8Chunk && kw == nf % KW) {
    // The last chunk's pieces: those past the row's end come from its start, and
    // every byte of x at or past K counts as 0 (of W there may be anything).
    Set q;
#pragma unroll
    for (int s = 0; s < P; ++s) {
      const int64_t k = (int64_t)nf * kQ8Chunk + s * 16;
      const int left = p.K - (int)k - g * (16 * P);  // bytes of this piece inside the row
      const int64_t o = left > 0 ? k : -g * (16 * P);
#pragma unroll
      for (int t = 0; t < NT; ++t) q.w[t][s] = *reinterpret_cast<const u32x4*>(wp[t] + o);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        u32x4 v = *reinterpret_cast<const u32x4*>(xp[i] + o);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = left - 4 * e;                // bytes of this word inside the row
          v[e] = n >= 4 ? v[e] : n <= 0 ? 0u : v[e] & ((1u << (8 * n)) - 1u);
        }
        q.x[i][s] = v;
      }
    }
    mma(q);
  }

  int* mine = red + wave * ROWS * PITCH;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < ACC; ++e) mine[(i * S + F::row(g, e)) * PITCH + t * S + r] = acc[i][t][e];
  __syncthreads();
  constexpr int GR = OCOLS / 8;                      // pieces of 8 columns a row and wave
  for (int j = tid; j < ROWS * GR * NW; j += 64 * KW * NW) {
    const int c = j % (GR * NW), row = j / (GR * NW), m = m0 + row;
    const int w = c / GR, o = c % GR * 8;            // (OCOLS of each wave follow each other)
    const int n = (ni * NW + w) * OCOLS + o;
    if (m >= p.M || n >= p.cols) continue;
    const int* src = red + w * KW * ROWS * PITCH + row * PITCH;
    const float xs = p.xs[m];
    auto sum8 = [&](int col, int (&a)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = 0;
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(src + k * ROWS * PITCH + col),
                    hi = *reinterpret_cast<const i32x4*>(src + k * ROWS * PITCH + col + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { a[i] += lo[i]; a[4 + i] += hi[i]; }
      }
    };
    int a[8];
    float v[8];
    if constexpr (SW) {
      float u[8];
      const int col = o / S * 2 * S + o % S;         // the gate's; the up's is S further on
      sum8(col, a);
      q8_scale8(p, xs, n, p.cols, a, v);
      sum8(col + S, a);
      q8_scale8(p, xs, p.cols + n, p.N, a, u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = q8_swiglu(v[i], u[i]);
    } else {
      sum8(o, a);
      q8_scale8(p, xs, n, p.N, a, v);
    }
    q8_out8(p, m, n, v);
  }
}

template <int S, int MT, int NT, int KW, int NW, bool SW>
int q8_direct(Q8LinParams p, hipStream_t st) {
  constexpr int OC = NW * S * NT / (SW ? 2 : 1);
  p.mt = (p.M + S * MT - 1) / (S * MT);
  p.nt = (p.cols + OC - 1) / OC;
  const int64_t wgs = (int64_t)p.mt * ((p.nt + kQ8Xcds - 1) / kQ8Xcds * kQ8Xcds);
  if (wgs >= INT_MAX || !launch_fits(wgs, 64 * KW * NW)) return VNX_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((k_q8_direct<S, MT, NT, KW, NW, SW>), dim3((unsigned)wgs), dim3(64 * KW * NW), 0, st, p);
  VNX_LAUNCH_CHECK();
  return VNX_OK;
}

// ---------------------------------------------------------------------------
// k_q8_tile: many rows.  BM x BN tiles of y, WM x WN waves, slabs of 64 bytes of
// k in a ring of NS buffers in LDS.
//
// The slabs come by direct copies from memory to LDS (1 KB an instruction: 16
// rows of 64 bytes, lane l's 16 bytes at 16 l), so the tile's layout is made by
// which piece of its row a lane asks for: piece c of row R lies at c ^ (R / 4 %
// 4), and the sixteen lanes that LDS serves together, four runs of four rows,
// read sixteen different 16-byte columns of its 256.  A wave holds two sets of operands: it reads slab c + 1
// while the products of slab c run, and slab c + NS comes into the buffer that
// slab c has left, so one barrier a slab does.
// ---------------------------------------------------------------------------
constexpr int kQ8Slab = 64;

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

// Waits until at most N of this wave's copies are under way.
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "i"(N) : "memory");
}

// Every wave's LDS reads so far are done, and every wave is here.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), in a form that the compiler counts with
  asm volatile("s_barrier" : : : "memory");
}

template <int S, int BM, int BN, int WM, int WN, int NS, int OCC, bool SW>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_q8_tile(Q8LinParams p) {
  using F = Mfma<S>;
  constexpr int NW = WM * WN, RT = BM / WM / S, CT = BN / WN / S, KT = S / 16;
  constexpr int STAGE = (BM + BN) * kQ8Slab, PW = (BM + BN) / 16 / NW;
  static_assert((BM + BN) / 16 % NW == 0 && (NS - 1) * PW < 64 && (!SW || CT % 2 == 0), "");
  constexpr int ACC = S * S / 64, WCOLS = CT * S, WOUT = SW ? WCOLS / 2 : WCOLS, OC = SW ? BN / 2 : BN;
  constexpr int TP = WOUT + 4;                       // row pitch (floats) of a wave's output strip
  constexpr int EPI = NW * S * TP * 4 + BM * 4;
  constexpr int SM = NS * STAGE > EPI ? NS * STAGE : EPI;
  __shared__ __attribute__((aligned(128))) char smem[SM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // Each XCD takes a run of tiles, in blocks of eight rows of tiles: the tiles
  // that run at once on it share rows of x and of W in its L2.
  int mi, ni;
  {
    const int total = p.mt * p.nt, run = (total + kQ8Xcds - 1) / kQ8Xcds;
    const int at = blockIdx.x / kQ8Xcds, i = blockIdx.x % kQ8Xcds * run + at;
    if (at >= run || i >= total) return;             // uniform over the workgroup
    const int blk = i / (8 * p.nt), in = i - blk * 8 * p.nt, h = min(8, p.mt - blk * 8);
    mi = blk * 8 + in % h;
    ni = in / h;
  }
  const int m0 = mi * BM, o0 = ni * OC;              // first row and column of y
  const int nsl = (p.K + kQ8Slab - 1) / kQ8Slab;
  const uint32_t lds0 = lds_addr(smem);

  // this wave's copies of a slab: rows 16 (wave PW + q) + lane / 4 of [x tile; W tile]
  const int piece = (lane & 3) ^ (-(lane >> 4) & 3);    // of the row's four in a slab
  uint32_t off[PW];
  const int8_t* base[PW];                            // uniform
#pragma unroll
  for (int q = 0; q < PW; ++q) {
    const int r0 = (wave * PW + q) * 16;
    if (r0 < BM) {
      base[q] = p.x + (int64_t)m0 * p.ldx;
      off[q] = (uint32_t)min(r0 + (lane >> 2), p.M - 1 - m0) * (uint32_t)p.ldx + piece * 16;
    } else {
      const int w0 = r0 - BM, up = SW ? w0 / S & 1 : 0, row = SW ? w0 / (2 * S) * S + w0 % S : w0;
      base[q] = p.w + (int64_t)(up ? p.cols + o0 : o0) * p.ldw;
      off[q] = (uint32_t)min(row + (lane >> 2), p.cols - 1 - o0) * (uint32_t)p.ldw + piece * 16;
    }
  }
  // copy q of slab c
  auto copy = [&](int c, int q) {
    // (a piece past the row's end: the slab's first instead)
    const uint32_t back = c * kQ8Slab + piece * 16 < p.K ? 0u : piece * 16u;
    copy_to_lds(lds0 + c % NS * STAGE + (wave * PW + q) * 1024, off[q] - back, base[q] + (int64_t)c * kQ8Slab);
  };
  auto fetch = [&](int c) {
#pragma unroll
    for (int q = 0; q < PW; ++q) copy(c, q);
  };
  // bytes of x at or past K count as 0, in the pieces that this lane copied
  auto clear = [&](int c) {
    const int left = p.K - c * kQ8Slab - piece * 16;
    if (left < 16) {
#pragma unroll
      for (int q = 0; q < PW; ++q) {
        if ((wave * PW + q) * 16 >= BM) continue;
        u32x4* d = reinterpret_cast<u32x4*>(smem + c % NS * STAGE + (wave * PW + q) * 1024 + lane * 16);
        u32x4 v = *d;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = left - 4 * e;
          v[e] = n >= 4 ? v[e] : n <= 0 ? 0u : v[e] & ((1u << (8 * n)) - 1u);
        }
        *d = v;
      }
    }
  };

  typename F::Acc acc[RT][CT];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int e = 0; e < ACC; ++e) acc[i][t][e] = 0;
  const int r = lane % S, g = lane / S;
  int xo[KT], wo[KT];
#pragma unroll
  for (int s = 0; s < KT; ++s) {
    const int col = ((64 / S * s + g) ^ (-(r >> 2) & 3)) * 16;
    xo[s] = (wm * RT * S + r) * kQ8Slab + col;
    wo[s] = (BM + wn * CT * S + r) * kQ8Slab + col;
  }
  struct Set { u32x4 x[KT][RT], w[KT][CT]; };
  // operand j of slab c, in the products' order of k, x before W
  constexpr int OPS = KT * (RT + CT);
  auto read1 = [&](const char* b, int j, Set& q) {
    const int s = j / (RT + CT), i = j % (RT + CT);
    if (i < RT) q.x[s][i] = *reinterpret_cast<const u32x4*>(b + xo[s] + i * S * kQ8Slab);
    else q.w[s][i - RT] = *reinterpret_cast<const u32x4*>(b + wo[s] + (i - RT) * S * kQ8Slab);
  };
  auto read = [&](int c, Set& q) {
#pragma unroll
    for (int j = 0; j < OPS; ++j) read1(smem + c % NS * STAGE, j, q);
  };
  auto product = [&](const Set& q, int j) {
    const int s = j / (RT * CT), t = j / RT % CT, i = j % RT;
    acc[i][t] = F::mma(q.x[s][i], q.w[s][t], acc[i][t]);
  };
  // Slab c's products; STEADY: slab c + NS is one more to fetch.  Its copies and
  // the reads of slab c + 1 are spread over the products, the reads early.
  auto step = [&](auto steady, int c, const Set& cur, Set& nxt) {
    constexpr int PROD = KT * RT * CT, G = PROD < 8 ? PROD : 8, PG = PROD / G, RG = (OPS + G * 3 / 4 - 1) / (G * 3 / 4);
    if constexpr (decltype(steady)::value) {
      wait_copies<(NS - 2) * PW>();
      lds_barrier();
      const char* b = smem + (c + 1) % NS * STAGE;
#pragma unroll
      for (int g = 0; g < G; ++g) {
#pragma unroll
        for (int q = g * PW / G; q < (g + 1) * PW / G; ++q) copy(c + NS, q);
#pragma unroll
        for (int j = 0; j < RG; ++j)
          if (g * RG + j < OPS) read1(b, g * RG + j, nxt);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < PG; ++j) product(cur, g * PG + j);
        __builtin_amdgcn_sched_barrier(0);
      }
      return;
    }
    if (c + 1 < nsl) {                               // uniform
      wait_copies<0>();
      if (c + 2 == nsl && p.K % kQ8Slab) clear(c + 1);
      lds_barrier();
      read(c + 1, nxt);
    }
#pragma unroll
    for (int j = 0; j < KT * RT * CT; ++j) product(cur, j);
  };
  for (int c = 0; c < NS && c < nsl; ++c) fetch(c);
  if (nsl >= NS) wait_copies<(NS - 1) * PW>();
  else wait_copies<0>();
  if (nsl == 1 && p.K % kQ8Slab) clear(0);
  lds_barrier();
  Set a, b;
  read(0, a);
  int c = 0;
  for (; c + 1 + NS < nsl; c += 2) {
    step(BoolC<true>{}, c, a, b);
    step(BoolC<true>{}, c + 1, b, a);
  }
  if (c + NS < nsl) {                                // an odd one: the sets change places
    step(BoolC<true>{}, c, a, b);
    a = b;
    ++c;
  }
  for (; c < nsl; c += 2) {
    step(BoolC<false>{}, c, a, b);
    if (c + 1 < nsl) step(BoolC<false>{}, c + 1, b, a);
  }

  // A strip of S rows at a time leaves through this wave's part of LDS: lane (r,
  // g) writes its column of each tile, then holds 8 columns of a row.
  lds_barrier();
  float* xs = reinterpret_cast<float*>(smem + NW * S * TP * 4);
  for (int i = tid; i < BM; i += 64 * NW) xs[i] = p.xs[min(m0 + i, p.M - 1)];
  float ws[CT], bias[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const int n = SW ? (t & 1) * p.cols + min(o0 + wn * WOUT + t / 2 * S + r, p.cols - 1)
                     : min(o0 + wn * WOUT + t * S + r, p.cols - 1);
    ws[t] = p.ws[n];
    bias[t] = p.bias ? p.bias[n] : 0.0f;
  }
  __syncthreads();
  float* tr = reinterpret_cast<float*>(smem) + wave * S * TP;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int row0 = (wm * RT + i) * S;          // of the tile
    if (m0 + row0 >= p.M) break;                     // uniform
#pragma unroll
    for (int ii = 0; ii < ACC / 4; ++ii) {
      const f32x4 sx = *reinterpret_cast<const f32x4*>(xs + row0 + F::row(g, 4 * ii));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float* d = tr + F::row(g, 4 * ii + e) * TP + r;
        auto val = [&](int t) {
          const float v = (float)acc[i][t][4 * ii + e] * sx[e] * ws[t];
          return p.bias ? v + bias[t] : v;
        };
        if constexpr (SW) {
#pragma unroll
          for (int t = 0; t < CT; t += 2) d[t / 2 * S] = q8_swiglu(val(t), val(t + 1));
        } else {
#pragma unroll
          for (int t = 0; t < CT; ++t) d[t * S] = val(t);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int LR = WOUT / 8, RP = 64 / LR;       // lanes a row, rows a pass
#pragma unroll 1
    for (int q = 0; q < S / RP; ++q) {
      const int row = q * RP + lane / LR, col = lane % LR * 8;
      float v[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x4 f = *reinterpret_cast<const f32x4*>(tr + row * TP + col + 4 * e);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * e + j] = f[j];
      }
      const int m = m0 + row0 + row, n = o0 + wn * WOUT + col;
      if (m < p.M && n < p.cols) q8_out8(p, m, n, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

template <int S, int BM, int BN, int WM, int WN, int NS, int OCC, bool SW>
int q8_tile(Q8LinParams p, hipStream_t st) {
  constexpr int OC = SW ? BN / 2 : BN;
  p.mt = (p.M + BM - 1) / BM;
  p.nt = (p.cols + OC - 1) / OC;
  const int64_t total = (int64_t)p.mt * p.nt;
  if (total >= INT_MAX - 64 || (int64_t)8 * p.nt >= INT_MAX || !launch_fits(total + 8, 64 * WM * WN))
    return VNX_ERR_UNSUPPORTED;
  const unsigned wgs = (unsigned)((total + kQ8Xcds - 1) / kQ8Xcds * kQ8Xcds);
  hipLaunchKernelGGL((k_q8_tile<S, BM, BN, WM, WN, NS, OCC, SW>), dim3(wgs), dim3(64 * WM * WN), 0, st, p);
  VNX_LAUNCH_CHECK();
  return VNX_OK;
}

constexpr int kQ8Shapes = 8;

template <bool SW>
int q8_linear(const Q8LinParams& p, int force, hipStream_t st) {
  auto tiles = [&](int bm, int bn) {
    const int oc = SW ? bn / 2 : bn;
    return (int64_t)((p.M + bm - 1) / bm) * ((p.cols + oc - 1) / oc);
  };
  int shape = p.M <= 16 ? 0 : tiles(256, 256) >= 2 * device_cus() && p.M > 256 ? 3 : p.M > 128 ? 2 : 1;
  if (force) shape = force - 1;
  switch (shape) {
    case 0: return q8_direct<16, 1, 2, 4, 1, SW>(p, st);
    case 1: return q8_direct<32, 2, 2, 2, 1, SW>(p, st);
    case 2: return q8_tile<32, 128, 128, 2, 2, 4, 2, SW>(p, st);
    case 3: return q8_tile<16, 256, 256, 2, 2, 4, 1, SW>(p, st);
    case 4: return q8_tile<32, 256, 256, 2, 4, 4, 1, SW>(p, st);
    case 5: return q8_tile<16, 256, 256, 2, 4, 4, 1, SW>(p, st);
    case 6: return q8_tile<16, 128, 128, 2, 2, 4, 2, SW>(p, st);
    default: return q8_tile<16, 256, 256, 2, 4, 5, 1, SW>(p, st);
  }
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

int vnx_q8_linear(const vnx_q8_linear_args* a, void* stream) {
  if (!a || a->M < 0 || a->N < 0 || a->K < 1 || a->ldx < a->K || a->ldw < a->K) return VNX_ERR_INVALID_ARG;
  if (a->epilogue != VNX_EPI_NONE && a->epilogue != VNX_EPI_SWIGLU) return VNX_ERR_INVALID_ARG;
  const bool sw = a->epilogue == VNX_EPI_SWIGLU;
  const int64_t cols = sw ? a->N / 2 : a->N;
  if ((sw && (a->N % 2 || a->res)) || a->ldy < cols || (a->res && a->ldr < cols)) return VNX_ERR_INVALID_ARG;
  if (!q8_float(a->y_dtype) || (a->res && !q8_float(a->res_dtype))) return VNX_ERR_UNSUPPORTED;
  // rows and columns are numbered to the end of their last tile in 32 bits
  if (a->K > kQ8MaxK || a->M >= INT_MAX - 4096 || a->N >= INT_MAX - 4096) return VNX_ERR_UNSUPPORTED;
  if (a->force_shape < 0 || a->force_shape > kQ8Shapes) return VNX_ERR_UNSUPPORTED;
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
  Q8LinParams p{};
  p.x = a->x; p.w = a->w; p.xs = a->x_scale; p.ws = a->w_scale; p.bias = a->bias; p.res = a->res; p.y = a->y;
  p.ldx = a->ldx; p.ldw = a->ldw; p.ldr = a->ldr; p.ldy = a->ldy;
  p.M = (int)a->M; p.N = (int)a->N; p.K = (int)a->K; p.cols = (int)cols;
  p.res_dtype = a->res_dtype; p.y_dtype = a->y_dtype;
  const auto st = static_cast<hipStream_t>(stream);
  return sw ? q8_linear<true>(p, a->force_shape, st) : q8_linear<false>(p, a->force_shape, st);
}

}  // extern "C"
