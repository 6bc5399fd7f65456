// y = residual + act((x W^T) [* x_scale[m] * w_scale[n]] + bias) on the matrix cores: x [M, K], W [N, K], both K-contiguous, 16-bit
// operands (bf16; fp16 under MVIT_F16) or e4m3 with a scale for each row of either.  f32 accumulation throughout.
//
// Everything below counts K in BYTES: a 128-byte row piece is 64 16-bit or 128 8-bit values, and the matrix instructions take equal time
// for equal bytes (v_mfma_f32_16x16x32 and the twice as wide v_mfma_f32_32x32x64_f8f6f4), so that one pipeline serves both.
//
// The e4m3 matrix instructions (all four shapes alike) add the products of neighbouring k with some 13 bits below the largest of them:
// 448 * 448 + 18 * 18 comes out as 448 * 448 + 320, and a product of 16-bit-like operands is off by 1 to 5e-5 of its norm.  Under a 16-bit
// output's own rounding (2^-9, 2^-12) that is nothing, and mode F8 uses them; an f32 output (a residual stream) would keep it, so mode F8X
// widens the e4m3 values to 16 bits in registers (exact) for the 16-bit instructions, at half the rate.  Few rows are bound by reading
// W, not by the matrix cores, and always take F8X.
#pragma once
#include "common.hpp"
#include "../../include/miphei_hip.h"

namespace mvit_linear {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((address_space(3))) void* lds_ptr;

enum Mode { H16, F8, F8X };   // 16-bit operands; e4m3 on the e4m3 instructions; e4m3 widened to 16 bits

struct Args {
  const char *x, *w;
  const void *bias, *res;
  void *y, *pre;
  const float *xs, *ws;
  long long ldr;     // residual's row stride in elements
  unsigned ldx, ldw; // row strides in bytes
  int M, N, kb;      // kb: bytes of a row of x and W
  int act, bias_f32, y_f32, vec;   // vec: rows of y, pre and res start on 16 bytes and N % 8 == 0
};

constexpr unsigned OOB = 0x80000000u;   // beyond every descriptor's range: the load returns zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const char* p) {
  // uniform by construction; readfirstlane lets the compiler see it and keep the descriptor in scalar registers
  const unsigned long long v = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), 0, 0x7fffffff, 0x00020000);
}

// ---------------------------------------------------------------- epilogue arithmetic
// erf by Abramowitz & Stegun 7.1.26 (|error| <= 1.5e-7, below f32 rounding of 1 + erf): one exp, one reciprocal and seven
// multiply-adds where the library's erff takes about forty instructions -- at 64 lanes a cycle and CU that is what the epilogue costs.
__device__ __forceinline__ float half_erfc(float a) {   // erfc(a / sqrt 2) / 2 for a >= 0
  const float t = __builtin_amdgcn_rcpf(1.f + 0.23164188684f * a);   // p / sqrt 2, p = 0.3275911
  const float e = __builtin_amdgcn_exp2f(-0.72134752044f * a * a);   // exp(-a^2 / 2)
  return 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
}
__device__ __forceinline__ float normal_cdf(float z) {
  const float q = half_erfc(fabsf(z));
  return z >= 0.f ? 1.f - q : q;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504089f * z)); }
constexpr float TANH_K = 1.5957691216f;   // 2 sqrt(2 / pi): (1 + tanh u) / 2 = sigmoid(2 u)

template <int V>
__device__ __forceinline__ void activate(float (&v)[V], int act) {
  switch (act) {
    case MVIT_ACT_RELU:
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];   // (a NaN stays one, as the definition has it)
      break;
    case MVIT_ACT_SILU:
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = v[e] * sigmoid(v[e]);
      break;
    case MVIT_ACT_GELU:
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = v[e] * normal_cdf(v[e]);
      break;
    case MVIT_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = v[e] * sigmoid(TANH_K * (v[e] + 0.044715f * v[e] * v[e] * v[e]));
      break;
    default:
      break;
  }
}

__device__ __forceinline__ float value_of(const void* p, size_t i, bool f32) { return f32 ? ((const float*)p)[i] : bf2f(((const bf16_t*)p)[i]); }

// The end of 8 columns of one row: column constants cs (w_scale) and cb (bias) of the lane's columns
template <bool OP8>
__device__ __forceinline__ void finish8(const Args& p, float (&v)[8], int row, int col, const float (&cs)[8], const float (&cb)[8]) {
  if (row >= p.M || col >= p.N) return;
  if constexpr (OP8) {
    const float s = p.xs[row];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * s * cs[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += cb[e];
  const size_t o = (size_t)row * p.N + col, r = (size_t)row * p.ldr + col;
  if (p.vec) {
    if (!OP8 && p.pre)
      *(uint4*)((bf16_t*)p.pre + o) = make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7]));
    activate(v, p.act);
    if (p.y_f32) {
      if (p.res) {
        const float4 a = *(const float4*)((const float*)p.res + r), b = *(const float4*)((const float*)p.res + r + 4);
        v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w, v[4] += b.x, v[5] += b.y, v[6] += b.z, v[7] += b.w;
      }
      *(float4*)((float*)p.y + o) = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)((float*)p.y + o + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      if (p.res) {
        const uint4 a = *(const uint4*)((const bf16_t*)p.res + r);
        v[0] += lo16f(a.x), v[1] += hi16f(a.x), v[2] += lo16f(a.y), v[3] += hi16f(a.y);
        v[4] += lo16f(a.z), v[5] += hi16f(a.z), v[6] += lo16f(a.w), v[7] += hi16f(a.w);
      }
      *(uint4*)((bf16_t*)p.y + o) = make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7]));
    }
  } else {
    const int n = min(8, p.N - col);
    if (!OP8 && p.pre)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) ((bf16_t*)p.pre)[o + e] = f2bf(v[e]);
    activate(v, p.act);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) {
        if (p.res) v[e] += value_of(p.res, r + e, p.y_f32);
        if (p.y_f32)
          ((float*)p.y)[o + e] = v[e];
        else
          ((bf16_t*)p.y)[o + e] = f2bf(v[e]);
      }
  }
}
template <bool OP8>
__device__ __forceinline__ void column_constants(const Args& p, int col, float (&cs)[8], float (&cb)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = OP8 && col + e < p.N ? p.ws[col + e] : 0.f;
    cb[e] = p.bias && col + e < p.N ? value_of(p.bias, col + e, p.bias_f32) : 0.f;
  }
}

// 16 e4m3 values -> two fragments of 8 16-bit ones (order kept; exact)
__device__ __forceinline__ void widen(const i32x4& v, bf16x8 (&out)[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    i32x4 r;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int w = v[h * 2 + q];
#ifdef MVIT_F16
      r[q * 2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
      r[q * 2 + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
#else
      r[q * 2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
      r[q * 2 + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true));
#endif
    }
    out[h] = __builtin_bit_cast(bf16x8, r);
  }
}

// ---------------------------------------------------------------- tiles
// A block of WM x WN waves forms BM x BN of y.  K goes by in tiles of BKB bytes a row; NST of them live in LDS, filled by DMA
// (buffer_load ... lds, 16 bytes a lane), NST - 1 ahead of the one being multiplied.  LDS rows are BKB bytes; the 16-byte piece c of row r
// lies at place c ^ (r / (256 / BKB) mod pieces), which puts the 16 rows that a fragment read touches on all 64 banks once.
// The fragments of the next sub-step are read into registers while the current one's matrix instructions run; the hand-over of a
// K tile (this wave's reads are back, its DMA of the next tile has landed, barrier, refill of the tile just read) stands in front of the
// last sub-step's instructions.
template <int MODE, int BM, int BN, int WM, int WN, int BKB, int NST>
struct Tile {
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int WTM = BM / WM, WTN = BN / WN;
  static constexpr int FR = MODE == F8 ? 32 : 16;       // rows of a fragment
  static constexpr int TM = WTM / FR, TN = WTN / FR;
  static constexpr int NSUB = BKB / 64;                 // sub-steps: 64 bytes of K each
  static constexpr int PIECES = BKB / 16;
  static constexpr int ROWS_PER_DMA = 1024 / BKB;       // rows of one wave's DMA instruction
  static constexpr int A_DMA = BM / ROWS_PER_DMA / NW, B_DMA = BN / ROWS_PER_DMA / NW, LPT = A_DMA + B_DMA;
  static constexpr int STAGE = (BM + BN) * BKB;
  static constexpr int PLD = WTN + 4;                   // floats in a row of the epilogue panel
  static constexpr size_t LDS = (size_t)NST * STAGE;
  static_assert(A_DMA >= 1 && B_DMA >= 1 && TM >= 1 && TN >= 1, "tile too small");
  static_assert((size_t)NW * 16 * PLD * 4 <= LDS, "the panels fit the stages");
};

template <int MODE, int BM, int BN, int WM, int WN, int BKB, int NST>
__global__ __launch_bounds__(64 * WM * WN) void linear_tile(const Args p) {
  using T = Tile<MODE, BM, BN, WM, WN, BKB, NST>;
  constexpr bool OP8 = MODE != H16, WIDE = MODE == F8;   // WIDE: 32 x 32 instructions
  using frag = std::conditional_t<WIDE, i32x8, i32x4>;
  using acc_t = std::conditional_t<WIDE, f32x16, f32x4>;
  constexpr int AR = WIDE ? 16 : 4;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // block -> tile: blocks go to the eight XCDs in turn, so the ids of one XCD are put on one contiguous run of tiles, and runs go down
  // 8 rows of tiles before the next column: the ~32 to 64 blocks that share an L2 share rows of x and of W
  const int tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN, nt = tm * tn;
  int id;
  {
    const int q = nt >> 3, r = nt & 7, xcd = blockIdx.x & 7;
    id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (blockIdx.x >> 3);
  }
  const int per = 8 * tn, g0 = id / per * 8, gsz = min(tm - g0, 8), in = id % per;
  const int m0 = (g0 + in % gsz) * BM, n0 = in / gsz * BN;

  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x + (size_t)m0 * p.ldx), rw = make_rsrc(p.w + (size_t)n0 * p.ldw);
  // this lane's part of a wave's DMA instruction: one 16-byte piece of row `dr`, at place lane % PIECES
  const int dr = lane / T::PIECES, dp = lane % T::PIECES;
  unsigned off[T::LPT];
  int src_piece;
  {
    // the places repeat every 16 rows, and a wave's instructions are a multiple of 16 rows apart: one piece for all of them
    static_assert(T::NW * T::ROWS_PER_DMA % 16 == 0, "places repeat every 16 rows");
    src_piece = (dp ^ (((wave * T::ROWS_PER_DMA + dr) / (256 / BKB)) % T::PIECES)) * 16;
#pragma unroll
    for (int j = 0; j < T::LPT; ++j) {
      const bool a = j < T::A_DMA;
      const int row = ((a ? j : j - T::A_DMA) * T::NW + wave) * T::ROWS_PER_DMA + dr;
      const bool ok = a ? m0 + row < p.M : n0 + row < p.N;
      off[j] = ok ? (unsigned)row * (a ? p.ldx : p.ldw) + (unsigned)src_piece : OOB;
    }
  }
  auto issue = [&](int t, auto) __attribute__((always_inline)) {   // K tile t into its stage; beyond the end: zeros
    char* s = smem + (t % NST) * T::STAGE;
    const int k = t * BKB;
    const bool ok = k + src_piece < p.kb;
#pragma unroll
    for (int j = 0; j < T::LPT; ++j) {
      const bool a = j < T::A_DMA;
      char* to = s + (a ? 0 : BM * BKB) + ((a ? j : j - T::A_DMA) * T::NW + wave) * 1024;
      unsigned o = ok ? off[j] : OOB;
      asm volatile("" : "+v"(o));   // one unconditional instruction a piece: the waits count them
      if (a)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)to, 16, o, k, 0, 0);
      else
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)to, 16, o, k, 0, 0);
    }
  };

  // fragment addresses.  A lane holds piece lane / 16 (of the sub-step's four) of row lane % 16; F8: pieces 2 (lane / 32) and the next
  // of row lane % 32.  Which K values those are does not matter as long as x and W agree.
  const int fr = lane % T::FR, fh = lane / T::FR;
  auto read = [&](const char* base, int rows0, int s) __attribute__((always_inline)) {
    const int sw = (fr / (256 / BKB)) % T::PIECES;   // rows0 is a multiple of 16
    const char* row = base + (rows0 + fr) * BKB;
    if constexpr (WIDE) {
      const int c = s * 4 + fh * 2;
      const i32x4 lo = *(const i32x4*)(row + ((c ^ sw) << 4)), hi = *(const i32x4*)(row + (((c + 1) ^ sw) << 4));
      return (frag){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    } else {
      return *(const frag*)(row + (((s * 4 + fh) ^ sw) << 4));
    }
  };
  frag fa[2][T::TM], fb[2][T::TN];
  acc_t acc[T::TM][T::TN];
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int j = 0; j < T::TN; ++j)
#pragma unroll
      for (int r = 0; r < AR; ++r) acc[i][j][r] = 0.f;
  auto load = [&](int t, int s, int f) __attribute__((always_inline)) {
    const char* st = smem + (t % NST) * T::STAGE;
#pragma unroll
    for (int j = 0; j < T::TN; ++j) fb[f][j] = read(st + BM * BKB, wn * T::WTN + j * T::FR, s);
#pragma unroll
    for (int i = 0; i < T::TM; ++i) fa[f][i] = read(st, wm * T::WTM + i * T::FR, s);
  };
  auto multiply = [&](int f) __attribute__((always_inline)) {
    if constexpr (MODE == F8X) {
      bf16x8 b[T::TN][2];
#pragma unroll
      for (int j = 0; j < T::TN; ++j) widen(fb[f][j], b[j]);
#pragma unroll
      for (int i = 0; i < T::TM; ++i) {
        bf16x8 a[2];
        widen(fa[f][i], a);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < T::TN; ++j) acc[i][j] = mvit_mfma16(a[h], b[j][h], acc[i][j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int jj = 0; jj < T::TN; ++jj) {
          const int j = i & 1 ? T::TN - 1 - jj : jj;   // neighbours share an operand
          if constexpr (WIDE)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[f][i], fb[f][j], acc[i][j], 0, 0, 0, 0, 0, 0);
          else
            acc[i][j] = mvit_mfma16(__builtin_bit_cast(bf16x8, fa[f][i]), __builtin_bit_cast(bf16x8, fb[f][j]), acc[i][j], 0, 0, 0);
        }
    }
  };
  auto hand_over = [&](int t, auto tag) __attribute__((always_inline)) {   // tile t is read, tile t + 1 comes
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * T::LPT) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue(t + NST, tag);
  };

  const int nk = (p.kb + BKB - 1) / BKB;
#pragma unroll
  for (int t = 0; t < NST; ++t) issue(t, 0);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * T::LPT) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  load(0, 0, 0);
  if constexpr (T::NSUB == 2) {
    for (int t = 0; t < nk; ++t) {
      load(t, 1, 1);
      multiply(0);
      hand_over(t, 0);
      load(t + 1, 0, 0);
      multiply(1);
    }
  } else {
    for (int t = 0; t < nk; t += 2) {   // an odd last tile is followed by one of zeros
      hand_over(t, 0);
      load(t + 1, 0, 1);
      multiply(0);
      hand_over(t + 1, 0);
      load(t + 2, 0, 0);
      multiply(1);
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // nothing of anybody's is on its way to or from the stages
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");

  // ---- epilogue: 16 rows at a time through a panel of this wave's own, so that a lane ends up with 8 columns of one row
  float* panel = (float*)smem + wave * 16 * T::PLD;
  constexpr int LPR = T::WTN / 8, RPP = 64 / LPR;   // lanes a row, rows a pass
  const int pr = lane / LPR, pc = lane % LPR * 8;
  const int col = n0 + wn * T::WTN + pc;
  float cs[8], cb[8];
  column_constants<OP8>(p, col, cs, cb);
#pragma unroll
  for (int i = 0; i < T::TM; ++i)
#pragma unroll
    for (int h = 0; h < T::FR / 16; ++h) {
#pragma unroll
      for (int j = 0; j < T::TN; ++j)
#pragma unroll
        for (int r = 0; r < AR / (T::FR / 16); ++r) {
          const int row = WIDE ? (r >> 2) * 8 + fh * 4 + (r & 3) : fh * 4 + r;
          panel[row * T::PLD + j * T::FR + fr] = acc[i][j][(WIDE ? h * 8 : 0) + r];
        }
#pragma unroll
      for (int q = 0; q < 16 / RPP; ++q) {
        const float* s = panel + (q * RPP + pr) * T::PLD + pc;
        const float4 a = *(const float4*)s, b = *(const float4*)(s + 4);
        float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        finish8<OP8>(p, v, m0 + wm * T::WTM + i * T::FR + h * 16 + q * RPP + pr, col, cs, cb);
      }
    }
}

// ---------------------------------------------------------------- few rows
// M <= 16 MT: what counts is to have W on its way at once.  A block forms 16 columns of all rows; its 8 waves share K in pieces of
// 128 bytes a row (wave w takes pieces w, w + 8, ...), load their fragments straight from memory into registers -- W is read by nobody
// else -- and join through LDS in wave order.
template <bool OP8, int MT>
__global__ __launch_bounds__(512) void linear_rows(const Args p) {
  constexpr int NWV = 8, U = 4;   // U pieces in flight
  __shared__ float part[NWV][MT * 16][17];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, fr = lane & 15, fh = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x), rw = make_rsrc(p.w + (size_t)n0 * p.ldw);
  const unsigned wo = n0 + fr < p.N ? (unsigned)fr * p.ldw : OOB;
  unsigned xo[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xo[m] = m * 16 + fr < p.M ? (unsigned)(m * 16 + fr) * p.ldx : OOB;
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int np = (p.kb + 127) / 128;
  for (int k0 = wave; k0 < np; k0 += NWV * U) {
    i32x4 b[U][2], a[U][MT][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int k = (k0 + u * NWV) * 128 + fh * 32 + c * 16;
        const bool ok = k < p.kb;
        b[u][c] = __builtin_amdgcn_raw_buffer_load_b128(rw, ok ? wo + k : OOB, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m) a[u][m][c] = __builtin_amdgcn_raw_buffer_load_b128(rx, ok ? xo[m] + k : OOB, 0, 0);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (OP8) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            bf16x8 x[2], w[2];
            widen(a[u][m][c], x);
            widen(b[u][c], w);
            acc[m] = mvit_mfma16(x[0], w[0], acc[m], 0, 0, 0);
            acc[m] = mvit_mfma16(x[1], w[1], acc[m], 0, 0, 0);
          }
        } else {
          acc[m] = mvit_mfma16(__builtin_bit_cast(bf16x8, a[u][m][0]), __builtin_bit_cast(bf16x8, b[u][0]), acc[m], 0, 0, 0);
          acc[m] = mvit_mfma16(__builtin_bit_cast(bf16x8, a[u][m][1]), __builtin_bit_cast(bf16x8, b[u][1]), acc[m], 0, 0, 0);
        }
      }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][m * 16 + fh * 4 + r][fr] = acc[m][r];
  __syncthreads();
  for (int i = tid; i < MT * 16 * 2; i += 512) {   // 8 columns of a row each
    const int row = i >> 1, c0 = (i & 1) * 8, col = n0 + c0;
    if (row >= p.M || col >= p.N) continue;
    float v[8], cs[8], cb[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = part[0][row][c0 + e];
#pragma unroll
      for (int k = 1; k < NWV; ++k) v[e] += part[k][row][c0 + e];
    }
    column_constants<OP8>(p, col, cs, cb);
    finish8<OP8>(p, v, row, col, cs, cb);
  }
}

}  // namespace mvit_linear
