// y = residual + act((x W^T) [* x_scale[m] * w_scale[n]] + bias) on the matrix cores: x [M, K], W [N, K], both K-contiguous, 16-bit
// operands (bf16; fp16 under MVIT_F16) or e4m3 with a scale for each row of either.  f32 accumulation, but for what mode F8 does (below).
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
#include <type_traits>
#include <utility>
#include "common.hpp"
#include "../../include/miphei_hip.h"

namespace mvit_linear {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((address_space(3))) void* lds_ptr;
typedef __attribute__((address_space(3))) i16x4* lds_4x16;

// 16-bit operands; e4m3 on the e4m3 instructions; e4m3 widened to 16 bits; and the gradients' products, whose K axis goes along the rows of
// memory of an operand: dx = dz W (DX: W [K, N] as it lies) and dW = dz^T x (DW: dz [K, M] and x [K, N])
enum Mode { H16, F8, F8X, DX, DW };

struct Args {
  const char *x, *w;
  const void *bias, *res;
  void *y, *pre;
  const float *xs, *ws;
  long long ldr;     // residual's row stride in elements
  unsigned ldx, ldw; // row strides in bytes
  int M, N, kb;      // kb: bytes of a row of x and W
  int act, bias_f32;
  float act_lo;   // -inf, or 0 for relu
  int krows;         // DX, DW: rows of the operands whose rows are K
  int kper, splits;  // K tiles of a part of K, and parts; their products f32 [splits][M][N] where there is more than one:
  float* part;       // DX, DW: here, else in y (f32)
};

// What a tile kernel is compiled for besides its operands.  The epilogue is unrolled over the accumulators: with every activation and
// output in one kernel it was 9800 instructions, more than the instruction cache holds, and cost 3 us a tile instead of 1.
enum Act { A_CLIP, A_SILU, A_TANH, A_ERF, A_ANY };
// VEC: rows of y, pre and res start on 16 bytes and N % 8 == 0; else pieces go to odd addresses (global memory takes 16-byte accesses at any)
// and a row's last one by elements
template <bool OUT32, int ACT, bool VEC>
struct End {
  static constexpr bool out32 = OUT32, vec = VEC;
  static constexpr int act = ACT;
};

constexpr unsigned OOB = 0x80000000u;   // a descriptor's size, and so beyond its range: the load returns zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const char* p) {
  // uniform by construction; readfirstlane lets the compiler see it and keep the descriptor in scalar registers
  const unsigned long long v = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)(((unsigned long long)hi << 32) | lo), 0, (int)OOB, 0x00020000);
}

// ---------------------------------------------------------------- epilogue arithmetic
// erf by Abramowitz & Stegun 7.1.26 (|error| <= 1.5e-7, below f32 rounding of 1 + erf): one exp, one reciprocal and seven
// multiply-adds where the library's erff takes about forty instructions -- at 64 lanes a cycle and CU that is what the epilogue costs.
__device__ __forceinline__ float gauss(float z) { return __builtin_amdgcn_exp2f(-0.72134752044f * z * z); }   // exp(-z^2 / 2)
__device__ __forceinline__ float normal_cdf(float z, float e) {   // e = gauss(z)
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.23164188684f, fabsf(z), 1.f));   // p / sqrt 2, p = 0.3275911
  // erfc(|z| / sqrt 2) / 2: half of 7.1.26's coefficients
  const float q = e * t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f))));
  return z >= 0.f ? 1.f - q : q;
}
constexpr float LOG2E = 1.44269504089f;
__device__ __forceinline__ float sigmoid2(float u) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-u)); }   // of u / log2 e

constexpr float TANH_A = LOG2E * 1.5957691216f, TANH_B = TANH_A * 0.044715f;   // 2 sqrt(2 / pi), log2 e

// none and relu clip at act_lo (a NaN stays one); silu is z s(z), gelu_tanh z s(2 sqrt(2 / pi) (z + 0.044715 z^3)), as
// (1 + tanh u) / 2 = s(2 u) for the logistic function s; gelu is z Phi(z)
template <int ACT>
__device__ __forceinline__ float activated(const Args& p, float z) {
  if constexpr (ACT == A_CLIP) return __builtin_elementwise_maximum(z, p.act_lo);
  if constexpr (ACT == A_SILU) return z * sigmoid2(LOG2E * z);
  if constexpr (ACT == A_TANH) return z * sigmoid2(z * __builtin_fmaf(z * z, TANH_B, TANH_A));
  if constexpr (ACT == A_ERF) return z * normal_cdf(z, gauss(z));
  return p.act == MVIT_ACT_GELU        ? activated<A_ERF>(p, z)
         : p.act == MVIT_ACT_SILU      ? activated<A_SILU>(p, z)
         : p.act == MVIT_ACT_GELU_TANH ? activated<A_TANH>(p, z)
                                       : activated<A_CLIP>(p, z);
}

__device__ __forceinline__ float value_of(const void* p, size_t i, bool f32) { return f32 ? ((const float*)p)[i] : bf2f(((const bf16_t*)p)[i]); }

// A piece is what a lane finishes at once: 16 bytes of y, W = 8 columns of a row (4 where y is f32).
// Column constants of a piece: the weight's scales and the bias
template <bool OP8, int W>
struct Columns {
  float s[W], b[W];
  __device__ __forceinline__ void load(const Args& p, int col) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = min(col + e, p.N - 1);
      s[e] = OP8 ? p.ws[c] : 1.f;
      b[e] = p.bias ? value_of(p.bias, c, p.bias_f32) : 0.f;
    }
  }
};
// The residual's piece, raw: loaded ahead of use, because a load that is waited for behind stores waits for these too
template <class E>
__device__ __forceinline__ uint4 residual_piece(const Args& p, int row, int col) {
  uint4 u = make_uint4(0, 0, 0, 0);
  if (!p.res || row >= p.M || col >= p.N) return u;
  const char* at = (const char*)p.res + ((size_t)row * p.ldr + col) * (E::out32 ? 4 : 2);
  if constexpr (E::vec) return *(const uint4*)at;
  if (p.N - col >= (E::out32 ? 4 : 8)) {
    __builtin_memcpy(&u, at, 16);
  } else if constexpr (E::out32) {
    u.x = ((const uint32_t*)at)[0];
    if (p.N - col > 1) u.y = ((const uint32_t*)at)[1];
    if (p.N - col > 2) u.z = ((const uint32_t*)at)[2];
  } else {
    const bf16_t* h = (const bf16_t*)at;
    auto two = [&](int e) __attribute__((always_inline)) {
      return (e < p.N - col ? (uint32_t)h[e] : 0u) | (e + 1 < p.N - col ? (uint32_t)h[e + 1] << 16 : 0u);
    };
    u = make_uint4(two(0), two(2), two(4), two(6));
  }
  return u;
}
// BYTES of bits to `at`, the first `left` of 4-byte (WORDS) or 2-byte values of them where that is fewer
template <class E, bool WORDS, int BYTES>
__device__ __forceinline__ void put(void* at, const uint32_t (&u)[BYTES / 4], int left) {
  if constexpr (E::vec) {
    if constexpr (BYTES == 16)
      *(uint4*)at = make_uint4(u[0], u[1], u[2], u[3]);
    else
      *(uint2*)at = make_uint2(u[0], u[1]);
  } else if (left >= BYTES / (WORDS ? 4 : 2)) {
    __builtin_memcpy(at, u, BYTES);
  } else {
#pragma unroll
    for (int e = 0; e < BYTES / (WORDS ? 4 : 2); ++e)
      if (e < left) {
        if constexpr (WORDS)
          ((uint32_t*)at)[e] = u[e];
        else
          ((bf16_t*)at)[e] = (bf16_t)(e & 1 ? u[e / 2] >> 16 : u[e / 2]);
      }
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7]));
}

// The end of a piece but for its store: v (products, times their row's scale) -> the bits of y
template <bool OP8, class E, int W>
__device__ __forceinline__ uint4 finish(const Args& p, float (&v)[W], int row, int col, const Columns<OP8, W>& c, const uint4& res) {
  static_assert(W == (E::out32 ? 4 : 8), "16 bytes of y");
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = OP8 ? __builtin_fmaf(v[e], c.s[e], c.b[e]) : v[e] + c.b[e];
  // (kept in 16 bits also beside an f32 y: what comes of it, dz, is rounded to the operands' 16 bits for the matrix instructions anyway, and f32 would
  // double what the forward pass writes and the backward pass reads again)
  if (!OP8 && p.pre && row < p.M && col < p.N) {
    uint32_t u[W / 2];
#pragma unroll
    for (int e = 0; e < W / 2; ++e) u[e] = pack2bf(v[2 * e], v[2 * e + 1]);
    put<E, false, W * 2>((bf16_t*)p.pre + (size_t)row * p.N + col, u, p.N - col);
  }
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = activated<E::act>(p, v[e]);
  if constexpr (W == 4) {
    if (p.res) v[0] += __uint_as_float(res.x), v[1] += __uint_as_float(res.y), v[2] += __uint_as_float(res.z), v[3] += __uint_as_float(res.w);
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    if (p.res) {
      v[0] += lo16f(res.x), v[1] += hi16f(res.x), v[2] += lo16f(res.y), v[3] += hi16f(res.y);
      v[4] += lo16f(res.z), v[5] += hi16f(res.z), v[6] += lo16f(res.w), v[7] += hi16f(res.w);
    }
    return pack8(v);
  }
}
template <class E>
__device__ __forceinline__ void store_piece(const Args& p, int part, int row, int col, const uint4& u) {   // of part `part` of K
  if (row < p.M && col < p.N) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    put<E, E::out32, 16>((char*)p.y + (((size_t)part * p.M + row) * p.N + col) * (E::out32 ? 4 : 2), w, p.N - col);
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
// WM x WN waves form BM x BN of y at a time.  K goes by in tiles of 128 bytes a row (BKB); NST of them live in LDS, filled by DMA
// (buffer_load ... lds, 16 bytes a lane).  The 16-byte piece c of LDS row r lies at place c ^ x_place(r) (w_place(r) for W), which
// puts the 16 rows that a fragment read touches on all 64 banks once.
//  * The fragments of the next sub-step (64 bytes of K) are read into registers behind the current one's matrix instructions; the
//    hand-over of a K tile (this wave's reads are back, its DMA of the next tile has landed, barrier) stands in front of the last
//    sub-step, and the refill of the tile just read is issued behind it.
//  * Blocks are persistent: a block walks output tiles, and the refill runs on into the next output tile's K tiles, so that neither
//    its first loads nor a launch stand between two tiles; they land while the epilogue runs.
//  * The products are formed as W x^T: a lane then holds groups of 4 consecutive columns of one row of y.  Which row of W is which row of
//    a fragment is free, and is chosen so that a lane's groups make up whole pieces of 16 bytes and the lanes of a row 64 bytes in a
//    line: y leaves from the registers.  (Through panels in LDS, whole lines a store, the epilogue took 6 to 8 us of a 256 x 256 tile:
//    a chain of LDS writes, reads and waits with two waves a SIMD to hide it.)
//  * An operand whose rows are K (DX, DW) lies in LDS as it does in memory, 64 rows of the tile's columns, and is turned by the transposing
//    LDS reads (ds_read_b64_tr_b16: 16 lanes read 4 rows of 16 columns, a lane gets the 4 values of its column), two for a fragment.
//    (With transposed copies of x, W and dz in memory forward and
//    backward of [5264, 1536] x [4096, 1536], gelu, took 266 us instead of 231.)
constexpr int BKB = 128;

// Layout of 64 rows of BN columns: the 16-byte piece c of row k at place c ^ fold(k).  What 32 lanes read at once -- 32 bytes each of rows
// k .. k + 3 and k + 8 .. k + 11 -- falls on all 64 banks once (rows of 128 bytes: two rows span them, so two bits of k are enough).
template <int COLS>
struct KRows {
  static constexpr int RL = COLS * 2, PER_DMA = 1024 / RL;   // bytes of a row, rows of a wave's DMA instruction
  static constexpr bool ok(int waves) { return (RL & (RL - 1)) == 0 && RL >= 128 && RL <= 512 && waves * PER_DMA % 16 == 0; }
  static __device__ __forceinline__ int fold(int k) { return RL == 128 ? (k & 2) | ((k >> 1) & 4) : (k & 3) << 1 | (k & 8); }
  // (__restrict: nothing else writes here in this function's scope.  DMA into LDS is waited for by hand, a stage at a time; without the word
  // the compiler waits for all that is in flight in front of every one of these reads, as it does not for ordinary ones.)
  static __device__ __forceinline__ i32x2 turned(lds_4x16 __restrict p) { return __builtin_bit_cast(i32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p)); }
  // 16 columns from `col` on (a multiple of 16), 32 rows from 32 s on: lane l gets column l % 16, rows 8 (l / 16) .. + 7
  static __device__ __forceinline__ i32x4 read(char* base, int col, int s) {
    const int lane = threadIdx.x & 63, i = lane & 15, k = (lane >> 4) * 8 + (i >> 2);
    const int at = k * RL + ((((i & 3) >> 1) ^ fold(k)) << 4) + (i & 1) * 8;
    char* p = base + s * 32 * RL + (at ^ (col * 2));
    const i32x2 a = turned((lds_4x16)p), b = turned((lds_4x16)(p + 4 * RL));
    return (i32x4){a.x, a.y, b.x, b.y};
  }
};

template <int MODE, int BM, int BN, int WM, int WN, int NST>
struct Tile {
  static constexpr int NW = WM * WN, NT = NW * 64;
  static constexpr int WTM = BM / WM, WTN = BN / WN;
  static constexpr int FR = MODE == F8 ? 32 : 16;       // rows of a fragment
  static constexpr int TM = WTM / FR, TN = WTN / FR;
  static constexpr int PIECES = BKB / 16;
  static constexpr int ROWS_PER_DMA = 1024 / BKB;       // rows of one wave's DMA instruction
  static constexpr int A_DMA = BM / ROWS_PER_DMA / NW, B_DMA = BN / ROWS_PER_DMA / NW, LPT = A_DMA + B_DMA;
  static constexpr bool XR = MODE == DW, WR = MODE == DX || MODE == DW;   // K along the rows of x, of W
  static constexpr int STAGE = (BM + BN) * BKB;
  static constexpr int TABLE = MODE == F8 ? 2 * WTN : 0;   // floats of a wave's table of column constants
  static constexpr size_t LDS = (size_t)NST * STAGE + (size_t)NW * TABLE * 4;
  static constexpr int BLOCKS_PER_CU = 160 * 1024 / LDS < 512 / NT ? 160 * 1024 / LDS : 512 / NT;   // two waves a SIMD
  static_assert(A_DMA >= 1 && B_DMA >= 1 && TM >= 1 && TN >= 1 && WTN <= 64, "sizes of a wave");
  static_assert(NW * ROWS_PER_DMA % 32 == 0, "LDS places repeat every 32 rows");
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static_assert(!WR || (TN % 2 == 0 && KRows<BN>::ok(NW) && (!XR || KRows<BM>::ok(NW))), "K along the rows");
};

template <int MODE, class E, int BM, int BN, int WM, int WN, int NST>
__global__ __launch_bounds__(64 * WM * WN, 2) void linear_tile(const Args p) {
  using T = Tile<MODE, BM, BN, WM, WN, NST>;
  constexpr bool OP8 = MODE == F8 || MODE == F8X, WIDE = MODE == F8;   // WIDE: 32 x 32 instructions
  using frag = std::conditional_t<WIDE, i32x8, i32x4>;
  using acc_t = std::conditional_t<WIDE, f32x16, f32x4>;
  constexpr int AR = WIDE ? 16 : 4, NR = T::TM + T::TN;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN, nt = tm * tn;
  const int nk = (p.kb + BKB - 1) / BKB;
  // K in parts: number v is part v / nt of tile v % nt, K tiles [first, end)
  constexpr bool PARTS = T::WR || (E::out32 && E::act == A_CLIP);
  const int nv = PARTS ? nt * p.splits : nt;
  auto first_k = [&](int v) __attribute__((always_inline)) { return PARTS ? v / nt * p.kper : 0; };
  auto end_k = [&](int v) __attribute__((always_inline)) { return PARTS ? min(nk, (v / nt + 1) * p.kper) : nk; };

  // tile number -> place: blocks go to the eight XCDs in turn, so the numbers of one XCD are put on one contiguous run of tiles, and runs
  // go down 8 rows of tiles before the next column: the blocks that share an L2 share rows of x and of W
  auto place = [&](int v, int& m0, int& n0) __attribute__((always_inline)) {
    if constexpr (PARTS) v %= nt;
    const int q = nt >> 3, r = nt & 7, xcd = v & 7;
    const int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (v >> 3);
    const int per = 8 * tn, g0 = id / per * 8, gsz = min(tm - g0, 8), in = id % per;
    m0 = (g0 + in % gsz) * BM, n0 = in / gsz * BN;
  };

  // the place of piece c of LDS row r is c ^ x_place(r), c ^ w_place(r): 16 lanes read 16 rows, for x 16 in a line, for W (H16 with 16-bit
  // y) those of bit 2 alike among 32
  constexpr bool PAIRED = MODE == H16 && !E::out32;
  auto x_place = [](int r) __attribute__((always_inline)) { return (r >> 1) & 7; };
  auto w_place = [](int r) __attribute__((always_inline)) { return PAIRED ? ((r >> 1) & 1) | ((r >> 2) & 6) : (r >> 1) & 7; };

  // ---- the DMA side: output tile `dv`, K tile `dk` of it come next
  const int dr = lane / T::PIECES;   // this lane's part of a wave's DMA instruction: one 16-byte piece of row `dr`
  const int drow = wave * T::ROWS_PER_DMA + dr;   // (further instructions of the wave are a multiple of 32 rows on: the same places)
  // (K along the rows: this lane's row kx, kw of the tile's 64 and its piece of it, for every instruction the next `step` rows)
  constexpr int XL = KRows<BM>::RL, WL = KRows<BN>::RL, x_step = T::NW * 1024 / XL, w_step = T::NW * 1024 / WL;
  const int kx = wave * (1024 / XL) + lane / (XL / 16), kw = wave * (1024 / WL) + lane / (WL / 16);
  const int x_piece = (T::XR ? lane % (XL / 16) ^ KRows<BM>::fold(kx) : lane % T::PIECES ^ x_place(drow)) * 16;
  const int w_piece = (T::WR ? lane % (WL / 16) ^ KRows<BN>::fold(kw) : lane % T::PIECES ^ w_place(drow)) * 16;
  __amdgpu_buffer_rsrc_t rx, rw;
  unsigned off[T::LPT];
  int dv = blockIdx.x, dk = 0, dk_end = 0;
  const char *bx = p.x, *bw = p.w;   // where the K tile's rows begin (K along the rows)
  auto aim = [&](auto) __attribute__((always_inline)) {
    int m0 = 0, n0 = 0;
    const bool any = dv < nv;
    dk = 0, dk_end = nk;
    if (any) place(dv, m0, n0), dk = first_k(dv), dk_end = end_k(dv);
    bx = p.x + (T::XR ? (size_t)m0 * 2 + (size_t)p.ldx * (BKB / 2) * dk : (size_t)m0 * p.ldx);
    bw = p.w + (T::WR ? (size_t)n0 * 2 + (size_t)p.ldw * (BKB / 2) * dk : (size_t)n0 * p.ldw);
    rx = make_rsrc(bx), rw = make_rsrc(bw);
#pragma unroll
    for (int j = 0; j < T::LPT; ++j) {
      const bool a = j < T::A_DMA;
      const int row = ((a ? j : j - T::A_DMA) * T::NW + wave) * T::ROWS_PER_DMA + dr;
      if (a ? T::XR : T::WR) {
        const bool in = any && (a ? m0 + x_piece / 2 < p.M : n0 + w_piece / 2 < p.N);
        off[j] = in ? (unsigned)(a ? kx + j * x_step : kw + (j - T::A_DMA) * w_step) * (a ? p.ldx : p.ldw) + (unsigned)(a ? x_piece : w_piece) : OOB;
      } else {
        const bool in = any && (a ? m0 + row < p.M : n0 + row < p.N);
        off[j] = in ? (unsigned)row * (a ? p.ldx : p.ldw) + (unsigned)(a ? x_piece : w_piece) : OOB;
      }
    }
  };
  auto issue = [&](int stage, int j, auto) __attribute__((always_inline)) {   // piece j of the next K tile; beyond K or M, N: zeros
    const bool a = j < T::A_DMA;
    char* to = smem + stage * T::STAGE + (a ? 0 : BM * BKB) + ((a ? j : j - T::A_DMA) * T::NW + wave) * 1024;
    const bool rows = a ? T::XR : T::WR;
    const int k = rows ? 0 : dk * BKB;
    const bool in = rows ? (a ? kx + j * x_step : kw + (j - T::A_DMA) * w_step) < p.krows - dk * (BKB / 2) : k + (a ? x_piece : w_piece) < p.kb;
    unsigned o = in ? off[j] : OOB;
    asm volatile("" : "+v"(o));   // one unconditional instruction a piece: the waits count them
    if (a)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_ptr)to, 16, o, k, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (lds_ptr)to, 16, o, k, 0, 0);
  };
  auto advance = [&]() __attribute__((always_inline)) {
    if (++dk == dk_end) {
      dv += gridDim.x;
      aim(0);
    } else {
      if constexpr (T::XR) rx = make_rsrc(bx += (size_t)p.ldx * (BKB / 2));
      if constexpr (T::WR) rw = make_rsrc(bw += (size_t)p.ldw * (BKB / 2));
    }
  };

  // ---- fragments.  A lane holds piece lane / 16 (of the sub-step's four) of row lane % 16; F8: pieces 2 (lane / 32) and the next of row
  // lane % 32.  Which K values those are does not matter as long as x and W agree.
  const int fr = lane % T::FR, fh = lane / T::FR;
  frag fa[2][T::TM], fb[2][T::TN];
  auto read = [&](const char* base, int row, int place, int s) __attribute__((always_inline)) {
    const char* at = base + row * BKB;
    if constexpr (WIDE) {
      const int c = s * 4 + fh * 2;
      const i32x4 lo = *(const i32x4*)(at + ((c ^ place) << 4)), hi = *(const i32x4*)(at + (((c + 1) ^ place) << 4));
      return (frag){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    } else {
      return *(const frag*)(at + (((s * 4 + fh) ^ place) << 4));
    }
  };
  // row of W (of the wave's WTN) that is row fr of fragment j.  A lane's results are, by row of the fragment, 4 fh .. + 3 (F8: + 8 g):
  //   H16, 16-bit y: of fragments 2 q and 2 q + 1 together the 8 columns from 32 q + 8 fh on
  //   F8:            of groups 2 k and 2 k + 1 together the 8 columns from 32 j + 16 k + 8 fh on
  //   f32 y:         the 4 columns from 16 j + 4 fh on
  const int w_row = PAIRED ? (fr >> 2) * 8 + (fr & 3) : WIDE ? (fr & 0x13) | (fr & 4) << 1 | (fr & 8) >> 1 : fr;
  auto w_row_of = [&](int j) __attribute__((always_inline)) { return w_row + (PAIRED ? (j >> 1) * 32 + (j & 1) * 4 : j * T::FR); };
  // fragment r of sub-step s of a stage into set f, in the order the products take them: x 0, all of W, x 1 ...
  auto load1 = [&](int stage, int s, int f, int r) __attribute__((always_inline)) {
    char* st = smem + stage * T::STAGE;
    const int i = r ? r - T::TN : 0;
    if (r >= 1 && r <= T::TN) {   // (the places of rows 32 or 4 apart agree where w_row_of() steps by them)
      if constexpr (T::WR)
        fb[f][r - 1] = KRows<BN>::read(st + BM * BKB, wn * T::WTN + (r - 1) * 16, s);
      else
        fb[f][r - 1] = read(st + BM * BKB + wn * T::WTN * BKB, w_row_of(r - 1), w_place(w_row), s);
    } else {
      if constexpr (T::XR)
        fa[f][i] = KRows<BM>::read(st, wm * T::WTM + i * 16, s);
      else
        fa[f][i] = read(st + wm * T::WTM * BKB, fr + i * T::FR, x_place(fr), s);
    }
  };
  acc_t acc[T::TM][T::TN];
  // One sub-step: the products of fragment set f, and behind each of them its share of the reads of the next set (sub-step s of a stage)
  // and of the DMA into stage d (d < 0: none).  Left to itself the compiler gathers the reads into bursts that the next products wait for.
  auto sub_step = [&](int f, int stage, int s, int d, auto dma) __attribute__((always_inline)) {
    constexpr int ND = decltype(dma)::value ? T::LPT : 0;
    auto behind = [&](int m, int NM) __attribute__((always_inline)) {
#pragma unroll
      for (int r = m * NR / NM; r < (m + 1) * NR / NM; ++r) load1(stage, s, f ^ 1, r);
#pragma unroll
      for (int j = m * ND / NM; j < (m + 1) * ND / NM; ++j) issue(d, j, 0);
      __builtin_amdgcn_sched_barrier(0);
    };
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
          for (int j = 0; j < T::TN; ++j) {
            acc[i][j] = mvit_mfma16(b[j][h], a[h], acc[i][j], 0, 0, 0);
            behind((i * 2 + h) * T::TN + j, T::TM * T::TN * 2);
          }
      }
    } else {
#pragma unroll
      for (int i = 0; i < T::TM; ++i)
#pragma unroll
        for (int jj = 0; jj < T::TN; ++jj) {
          const int j = i & 1 ? T::TN - 1 - jj : jj;   // neighbours share an operand
          if constexpr (WIDE)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[f][j], fa[f][i], acc[i][j], 0, 0, 0, 0, 0, 0);
          else
            acc[i][j] = mvit_mfma16(__builtin_bit_cast(bf16x8, fb[f][j]), __builtin_bit_cast(bf16x8, fa[f][i]), acc[i][j], 0, 0, 0);
          behind(i * T::TN + jj, T::TM * T::TN);
        }
    }
  };
  auto barrier = [&]() __attribute__((always_inline)) {   // this wave's LDS reads are back: behind it others' DMA may overwrite what they read
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  aim(0);
#pragma unroll
  for (int t = 0; t < NST; ++t) {
#pragma unroll
    for (int j = 0; j < T::LPT; ++j) issue(t, j, 0);
    advance();
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 1) * T::LPT) : "memory");
  barrier();
#pragma unroll
  for (int r = 0; r < NR; ++r) load1(0, 0, 0, r);

  int stage = 0, landed = 0;   // landed: K tiles behind the current one whose DMA has been waited for already
  for (int v = blockIdx.x; v < nv; v += gridDim.x) {
#pragma unroll
    for (int i = 0; i < T::TM; ++i)
#pragma unroll
      for (int j = 0; j < T::TN; ++j)
#pragma unroll
        for (int r = 0; r < AR; ++r) acc[i][j][r] = 0.f;
    for (int t = first_k(v), end = end_k(v); t < end; ++t) {
      const int next = stage + 1 == NST ? 0 : stage + 1;
      sub_step(0, stage, 1, -1, std::false_type{});
      if (landed <= 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NST - 2) * T::LPT) : "memory");
      --landed;
      barrier();
      sub_step(1, next, 0, stage, std::true_type{});
      advance();
      stage = next;
    }
    // ---- epilogue, from the registers.  The DMA of the next tile's first K tiles is waited for in front of its stores: loads, DMA and
    // stores share one counter, and behind the stores it could not be told any more.
    int m0, n0;
    place(v, m0, n0);
    if constexpr (T::WR) {
      // nothing to add: y's 16 bits as they are.  A lane has 4 columns of two neighbouring fragments; traded with the next 16 lanes they make 8
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      landed = NST - 1;
      if (p.splits > 1) {
        float* part = p.part + (size_t)(v / nt) * p.M * p.N;
#pragma unroll
        for (int i = 0; i < T::TM; ++i) {
          const int row = m0 + wm * T::WTM + i * 16 + fr;
#pragma unroll
          for (int j = 0; j < T::TN; ++j) {
            const int col = n0 + wn * T::WTN + j * 16 + fh * 4;
            if (row < p.M && col < p.N) *(f32x4*)(part + (size_t)row * p.N + col) = acc[i][j];
          }
        }
      } else
#pragma unroll
      for (int i = 0; i < T::TM; ++i) {
#pragma unroll
        for (int j = 0; j < T::TN; j += 2) {
          const acc_t &c0 = acc[i][j], &c1 = acc[i][j + 1];
          const auto lo = __builtin_amdgcn_permlane16_swap(pack2bf(c0[0], c0[1]), pack2bf(c1[0], c1[1]), false, false);
          const auto hi = __builtin_amdgcn_permlane16_swap(pack2bf(c0[2], c0[3]), pack2bf(c1[2], c1[3]), false, false);
          store_piece<E>(p, 0, m0 + wm * T::WTM + i * 16 + fr, n0 + wn * T::WTN + (j + (fh & 1)) * 16 + (fh >> 1) * 8, make_uint4(lo[0], hi[0], lo[1], hi[1]));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      constexpr int W = E::out32 ? 4 : 8, NP = T::TN * AR / W;   // pieces of a lane in one row of fragments
      const int row0 = m0 + wm * T::WTM + fr, col0 = n0 + wn * T::WTN, part = PARTS ? v / nt : 0;
      auto col_of = [&](int q) __attribute__((always_inline)) {
        return col0 + (PAIRED ? q * 32 + fh * 8 : WIDE ? (q >> 1) * 32 + (q & 1) * 16 + fh * 8 : q * 16 + fh * 4);
      };
      // column constants: in registers, or (F8: 64 of them, beside 128 accumulators) in a table of the wave's own
      Columns<OP8, W> cols[NP];
      float rs[T::TM];
      float* table = (float*)(smem + NST * T::STAGE) + wave * T::TABLE;
      if constexpr (WIDE) {
        const int c = min(col0 + lane, p.N - 1);
        if (lane < T::WTN) {
          table[lane] = p.ws[c];
          table[T::WTN + lane] = p.bias ? value_of(p.bias, c, p.bias_f32) : 0.f;
        }
      } else {
#pragma unroll
        for (int q = 0; q < NP; ++q) cols[q].load(p, col_of(q));
      }
#pragma unroll
      for (int i = 0; i < T::TM; ++i) rs[i] = OP8 ? p.xs[min(row0 + i * T::FR, p.M - 1)] : 1.f;
      uint4 res[2][NP];   // of this row of fragments and the next
#pragma unroll
      for (int q = 0; q < NP; ++q) res[0][q] = residual_piece<E>(p, row0, col_of(q));
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      landed = NST - 1;
#pragma unroll
      for (int i = 0; i < T::TM; ++i) {
        const int row = row0 + i * T::FR;
        if (i + 1 < T::TM)
#pragma unroll
          for (int q = 0; q < NP; ++q) res[(i + 1) & 1][q] = residual_piece<E>(p, row + T::FR, col_of(q));
        uint4 out[NP];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          if constexpr (WIDE) {
            const float* t = table + (col_of(q) - col0);
#pragma unroll
            for (int e = 0; e < W; ++e) cols[q].s[e] = t[e], cols[q].b[e] = t[T::WTN + e];
          }
          float o[W];
#pragma unroll
          for (int e = 0; e < W; ++e)
            o[e] = (WIDE ? acc[i][q >> 1][(q & 1) * 8 + e] : PAIRED ? acc[i][q * 2 + (e >> 2)][e & 3] : acc[i][q][e & 3]) * (OP8 ? rs[i] : 1.f);
          out[q] = finish<OP8, E, W>(p, o, row, col_of(q), cols[q], res[i & 1][q]);
          if constexpr (!WIDE) store_piece<E>(p, part, row, col_of(q), out[q]);
        }
        if constexpr (WIDE) {
          // two lanes of a row, 32 bytes a store: trade pieces between rows r and r + 16, so that four lanes have 64 bytes of one row
#pragma unroll
          for (int q = 0; q < NP; q += 2) {
            uint32_t *a = (uint32_t*)&out[q], *b = (uint32_t*)&out[q + 1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const auto s = __builtin_amdgcn_permlane16_swap(a[e], b[e], false, false);
              a[e] = s[0], b[e] = s[1];
            }
            const int r = row - fr + (lane & 15), c = col0 + (q >> 1) * 32 + ((lane >> 4) & 1) * 16 + (lane >> 5) * 8;
            store_piece<E>(p, part, r, c, out[q]);
            store_piece<E>(p, part, r + 16, c, out[q + 1]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);   // (rows of fragments pulled together cost registers that are not there)
      }
    }
    // the next tile's first fragments again: read once more, they need no registers during the epilogue
#pragma unroll
    for (int r = 0; r < NR; ++r) load1(stage, 0, 0, r);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (the zeros behind the last tile: nothing of this block's is on its way to LDS)
}

// ---------------------------------------------------------------- few rows
// M <= 16 MT: what counts is to have W on its way at once.  A block forms 16 columns of all rows; its 8 waves share K in pieces of
// 128 bytes a row (wave w takes pieces w, w + 8, ...), load their fragments straight from memory into registers -- W is read by nobody
// else -- and join through LDS in wave order.
template <bool OP8, class E, int MT>
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
  const int part_k = blockIdx.y, np = min((p.kb + 127) / 128, (part_k + 1) * p.kper);   // this block's part of K: pieces [kper part_k, np)
  for (int k0 = part_k * p.kper + wave; k0 < np; k0 += NWV * U) {
    i32x4 b[U][2], a[U][MT][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int k = (k0 + u * NWV) * 128 + fh * 32 + c * 16;
        const bool ok = k < p.kb && k0 + u * NWV < np;
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
  constexpr int W = E::out32 ? 4 : 8;
  for (int i = tid; i < MT * 16 * (16 / W); i += 512) {   // a piece each
    const int row = i / (16 / W), c0 = i % (16 / W) * W, col = n0 + c0;
    if (row >= p.M || col >= p.N) continue;
    Columns<OP8, W> cols;
    cols.load(p, col);
    const uint4 res = residual_piece<E>(p, row, col);
    float v[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      v[e] = part[0][row][c0 + e];
#pragma unroll
      for (int k = 1; k < NWV; ++k) v[e] += part[k][row][c0 + e];
      if constexpr (OP8) v[e] *= p.xs[row];
    }
    store_piece<E>(p, part_k, row, col, finish<OP8, E, W>(p, v, row, col, cols, res));
  }
}

}  // namespace mvit_linear
