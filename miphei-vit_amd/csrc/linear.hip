// The linear layer with activation and residual in its epilogue (kernels in linear_kernel.hpp), 16-bit and 8-bit operands.
#include <cmath>
#include "column_sums.hpp"
#include "linear_kernel.hpp"

using namespace mvit_linear;

namespace mvit_linear {
template <int MODE, bool OUT32>
int dispatch(const Args& a, bool vec, hipStream_t s);   // linear_launch.hpp
template <int MODE>
int dispatch_parts(const Args& a, bool vec, int kind, hipStream_t s);
template <int MODE>
int dispatch_grad(const Args& a, int tile, hipStream_t s);
extern template int dispatch<H16, false>(const Args&, bool, hipStream_t);
extern template int dispatch<H16, true>(const Args&, bool, hipStream_t);
extern template int dispatch<F8, false>(const Args&, bool, hipStream_t);
extern template int dispatch<F8X, true>(const Args&, bool, hipStream_t);
extern template int dispatch_parts<H16>(const Args&, bool, int, hipStream_t);
extern template int dispatch_parts<F8X>(const Args&, bool, int, hipStream_t);
extern template int dispatch_grad<DX>(const Args&, int, hipStream_t);
extern template int dispatch_grad<DW>(const Args&, int, hipStream_t);
}  // namespace mvit_linear

namespace {

constexpr int MAX_M = 1 << 30, MAX_N = 1 << 24, MAX_K = 1 << 29;   // tile numbers, grids and bytes of K stay in 31 bits

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 0: go on, 1: nothing to do, < 0: refused.  es: bytes of an operand's value.
int check(const mvit_linear_args* g, int es, Args& a, bool& vec) {
  if (!g || g->M < 0 || g->M > MAX_M || g->N <= 0 || g->N > MAX_N || g->K <= 0) return MVIT_EINVAL;
  if (g->M == 0) return 1;   // (an empty tensor has no address)
  if (!g->x || !g->w || !g->y) return MVIT_EINVAL;
  if (g->act < MVIT_ACT_NONE || g->act > MVIT_ACT_GELU_TANH) return MVIT_EINVAL;
  const long long kb = (long long)g->K * es, lx = g->ldx * es, lw = g->ldw * es;
  // 16-byte pieces of K; the offsets inside a block's 256 rows are 31-bit
  if (kb % 16 || lx % 16 || lw % 16 || lx < kb || lw < kb || !aligned16(g->x) || !aligned16(g->w)) return MVIT_EINVAL;
  if (kb > (1 << 23) || lx > (1 << 23) || lw > (1 << 23)) return MVIT_EINVAL;
  if (g->res && g->ldr < g->N) return MVIT_EINVAL;
  const int ye = g->y_f32 ? 4 : 2;
  a = {(const char*)g->x, (const char*)g->w, g->bias, g->res, g->y, g->pre, g->x_scale, g->w_scale, g->res ? g->ldr : 0, (unsigned)lx, (unsigned)lw,
       g->M, g->N, (int)kb, g->act, g->bias_f32, g->act == MVIT_ACT_RELU ? 0.f : -INFINITY, 0, 1 << 20, 1, nullptr};
  vec = g->N % 8 == 0 && aligned16(g->y) && aligned16(g->pre) && aligned16(g->res) && (!g->res || g->ldr * ye % 16 == 0);
  return 0;
}

// Few tiles or few columns and a long K: K in parts, whose f32 products a second launch adds in order and finishes.  By what it costs, in
// tenths of a microsecond: 40 for a round of blocks and for each of its K tiles of 128 bytes 10 and 4 with tiles of 128 x 128 and 64 x 64 (7 and 3
// with one block a CU), 22 for every 32 of them by rows; 50 for the second launch and 8 bytes an output and part at 5 TB/s.  Taken where that
// says a quarter less (at a seventh, [134, 2352] x [395, 2352] lost 1 us).  us without and with: bf16 [1, 16384] x [512, 16384] 22 / 10,
// [64, 7792] x [2558, 7792] 35 / 21, the same in e4m3 20 / 16, [66, 6784] x [146, 6784] 25 / 14, [37, 2560] x [2044, 2560] 11.4 / 9.0,
// [513, 14336] x [4096, 14336] 138 / 74, [1400, 8192] x [1536, 8192] 77 / 48.  e4m3 with a 16-bit y leaves the e4m3 instructions for it and gains the least:
// [513, 14336] x [4096, 14336] 71 / 71, onto an f32 stream 104 / 72
struct Parts {
  int kind, splits, kper;
};
Parts plan_parts(int M, int N, long long kb) {
  const int cus = mvit_num_cus(), nk = (int)((kb + 127) / 128);
  Parts best = {0, 1, 1 << 20};
  if (nk < 8) return best;
  const bool rows = M <= 16 || (M <= 32 && N <= 16 * cus);
  double whole = 1e300, least = 1e300;
  for (int kind = rows ? 0 : 2; kind <= (rows ? 0 : 3); ++kind) {
    const int b = kind == 0 ? 16 : kind == 2 ? 128 : 64;
    const long long tiles = (kind == 0 ? 1 : ((long long)M + b - 1) / b) * ((N + b - 1) / b);
    const int slots = 2 * cus;
    if (tiles > slots) continue;   // (no room for parts here; and by_size forms nothing whole of them where 128 x 128 tiles are one a CU at most)
    for (int want = 1; want <= 16 && tiles * want <= slots && nk >= 4 * want; ++want) {
      const int kper = (nk + want - 1) / want, s = (nk + kper - 1) / kper;
      double c = 40. + (kind == 0 ? 22. * ((kper + 31) / 32) : (double)kper * (kind == 2 ? (tiles * s <= cus ? 7 : 10) : (tiles * s <= cus ? 3 : 4)));
      if (want == 1) {
        whole = c < whole ? c : whole;
        continue;
      }
      c += 50. + (double)s * M * N * (8. / 5e5);
      if (s > 1 && c < least) least = c, best = {kind, s, kper};
    }
  }
  return least < whole * 0.73 ? best : Parts{0, 1, 1 << 20};
}
long long parts_bytes(const Parts& p, int M, int N) { return p.splits > 1 ? (long long)p.splits * M * N * 4 : 0; }

// Sum of `splits` groups of 4 values, `stride` apart, in order; eight of them on their way at a time (f32, at any 4-byte address)
__device__ __forceinline__ f32x4 sum_of_parts(const float* at, size_t stride, int splits) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < splits; k += 8) {
    f32x4 u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) __builtin_memcpy(&u[j], at + (size_t)min(k + j, splits - 1) * stride, 16);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < splits) s += u[j];
  }
  return s;
}

// y = res + act(sum of the parts + bias), 4 columns a thread, 64 threads by 4 rows a block
template <bool OUT32>
__global__ __launch_bounds__(256) void finish_parts(const Args p, const float* part, int splits) {
  using E = End<OUT32, A_ANY, false>;
  const int col = (blockIdx.x * 64 + threadIdx.x) * 4, left = p.N - col;
  if (left <= 0) return;
  float bias[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) bias[e] = p.bias && e < left ? value_of(p.bias, col + e, p.bias_f32) : 0.f;
  for (int row = blockIdx.y * 4 + threadIdx.y; row < p.M; row += gridDim.y * 4) {
    float v[4] = {}, res[4] = {};
    const float* at = part + (size_t)row * p.N + col;
    if (p.res)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) res[e] = value_of(p.res, (size_t)row * p.ldr + col + e, OUT32);
    if (left >= 4) {
      const f32x4 s = sum_of_parts(at, (size_t)p.M * p.N, splits);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = s[e];
    } else {
      for (int k = 0; k < splits; ++k)
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (e < left) v[e] += at[(size_t)k * p.M * p.N + e];
    }
    const size_t o = (size_t)row * p.N + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += bias[e];
    if (p.pre) {
      const uint32_t u[2] = {pack2bf(v[0], v[1]), pack2bf(v[2], v[3])};
      put<E, false, 8>((bf16_t*)p.pre + o, u, left);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = activated<A_ANY>(p, v[e]) + res[e];
    if constexpr (OUT32) {
      const uint32_t u[4] = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
      put<E, true, 16>((float*)p.y + o, u, left);
    } else {
      const uint32_t u[2] = {pack2bf(v[0], v[1]), pack2bf(v[2], v[3])};
      put<E, false, 8>((bf16_t*)p.y + o, u, left);
    }
  }
}

// MODE: the kernels whose f32 outputs are not rounded before they are added
template <int MODE>
int in_parts(const mvit_linear_args* g, const Args& a, const Parts& plan, hipStream_t s) {
  Args b = a;
  b.y = g->scratch, b.bias = b.res = nullptr, b.pre = nullptr, b.act = MVIT_ACT_NONE, b.act_lo = -INFINITY, b.kper = plan.kper, b.splits = plan.splits;
  if (const int rc = dispatch_parts<MODE>(b, a.N % 8 == 0, plan.kind, s)) return rc;
  const int row_blocks = (a.M + 3) / 4;
  const dim3 grid((a.N + 255) / 256, row_blocks < 4096 ? row_blocks : 4096);
  if (g->y_f32)
    hipLaunchKernelGGL((finish_parts<true>), grid, dim3(64, 4), 0, s, a, (const float*)g->scratch, plan.splits);
  else
    hipLaunchKernelGGL((finish_parts<false>), grid, dim3(64, 4), 0, s, a, (const float*)g->scratch, plan.splits);
  return MVIT_LAUNCH_CHECK();
}
// in parts where that pays and there is room for them
bool parts_fit(const mvit_linear_args* g, const Args& a, Parts& plan) {
  if (!g->scratch || !aligned16(g->scratch)) return false;
  plan = plan_parts(a.M, a.N, a.kb);
  return plan.splits > 1 && g->scratch_bytes >= parts_bytes(plan, a.M, a.N);
}

}  // namespace

extern "C" MVIT_API long long mvit_linear_scratch_bytes(int M, int N, long long k_bytes) {
  if (M <= 0 || M > MAX_M || N <= 0 || N > MAX_N || k_bytes <= 0 || k_bytes > (1 << 23)) return 0;
  return parts_bytes(plan_parts(M, N, k_bytes), M, N);
}

extern "C" MVIT_API int mvit_linear_act(const mvit_linear_args* args, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  Args a;
  bool vec;
  if (const int rc = check(args, 2, a, vec)) return rc < 0 ? rc : MVIT_OK;
  Parts plan;
  if (parts_fit(args, a, plan)) return in_parts<H16>(args, a, plan, (hipStream_t)stream);
  return args->y_f32 ? dispatch<H16, true>(a, vec, (hipStream_t)stream) : dispatch<H16, false>(a, vec, (hipStream_t)stream);
}

extern "C" MVIT_API int mvit_linear_fp8(const mvit_linear_args* args, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  Args a;
  bool vec;
  if (const int rc = check(args, 1, a, vec)) return rc < 0 ? rc : MVIT_OK;
  if (!a.xs || !a.ws || a.pre) return MVIT_EINVAL;
  Parts plan;
  if (parts_fit(args, a, plan)) return in_parts<F8X>(args, a, plan, (hipStream_t)stream);
  return args->y_f32 ? dispatch<F8X, true>(a, vec, (hipStream_t)stream) : dispatch<F8, false>(a, vec, (hipStream_t)stream);
}

// ---------------------------------------------------------------- the gradients' products
namespace {

// Which tile, and K in how many parts: dW has few tiles and a K axis of all rows, dx of few rows few tiles.  The parts' f32 products are added
// by a second launch, in order.  By what it costs, in tenths of a microsecond: 40 for a round of blocks and, for each of its K tiles of 64, with
// the tiles of 256 x 256, 128 x 256, 128 x 128 and 64 x 64, 16, 10, 10 and 4 (7 and 3 with one block a CU); 50 for the second launch and
// 8 bytes an output and part at 5 TB/s.  us without and with splits: dW
// [1536, 1536] of 21056 rows 252 / 96, of 5264 rows 52 / 39, [64, 512] of 20816 rows 86 / 13, [4096, 1536] of 21056 rows 289 / 251; dx [33, 1536] of
// 4096 columns 18 / 10, [329, 1536] 19 / 15
struct Plan {
  int tile, splits, kper;
};
Plan plan_grad(int M, int N, int K) {
  static constexpr int BM[4] = {256, 128, 128, 64}, BN[4] = {256, 256, 128, 64}, full[4] = {16, 10, 10, 4}, alone[4] = {16, 10, 7, 3};
  const int cus = mvit_num_cus(), nk = (int)(((long long)K + 63) / 64);
  Plan best = {0, 1, nk};
  double least = 1e300;
  for (int t = 0; t < 4; ++t) {
    const long long tiles = (((long long)M + BM[t] - 1) / BM[t]) * ((N + BN[t] - 1) / BN[t]);
    const int slots = t < 2 ? cus : 2 * cus;
    // up to two rounds and a part; four K tiles a part at least
    const int most = tiles > 2 * slots ? 1 : 1 + 2 * slots / (int)tiles;
    for (int want = 1; want <= 64 && want <= most && (want == 1 || nk >= 4 * want); ++want) {
      const int kper = (nk + want - 1) / want, s = want == 1 ? 1 : (nk + kper - 1) / kper;
      const long long n = tiles * s, rounds = want == 1 ? (n + slots - 1) / slots : ((int)n + slots - 1) / slots;
      double c = (double)rounds * (40. + (double)(n <= cus ? alone[t] : full[t]) * kper);
      if (s > 1) c += 50. + (double)s * M * N * (8. / 5e5);
      if (c < least) least = c, best = {t, s, kper};
    }
  }
  return best;
}

long long split_bytes(const Plan& p, int M, int N) { return p.splits > 1 ? (long long)p.splits * M * N * 4 : 0; }

// 4 outputs a thread
__global__ __launch_bounds__(256) void sum_splits(const float* part, bf16_t* y, int splits, long long n4) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) {
    const f32x4 s = sum_of_parts(part + i * 4, (size_t)n4 * 4, splits);
    *(uint2*)(y + i * 4) = make_uint2(pack2bf(s[0], s[1]), pack2bf(s[2], s[3]));
  }
}

}  // namespace

extern "C" MVIT_API long long mvit_linear_grad_scratch_bytes(int M, int N, int K) {
  if (M <= 0 || M > MAX_M || N <= 0 || N > MAX_N || K <= 0 || K > MAX_K) return 0;
  return split_bytes(plan_grad(M, N, K), M, N);
}

extern "C" MVIT_API int mvit_linear_grad(const mvit_linear_args* g, int x_rows, void* scratch, long long scratch_bytes, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  if (!g || g->M <= 0 || g->M > MAX_M || g->N <= 0 || g->N > MAX_N || g->K <= 0 || g->K > MAX_K || !g->x || !g->w || !g->y) return MVIT_EINVAL;
  if (g->bias || g->res || g->pre || g->x_scale || g->w_scale || g->act != MVIT_ACT_NONE || g->y_f32) return MVIT_EINVAL;
  // 16-byte pieces of the rows in memory; 31-bit offsets inside a block's rows
  const long long lx = g->ldx * 2, lw = g->ldw * 2, up8 = (g->K + 7LL) / 8 * 8;
  if (lx % 16 || lw % 16 || lx > (1 << 23) || lw > (1 << 23) || g->N % 8 || g->ldw < g->N || !aligned16(g->x) || !aligned16(g->w) || !aligned16(g->y))
    return MVIT_EINVAL;
  if (g->ldx < (x_rows ? (g->M + 7LL) / 8 * 8 : up8)) return MVIT_EINVAL;   // (x_rows = 0: and so K is at most 2^22)
  const Plan plan = plan_grad(g->M, g->N, g->K);
  if (plan.splits > 1 && (!scratch || !aligned16(scratch) || scratch_bytes < split_bytes(plan, g->M, g->N))) return MVIT_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  const Args a = {(const char*)g->x, (const char*)g->w, nullptr, nullptr, g->y, nullptr, nullptr, nullptr, 0, (unsigned)lx, (unsigned)lw,
                  g->M, g->N, (int)(up8 * 2), MVIT_ACT_NONE, 0, -INFINITY, g->K, plan.kper, plan.splits, (float*)scratch};
  if (const int rc = x_rows ? dispatch_grad<DW>(a, plan.tile, s) : dispatch_grad<DX>(a, plan.tile, s)) return rc;
  if (plan.splits == 1) return MVIT_OK;
  const long long n4 = (long long)g->M * g->N / 4, blocks = (n4 + 255) / 256, most = (long long)mvit_num_cus() * 16;
  hipLaunchKernelGGL(sum_splits, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, s, (const float*)scratch, (bf16_t*)g->y, plan.splits, n4);
  return MVIT_LAUNCH_CHECK();
}

// ---------------------------------------------------------------- backward of the epilogue
// dz = dy act'(pre) and its column sums, in one pass over dy and pre.  dz is rounded to 16 bits, as the operand of dx = dz W and dW = dz^T x that it is;
// the sums are taken before that.  With z as it is kept this makes the gradients' error against 64 bits 2.4e-3 of their norm where one rounding at
// the end gives 1.7e-3 ([5264, 1536] x [4096, 1536], bf16, gelu).  Bound by HBM ([5264, 4096] bf16, gelu: 24 us, 129 MB, 5.3 TB/s).  A block owns 256
// columns and a run of rows: 32 lanes of 8 columns (16-byte loads) by 8 rows at a time.  Sums over a run stay in registers, then LDS; the
// runs meet in a f32 workspace (column_sums.hpp): a fixed order, no atomics.
namespace {

enum Slope { S_ONE, S_CLIP, S_SILU, S_TANH, S_ERF };

template <int SL>
__device__ __forceinline__ float slope(float z) {
  if constexpr (SL == S_ONE) return 1.f;
  // (an infinity, as a z beyond fp16 is kept, has the slope of the far values: bounded, no infinity meets a zero.  A NaN stays one.)
  z = __builtin_elementwise_minimum(__builtin_elementwise_maximum(z, -1e15f), 1e15f);
  if constexpr (SL == S_CLIP) return z > 0.f ? 1.f : z != z ? z : 0.f;
  if constexpr (SL == S_SILU) {   // z s(z): s + z s (1 - s)
    const float p = sigmoid2(LOG2E * z);
    return p + z * p * (1.f - p);
  }
  if constexpr (SL == S_TANH) {   // z s(u), u = z (a + b z^2): s + z s (1 - s) (a + 3 b z^2)
    const float z2 = z * z, p = sigmoid2(z * __builtin_fmaf(z2, TANH_B, TANH_A));
    return p + z * p * (1.f - p) * __builtin_fmaf(z2, 3.f * TANH_B / LOG2E, TANH_A / LOG2E);
  }
  if constexpr (SL == S_ERF) {   // z Phi(z): Phi + z phi
    const float e = gauss(z);
    return normal_cdf(z, e) + z * e * 0.39894228040f;
  }
}

struct SlopeArgs {
  const void* dy;
  const bf16_t* pre;
  bf16_t* dz;
  float* part;
  long long ld_dz;          // dy and pre are dense
  int M, N, rows, act;      // rows: of a run
};

// 8 values of a row, `left` of them in it; ODD: at any address
template <bool F32, bool ODD>
__device__ __forceinline__ void values8(const void* p, size_t i, int left, float (&v)[8]) {
  if (ODD && left < 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? value_of(p, i + e, F32) : 0.f;
  } else if constexpr (F32) {
    float4 a, b;
    __builtin_memcpy(&a, __builtin_assume_aligned((const float*)p + i, ODD ? 4 : 16), 16);
    __builtin_memcpy(&b, __builtin_assume_aligned((const float*)p + i + 4, ODD ? 4 : 16), 16);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    uint4 u;
    __builtin_memcpy(&u, __builtin_assume_aligned((const bf16_t*)p + i, ODD ? 2 : 16), 16);
    v[0] = lo16f(u.x), v[1] = hi16f(u.x), v[2] = lo16f(u.y), v[3] = hi16f(u.y), v[4] = lo16f(u.z), v[5] = hi16f(u.z), v[6] = lo16f(u.w), v[7] = hi16f(u.w);
  }
}

template <int SL, bool F32, bool ODD>
__global__ __launch_bounds__(256) void act_bwd_rows(const SlopeArgs p) {
  __shared__ float sums[8][256];
  const int cg = threadIdx.x & 31, rg = threadIdx.x >> 5, c0 = blockIdx.x * 256 + cg * 8;
  const int r0 = blockIdx.y * p.rows, r1 = min(r0 + p.rows, p.M);
  float sum[8] = {};
  if (c0 < p.N) {
#pragma unroll 2
    for (int r = r0 + rg; r < r1; r += 8) {
      const size_t o = (size_t)r * p.N + c0;
      float g[8];
      values8<F32, ODD>(p.dy, o, p.N - c0, g);
      if constexpr (SL != S_ONE) {
        float z[8];
        values8<false, ODD>(p.pre, o, p.N - c0, z);
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] *= slope<SL>(z[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += g[e];
      if (p.dz) *(uint4*)(p.dz + (size_t)r * p.ld_dz + c0) = pack8(g);
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[rg][cg * 8 + e] = sum[e];
  __syncthreads();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c < p.N) {
    float s = sums[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sums[k][threadIdx.x];
    p.part[(size_t)blockIdx.y * p.N + c] = s;
  }
}

// rows of a run: blocks enough for eight a CU, no more than 128 runs to add up, no fewer than 8 rows
int run_rows(int M, int N) {
  const int cols = (N + 255) / 256;
  int runs = (mvit_num_cus() * 8 + cols - 1) / cols;
  runs = runs > 128 ? 128 : runs;
  const int rows = (M + runs - 1) / runs;
  return rows < 8 ? 8 : rows;
}
int run_count(int M, int N) { return M <= 0 ? 0 : (M + run_rows(M, N) - 1) / run_rows(M, N); }

template <bool F32, bool ODD>
void launch_rows_bwd(const SlopeArgs& a, dim3 grid, hipStream_t s) {
  if (a.act == MVIT_ACT_NONE)
    hipLaunchKernelGGL((act_bwd_rows<S_ONE, F32, ODD>), grid, dim3(256), 0, s, a);
  else if (a.act == MVIT_ACT_RELU)
    hipLaunchKernelGGL((act_bwd_rows<S_CLIP, F32, ODD>), grid, dim3(256), 0, s, a);
  else if (a.act == MVIT_ACT_GELU)
    hipLaunchKernelGGL((act_bwd_rows<S_ERF, F32, ODD>), grid, dim3(256), 0, s, a);
  else if (a.act == MVIT_ACT_SILU)
    hipLaunchKernelGGL((act_bwd_rows<S_SILU, F32, ODD>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((act_bwd_rows<S_TANH, F32, ODD>), grid, dim3(256), 0, s, a);
}

}  // namespace

extern "C" MVIT_API long long mvit_act_bwd_scratch_bytes(int M, int N) { return M <= 0 || N <= 0 ? 0 : (long long)run_count(M, N) * N * 4; }

extern "C" MVIT_API int mvit_act_bwd(const void* dy, int dy_f32, const void* pre, int act, void* dz, long long ld_dz, void* dbias, int dbias_f32,
                                     void* scratch, int M, int N, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  if (M < 0 || M > MAX_M || N <= 0 || N > MAX_N || (M > 0 && !dy) || act < MVIT_ACT_NONE || act > MVIT_ACT_GELU_TANH || (act != MVIT_ACT_NONE && M > 0 && !pre)) return MVIT_EINVAL;
  if (dbias && M > 0 && !scratch) return MVIT_EINVAL;
  if (dz && (ld_dz < N || ld_dz % 8 || !aligned16(dz))) return MVIT_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  const int runs = run_count(M, N);
  if (M > 0) {
    const SlopeArgs a = {dy, (const bf16_t*)pre, (bf16_t*)dz, dbias ? (float*)scratch : nullptr, ld_dz, M, N, run_rows(M, N), act};
    const dim3 grid((N + 255) / 256, runs);
    if (N % 8 == 0 && aligned16(dy) && aligned16(pre))
      dy_f32 ? launch_rows_bwd<true, false>(a, grid, s) : launch_rows_bwd<false, false>(a, grid, s);
    else
      dy_f32 ? launch_rows_bwd<true, true>(a, grid, s) : launch_rows_bwd<false, true>(a, grid, s);
    if (const int rc = MVIT_LAUNCH_CHECK()) return rc;
  }
  return dbias ? launch_sum_parts((const float*)scratch, dbias, runs, N, dbias_f32, s) : MVIT_OK;
}
