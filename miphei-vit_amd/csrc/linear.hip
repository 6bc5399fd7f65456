// The linear layer with activation and residual in its epilogue (kernels in linear_kernel.hpp), 16-bit and 8-bit operands.
#include <cmath>
#include "column_sums.hpp"
#include "linear_kernel.hpp"

using namespace mvit_linear;

namespace mvit_linear {
template <int MODE, bool OUT32>
int dispatch(const Args& a, bool vec, hipStream_t s);   // linear_launch.hpp
extern template int dispatch<H16, false>(const Args&, bool, hipStream_t);
extern template int dispatch<H16, true>(const Args&, bool, hipStream_t);
extern template int dispatch<F8, false>(const Args&, bool, hipStream_t);
extern template int dispatch<F8X, true>(const Args&, bool, hipStream_t);
}  // namespace mvit_linear

namespace {

constexpr int MAX_M = 1 << 30, MAX_N = 1 << 24;   // tile numbers and grids stay in 31 bits

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
       g->M, g->N, (int)kb, g->act, g->bias_f32, g->act == MVIT_ACT_RELU ? 0.f : -INFINITY};
  vec = g->N % 8 == 0 && aligned16(g->y) && aligned16(g->pre) && aligned16(g->res) && (!g->res || g->ldr * ye % 16 == 0);
  return 0;
}

}  // namespace

extern "C" MVIT_API int mvit_linear_act(const mvit_linear_args* args, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  Args a;
  bool vec;
  if (const int rc = check(args, 2, a, vec)) return rc < 0 ? rc : MVIT_OK;
  return args->y_f32 ? dispatch<H16, true>(a, vec, (hipStream_t)stream) : dispatch<H16, false>(a, vec, (hipStream_t)stream);
}

extern "C" MVIT_API int mvit_linear_fp8(const mvit_linear_args* args, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  Args a;
  bool vec;
  if (const int rc = check(args, 1, a, vec)) return rc < 0 ? rc : MVIT_OK;
  if (!a.xs || !a.ws || a.pre) return MVIT_EINVAL;
  return args->y_f32 ? dispatch<F8X, true>(a, vec, (hipStream_t)stream) : dispatch<F8, false>(a, vec, (hipStream_t)stream);
}

// ---------------------------------------------------------------- backward of the epilogue
// dz = dy act'(pre), as rows and transposed, and its column sums, in one pass over dy and pre: bound by HBM.  The transposed copy is an
// operand of dW = dz^T x, whose K axis is the rows; made from the values at hand it costs its write alone, a third of a transposition
// by itself.  A block owns 64 columns and a run of rows, and goes down it by 64 x 64 tiles: a thread takes 8 columns of rows 2 r and
// 2 r + 1 (16-byte loads), packs pairs of rows into LDS [column][row], and reads 8 rows of a column back.  Column stride 136 bytes: the 64
// writes of a wave fall on 64 banks.  Sums over a run stay in registers, the runs meet in a f32 workspace (column_sums.hpp).
// The same kernel with the identity and no sums transposes x and W.
namespace {

enum Slope { S_ONE, S_CLIP, S_SILU, S_TANH, S_ERF, S_ANY };

template <int SL>
__device__ __forceinline__ float slope(float z, int act) {
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
  return act == MVIT_ACT_NONE        ? 1.f
         : act == MVIT_ACT_RELU      ? slope<S_CLIP>(z, act)
         : act == MVIT_ACT_SILU      ? slope<S_SILU>(z, act)
         : act == MVIT_ACT_GELU_TANH ? slope<S_TANH>(z, act)
                                     : slope<S_ERF>(z, act);
}

struct SlopeArgs {
  const void* dy;
  const bf16_t* pre;
  bf16_t *dz, *dzt;
  float* part;
  long long ld, ld_dz, ld_dzt;   // ld: of dy (and of the source of a transposition); pre is dense
  int M, N, rows, act;           // rows: of a run, a multiple of 64
};

template <int SL, bool F32>
__global__ __launch_bounds__(256) void act_bwd_tiles(const SlopeArgs p) {
  constexpr int LDT = 68;   // 16-bit values of a column in LDS
  __shared__ __attribute__((aligned(16))) bf16_t tile[2][64 * LDT];
  __shared__ float sums[32][65];
  const int cg = threadIdx.x & 7, rp = threadIdx.x >> 3;
  const int c0 = blockIdx.x * 64 + cg * 8;
  const int r0 = blockIdx.y * p.rows, r1 = min(r0 + p.rows, (p.M + 63) / 64 * 64);
  float sum[8] = {};
  int buf = 0;
  for (int t = r0; t < r1; t += 64, buf ^= 1) {
    float g[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = t + rp * 2 + h;
      const bool in = r < p.M && c0 < p.N;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[h][e] = 0.f;
      if (in) {
        const size_t o = (size_t)r * p.ld + c0;
        if constexpr (F32) {
          const float4 u = *(const float4*)((const float*)p.dy + o), v = *(const float4*)((const float*)p.dy + o + 4);
          g[h][0] = u.x, g[h][1] = u.y, g[h][2] = u.z, g[h][3] = u.w, g[h][4] = v.x, g[h][5] = v.y, g[h][6] = v.z, g[h][7] = v.w;
        } else {
          const uint4 u = *(const uint4*)((const bf16_t*)p.dy + o);
          g[h][0] = lo16f(u.x), g[h][1] = hi16f(u.x), g[h][2] = lo16f(u.y), g[h][3] = hi16f(u.y);
          g[h][4] = lo16f(u.z), g[h][5] = hi16f(u.z), g[h][6] = lo16f(u.w), g[h][7] = hi16f(u.w);
        }
        if constexpr (SL != S_ONE) {
          const uint4 u = *(const uint4*)(p.pre + (size_t)r * p.N + c0);
          const float z[8] = {lo16f(u.x), hi16f(u.x), lo16f(u.y), hi16f(u.y), lo16f(u.z), hi16f(u.z), lo16f(u.w), hi16f(u.w)};
#pragma unroll
          for (int e = 0; e < 8; ++e) g[h][e] *= slope<SL>(z[e], 0);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += g[h][e];
        if (p.dz) *(uint4*)(p.dz + (size_t)r * p.ld_dz + c0) = pack8(g[h]);
      }
    }
    if (p.dzt) {
#pragma unroll
      for (int e = 0; e < 8; ++e) *(uint32_t*)&tile[buf][(cg * 8 + e) * LDT + rp * 2] = pack2bf(g[0][e], g[1][e]);
      __syncthreads();   // (the other buffer's reads are two barriers away from its next writes)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = rp + h * 32, r = t + cg * 8;   // 8 lanes a column: 128 bytes in a line; rows from M to the end of the last piece: zeros
        if (blockIdx.x * 64 + c < p.N && r < p.ld_dzt) {
          const uint2 *s = (const uint2*)&tile[buf][c * LDT + cg * 8], u = s[0], v = s[1];
          *(uint4*)(p.dzt + (size_t)(blockIdx.x * 64 + c) * p.ld_dzt + r) = make_uint4(u.x, u.y, v.x, v.y);
        }
      }
    }
  }
  if (!p.part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[rp][cg * 8 + e] = sum[e];
  __syncthreads();
  if (threadIdx.x < 64 && blockIdx.x * 64 + (int)threadIdx.x < p.N) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += sums[k][threadIdx.x];
    p.part[(size_t)blockIdx.y * p.N + blockIdx.x * 64 + threadIdx.x] = s;
  }
}

// by elements, where N or an address is not a multiple of 8 values: a thread a column, dz with its rows padded by zeros to ld_dz
template <bool F32>
__global__ __launch_bounds__(256) void act_bwd_elements(const SlopeArgs p) {
  const int c = blockIdx.x * 256 + threadIdx.x, r0 = blockIdx.y * p.rows, r1 = min(r0 + p.rows, p.M);
  float sum = 0.f;
  for (int r = r0; r < r1; ++r) {
    float g = 0.f;
    if (c < p.N) {
      const size_t o = (size_t)r * p.N + c;
      g = value_of(p.dy, o, F32);
      if (p.act != MVIT_ACT_NONE) g *= slope<S_ANY>(bf2f(p.pre[o]), p.act);
      sum += g;
    }
    if (p.dz && c < p.ld_dz) p.dz[(size_t)r * p.ld_dz + c] = f2bf(g);
  }
  if (p.part && c < p.N) p.part[(size_t)blockIdx.y * p.N + c] = sum;
}

// rows of a run: blocks enough for sixteen a CU, no more than 128 runs to add up
int run_rows(int M, int N) {
  const int tiles = (M + 63) / 64, cols = (N + 63) / 64;
  int runs = (mvit_num_cus() * 16 + cols - 1) / cols;
  runs = runs > 128 ? 128 : runs;
  runs = runs > tiles ? tiles : runs;
  return (tiles + runs - 1) / runs * 64;
}
int run_count(int M, int N) { return M <= 0 ? 0 : (M + run_rows(M, N) - 1) / run_rows(M, N); }

template <bool F32>
void launch_tiles(const SlopeArgs& a, dim3 grid, hipStream_t s) {
  if (a.act == MVIT_ACT_NONE)
    hipLaunchKernelGGL((act_bwd_tiles<S_ONE, F32>), grid, dim3(256), 0, s, a);
  else if (a.act == MVIT_ACT_RELU)
    hipLaunchKernelGGL((act_bwd_tiles<S_CLIP, F32>), grid, dim3(256), 0, s, a);
  else if (a.act == MVIT_ACT_GELU)
    hipLaunchKernelGGL((act_bwd_tiles<S_ERF, F32>), grid, dim3(256), 0, s, a);
  else if (a.act == MVIT_ACT_SILU)
    hipLaunchKernelGGL((act_bwd_tiles<S_SILU, F32>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((act_bwd_tiles<S_TANH, F32>), grid, dim3(256), 0, s, a);
}

}  // namespace

extern "C" MVIT_API int mvit_transpose_padded(const void* src, long long ld, void* dst, long long ld_dst, int R, int Cc, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  if (!src || !dst || R <= 0 || R > MAX_M || Cc <= 0 || Cc > MAX_N || ld % 8 || ld_dst % 8 || ld < (Cc + 7) / 8 * 8 || ld_dst < R || ld_dst >= R + 8 || !aligned16(src) || !aligned16(dst))
    return MVIT_EINVAL;
  SlopeArgs a = {};
  a.dy = src, a.dzt = (bf16_t*)dst, a.ld = ld, a.ld_dzt = ld_dst, a.M = R, a.N = Cc, a.rows = run_rows(R, Cc), a.act = MVIT_ACT_NONE;
  launch_tiles<false>(a, dim3((Cc + 63) / 64, run_count(R, Cc)), (hipStream_t)stream);
  return MVIT_LAUNCH_CHECK();
}

extern "C" MVIT_API long long mvit_act_bwd_scratch_bytes(int M, int N) { return M <= 0 || N <= 0 ? 0 : (long long)run_count(M, N) * N * 4; }

extern "C" MVIT_API int mvit_act_bwd(const void* dy, int dy_f32, const void* pre, int act, void* dz, long long ld_dz, void* dzt, long long ld_dzt,
                                     void* dbias, int dbias_f32, void* scratch, int M, int N, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  if (M < 0 || M > MAX_M || N <= 0 || N > MAX_N || (M > 0 && !dy) || act < MVIT_ACT_NONE || act > MVIT_ACT_GELU_TANH || (act != MVIT_ACT_NONE && M > 0 && !pre)) return MVIT_EINVAL;
  if (dbias && M > 0 && !scratch) return MVIT_EINVAL;
  if ((dz && (ld_dz < N || ld_dz % 8 || !aligned16(dz))) || (dzt && (!dz || ld_dzt < M || ld_dzt >= M + 8 || ld_dzt % 8 || !aligned16(dzt))))
    return MVIT_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  const int runs = run_count(M, N);
  if (M > 0) {
    const SlopeArgs a = {dy, (const bf16_t*)pre, (bf16_t*)dz, (bf16_t*)dzt, dbias ? (float*)scratch : nullptr, N, ld_dz, ld_dzt, M, N, run_rows(M, N), act};
    if (N % 8 == 0 && aligned16(dy) && aligned16(pre)) {
      const dim3 grid((N + 63) / 64, runs);
      dy_f32 ? launch_tiles<true>(a, grid, s) : launch_tiles<false>(a, grid, s);
    } else {
      const dim3 grid((unsigned)(((dz ? ld_dz : N) + 255) / 256), runs);
      if (dy_f32)
        hipLaunchKernelGGL((act_bwd_elements<true>), grid, dim3(256), 0, s, a);
      else
        hipLaunchKernelGGL((act_bwd_elements<false>), grid, dim3(256), 0, s, a);
      if (const int rc = MVIT_LAUNCH_CHECK()) return rc;
      if (dzt)
        if (const int rc = mvit_transpose_padded(dz, ld_dz, dzt, ld_dzt, M, N, stream)) return rc;
    }
    if (const int rc = MVIT_LAUNCH_CHECK()) return rc;
  }
  return dbias ? launch_sum_parts((const float*)scratch, dbias, runs, N, dbias_f32, s) : MVIT_OK;
}
