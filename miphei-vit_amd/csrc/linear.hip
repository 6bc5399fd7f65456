// The linear layer with activation and residual in its epilogue (kernels in linear_kernel.hpp), 16-bit and 8-bit operands.
#include <cmath>
#include "linear_kernel.hpp"

using namespace mvit_linear;

namespace {

template <int MODE, class E, int BM, int BN, int WM, int WN, int BKB, int NST>
int launch_tile(const Args& a, hipStream_t s) {
  using T = Tile<MODE, BM, BN, WM, WN, BKB, NST>;
  const long long nt = (long long)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  if (nt > 0x7fffffff) return MVIT_EINVAL;
  static mvit_per_device_size raised;
  const auto fn = linear_tile<MODE, E, BM, BN, WM, WN, BKB, NST>;
  if (const int rc = mvit_ensure_dynamic_lds((const void*)fn, T::LDS, raised)) return rc;
  const long long slots = (long long)mvit_num_cus() * T::BLOCKS_PER_CU;
  hipLaunchKernelGGL(fn, dim3((unsigned)(nt < slots ? nt : slots)), dim3(T::NT), T::LDS, s, a);
  return MVIT_LAUNCH_CHECK();
}

template <bool OP8, class E, int MT>
int launch_rows(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((linear_rows<OP8, E, MT>), dim3((a.N + 15) / 16), dim3(512), 0, s, a);
  return MVIT_LAUNCH_CHECK();
}

// Rows or tiles, and which: by what a round of blocks costs.  A round is every CU's share at once (one 256 x 256 tile, two of the others);
// measured at K = 1536, bf16, it takes 40 us with tiles of 256 x 256, 27 of 128 x 128 (20 with one a CU) and 12 of 64 x 64, and the
// ratios hold for e4m3 and other K within some per cent.  Large tiles read less of x and W; small ones leave less of the chip idle in the
// last round: [5264, 1536] x [4608, 1536]: 75 / 79 / 130 us, [5264, 4096] x [1536, 4096]: 80 / 62 / 104, [1301, 1536] x [4608, 1536]:
// 36 / 26 / 35, [329, 1536] x [4608, 1536]: 34 / 20 / 13.
template <int MODE, class E>
int by_size(const Args& a, hipStream_t s) {
  using Any = End<E::out32, A_ANY, E::vec>;   // (the row kernels' epilogue is not unrolled)
  const long long cus = mvit_num_cus();
  // few rows: [1, 1536] x [1536, 1536] bf16 5.8 us against 9.0 with tiles, [17, ..] 6.7 / 9.1, [32, 4096] x [1536, 4096] 14 / 18; from 33
  // rows on (9.0 / 9.2) and, from 17 on, with more than one block a CU (N > 4096) the tiles are as fast or faster
  if (a.M <= 16) return launch_rows<MODE != H16, Any, 1>(a, s);
  if (a.M <= 32 && a.N <= 16 * cus) return launch_rows<MODE != H16, Any, 2>(a, s);
  auto rounds = [&](long long edge, long long at_once) {
    const long long t = ((a.M + edge - 1) / edge) * ((a.N + edge - 1) / edge);
    return (t + at_once - 1) / at_once;
  };
  const long long c256 = 40 * rounds(256, cus), c128 = rounds(128, cus) == 1 ? 20 : 27 * rounds(128, 2 * cus), c64 = 12 * rounds(64, 2 * cus);
  if (c256 < c128 && c256 < c64) return launch_tile<MODE, E, 256, 256, 2, 4, 128, 2>(a, s);
  if (c128 < c64) return launch_tile<MODE, E, 128, 128, 2, 2, 128, 2>(a, s);
  return launch_tile<MODE, E, 64, 64, 2, 2, 128, 4>(a, s);
}

template <int MODE, bool OUT32>
int dispatch(Args& a, bool vec, hipStream_t s) {
  if (!vec) return by_size<MODE, End<OUT32, A_ANY, false>>(a, s);
  switch (a.act) {
    case MVIT_ACT_NONE:
    case MVIT_ACT_RELU:
      return by_size<MODE, End<OUT32, A_CLIP, true>>(a, s);
    case MVIT_ACT_GELU:
      return by_size<MODE, End<OUT32, A_ERF, true>>(a, s);
    default:
      return by_size<MODE, End<OUT32, A_SIGMOID, true>>(a, s);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 0: go on, 1: nothing to do, < 0: refused.  es: bytes of an operand's value.
int check(const mvit_linear_args* g, int es, Args& a, bool& vec) {
  if (!g || g->M < 0 || g->N <= 0 || g->K <= 0) return MVIT_EINVAL;
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
       g->M, g->N, (int)kb, g->act, g->bias_f32, g->act == MVIT_ACT_RELU ? 0.f : -INFINITY, g->act == MVIT_ACT_SILU ? 1.f : TANH_K,
       g->act == MVIT_ACT_SILU ? 0.f : TANH_K * 0.044715f};
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
// dz = dy act'(pre) and its column sums, in one pass over dy and pre (HBM-bound).  A block owns 512 columns (64 lanes x 8; by elements
// where N or an address is odd) and a run of rows, its 4 waves every fourth one; the sums of a run go through LDS in wave order to a
// [runs][N] f32 workspace, which a second launch adds up in order.
namespace {

__device__ __forceinline__ float act_grad(float z, int act) {
  switch (act) {
    case MVIT_ACT_RELU:
      return z > 0.f ? 1.f : z != z ? z : 0.f;
    case MVIT_ACT_SILU: {
      const float p = sigmoid(z);
      return p + z * p * (1.f - p);
    }
    case MVIT_ACT_GELU:
      return normal_cdf(z) + z * 0.39894228040f * __builtin_amdgcn_exp2f(-0.72134752044f * z * z);
    case MVIT_ACT_GELU_TANH: {
      const float p = sigmoid(TANH_K * (z + 0.044715f * z * z * z));
      return p + z * p * (1.f - p) * TANH_K * (1.f + 0.134145f * z * z);
    }
    default:
      return 1.f;
  }
}

template <bool F32, bool VEC>
__global__ __launch_bounds__(256) void act_bwd(const void* dy, const bf16_t* pre, int act, bf16_t* dz, float* part, int M, int N, int rows) {
  __shared__ float lds[4][512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r0 = blockIdx.y * rows, r1 = min(M, r0 + rows);
  // VEC: lane owns columns c0 .. c0 + 7; else column c0 + 64 e
  const int c0 = blockIdx.x * 512 + (VEC ? lane * 8 : lane);
  float sum[8] = {};
  for (int r = r0 + wave; r < r1; r += 4) {
    const size_t o = (size_t)r * N + c0;
    float g[8], z[8];
    if constexpr (VEC) {
      if (c0 >= N) break;
      if constexpr (F32) {
        const float4 a = *(const float4*)((const float*)dy + o), b = *(const float4*)((const float*)dy + o + 4);
        g[0] = a.x, g[1] = a.y, g[2] = a.z, g[3] = a.w, g[4] = b.x, g[5] = b.y, g[6] = b.z, g[7] = b.w;
      } else {
        const uint4 a = *(const uint4*)((const bf16_t*)dy + o);
        g[0] = lo16f(a.x), g[1] = hi16f(a.x), g[2] = lo16f(a.y), g[3] = hi16f(a.y);
        g[4] = lo16f(a.z), g[5] = hi16f(a.z), g[6] = lo16f(a.w), g[7] = hi16f(a.w);
      }
      if (pre) {
        const uint4 a = *(const uint4*)(pre + o);
        z[0] = lo16f(a.x), z[1] = hi16f(a.x), z[2] = lo16f(a.y), z[3] = hi16f(a.y);
        z[4] = lo16f(a.z), z[5] = hi16f(a.z), z[6] = lo16f(a.w), z[7] = hi16f(a.w);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool ok = c0 + 64 * e < N;
        g[e] = ok ? value_of(dy, o + 64 * e, F32) : 0.f;
        if (pre) z[e] = ok ? bf2f(pre[o + 64 * e]) : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (pre) g[e] *= act_grad(z[e], act);
      sum[e] += g[e];
    }
    if (dz) {
      if constexpr (VEC) {
        *(uint4*)(dz + o) = make_uint4(pack2bf(g[0], g[1]), pack2bf(g[2], g[3]), pack2bf(g[4], g[5]), pack2bf(g[6], g[7]));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c0 + 64 * e < N) dz[o + 64 * e] = f2bf(g[e]);
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) lds[wave][VEC ? lane * 8 + e : lane + 64 * e] = sum[e];
  __syncthreads();
  for (int c = threadIdx.x; c < 512; c += 256)
    if (blockIdx.x * 512 + c < N) part[(size_t)blockIdx.y * N + blockIdx.x * 512 + c] = lds[0][c] + lds[1][c] + lds[2][c] + lds[3][c];
}

// out[c] = sum over the runs in order
__global__ __launch_bounds__(256) void add_runs(const float* part, void* out, int runs, int N, int out_f32) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < runs; ++k) s += part[(size_t)k * N + c];
  if (out_f32)
    ((float*)out)[c] = s;
  else
    ((bf16_t*)out)[c] = f2bf(s);
}

// rows of a run: runs enough to fill the chip, but no more than 64 of them to add up
int run_rows(int M) {
  const int r = (M + 63) / 64;
  return r < 16 ? 16 : r;
}
int run_count(int M) { return M <= 0 ? 0 : (M + run_rows(M) - 1) / run_rows(M); }

}  // namespace

extern "C" MVIT_API long long mvit_act_bwd_scratch_bytes(int M, int N) { return M <= 0 || N <= 0 ? 0 : (long long)run_count(M) * N * 4; }

extern "C" MVIT_API int mvit_act_bwd(const void* dy, int dy_f32, const void* pre, int act, void* dz, void* dbias, int dbias_f32, void* scratch,
                                     int M, int N, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  if (M < 0 || N <= 0 || (M > 0 && !dy) || act < MVIT_ACT_NONE || act > MVIT_ACT_GELU_TANH || (act != MVIT_ACT_NONE && M > 0 && !pre)) return MVIT_EINVAL;
  if (dbias && M > 0 && !scratch) return MVIT_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  const int runs = run_count(M), rows = M > 0 ? run_rows(M) : 0;
  if (M > 0) {
    const bool vec = N % 8 == 0 && aligned16(dy) && aligned16(pre) && aligned16(dz);
    const dim3 grid((N + 511) / 512, runs);
    float* part = dbias ? (float*)scratch : nullptr;
    const bf16_t* z = act == MVIT_ACT_NONE ? nullptr : (const bf16_t*)pre;
    if (dy_f32)
      hipLaunchKernelGGL((vec ? act_bwd<true, true> : act_bwd<true, false>), grid, dim3(256), 0, s, dy, z, act, (bf16_t*)dz, part, M, N, rows);
    else
      hipLaunchKernelGGL((vec ? act_bwd<false, true> : act_bwd<false, false>), grid, dim3(256), 0, s, dy, z, act, (bf16_t*)dz, part, M, N, rows);
    if (const int rc = MVIT_LAUNCH_CHECK()) return rc;
  }
  if (dbias) {
    hipLaunchKernelGGL(add_runs, dim3((N + 255) / 256), dim3(256), 0, s, (const float*)scratch, dbias, runs, N, dbias_f32);
    return MVIT_LAUNCH_CHECK();
  }
  return MVIT_OK;
}
