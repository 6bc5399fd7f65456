// Root-mean-square norm of a residual stream, with its backward pass and its 8-bit form, and the 8-bit quantisation of rows.
//
//   h = x + residual                              kept in the residual stream's type: what the next layer reads is what is normed
//   y = h * r * w,  r = 1 / sqrt(mean(h^2) + eps)
//   8 bits: scale = max(max |y|, 1e-30) / 448 (one per row), q = e4m3(y / scale); 448 is the largest e4m3 value
//   d h = d h_out + r (w dy - xhat mean(w dy xhat)),  xhat = h r;   d w = sum over rows of dy xhat
//
// All of it is bound by HBM: a row is read once, lives in registers (f32) while its sum of squares, its largest value and its outputs
// are formed, and is written once.
//  * A row belongs to TPR = 64 threads (one wave: no barrier) or to a block (fewer registers and loads a thread: for wide rows, and for
//    few, whose latency counts).
//  * Each thread holds NV pieces of 8 values (16-byte loads).  Where D is no multiple of 8, or a row starts off 16 bytes (ODD), they go to odd
//    addresses and a row's last piece goes by elements; with all of it by elements an f32 stream of [16623, 1053] to 8 bits took 106 us
//    instead of 46, of [2032, 7956] 257 instead of 40.
//  * Rows are walked with a grid stride, so that w is loaded once per thread and not once per row.
// Measured against a 1 GiB copy's 5.05 TB/s (one MI355X, kernels by themselves): f32 stream of [21056, 1536] forward 71 us (388 MB, 5.5 TB/s), backward
// 97 us (517 MB, 5.3 TB/s) and 5 for d w's partial sums; 16-bit stream to 8 bits [20816, 1536] 34 us (6.6 TB/s); quantisation [21056, 4096] 39 us
// (6.6 TB/s).  Among other calls a pass takes some 10 us more, in 8 bits 43 and 48.
// Sums and statistics are f32; sums over the rows (d w) go row by row in registers, over the waves of a block in LDS, over the blocks
// through a [blocks][D] f32 workspace that a second launch adds up: a fixed order, no atomics, bit-identical from run to run.
#include "column_sums.hpp"
#include "common.hpp"
#include "../../include/miphei_hip.h"

namespace {

enum { T16 = 0, F32 = 1, NONE = 2, F8 = 3 };

constexpr float E4M3_MAX = 448.f, AMAX_MIN = 1e-30f;

// 8 values from element `i` of a 16-bit or f32 array (f32: 8 from 4-byte, 16-bit: from 2-byte addresses where ODD; global memory takes
// 16-byte accesses at any address), of which the last `left` .. 8 lie behind the row where ODD: not touched, and zeros.
constexpr int VEC = 8;
template <bool ODD, class V>
__device__ __forceinline__ V load_raw(const void* p) {
  V u;
  if constexpr (ODD)
    __builtin_memcpy(&u, p, sizeof(V));
  else
    u = *(const V*)p;
  return u;
}
template <bool ODD, class V>
__device__ __forceinline__ void store_raw(void* p, const V& u) {
  if constexpr (ODD)
    __builtin_memcpy(p, &u, sizeof(V));
  else
    *(V*)p = u;
}
template <int T, bool ODD>
__device__ __forceinline__ void load_vec(const void* p, size_t i, int left, float* v) {
  if (ODD && left < VEC) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = e >= left ? 0.f : T == T16 ? bf2f(((const bf16_t*)p)[i + e]) : ((const float*)p)[i + e];
  } else if constexpr (T == T16) {
    const uint4 u = load_raw<ODD, uint4>((const bf16_t*)p + i);
    v[0] = lo16f(u.x), v[1] = hi16f(u.x), v[2] = lo16f(u.y), v[3] = hi16f(u.y);
    v[4] = lo16f(u.z), v[5] = hi16f(u.z), v[6] = lo16f(u.w), v[7] = hi16f(u.w);
  } else {
    const float4 a = load_raw<ODD, float4>((const float*)p + i), b = load_raw<ODD, float4>((const float*)p + i + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}
template <int T, bool ODD>
__device__ __forceinline__ void store_vec(void* p, size_t i, int left, const float* v) {
  if (ODD && left < VEC) {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e < left) {
        if constexpr (T == T16)
          ((bf16_t*)p)[i + e] = f2bf(v[e]);
        else if constexpr (T == F32)
          ((float*)p)[i + e] = v[e];
        else
          ((uint8_t*)p)[i + e] = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v[e], v[e], 0, false) & 0xff);
      }
  } else if constexpr (T == T16) {
    store_raw<ODD>((bf16_t*)p + i, make_uint4(pack2bf(v[0], v[1]), pack2bf(v[2], v[3]), pack2bf(v[4], v[5]), pack2bf(v[6], v[7])));
  } else if constexpr (T == F32) {
    store_raw<ODD>((float*)p + i, make_float4(v[0], v[1], v[2], v[3]));
    store_raw<ODD>((float*)p + i + 4, make_float4(v[4], v[5], v[6], v[7]));
  } else {
    int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], a, true), b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], b, true);
    store_raw<ODD>((uint8_t*)p + i, make_int2(a, b));
  }
}
// the value as it reads back from the stream's own type (16-bit streams are normed as they are stored)
template <int T>
__device__ __forceinline__ float as_stored(float v) {
  if constexpr (T == T16) return bf2f(f2bf(v));
  return v;
}

__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
  return v;
}

// Sum and maximum over the TPR threads of a row.  TPR = 256: through 4 words of LDS, one set of them for each turn (`odd`), so that
// the next reduction's writes never meet this one's reads: one barrier a reduction.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* lds, int& turn) {
  v = wave_sum(v);
  if constexpr (TPR > 64) {
    float* s = lds + (turn & 1) * (TPR / 64);
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int k = 0; k < TPR / 64; ++k) v += s[k];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ unsigned row_umax(unsigned v, float* lds, int& turn) {
  v = wave_umax(v);
  if constexpr (TPR > 64) {
    unsigned* s = (unsigned*)lds + (turn & 1) * (TPR / 64);
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int k = 0; k < TPR / 64; ++k) v = max(v, s[k]);
  }
  return v;
}

struct RowArgs {
  const void *x, *res;
  const void* w;
  void *h, *y;
  float *rstd, *scale;
  long long ldx, ldr;
  int M, D, w_f32;
  float eps;
};

// NORM = false: y is x itself (the quantisation alone)
template <int TPR, int NV, bool ODD, int XT, int RT, int YT, bool NORM>
__global__ __launch_bounds__(256) void rms_fwd(const RowArgs p) {
  constexpr int RPB = 256 / TPR;
  __shared__ float lds[2 * 4];
  int turn = 0;
  const int t = threadIdx.x % TPR;
  float w[NV][VEC];
  if constexpr (NORM) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + t) * VEC;
      if (c < p.D) {
        if (p.w_f32)
          load_vec<F32, ODD>(p.w, c, p.D - c, w[v]);
        else
          load_vec<T16, ODD>(p.w, c, p.D - c, w[v]);
      }
    }
  }
  const float inv_d = 1.f / (float)p.D;
  for (int row = blockIdx.x * RPB + threadIdx.x / TPR; row < p.M; row += gridDim.x * RPB) {
    float a[NV][VEC];
    const size_t xo = (size_t)row * p.ldx, ro = (size_t)row * p.ldr, o = (size_t)row * p.D;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + t) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[v][e] = 0.f;
      if (c < p.D) load_vec<XT, ODD>(p.x, xo + c, p.D - c, a[v]);
    }
    if constexpr (RT != NONE) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + t) * VEC;
        if (c < p.D) {
          float r[VEC];
          load_vec<RT, ODD>(p.res, ro + c, p.D - c, r);
#pragma unroll
          for (int e = 0; e < VEC; ++e) a[v][e] = as_stored<RT>(a[v][e] + r[e]);
          store_vec<RT, ODD>(p.h, o + c, p.D - c, a[v]);
        }
      }
    }
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += a[v][e] * a[v][e];
      const float r = rsqrtf(row_sum<TPR>(ss, lds, turn) * inv_d + p.eps);
      if (p.rstd && t == 0) p.rstd[row] = r;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + t) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[v][e] = c + (ODD ? e : 0) < p.D ? a[v][e] * r * w[v][e] : 0.f;
      }
    }
    if constexpr (YT == F8) {
      // the largest |y| as the largest bit pattern without its sign: a NaN's is above every number's, so that a row with a NaN gets a
      // NaN as its scale and reads back as NaN (fmaxf would drop it)
      unsigned m = 0;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = max(m, __float_as_uint(a[v][e]) & 0x7fffffffu);
      const float amax = __uint_as_float(row_umax<TPR>(m, lds, turn));
      const float scale = (amax < AMAX_MIN ? AMAX_MIN : amax) / E4M3_MAX, inv = 1.f / scale;
      if (t == 0) p.scale[row] = scale;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          // y / scale to the last bit by one correction of y * inv (Markstein): 16-bit values quantised by a power-of-two multiple of
          // 7 lie exactly between two e4m3 values often enough that the last bit shows
          const float q = a[v][e] * inv;
          const float c = __builtin_fmaf(__builtin_fmaf(-q, scale, a[v][e]), inv, q);
          a[v][e] = c;
        }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + t) * VEC;
      if (c < p.D) store_vec<YT, ODD>(p.y, o + c, p.D - c, a[v]);
    }
  }
}

struct BwdArgs {
  const void *dy, *dh, *h, *w;
  const float* rstd;
  void *dx, *dres;
  float* part;   // [gridDim.x][D]
  int M, D, w_f32;
};

// XT: the type of dy and dx; HT: the type of h, dh and dres.  Blocks of NT threads, a row to a wave (TPR = 64) or to the block (TPR = NT).
template <int NT, int TPR, int NV, bool ODD, int XT, int HT>
__global__ __launch_bounds__(NT) void rms_bwd(const BwdArgs p) {
  constexpr int RPB = NT / TPR;
  static_assert(RPB == 1 || TPR == 64, "rows that share a barrier would have to end together");
  extern __shared__ float lds[];   // TPR = 64: D floats (the block's sum of d w); else 2 * 8 words of the row sums
  int turn = 0;
  const int t = threadIdx.x % TPR;
  float w[NV][VEC], acc[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * TPR + t) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[v][e] = acc[v][e] = 0.f;
    if (c < p.D) {
      if (p.w_f32)
        load_vec<F32, ODD>(p.w, c, p.D - c, w[v]);
      else
        load_vec<T16, ODD>(p.w, c, p.D - c, w[v]);
    }
  }
  const float inv_d = 1.f / (float)p.D;
  for (int row = blockIdx.x * RPB + threadIdx.x / TPR; row < p.M; row += gridDim.x * RPB) {
    float g[NV][VEC], h[NV][VEC];
    const size_t o = (size_t)row * p.D;
    const float r = p.rstd[row];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + t) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[v][e] = h[v][e] = 0.f;
      if (c < p.D) {
        load_vec<HT, ODD>(p.h, o + c, p.D - c, h[v]);
        load_vec<XT, ODD>(p.dy, o + c, p.D - c, g[v]);
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        h[v][e] *= r;
        acc[v][e] += g[v][e] * h[v][e];
        g[v][e] *= w[v][e];
        dot += g[v][e] * h[v][e];
      }
    const float mean = row_sum<TPR>(dot, lds, turn) * inv_d;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + t) * VEC;
      if (c < p.D) {
        float d[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] = 0.f;
        if (p.dh) load_vec<HT, ODD>(p.dh, o + c, p.D - c, d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[e] += r * (g[v][e] - h[v][e] * mean);
        if (p.dx) store_vec<XT, ODD>(p.dx, o + c, p.D - c, d);
        if (p.dres) store_vec<HT, ODD>(p.dres, o + c, p.D - c, d);
      }
    }
  }
  if (!p.part) return;
  float* out = p.part + (size_t)blockIdx.x * p.D;
  if constexpr (TPR == 64) {
    for (int c = threadIdx.x; c < p.D; c += NT) lds[c] = 0.f;
    __syncthreads();
    for (int k = 0; k < NT / 64; ++k) {   // wave after wave: a fixed order
      if ((int)(threadIdx.x >> 6) == k) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const int c = (v * TPR + t) * VEC;
          if (c < p.D)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
              if (!ODD || c + e < p.D) lds[c + e] += acc[v][e];
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < p.D; c += NT) out[c] = lds[c];
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + t) * VEC;
      if (c < p.D) store_vec<F32, ODD>(out, c, p.D - c, acc[v]);
    }
  }
}

constexpr int MAX_D = 16384, MAX_M = 1 << 30;   // (row numbers run past M by a grid's stride)

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <int TPR, int NV, bool ODD, int XT, int RT, int YT, bool NORM>
int launch_fwd(const RowArgs& a, hipStream_t s) {
  const int rpb = 256 / TPR;
  // rounds of the grid stride: [20816, 1536] bf16 to 8 bits 40 us with 8 blocks a CU, 37 with 16, 39 with as many as there are rows for
  const long long need = ((long long)a.M + rpb - 1) / rpb, most = (long long)mvit_num_cus() * 16;
  hipLaunchKernelGGL((rms_fwd<TPR, NV, ODD, XT, RT, YT, NORM>), dim3((unsigned)(need < most ? need : most)), dim3(256), 0, s, a);
  return MVIT_LAUNCH_CHECK();
}

template <bool ODD, int XT, int RT, int YT, bool NORM>
int fwd_layout(const RowArgs& a, hipStream_t s) {
  const int D = a.D;
  // a wave a row, or 256 threads (f32 stream to 8 bits, us): rows of 512: 1024 of them 3.1 / 3.8, 8192 9.1 / 12.1; of 1024: 256 3.4 / 3.2,
  // 1024 4.1 / 4.3, 8192 15.7 / 16.5; of 1536: 256 4.1 / 3.4, 2048 7.6 / 6.9, 4096 12.0 / 13.2; of 4096: 64 6.9 / 3.7,
  // 8192 83 / 75
  if (D <= 512) return launch_fwd<64, 1, ODD, XT, RT, YT, NORM>(a, s);
  if (D <= 2048 && a.M >= (D <= 1024 ? 4 : 12) * mvit_num_cus()) {
    if (D <= 1024) return launch_fwd<64, 2, ODD, XT, RT, YT, NORM>(a, s);
    if (D <= 1536) return launch_fwd<64, 3, ODD, XT, RT, YT, NORM>(a, s);
    return launch_fwd<64, 4, ODD, XT, RT, YT, NORM>(a, s);
  }
  if (D <= 2048) return launch_fwd<256, 1, ODD, XT, RT, YT, NORM>(a, s);
  if (D <= 4096) return launch_fwd<256, 2, ODD, XT, RT, YT, NORM>(a, s);
  if (D <= 8192) return launch_fwd<256, 4, ODD, XT, RT, YT, NORM>(a, s);
  return launch_fwd<256, 8, ODD, XT, RT, YT, NORM>(a, s);
}
template <int XT, int RT, int YT, bool NORM>
int fwd_layout(const RowArgs& a, bool even, hipStream_t s) {
  return even ? fwd_layout<false, XT, RT, YT, NORM>(a, s) : fwd_layout<true, XT, RT, YT, NORM>(a, s);
}

// every row of every operand starts on 16 bytes (8 for the e4m3 output, whose rows are D bytes)
bool vec_ok(const RowArgs& a) {
  return a.D % 8 == 0 && a.ldx % 8 == 0 && (!a.res || a.ldr % 8 == 0) && aligned16(a.x) && aligned16(a.res) && aligned16(a.h) && aligned16(a.y) &&
         aligned16(a.w);
}

// (an empty tensor has no address: pointers are asked for where there are rows)
bool rows_bad(const RowArgs& a) {
  if (a.M < 0 || a.M > MAX_M || a.D <= 0 || a.D > MAX_D) return true;
  return a.M > 0 && (!a.x || !a.y || a.ldx < a.D || (a.res && (!a.h || a.ldr < a.D)));
}

// blocks of the backward pass at most, and so partial sums of d w: a CU's 1024 threads
int bwd_blocks(int M, int nt) {
  const long long most = (long long)mvit_num_cus() * (1024 / nt);
  return (int)(M < most ? M : most);
}

template <int NT, int TPR, int NV, bool ODD, int XT, int HT>
int launch_bwd(const BwdArgs& a, int& grid, hipStream_t s) {
  const size_t lds = TPR == 64 ? (size_t)a.D * 4 : 64;
  constexpr int RPB = NT / TPR;
  grid = bwd_blocks((a.M + RPB - 1) / RPB, NT);
  hipLaunchKernelGGL((rms_bwd<NT, TPR, NV, ODD, XT, HT>), dim3(grid), dim3(NT), lds, s, a);
  return MVIT_LAUNCH_CHECK();
}

template <bool ODD, int XT, int HT>
int bwd_layout(const BwdArgs& a, int& grid, hipStream_t s) {
  const int D = a.D;
  // f32 stream, with d w, us.  A wave a row or a block: rows of 1024: 1024 of them 9.6 / 8.1, 4096 17.5 / 17.7, 8192 26 / 28, 21056 69 / 87;
  // of 1536: 21056 107 / 105; of 2048: 140 / 127.  A row to 256 threads or to 512: of 1536: 1024 11.1 / 9.0 (twice the partial sums of
  // d w), 8192 35 / 34, 21056 96 / 105; of 2048: 131 / 126.  Rows that leave most of 512 threads without a piece go to 256 sooner: of 520: 2000 10.7 /
  // 10.7, 4000 12.2 / 15.0; of 768: 4000 13.5 / 15.3; of 1053 (odd): 1000 13.3 / 11.1, 4000 22.8 / 28.0, 8000 36 / 49; of 1280: 2000 12.4 / 11.6,
  // 4000 18.0 / 18.2
  if (D <= 512) return launch_bwd<512, 64, 1, ODD, XT, HT>(a, grid, s);
  if (D <= 1024 && a.M >= 16 * mvit_num_cus()) return launch_bwd<512, 64, 2, ODD, XT, HT>(a, grid, s);
  if (D <= 1920 && a.M >= (D <= 1280 ? 8 : 32) * mvit_num_cus()) return launch_bwd<256, 256, 1, ODD, XT, HT>(a, grid, s);
  if (D <= 4096) return launch_bwd<512, 512, 1, ODD, XT, HT>(a, grid, s);
  if (D <= 8192) return launch_bwd<512, 512, 2, ODD, XT, HT>(a, grid, s);
  return launch_bwd<512, 512, 4, ODD, XT, HT>(a, grid, s);
}
template <int XT, int HT>
int bwd_layout(const BwdArgs& a, bool even, int& grid, hipStream_t s) {
  return even ? bwd_layout<false, XT, HT>(a, grid, s) : bwd_layout<true, XT, HT>(a, grid, s);
}

}  // namespace

extern "C" MVIT_API int mvit_rmsnorm_fwd(const void* x, int x_f32, long long ldx, const void* res, int res_f32, long long ldr, const void* w,
                                         int w_f32, void* h, void* y, int y_f32, float* rstd, int M, int D, float eps, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  const RowArgs a = {x, res, w, h, y, rstd, nullptr, ldx, ldr, M, D, w_f32, eps};
  if (rows_bad(a) || !w || (!x_f32 && y_f32) || (x_f32 && res && !res_f32)) return MVIT_EINVAL;
  if (M == 0) return MVIT_OK;
  const bool v = vec_ok(a);
  hipStream_t s = (hipStream_t)stream;
  if (!x_f32) {
    if (!res) return fwd_layout<T16, NONE, T16, true>(a, v, s);
    return res_f32 ? fwd_layout<T16, F32, T16, true>(a, v, s) : fwd_layout<T16, T16, T16, true>(a, v, s);
  }
  if (!res) return y_f32 ? fwd_layout<F32, NONE, F32, true>(a, v, s) : fwd_layout<F32, NONE, T16, true>(a, v, s);
  return y_f32 ? fwd_layout<F32, F32, F32, true>(a, v, s) : fwd_layout<F32, F32, T16, true>(a, v, s);
}

extern "C" MVIT_API int mvit_rmsnorm_fp8_fwd(const void* x, int x_f32, long long ldx, const void* res, int res_f32, long long ldr,
                                             const void* w, int w_f32, void* h, void* q, float* scale, int M, int D, float eps,
                                             mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  const RowArgs a = {x, res, w, h, q, nullptr, scale, ldx, ldr, M, D, w_f32, eps};
  if (rows_bad(a) || !w || (M > 0 && !scale) || (x_f32 && res && !res_f32)) return MVIT_EINVAL;
  if (M == 0) return MVIT_OK;
  const bool v = vec_ok(a);
  hipStream_t s = (hipStream_t)stream;
  if (!x_f32) {
    if (!res) return fwd_layout<T16, NONE, F8, true>(a, v, s);
    return res_f32 ? fwd_layout<T16, F32, F8, true>(a, v, s) : fwd_layout<T16, T16, F8, true>(a, v, s);
  }
  return res ? fwd_layout<F32, F32, F8, true>(a, v, s) : fwd_layout<F32, NONE, F8, true>(a, v, s);
}

extern "C" MVIT_API int mvit_quantize_rows_fp8(const void* x, int x_f32, long long ldx, void* q, float* scale, int M, int D,
                                               mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  const RowArgs a = {x, nullptr, nullptr, nullptr, q, nullptr, scale, ldx, 0, M, D, 0, 0.f};
  if (rows_bad(a) || (M > 0 && !scale)) return MVIT_EINVAL;
  if (M == 0) return MVIT_OK;
  const bool v = vec_ok(a);
  return x_f32 ? fwd_layout<F32, NONE, F8, false>(a, v, (hipStream_t)stream) : fwd_layout<T16, NONE, F8, false>(a, v, (hipStream_t)stream);
}

extern "C" MVIT_API long long mvit_rmsnorm_bwd_scratch_bytes(int M, int D) {
  return M <= 0 || D <= 0 ? 0 : (long long)bwd_blocks(M, 256) * D * 4;
}

extern "C" MVIT_API int mvit_rmsnorm_bwd(const void* dy, int x_f32, const void* dh, const void* h, int h_f32, const void* w, int w_f32,
                                         const float* rstd, void* dx, void* dres, void* dw, void* scratch, long long scratch_bytes, int M,
                                         int D, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  if (M < 0 || M > MAX_M || D <= 0 || D > MAX_D || !w || (M > 0 && (!dy || !h || !rstd)) || (x_f32 && !h_f32)) return MVIT_EINVAL;
  if (dw && M > 0 && (!scratch || scratch_bytes < mvit_rmsnorm_bwd_scratch_bytes(M, D))) return MVIT_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  int grid = 0;
  if (M > 0) {
    const BwdArgs a = {dy, dh, h, w, rstd, dx, dres, dw ? (float*)scratch : nullptr, M, D, w_f32};
    const bool v = D % 8 == 0 && aligned16(dy) && aligned16(dh) && aligned16(h) && aligned16(w) && aligned16(dx) && aligned16(dres) && aligned16(scratch);
    int rc;
    if (x_f32)
      rc = bwd_layout<F32, F32>(a, v, grid, s);
    else
      rc = h_f32 ? bwd_layout<T16, F32>(a, v, grid, s) : bwd_layout<T16, T16>(a, v, grid, s);
    if (rc) return rc;
  }
  if (dw) {
    return launch_sum_parts((const float*)scratch, dw, grid, D, w_f32, s);
  }
  return MVIT_OK;
}
