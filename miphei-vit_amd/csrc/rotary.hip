// Rotary positions with several axes (row and column of a patch; time, height and width of a focal stack or a video).
//
// Pair i of a head's leading 2P values turns by angle = position[axis(i)] * inv_freq[i], the pairs shared out to the axes in `sections`:
//   (a, b) -> (a cos - b sin, b cos + a sin)
// with (a, b) = values (i, i + P), or (2i, 2i + 1) where interleaved.  The gradient is the same turn by the negative angle.
//
// Bound by HBM (each value in once, out once); the sines cost as much as the rest if every head computed them again, so
//  * a block takes one token (as many as give its 256 threads work, where heads are few) and writes its P (cos, sin) pairs into LDS
//    once; all heads of q and k read them from there.  One token a block keeps the most loads on their way: packed bf16 [64, 329, 72, 64]
//    forward and backward 135 us, 144 with two tokens a block, 152 with four; f32 [1, 10376, 16, 128] head-major 32 / 36 / 40 us
//    (5.7 and 5.4 TB/s);
//  * an angle is formed and reduced to one revolution in f64 (position * inv_freq / 2 pi: a far position's angle in f32 is off by more
//    than a bf16 step from position 2^14 on), the sine of the remainder in f32;
//  * a thread moves VEC values of both halves of a pair block (16-byte loads at VEC = 8 and 16-bit values).
// Tokens before `prefix` (class and register tokens), heads from `rotate_heads` on (v of a packed projection) and values from 2P on pass
// through; where the output is the input, they are not touched at all.
#include "common.hpp"
#include "../../include/miphei_hip.h"

namespace {

struct RotArgs {
  const void* x;
  void* y;
  const void* pos;
  const void* freq;
  long long xb, xn, xh, yb, yn, yh;   // strides in elements of [B, N, H, Dh] (the last one is 1)
  long long pos_b;                    // elements between the positions of two batch entries (0: shared)
  int B, N, H, Dh, rot, prefix, P, axes;
  int end[4];                         // pair index where each axis' section ends
  int pos_type, freq_f64;             // 0 int32, 1 int64, 2 f32
  float sign;
  int copy;                           // 0: in place, nothing passes through
  unsigned rot_units, pass_units;     // units of a token: a thread's work at once
  int tokens;                         // of a block
  unsigned per_magic;
  unsigned rpu, rpu_magic;            // rotated units of a head
  unsigned tail, tail_magic;          // passing units of a rotated head
  unsigned full, full_magic;          // units of a whole head
};

template <bool F, int VEC>
struct Piece {
  float v[VEC];
  __device__ __forceinline__ void load(const void* p, size_t i) {
    if constexpr (F) {
      if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
          const float4 a = *(const float4*)((const float*)p + i + e);
          v[e] = a.x, v[e + 1] = a.y, v[e + 2] = a.z, v[e + 3] = a.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = ((const float*)p)[i + e];
      }
    } else if constexpr (VEC % 2 == 0) {
      uint32_t u[VEC / 2];
      if constexpr (VEC == 8)
        *(uint4*)u = *(const uint4*)((const bf16_t*)p + i);
      else if constexpr (VEC == 4)
        *(uint2*)u = *(const uint2*)((const bf16_t*)p + i);
      else
        u[0] = (uint32_t)((const bf16_t*)p)[i] | ((uint32_t)((const bf16_t*)p)[i + 1] << 16);
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) v[2 * e] = lo16f(u[e]), v[2 * e + 1] = hi16f(u[e]);
    } else {
      v[0] = bf2f(((const bf16_t*)p)[i]);
    }
  }
  __device__ __forceinline__ void store(void* p, size_t i) const {
    if constexpr (F) {
      if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) *(float4*)((float*)p + i + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) ((float*)p)[i + e] = v[e];
      }
    } else if constexpr (VEC % 2 == 0) {
      uint32_t u[VEC / 2];
#pragma unroll
      for (int e = 0; e < VEC / 2; ++e) u[e] = pack2bf(v[2 * e], v[2 * e + 1]);
      if constexpr (VEC == 8)
        *(uint4*)((bf16_t*)p + i) = *(uint4*)u;
      else if constexpr (VEC == 4)
        *(uint2*)((bf16_t*)p + i) = *(uint2*)u;
      else
        ((bf16_t*)p)[i] = (bf16_t)(u[0] & 0xffffu), ((bf16_t*)p)[i + 1] = (bf16_t)(u[0] >> 16);
    } else {
      ((bf16_t*)p)[i] = f2bf(v[0]);
    }
  }
};

// the bits themselves for what passes through (a NaN's payload survives)
template <bool F, int VEC>
__device__ __forceinline__ void copy_piece(const void* x, size_t i, void* y, size_t o) {
  constexpr int BYTES = VEC * (F ? 4 : 2);
  const char* s = (const char*)x + i * (F ? 4 : 2);
  char* d = (char*)y + o * (F ? 4 : 2);
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int e = 0; e < BYTES; e += 16) *(uint4*)(d + e) = *(const uint4*)(s + e);
  } else if constexpr (VEC == 4) {
    *(uint2*)d = *(const uint2*)s;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if constexpr (F)
        ((uint32_t*)d)[e] = ((const uint32_t*)s)[e];
      else
        ((bf16_t*)d)[e] = ((const bf16_t*)s)[e];
    }
  }
}

template <bool F, int VEC, bool IL>
__global__ __launch_bounds__(256) void rotary_kernel(const RotArgs p) {
  extern __shared__ float2 turn[];   // [tokens of the block][P]
  const int tid = threadIdx.x, b = blockIdx.y;
  for (int n0 = blockIdx.x * p.tokens; n0 < p.N; n0 += gridDim.x * p.tokens) {   // (once, but for millions of tokens)
    const int nt = min(p.tokens, p.N - n0);
    for (int i = tid; i < nt * p.P; i += 256) {
      const int k = i / p.P, pair = i - k * p.P, n = n0 + k - p.prefix;
      if (n < 0) continue;
      const int axis = (pair >= p.end[0]) + (pair >= p.end[1]) + (pair >= p.end[2]);
      const size_t at = (size_t)b * p.pos_b + (size_t)n * p.axes + axis;
      const double f = p.freq_f64 ? ((const double*)p.freq)[pair] : (double)((const float*)p.freq)[pair];
      const double q = p.pos_type == 0 ? (double)((const int*)p.pos)[at] : p.pos_type == 1 ? (double)((const long long*)p.pos)[at] : (double)((const float*)p.pos)[at];
      double rev = q * f * 0.15915494309189533577;   // 1 / 2 pi
      rev -= rint(rev);
      float s, c;
      sincospif((float)(2.0 * rev), &s, &c);
      turn[i] = make_float2(c, s * p.sign);
    }
    __syncthreads();
    const unsigned per = p.rot_units + p.pass_units;
    for (unsigned i = tid; i < (unsigned)nt * per; i += 256) {
      const unsigned k = p.tokens == 1 ? 0u : mvit_fast_div(i, per, p.per_magic), u = i - k * per;
      const int n = n0 + (int)k;
      const size_t xt = (size_t)b * p.xb + (size_t)n * p.xn, yt = (size_t)b * p.yb + (size_t)n * p.yn;
      if (u < p.rot_units) {
        const unsigned h = mvit_fast_div(u, p.rpu, p.rpu_magic), j = (u - h * p.rpu) * VEC;
        const size_t xi = xt + (size_t)h * p.xh + j, yi = yt + (size_t)h * p.yh + j;
        if (n < p.prefix) {   // the whole token passes
          if (p.copy) {
            copy_piece<F, VEC>(p.x, xi, p.y, yi);
            if constexpr (!IL) copy_piece<F, VEC>(p.x, xi + p.P, p.y, yi + p.P);
          }
          continue;
        }
        const float2* cs = turn + k * p.P + (IL ? j / 2 : j);
        Piece<F, VEC> a;
        a.load(p.x, xi);
        if constexpr (IL) {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            const float2 t = cs[e / 2];
            const float u0 = a.v[e], u1 = a.v[e + 1];
            a.v[e] = u0 * t.x - u1 * t.y;
            a.v[e + 1] = u1 * t.x + u0 * t.y;
          }
        } else {
          Piece<F, VEC> c;
          c.load(p.x, xi + p.P);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float2 t = cs[e];
            const float u0 = a.v[e], u1 = c.v[e];
            a.v[e] = u0 * t.x - u1 * t.y;
            c.v[e] = u1 * t.x + u0 * t.y;
          }
          c.store(p.y, yi + p.P);
        }
        a.store(p.y, yi);
      } else {
        unsigned v = u - p.rot_units, h, j;
        if (v < (unsigned)p.rot * p.tail) {   // tails of the rotated heads
          h = mvit_fast_div(v, p.tail, p.tail_magic);
          j = 2 * p.P + (v - h * p.tail) * VEC;
        } else {                              // heads that pass
          v -= (unsigned)p.rot * p.tail;
          h = mvit_fast_div(v, p.full, p.full_magic);
          j = (v - h * p.full) * VEC;
          h += p.rot;
        }
        copy_piece<F, VEC>(p.x, xt + (size_t)h * p.xh + j, p.y, yt + (size_t)h * p.yh + j);
      }
    }
    __syncthreads();
  }
}

template <bool F, int VEC, bool IL>
int launch(RotArgs a, hipStream_t s) {
  const unsigned rpu = (unsigned)(IL ? 2 * a.P : a.P) / VEC, tail = (unsigned)(a.Dh - 2 * a.P) / VEC, full = (unsigned)a.Dh / VEC;
  a.rpu = rpu, a.rpu_magic = mvit_div_magic(rpu);
  a.tail = tail, a.tail_magic = mvit_div_magic(tail);
  a.full = full, a.full_magic = mvit_div_magic(full);
  a.rot_units = (unsigned)a.rot * rpu;
  a.pass_units = a.copy ? (unsigned)a.rot * tail + (unsigned)(a.H - a.rot) * full : 0u;
  const unsigned per = a.rot_units + a.pass_units;
  if (per == 0) return MVIT_OK;   // (in place with no head to turn)
  a.tokens = per >= 256 ? 1 : 256 / per < 32 ? 256 / per : 32;
  a.per_magic = mvit_div_magic(per);
  const int groups = (a.N + a.tokens - 1) / a.tokens;
  const dim3 grid(groups < (1 << 22) ? groups : 1 << 22, a.B);   // (a grid has fewer than 2^32 threads in a dimension)
  hipLaunchKernelGGL((rotary_kernel<F, VEC, IL>), grid, dim3(256), (size_t)a.tokens * a.P * sizeof(float2), s, a);
  return MVIT_LAUNCH_CHECK();
}

template <bool F, bool IL>
int layout(const RotArgs& a, hipStream_t s) {
  // the widest piece that divides every stride, the rotated part and the head, and that the addresses are aligned to
  const long long strides = a.xb | a.xn | a.xh | a.yb | a.yn | a.yh | a.Dh | (IL ? 2 * a.P : a.P);
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.y;
  auto fits = [&](int vec) { return strides % vec == 0 && (at & (uintptr_t)((vec * (F ? 4 : 2) > 16 ? 16 : vec * (F ? 4 : 2)) - 1)) == 0; };
  if (fits(8)) return launch<F, 8, IL>(a, s);
  if (fits(4)) return launch<F, 4, IL>(a, s);
  return launch<F, IL ? 2 : 1, IL>(a, s);
}

}  // namespace

extern "C" MVIT_API int mvit_rotary(const mvit_rotary_args* args, mvit_stream_t stream) {
  MVIT_CLEAR_ERROR();
  if (!args) return MVIT_EINVAL;
  const mvit_rotary_args& g = *args;
  if (!g.x || !g.y || !g.inv_freq || g.B < 0 || g.N < 0 || g.H <= 0 || g.Dh <= 0 || (g.Dh & 1) || g.Dh > 1024 || g.H > 1024 || g.B > 65535 || g.N > (1 << 30))
    return MVIT_EINVAL;   // H, Dh: the divisions by multiplication are exact below H * Dh^2 = 2^32
  if (g.rotate_heads < 0 || g.rotate_heads > g.H || g.prefix < 0 || g.prefix > g.N || g.axes < 1 || g.axes > 4) return MVIT_EINVAL;
  if (g.pos_type < 0 || g.pos_type > 2 || (g.prefix < g.N && !g.positions)) return MVIT_EINVAL;
  RotArgs a = {};
  int P = 0;
  for (int k = 0; k < 4; ++k) {
    if (k < g.axes) {
      if (g.sections[k] < 0) return MVIT_EINVAL;
      P += g.sections[k];
      if (2 * P > g.Dh) return MVIT_EINVAL;
    }
    a.end[k] = k < g.axes - 1 ? P : 1 << 30;   // the last axis' section has no end to pass
  }
  if (P <= 0) return MVIT_EINVAL;
  if (g.B == 0 || g.N == 0) return MVIT_OK;
  a.x = g.x, a.y = g.y, a.pos = g.positions, a.freq = g.inv_freq;
  a.xb = g.xb, a.xn = g.xn, a.xh = g.xh, a.yb = g.yb, a.yn = g.yn, a.yh = g.yh, a.pos_b = g.pos_b;
  a.B = g.B, a.N = g.N, a.H = g.H, a.Dh = g.Dh, a.rot = g.rotate_heads, a.prefix = g.prefix, a.P = P, a.axes = g.axes;
  a.pos_type = g.pos_type, a.freq_f64 = g.freq_f64, a.sign = g.inverse ? -1.f : 1.f, a.copy = g.x != g.y;
  hipStream_t s = (hipStream_t)stream;
  if (g.x_f32) return g.interleaved ? layout<true, true>(a, s) : layout<true, false>(a, s);
  return g.interleaved ? layout<false, true>(a, s) : layout<false, false>(a, s);
}
