// Sums of columns that many blocks have formed in part: out[c] = sum over k of part[k][c], part f32 [parts][n].  A block takes 32 columns
// with 32 groups of lanes, group g the parts g, g + 32, ... in order, and adds the groups in order: no atomics, the same bits every time.
#pragma once
#include "common.hpp"

namespace {

__global__ __launch_bounds__(1024) void sum_parts(const float* part, void* out, int parts, int n, int out_f32) {
  __shared__ float lds[32][33];
  const int l = threadIdx.x & 31, c = blockIdx.x * 32 + l, g = threadIdx.x >> 5;
  float s = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int k = g; k < parts; k += 32) s += part[(size_t)k * n + c];
  }
  lds[g][l] = s;
  __syncthreads();
  if (g == 0 && c < n) {
#pragma unroll
    for (int k = 1; k < 32; ++k) s += lds[k][l];
    if (out_f32)
      ((float*)out)[c] = s;
    else
      ((bf16_t*)out)[c] = f2bf(s);
  }
}

int launch_sum_parts(const float* part, void* out, int parts, int n, int out_f32, hipStream_t s) {
  hipLaunchKernelGGL(sum_parts, dim3((n + 31) / 32), dim3(1024), 0, s, part, out, parts, n, out_f32);
  return MVIT_LAUNCH_CHECK();
}

}  // namespace
