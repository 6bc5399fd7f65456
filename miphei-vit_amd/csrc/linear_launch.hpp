// Launches of linear_kernel.hpp: which kernel forms a product.  One translation unit for each kind of operands and output includes this
// and instantiates its dispatch (linear_h16.hip and so on): the kernels of all are a minute of compilation.
#pragma once
#include "linear_kernel.hpp"

namespace mvit_linear {

template <int MODE, class E, int BM, int BN, int WM, int WN, int NST>
int launch_tile(const Args& a, hipStream_t s) {
  using T = Tile<MODE, BM, BN, WM, WN, NST>;
  const long long nt = (long long)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN) * a.splits;
  if (nt > 0x7fffffff) return MVIT_EINVAL;
  static mvit_per_device_size raised;
  const auto fn = linear_tile<MODE, E, BM, BN, WM, WN, NST>;
  if (const int rc = mvit_ensure_dynamic_lds((const void*)fn, T::LDS, raised)) return rc;
  const long long slots = (long long)mvit_num_cus() * T::BLOCKS_PER_CU;
  hipLaunchKernelGGL(fn, dim3((unsigned)(nt < slots ? nt : slots)), dim3(T::NT), T::LDS, s, a);
  return MVIT_LAUNCH_CHECK();
}

template <bool OP8, class E, int MT>
int launch_rows(const Args& a, hipStream_t s) {
  hipLaunchKernelGGL((linear_rows<OP8, E, MT>), dim3((a.N + 15) / 16, a.splits), dim3(512), 0, s, a);
  return MVIT_LAUNCH_CHECK();
}

// Rows or tiles, and which: by what a round of blocks costs.  A round is every CU's share at once (one tile of 256 columns, two of the
// others); measured at K = 1536, bf16, it takes 43 us with tiles of 256 x 256, 35 of 192 x 256, 24 of 128 x 256, 26 of 128 x 128 (20 with one
// a CU) and 12 of 64 x 64, and the ratios hold for e4m3 and other K within some per cent.  Large tiles read less of x and W; small ones
// leave less of the chip idle in the last round.  us, in that order:
//   [5264, 1536] x [4096, 1536]   72  63  72  76 113      [5264, 4096] x [1536, 4096]   78  68  58  60 104
//   [5264, 1536] x [8192, 1536]  115 125 140              [21056, 1536] x [1536, 1536]  88 102  99 109 174
//   [1301, 1536] x [4608, 1536]   36      24  25  34      [700, 1536] x [4096, 1536]            22  20  20
//   [329, 1536] x [4608, 1536]    34      22  20  13
template <int MODE, class E>
int by_size(const Args& a, hipStream_t s) {
  using Any = End<E::out32, A_ANY, E::vec>;   // (the row kernels' epilogue is not unrolled)
  const long long cus = mvit_num_cus();
  // few rows: [1, 1536] x [1536, 1536] bf16 5.8 us against 9.0 with tiles, [17, ..] 6.7 / 9.1, [32, 4096] x [1536, 4096] 14 / 18; from 33
  // rows on (9.0 / 9.2) and, from 17 on, with more than one block a CU (N > 4096) the tiles are as fast or faster
  if (a.M <= 16) return launch_rows<MODE != H16, Any, 1>(a, s);
  if (a.M <= 32 && a.N <= 16 * cus) return launch_rows<MODE != H16, Any, 2>(a, s);
  auto tiles = [&](long long bm, long long bn) { return ((a.M + bm - 1) / bm) * ((a.N + bn - 1) / bn); };
  auto rounds = [&](long long t, long long at_once) { return (t + at_once - 1) / at_once; };
  const long long t128 = tiles(128, 128);
  const long long cost[5] = {43 * rounds(tiles(256, 256), cus), 35 * rounds(tiles(192, 256), cus), 24 * rounds(tiles(128, 256), cus),
                             t128 <= cus ? 20 : 26 * rounds(t128, 2 * cus), 12 * rounds(tiles(64, 64), 2 * cus)};
  int best = 0;
  for (int k = 1; k < 5; ++k)
    if (cost[k] < cost[best]) best = k;
  switch (best) {
    case 0:
      return launch_tile<MODE, E, 256, 256, 2, 4, 2>(a, s);
    case 1:
      return launch_tile<MODE, E, 192, 256, 2, 4, 2>(a, s);
    case 2:
      return launch_tile<MODE, E, 128, 256, 2, 4, 3>(a, s);
    case 3:
      return launch_tile<MODE, E, 128, 128, 2, 2, 2>(a, s);
    default:
      return launch_tile<MODE, E, 64, 64, 2, 2, 4>(a, s);
  }
}

// The gradients' products: one of four tiles (plan_grad in linear.hip)
template <int MODE>
int dispatch_grad(const Args& a, int tile, hipStream_t s) {
  using E = End<false, A_CLIP, true>;
  switch (tile) {
    case 0:
      return launch_tile<MODE, E, 256, 256, 2, 4, 2>(a, s);
    case 1:
      return launch_tile<MODE, E, 128, 256, 2, 4, 3>(a, s);
    case 2:
      return launch_tile<MODE, E, 128, 128, 2, 2, 2>(a, s);
    default:
      return launch_tile<MODE, E, 64, 64, 2, 2, 4>(a, s);
  }
}

template <int MODE, bool OUT32, bool VEC>
int by_activation(const Args& a, hipStream_t s) {
  switch (a.act) {
    case MVIT_ACT_NONE:
    case MVIT_ACT_RELU:
      return by_size<MODE, End<OUT32, A_CLIP, VEC>>(a, s);
    case MVIT_ACT_GELU:
      return by_size<MODE, End<OUT32, A_ERF, VEC>>(a, s);
    case MVIT_ACT_SILU:
      return by_size<MODE, End<OUT32, A_SILU, VEC>>(a, s);
    default:
      return by_size<MODE, End<OUT32, A_TANH, VEC>>(a, s);
  }
}
// The products of parts of K, f32 (plan_parts in linear.hip): kind 0 by rows, else tiles of 128 x 128 (2) or 64 x 64 (3)
template <int MODE, bool VEC>
int parts_of(const Args& a, int kind, hipStream_t s) {
  using Any = End<true, A_ANY, VEC>;
  using Sum = End<true, A_CLIP, VEC>;
  if (kind == 0) return a.M <= 16 ? launch_rows<MODE != H16, Any, 1>(a, s) : launch_rows<MODE != H16, Any, 2>(a, s);
  return kind == 2 ? launch_tile<MODE, Sum, 128, 128, 2, 2, 2>(a, s) : launch_tile<MODE, Sum, 64, 64, 2, 2, 4>(a, s);
}
template <int MODE>
int dispatch_parts(const Args& a, bool vec, int kind, hipStream_t s) {
  return vec ? parts_of<MODE, true>(a, kind, s) : parts_of<MODE, false>(a, kind, s);
}
template <int MODE, bool OUT32>
int dispatch(const Args& a, bool vec, hipStream_t s) {
  return vec ? by_activation<MODE, OUT32, true>(a, s) : by_activation<MODE, OUT32, false>(a, s);
}

}  // namespace mvit_linear
