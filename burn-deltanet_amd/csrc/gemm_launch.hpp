// Launches of the tile kernel for one operand type (included by the files
// that hold its instantiations).
#pragma once

#include "gemm.hpp"
#include "layer.hpp"

namespace dn {
namespace {

template <class T, class TO, bool ACOL, bool BCOL, int BM, int BN, int WM, int WN, int WK,
          int RING, int EPI, bool STAGED>
hipError_t gemm_go(const GemmArgs& g, hipStream_t stream) {
  const auto fn = gemm_kernel<T, TO, ACOL, BCOL, BM, BN, WM, WN, WK, RING, EPI, STAGED>;
  const int64_t total = int64_t(g.tiles_m) * g.tiles_n * g.npair * g.split;
  hipLaunchKernelGGL(fn, dim3(unsigned(total)), dim3(64 * WM * WN * WK), 0, stream, g);
  return hipGetLastError();
}

template <class T, class TO, bool ACOL, bool BCOL, int EPI, bool STAGED>
hipError_t gemm_tile(const GemmArgs& g, GemmTile tile, hipStream_t stream) {
  if constexpr (!STAGED && sizeof(T) < 4) {
    if (tile == kTileWide) {
      hipLaunchKernelGGL((gemm_wide_kernel<T, TO, ACOL, BCOL, EPI>), dim3(unsigned(g.split)),
                         dim3(256), 0, stream, g);
      return hipGetLastError();
    }
  }
  // Two tiles in flight: bf16 512 x 2048 x 4096 20.1 -> 18.1 us. 8-bit and fp32
  // products are bound by widening and the matrix unit, and have more workgroups
  // to a CU with one: 8-bit 4096 x 4096 x 2048 74 -> 69 us.
  constexpr int kRing = !STAGED && sizeof(T) == 2 ? 3 : 2;
  if (tile == kTile64)
    return gemm_go<T, TO, ACOL, BCOL, 64, 64, 2, 1, 2, kRing, EPI, STAGED>(g, stream);
  if constexpr (!STAGED && sizeof(T) < 4)
    if (tile == kTileLone)
      return gemm_go<T, TO, ACOL, BCOL, 128, 128, 2, 2, 2, kRing, EPI, STAGED>(g, stream);
  return gemm_go<T, TO, ACOL, BCOL, 128, 128, 2, 2, 1, 2, EPI, STAGED>(g, stream);
}

}  // namespace
}  // namespace dn
