// The tile kernel on 8-bit (e4m3) operands, both with k fastest.
#include "gemm_launch.hpp"

namespace dn {
hipError_t gemm_f8(const GemmArgs& g, int out_dtype, GemmTile tile, hipStream_t stream) {
  if (out_dtype == DN_BF16)
    return gemm_tile<f8, bf16, false, false, kEpiLinear, false>(g, tile, stream);
  return gemm_tile<f8, float, false, false, kEpiLinear, false>(g, tile, stream);
}
}  // namespace dn
