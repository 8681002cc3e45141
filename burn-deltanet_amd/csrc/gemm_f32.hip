// The tile kernel on fp32 operands (fp32 matrix cores).
#include "gemm_launch.hpp"

namespace dn {
namespace {
template <bool STAGED>
hipError_t go(const GemmArgs& g, GemmForm form, GemmEpi epi, GemmTile tile, hipStream_t stream) {
  if (form == kFormNN && epi == kEpiGated)
    return gemm_tile<float, float, false, true, kEpiGated, STAGED>(g, tile, stream);
  if (form == kFormNN) return gemm_tile<float, float, false, true, kEpiLinear, STAGED>(g, tile, stream);
  if (form == kFormNT && epi == kEpiDGated)
    return gemm_tile<float, float, false, false, kEpiDGated, STAGED>(g, tile, stream);
  if (form == kFormNT) return gemm_tile<float, float, false, false, kEpiLinear, STAGED>(g, tile, stream);
  return gemm_tile<float, float, true, true, kEpiLinear, STAGED>(g, tile, stream);
}
}  // namespace

hipError_t gemm_f32(const GemmArgs& g, GemmForm form, GemmEpi epi, GemmTile tile, bool staged,
                     hipStream_t stream) {
  return staged ? go<true>(g, form, epi, tile, stream) : go<false>(g, form, epi, tile, stream);
}
}  // namespace dn
