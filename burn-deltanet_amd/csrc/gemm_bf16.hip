// The tile kernel on bf16 operands.
#include "gemm_launch.hpp"

namespace dn {
namespace {
template <bool STAGED>
hipError_t go(const GemmArgs& g, GemmForm form, GemmEpi epi, GemmTile tile, hipStream_t stream) {
  if (form == kFormNN && epi == kEpiGated)
    return gemm_tile<bf16, bf16, false, true, kEpiGated, STAGED>(g, tile, stream);
  if (form == kFormNN) return gemm_tile<bf16, bf16, false, true, kEpiLinear, STAGED>(g, tile, stream);
  if (form == kFormNT && epi == kEpiDGated)
    return gemm_tile<bf16, bf16, false, false, kEpiDGated, STAGED>(g, tile, stream);
  if (form == kFormNT) return gemm_tile<bf16, bf16, false, false, kEpiLinear, STAGED>(g, tile, stream);
  return gemm_tile<bf16, bf16, true, true, kEpiLinear, STAGED>(g, tile, stream);
}
}  // namespace

hipError_t gemm_bf16(const GemmArgs& g, GemmForm form, GemmEpi epi, GemmTile tile, bool staged,
                     hipStream_t stream) {
  return staged ? go<true>(g, form, epi, tile, stream) : go<false>(g, form, epi, tile, stream);
}
}  // namespace dn
