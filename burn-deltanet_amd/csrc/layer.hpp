// The operators around the mixer: plans and launches shared by their files.
#pragma once

#include "gemm.hpp"

namespace dn {

// gemm_wide_kernel; gemm_kernel, 128 × 128 and 64 × 64; few_rows_kernel.
enum GemmTile { kTileWide, kTile128, kTileLone, kTile64, kTileFew };
// Operand layouts of a product (gemm.hpp): x·W, dz·Wᵀ, xᵀ·dz.
enum GemmForm { kFormNN, kFormNT, kFormTN };

hipError_t gemm_bf16(const GemmArgs& g, GemmForm form, GemmEpi epi, GemmTile tile, bool staged,
                     hipStream_t stream);
hipError_t gemm_f32(const GemmArgs& g, GemmForm form, GemmEpi epi, GemmTile tile, bool staged,
                    hipStream_t stream);
// dz·Wᵀ's form only, 16-byte rows.
hipError_t gemm_f8(const GemmArgs& g, int out_dtype, GemmTile tile, hipStream_t stream);

// Forwards of few rows (few_rows.hip): x·W, 8-bit x·Wᵀ, the gated pair.
int few_rows_most(GemmEpi epi);
int few_rows_split(const GemmArgs& g, GemmEpi epi, int dtype, bool copyable);
hipError_t few_rows(const GemmArgs& g, GemmEpi epi, int dtype, int out_dtype, bool copyable,
                    hipStream_t stream);

hipError_t launch_add_rms_norm(const dn_add_rms_norm_args& a, hipStream_t stream);
size_t add_rms_norm_bwd_workspace(const dn_add_rms_norm_bwd_args& a);
hipError_t launch_add_rms_norm_bwd(const dn_add_rms_norm_bwd_args& a, void* ws, hipStream_t stream);
size_t linear_workspace(const dn_linear_args& a);
hipError_t launch_linear(const dn_linear_args& a, void* ws, hipStream_t stream);
size_t linear_bwd_workspace(const dn_linear_bwd_args& a);
hipError_t launch_linear_bwd(const dn_linear_bwd_args& a, void* ws, hipStream_t stream);
size_t gated_ffn_workspace(const dn_gated_ffn_args& a);
hipError_t launch_gated_ffn(const dn_gated_ffn_args& a, void* ws, hipStream_t stream);
size_t gated_ffn_bwd_workspace(const dn_gated_ffn_bwd_args& a);
hipError_t launch_gated_ffn_bwd(const dn_gated_ffn_bwd_args& a, void* ws, hipStream_t stream);

}  // namespace dn
