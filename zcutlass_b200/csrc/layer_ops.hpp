// Launchers of the operators beside the GEMM: 8-bit quantisation, the 8-bit
// block-scaled product and rotary positions. Arguments have passed the checks
// in c_abi.cpp; each launcher only chooses a kernel and enqueues it.
#pragma once

#include "zcutlass_c.h"

#include <cuda_runtime_api.h>

namespace zcb {

cudaError_t launch_quantize_fp8(const zcutlass_quantize_desc& d, const void* x, void* q, float* scale, void* qt,
                                float* scale_t, float* col_sums);
cudaError_t launch_sum_rows(const float* part, int64_t rows, int64_t cols, void* out, int32_t out_type,
                            cudaStream_t stream);
cudaError_t launch_gemm_fp8(const zcutlass_fp8_gemm_desc& d, const void* a, const float* a_scale, const void* b,
                            const float* b_scale, void* out);
cudaError_t launch_rotary(const zcutlass_rotary_desc& d, const void* q, void* q_out, const void* k, void* k_out,
                          const void* positions, const float* table);

}  // namespace zcb
