// Products of 8-bit integers with rows at any byte (gemm_int8_any.hip).
#pragma once

#include "gemm_kernel.hpp"

namespace aitamd {

// K, lda and ldb of p count bytes (unlike those of the instances for i8x2, which count pairs)
hipError_t launch_gemm_int8_any(const GemmParams& p, bool bf16_out, int cus, hipStream_t stream);

}  // namespace aitamd
