// Products of 8-bit integers with rows at any byte (gemm_int8_any.hip).
#pragma once

#include "gemm_kernel.hpp"

namespace aitamd {

// K, lda and ldb of p count bytes (unlike those of the instances for i8x2, which count pairs)
hipError_t launch_gemm_int8_any(const GemmParams& p, bool bf16_out, int cus, hipStream_t stream);

// Rows of a [M, K] and of b [N, K] to `to_a` and `to_b`, (K + 15) / 16 * 16 bytes apart and zero behind byte K (M or N: 0 for an
// operand that stays where it is)
hipError_t launch_int8_align(const int8_t* a, int64_t lda, int64_t M, void* to_a, const int8_t* b, int64_t ldb, int64_t N, void* to_b, int64_t K,
                             hipStream_t stream);
// Whether that is worth it for rows of K bytes.  us, as they lie / laid out first: 1 x 4097, K 513 5.7 / 7.4, 1101 8.0 / 8.8, 4095
// 26.6 / 14.8; 64 x 1001 6.9 / 6.9, 9.6 / 7.1, 25.0 / 12.4; 777 x 2731 11.7 / 11.3, 17.1 / 14.7, 44.9 / 27.0; 2048 x 4096 19.9 / 22.4,
// 30.8 / 26.6, 74.0 / 48.1; K 257: 4.5 / 7.1, 5.5 / 6.8, 9.6 / 10.1, 15.6 / 14.3.
inline bool int8_align_pays(int64_t K) { return K > 512; }

}  // namespace aitamd
