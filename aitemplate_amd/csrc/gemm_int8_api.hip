// C ABI of the products of 8-bit integers (apart from gemm_api.hip: a model library takes only what it calls).
#include "../../include/aitemplate_amd_kernels.h"
#include "errors.hpp"
#include "gemm_host.hpp"
#include "gemm_int8_any.hpp"

using namespace aitamd;

namespace {

// (of the scratch memory: what its users leave zero)
constexpr int64_t kCounterBytes = 4096;

// rows of K bytes of an operand laid out in scratch memory
int64_t laid_out(int64_t rows, int64_t K) { return rows * ((K + 15) / 16 * 16); }
// whether rows of K bytes, `pitch` apart, are no whole dwords
bool off_dwords(const int8_t* x, int64_t rows, int64_t K, int64_t pitch) {
  return ((K | (int64_t)reinterpret_cast<uintptr_t>(x) | (rows > 1 ? pitch : 0)) & 3) != 0;
}

}  // namespace

extern "C" {

int aitamd_gemm_rcr_int8(int dtype, int algo, const int8_t* a, const int8_t* b, const float* scale_a, const float* scale_b, const void* bias,
                         void* c, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int64_t ldc, void* workspace,
                         int64_t workspace_bytes, void* stream) {
  const char* who = "aitamd_gemm_rcr_int8";
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  if (M < 0 || N < 0 || K < 0) return fail("%s: negative dimension", who);
  if (M > 0x7fffffffll || N > 0x7fffffffll) return fail("%s: dimension too large", who);
  // (the sum of K products of -128 by -128 has to fit 32 bits)
  if (K > 131071) return fail("%s: K = %lld: up to 131071 products fit a 32-bit sum", who, (long long)K);
  if (M == 0 || N == 0) return 0;
  if (!c || !scale_a || !scale_b || (K > 0 && (!a || !b))) return fail("%s: null pointer", who);
  if (lda < K || ldb < K || ldc < N) return fail("%s: row pitch smaller than the row", who);
  if ((reinterpret_cast<uintptr_t>(scale_a) | reinterpret_cast<uintptr_t>(scale_b)) & 3) return fail("%s: the scales have to be 4-byte aligned", who);
  GemmParams p{};
  p.a = a, p.b = b, p.c = c, p.bias = bias;
  p.scale_a = scale_a, p.scale_b = scale_b;
  p.M = (int32_t)M, p.N = (int32_t)N, p.K = (int32_t)K;
  p.batch = 1;
  p.lda = lda, p.ldb = ldb, p.ldc = ldc;
  p.ws = workspace, p.ws_bytes = workspace ? workspace_bytes : 0;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // rows that are no whole dwords
  const bool odd_k = (K & 3) != 0, odd_a = off_dwords(a, M, K, lda), odd_b = off_dwords(b, N, K, ldb);
  if (odd_a || odd_b) {
    if (algo >= 0) return fail("%s: instance %d takes rows of whole dwords only", who, algo);
    // to the scratch memory, behind the counters of the instances that share tiles, which are zero and stay zero
    const int64_t row = laid_out(1, K), bytes_a = odd_a ? M * row : 0, bytes_b = odd_b ? N * row : 0;
    if (!int8_align_pays(K) || kCounterBytes + bytes_a + bytes_b > p.ws_bytes || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0) {
      const hipError_t e = launch_gemm_int8_any(p, dtype == AITAMD_BF16, current_device_cus(), s);
      return e == hipSuccess ? 0 : fail("%s: launch failed: %s", who, hipGetErrorString(e));
    }
    unsigned char* const at = static_cast<unsigned char*>(workspace) + kCounterBytes;
    const hipError_t e = launch_int8_align(a, lda, odd_a ? M : 0, at, b, ldb, odd_b ? N : 0, at + bytes_a, K, s);
    if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
    if (odd_a) p.a = at, lda = row;
    if (odd_b) p.b = at + bytes_a, ldb = row;
    if (odd_k) K = row;
    p.ws = nullptr, p.ws_bytes = 0;
  }
  // (rows further apart than the instances' 32-bit offsets reach over a tile of them)
  constexpr int64_t kFar = 1 << 22;
  if (algo < 0 && ((M > 1 && lda > kFar) || (N > 1 && ldb > kFar))) {
    p.lda = lda, p.ldb = ldb, p.K = (int32_t)K;
    const hipError_t e = launch_gemm_int8_any(p, dtype == AITAMD_BF16, current_device_cus(), s);
    return e == hipSuccess ? 0 : fail("%s: launch failed: %s", who, hipGetErrorString(e));
  }
  p.K = (int32_t)(K / 2), p.lda = M > 1 ? lda / 2 : K / 2, p.ldb = N > 1 ? ldb / 2 : K / 2;
  return run_gemm(bias ? kEpiBias : kEpiNone, dtype + kNumDTypes, algo, p, s);
}

int64_t aitamd_gemm_int8_layout_bytes(int64_t rows_a, int64_t rows_b, int64_t K) {
  if (rows_a < 0 || rows_b < 0 || rows_a + rows_b == 0 || K <= 0 || rows_a > 0x7fffffffll || rows_b > 0x7fffffffll || K > 131071) return 0;
  return int8_align_pays(K) ? kCounterBytes + laid_out(rows_a + rows_b, K) : 0;
}

int64_t aitamd_gemm_int8_workspace_bytes(int dtype, int algo, int bias, int64_t M, int64_t N, int64_t K) {
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return 0;
  const int epilogue = bias ? kEpiBias : kEpiNone;
  if (algo >= 0) return aitamd_gemm_workspace_bytes(epilogue, dtype + kNumDTypes, algo, 1, M, N, K / 2);
  if (M <= 0 || N <= 0 || K <= 0 || M > 0x7fffffffll || N > 0x7fffffffll || K > 131071) return 0;
  if ((K & 3) != 0)  // (no instance shares tiles of such rows: they are laid out anew)
    return aitamd_gemm_int8_layout_bytes(M, N, K);
  int64_t most = 0;
  for (int i = 0; i < gemm_table(epilogue, dtype + kNumDTypes).count; ++i) {
    const int64_t n = aitamd_gemm_workspace_bytes(epilogue, dtype + kNumDTypes, i, 1, M, N, K / 2);
    most = n > most ? n : most;
  }
  return most;
}

}  // extern "C"
