// C ABI launchers of aitamd_gemm_rcr_lora: the adapters' first halves here, the product with their second halves in the tiles of
// the GEMM (lora.hpp, gemm_inst.hip with AITAMD_DT 4 and 5).
#include "../../include/aitemplate_amd_kernels.h"
#include "device.hpp"
#include "errors.hpp"
#include "gemm_host.hpp"
#include "lora.hpp"

namespace aitamd {
namespace {

struct LowParams {
  const void *x, *a;
  const int32_t* of;
  const float* scales;
  bf16* t;
  uint32_t* zeroed;  // the words that the GEMM's instances which share tiles count in
  int64_t ldx;
  int32_t M, K, n, rank, first;  // first: the launch's first row
};
constexpr int kZeroedWords = 1024;

template <class T>
AITAMD_DEVICE int adapter_of(const T& p, int m) {
  const int id = p.of[m];
  return (uint32_t)id < (uint32_t)p.n ? id : -1;
}
template <class P>
AITAMD_DEVICE void clear_counters(const P& p, int threads) {
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < kZeroedWords; i += threads) p.zeroed[i] = 0u;
}
// t = scale * sum, in two numbers that add up to it.  (An infinity or a NaN is the first one.)
AITAMD_DEVICE void put_low(bf16* row, int j, float v) {
  const bf16 one = (bf16)v;
  const float rest = v - (float)one;
  row[(j >> 3) * 16 + (j & 7)] = one;
  row[(j >> 3) * 16 + 8 + (j & 7)] = (bf16)(__builtin_isfinite((float)one) ? rest : 0.0f);
}

template <class T>
AITAMD_DEVICE float dot8(typename ElemTraits<T>::vec8 a, typename ElemTraits<T>::vec8 b, float s) {
#pragma unroll
  for (int e = 0; e < 8; ++e) s = __builtin_fmaf(ElemTraits<T>::to_float(a[e]), ElemTraits<T>::to_float(b[e]), s);
  return s;
}
// sum over the 64 lanes, in all of them
AITAMD_DEVICE float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
// x . a over K, by a wave
template <class T>
AITAMD_DEVICE float wave_dot(const T* x, const T* a, int K, int lane) {
  using vec8 = typename ElemTraits<T>::vec8;
  constexpr int AHEAD = 4;
  float s[AHEAD] = {};
  int k = lane * 8;
  for (; k + (AHEAD - 1) * 512 + 8 <= K; k += AHEAD * 512) {
    vec8 xv[AHEAD], av[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) xv[i] = load_vec<vec8>(x + k + i * 512), av[i] = load_vec<vec8>(a + k + i * 512);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) s[i] = dot8<T>(xv[i], av[i], s[i]);
  }
  for (; k + 8 <= K; k += 512) s[0] = dot8<T>(load_vec<vec8>(x + k), load_vec<vec8>(a + k), s[0]);
  for (int e = k; e < K && e < k + 8; ++e) s[1] = __builtin_fmaf(ElemTraits<T>::to_float(x[e]), ElemTraits<T>::to_float(a[e]), s[1]);
  return wave_sum((s[0] + s[1]) + (s[2] + s[3]));
}

constexpr int kRowThreads = 256;
// Few rows, which may all have adapters of their own: a wave for a rank of a row.  Bound: the latency of two trips to memory
// (adapter, then the rows of x and a together).
template <class T>
__global__ void __launch_bounds__(kRowThreads) low_rows_kernel(const LowParams p) {
  clear_counters(p, kRowThreads);
  const int lane = threadIdx.x & 63, m = p.first + blockIdx.x;
  const int padded = lora_chunks(p.rank) * 8;
  const int j = blockIdx.y * (kRowThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (j >= padded) return;
  const int id = __builtin_amdgcn_readfirstlane(adapter_of(p, m));
  float v = 0.0f;
  if (id >= 0 && j < p.rank) {
    v = wave_dot(reinterpret_cast<const T*>(p.x) + (int64_t)m * p.ldx, reinterpret_cast<const T*>(p.a) + ((int64_t)id * p.rank + j) * p.K, p.K, lane);
    v *= p.scales != nullptr ? p.scales[id] : 1.0f;
  }
  if (lane == 0) put_low(p.t + (int64_t)m * padded * 2, j, v);
}

// Rows of prompts, neighbours of one adapter mostly: ROWS of them and up to 64 ranks a workgroup, on matrix instructions, every
// wave with a part of K; a step is 64 deep, each lane with 32 neighbouring bytes of a row for two matrix instructions (which k is
// which does not matter where both operands have it alike), so that a row's share of a step is a line.  Bound: memory, x once.
// Several adapters among the rows: one after the other; more than kLoraFew: row by row.
constexpr int kTileWaves = 8, kTileRows = 32, kTileRanks = 64;
template <class T, int NR>
__global__ void __launch_bounds__(kTileWaves * 64) low_tile_kernel(const LowParams p) {
  using Tr = ElemTraits<T>;
  using vec8 = typename Tr::vec8;
  constexpr int MB = kTileRows / 16;
  __shared__ float part[kTileWaves][kTileRows][NR * 16 + 1];
  clear_counters(p, kTileWaves * 64);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int m0 = p.first + blockIdx.x * kTileRows, j0 = blockIdx.y * (NR * 16);
  const int padded = lora_chunks(p.rank) * 8;
  // (rows past the last: of the last one, with no adapter)
  int left[1];
  left[0] = lane < kTileRows && m0 + lane < p.M ? adapter_of(p, m0 + lane) : -1;
  const int mine = left[0];
  auto first_of = [&]() __attribute__((always_inline)) {
    const uint64_t some = __builtin_amdgcn_ballot_w64(left[0] >= 0);
    return some == 0 ? -1 : __builtin_amdgcn_readlane(left[0], __builtin_ctzll(some));
  };
  int distinct = 0;
  for (int id = first_of(); id >= 0 && distinct <= kLoraFew; id = first_of(), ++distinct)
    if (left[0] == id) left[0] = -1;
  left[0] = mine;
  const T* x = reinterpret_cast<const T*>(p.x);
  const T* a = reinterpret_cast<const T*>(p.a);
  bf16* const t = p.t + (int64_t)m0 * padded * 2;
  const int rows = p.M - m0 < kTileRows ? p.M - m0 : kTileRows;
  const int ranks = padded - j0 < NR * 16 ? padded - j0 : NR * 16;
  // zeros: rows without an adapter, ranks from p.rank on
  for (int i = tid; i < rows * ranks; i += kTileWaves * 64) {
    const int r = i / ranks, j = j0 + i - r * ranks;
    if (j >= p.rank || adapter_of(p, m0 + r) < 0) put_low(t + (int64_t)r * padded * 2, j, 0.0f);
  }
  if (distinct > kLoraFew) {
    for (int i = wave; i < rows * ranks; i += kTileWaves) {
      const int r = i / ranks, j = j0 + i - r * ranks;
      const int id = __builtin_amdgcn_readlane(mine, r);
      if (id < 0 || j >= p.rank) continue;
      const float v = wave_dot(x + (int64_t)(m0 + r) * p.ldx, a + ((int64_t)id * p.rank + j) * p.K, p.K, lane);
      if (lane == 0) put_low(t + (int64_t)r * padded * 2, j, v * (p.scales != nullptr ? p.scales[id] : 1.0f));
    }
    return;
  }
  const T* xr[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const int m = m0 + b * 16 + fr;
    xr[b] = x + (int64_t)(m < p.M ? m : p.M - 1) * p.ldx + fq * 16;
  }
  const int steps = p.K / 64, per = (steps + kTileWaves - 1) / kTileWaves;
  const int s0 = wave * per < steps ? wave * per : steps, s1 = s0 + per < steps ? s0 + per : steps;
  for (;;) {
    const int id = first_of();
    if (id < 0) break;
    const T* ar[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int j = j0 + r * 16 + fr;
      ar[r] = a + ((int64_t)id * p.rank + (j < p.rank ? j : p.rank - 1)) * p.K + fq * 16;
    }
    f32x4 acc[MB][NR] = {};
    auto step = [&](int k, auto whole) __attribute__((always_inline)) {
      vec8 xv[MB][2], av[NR][2];
      auto load = [&](const T* row, int h) __attribute__((always_inline)) {
        if constexpr (decltype(whole)::value) return load_vec<vec8>(row + k + h * 8);
        vec8 v = {};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + fq * 16 + h * 8 + e < p.K) v[e] = row[k + h * 8 + e];
        return v;
      };
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 0; b < MB; ++b) xv[b][h] = load(xr[b], h);
#pragma unroll
        for (int r = 0; r < NR; ++r) av[r][h] = load(ar[r], h);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
          for (int r = 0; r < NR; ++r) acc[b][r] = Tr::mfma16(av[r][h], xv[b][h], acc[b][r]);
    };
    for (int s = s0; s < s1; ++s) step(s * 64, std::true_type{});
    if (wave == kTileWaves - 1 && steps * 64 < p.K) step(steps * 64, std::false_type{});
    // (the operands swapped: a lane has four neighbouring ranks of one row)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][b * 16 + fr][r * 16 + fq * 4 + e] = acc[b][r][e];
    __syncthreads();
    const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;
    for (int i = tid; i < rows * ranks; i += kTileWaves * 64) {
      const int r = i / ranks, j = i - r * ranks;
      if (adapter_of(p, m0 + r) != id || j0 + j >= p.rank) continue;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kTileWaves; ++w) v += part[w][r][j];
      put_low(t + (int64_t)r * padded * 2, j0 + j, v * scale);
    }
    __syncthreads();
    if (left[0] == id) left[0] = -1;
  }
}

template <class T>
hipError_t launch_low(LowParams p, hipStream_t stream) {
  const int padded = lora_chunks(p.rank) * 8;
  // A row by itself reads its adapter alone, from the caches where others have read it; a tile reads x once and an adapter once
  // for 32 rows.
  constexpr int kFewRows = 256;
  if (p.M <= kFewRows) {
    hipLaunchKernelGGL(low_rows_kernel<T>, dim3(p.M, (padded + kRowThreads / 64 - 1) / (kRowThreads / 64)), dim3(kRowThreads), 0, stream, p);
    return hipGetLastError();
  }
  const int nr = padded > 32 ? 4 : (padded > 16 ? 2 : 1);
  auto kernel = nr == 4 ? low_tile_kernel<T, 4> : (nr == 2 ? low_tile_kernel<T, 2> : low_tile_kernel<T, 1>);
  const int64_t tiles = ((int64_t)p.M + kTileRows - 1) / kTileRows, groups = (padded + nr * 16 - 1) / (nr * 16);
  const int64_t most = most_workgroups(kTileWaves * 64) / groups;
  for (int64_t at = 0; at < tiles; at += most) {
    p.first = (int32_t)(at * kTileRows);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles - at < most ? tiles - at : most), (unsigned)groups), dim3(kTileWaves * 64), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

constexpr int64_t kMostRank = 1024;
int64_t t_bytes(int64_t M, int64_t rank) { return M * lora_chunks((int)rank) * 32; }

}  // namespace
}  // namespace aitamd

using namespace aitamd;

extern "C" int64_t aitamd_gemm_lora_workspace_bytes(int dtype, int algo, int bias, int64_t M, int64_t N, int64_t K, int64_t rank) {
  if ((dtype != AITAMD_F16 && dtype != AITAMD_BF16) || M <= 0 || N <= 0 || rank <= 0 || rank > kMostRank || M > 0x7fffffffll) return 0;
  const int epilogue = bias ? kEpiBias : kEpiNone, table = 2 * kNumDTypes + dtype;
  int64_t shared = kZeroedWords * 4;
  const int count = gemm_table(epilogue, table).count;
  for (int i = algo >= 0 ? algo : 0; i < (algo >= 0 && algo + 1 < count ? algo + 1 : count); ++i) {
    const int64_t n = aitamd_gemm_workspace_bytes(epilogue, table, i, 1, M, N, K);
    shared = n > shared ? n : shared;
  }
  return (shared + 15) / 16 * 16 + t_bytes(M, rank);
}

extern "C" int aitamd_gemm_rcr_lora(int dtype, int algo, const void* x, const void* w, const void* bias, const void* lora_a, const void* lora_b,
                                    const int32_t* adapters, const float* scales, void* y, int64_t M, int64_t N, int64_t K, int64_t rank,
                                    int64_t num_adapters, int64_t ldx, int64_t ldw, int64_t ldy, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  const char* who = "aitamd_gemm_rcr_lora";
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  if (M < 0 || N < 0 || K < 0 || num_adapters < 0) return fail("%s: negative dimension", who);
  if (rank < 1 || rank > kMostRank) return fail("%s: rank %lld: 1 to %lld are wanted", who, (long long)rank, (long long)kMostRank);
  if (M > 0x7fffffffll || N > 0x7fffffffll || K > 0x7fffffffll || num_adapters > 0x7fffffffll) return fail("%s: dimension too large", who);
  if (M == 0 || N == 0) return 0;
  if (!y || !adapters || (K > 0 && (!x || !w)) || (num_adapters > 0 && (!lora_b || (K > 0 && !lora_a)))) return fail("%s: null pointer", who);
  if (ldx < K || ldw < K || ldy < N) return fail("%s: row pitch smaller than the row", who);
  if ((reinterpret_cast<uintptr_t>(adapters) | reinterpret_cast<uintptr_t>(scales)) & 3)
    return fail("%s: adapters and scales have to be 4-byte aligned", who);
  const int64_t need = kZeroedWords * 4 + t_bytes(M, rank);
  if (!workspace || workspace_bytes < need)
    return fail("%s: a workspace of %lld bytes at least is wanted, got %lld", who, (long long)need, workspace ? (long long)workspace_bytes : 0ll);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail("%s: the workspace must be 16-byte aligned", who);
  // t behind what the instances that share tiles have
  const int64_t at = (workspace_bytes - t_bytes(M, rank)) & ~15ll;
  unsigned char* const base = static_cast<unsigned char*>(workspace);
  GemmParams p{};
  p.a = x, p.b = w, p.c = y, p.bias = bias;
  p.M = (int32_t)M, p.N = (int32_t)N, p.K = (int32_t)K;
  p.batch = 1;
  p.lda = ldx, p.ldb = ldw, p.ldc = ldy;
  p.ws = workspace, p.ws_bytes = at;
  p.lora_t = base + at, p.lora_b = lora_b, p.lora_of = adapters;
  p.lora_n = (int32_t)num_adapters, p.lora_rank = (int32_t)rank;
  LowParams low{};
  low.x = x, low.a = lora_a, low.of = adapters, low.scales = scales;
  low.t = reinterpret_cast<bf16*>(base + at), low.zeroed = reinterpret_cast<uint32_t*>(base);
  low.ldx = ldx;
  low.M = (int32_t)M, low.K = (int32_t)K, low.n = (int32_t)num_adapters, low.rank = (int32_t)rank;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F16 ? launch_low<f16>(low, s) : launch_low<bf16>(low, s);
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return run_gemm(bias ? kEpiBias : kEpiNone, 2 * kNumDTypes + dtype, algo, p, s);
}
