// C ABI launchers of aitamd_gemm_rcr_lora: the adapters' first halves here, the product with their second halves in the tiles of
// the GEMM (lora.hpp, gemm_inst.hip with AITAMD_DT 4 and 5).
#include <mutex>

#include "../../include/aitemplate_amd_kernels.h"
#include "device.hpp"
#include "errors.hpp"
#include "gemm_host.hpp"
#include "gemm_kernel_dma.hpp"
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
// x . a[e] over K, by a wave
template <class T>
AITAMD_DEVICE void wave_dots(const T* x, const T* const (&a)[4], int K, int lane, float (&v)[4]) {
  using vec8 = typename ElemTraits<T>::vec8;
  constexpr int AHEAD = 2;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = 0.0f;
  int k = lane * 8;
  for (; k + (AHEAD - 1) * 512 + 8 <= K; k += AHEAD * 512) {
    vec8 xv[AHEAD], av[AHEAD][4];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      xv[i] = load_vec<vec8>(x + k + i * 512);
#pragma unroll
      for (int e = 0; e < 4; ++e) av[i][e] = load_vec<vec8>(a[e] + k + i * 512);
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = dot8<T>(xv[i], av[i][e], v[e]);
  }
  for (; k < K; k += 512) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (k + 8 <= K) {
        v[e] = dot8<T>(load_vec<vec8>(x + k), load_vec<vec8>(a[e] + k), v[e]);
      } else {
        for (int i = k; i < K; ++i) v[e] = __builtin_fmaf(ElemTraits<T>::to_float(x[i]), ElemTraits<T>::to_float(a[e][i]), v[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = wave_sum(v[e]);
}

constexpr int kRowThreads = 256;
// Few rows, which may all have adapters of their own: a wave for RANKS ranks of a row.  Bound: the latency of two trips to memory
// (the row and its adapter's number, then the adapter; AHEAD x 512 of K at once).
template <class T, int RANKS>
__global__ void __launch_bounds__(kRowThreads) low_rows_kernel(const LowParams p) {
  using vec8 = typename ElemTraits<T>::vec8;
  constexpr int AHEAD = 8;
  const int lane = threadIdx.x & 63, m = p.first + blockIdx.x;
  const int padded = lora_chunks(p.rank) * 8;
  const int j0 = (blockIdx.y * (kRowThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * RANKS;
  const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)m * p.ldx;
  // whole pieces from k on
  auto load = [&](vec8 (&v)[AHEAD], const T* row, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      v[i] = vec8{};
      if (k + i * 512 + lane * 8 + 8 <= p.K) v[i] = load_vec<vec8>(row + k + i * 512 + lane * 8);
    }
  };
  vec8 xv[AHEAD], av[RANKS][AHEAD];
  load(xv, x, 0);
  const int id = __builtin_amdgcn_readfirstlane(adapter_of(p, m));
  clear_counters(p, kRowThreads);
  if (j0 >= padded) return;
  float v[RANKS] = {};
  if (id >= 0) {
    const T* a[RANKS];
    const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;
    // (ranks from p.rank on: of the last one, and zeros)
#pragma unroll
    for (int r = 0; r < RANKS; ++r) a[r] = reinterpret_cast<const T*>(p.a) + ((int64_t)id * p.rank + (j0 + r < p.rank ? j0 + r : p.rank - 1)) * p.K;
    for (int k = 0;;) {
#pragma unroll
      for (int r = 0; r < RANKS; ++r) load(av[r], a[r], k);
#pragma unroll
      for (int r = 0; r < RANKS; ++r)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          if (RANKS == 1 || k + i * 512 < p.K) v[r] = dot8<T>(xv[i], av[r][i], v[r]);
      k += AHEAD * 512;
      if (k >= p.K) break;
      load(xv, x, k);
    }
    const int whole = p.K & ~7;
#pragma unroll
    for (int r = 0; r < RANKS; ++r) {
      if (whole + lane < p.K) v[r] = __builtin_fmaf(ElemTraits<T>::to_float(x[whole + lane]), ElemTraits<T>::to_float(a[r][whole + lane]), v[r]);
      v[r] = j0 + r < p.rank ? wave_sum(v[r]) * scale : 0.0f;
    }
  }
#pragma unroll
  for (int r = 0; r < RANKS; ++r)
    if (lane == r) put_low(p.t + (int64_t)m * padded * 2, j0 + r, v[r]);
}

// Rows of prompts, neighbours of one adapter mostly: ROWS of them and NR x 16 ranks a workgroup.  Several adapters among the rows:
// where the grid is kLoraFew deep, each by a workgroup of its own (8192 x 4096, rank 64, tiles with two: 38 us one after the other, 31
// so), which leaves at once where there is none for it; more than kLoraFew: row by row, by all of them (2048 x 4096, rank 16, 48 at
// random: 168 us by one, 50 by four).
constexpr int kLoraFew = 4;
struct LowTile {
  int mine, left, distinct;  // the lane's row's adapter, that or -1, how many there are among the rows
  AITAMD_DEVICE int first() const {
    const uint64_t some = __builtin_amdgcn_ballot_w64(left >= 0);
    return some == 0 ? -1 : __builtin_amdgcn_readlane(left, __builtin_ctzll(some));
  }
  AITAMD_DEVICE void drop(int id) { left = left == id ? -1 : left; }
};
// Zeros where there is no adapter, and all rows where there are many adapters; false if that was all for this workgroup.  of: the rows'
// adapters, in LDS.
template <class T, int THREADS>
AITAMD_DEVICE bool low_begin(const LowParams& p, LowTile& l, int* of, int m0, int rows, int j0, int ranks, int padded) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  l.mine = l.left = lane < rows ? adapter_of(p, m0 + lane) : -1;
  clear_counters(p, THREADS);
  if (tid < rows) of[tid] = l.mine;
  l.distinct = 0;
  for (int id = l.first(); id >= 0 && l.distinct <= kLoraFew; id = l.first(), ++l.distinct) l.drop(id);
  l.left = l.mine;
  const int turn = blockIdx.z, turns = gridDim.z;
  if (turn != 0 && l.distinct <= kLoraFew) return l.distinct > turn;
  bf16* const t = p.t + ((int64_t)m0 * padded + j0) * 2;
  if (turn == 0 && __builtin_amdgcn_ballot_w64(lane < rows && l.mine < 0) != 0) {
    __syncthreads();
    const int chunks = ranks / 8;
    for (int i = tid; i < rows * chunks; i += THREADS) {
      const int r = i / chunks, c = i - r * chunks;
      if (of[r] < 0) {
        bf16* const at = t + ((int64_t)r * padded + c * 8) * 2;
        store_vec(at, bf16x8{});
        store_vec(at + 8, bf16x8{});
      }
    }
  }
  if (l.distinct <= kLoraFew) return l.distinct > 0;
  // four ranks of a row at a time (those from p.rank on: of the last one, and zeros)
  for (int i = wave + turn * (THREADS / 64); i < rows * (ranks / 4); i += turns * (THREADS / 64)) {
    const int r = i / (ranks / 4), j = j0 + (i - r * (ranks / 4)) * 4;
    const int id = __builtin_amdgcn_readlane(l.mine, r);
    if (id < 0) continue;
    const T* a = reinterpret_cast<const T*>(p.a) + (int64_t)id * p.rank * p.K;
    const T* row[4];
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) row[e] = a + (int64_t)(j + e < p.rank ? j + e : p.rank - 1) * p.K;
    wave_dots(reinterpret_cast<const T*>(p.x) + (int64_t)(m0 + r) * p.ldx, row, p.K, lane, v);
    const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (lane == e) put_low(p.t + (int64_t)(m0 + r) * padded * 2, j + e, j + e < p.rank ? v[e] * scale : 0.0f);
  }
  return false;
}
// The waves' sums part[wave][row][rank], PITCH floats a row, of the rows that belong to `id`: a chunk of a row for a thread
template <int WAVES, int PITCH>
AITAMD_DEVICE void low_end(const LowParams& p, const float* part, const int* of, int id, int m0, int rows, int j0, int ranks, int padded, int tile_rows) {
  const float scale = p.scales != nullptr ? p.scales[id] : 1.0f;
  const int chunks = ranks / 8;
  for (int i = threadIdx.x; i < rows * chunks; i += WAVES * 64) {
    const int r = i / chunks, c = i - r * chunks;
    if (of[r] != id) continue;
    float v[8] = {};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float* at = part + (w * tile_rows + r) * PITCH + c * 8;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(at), hi = *reinterpret_cast<const f32x4*>(at + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += lo[e], v[4 + e] += hi[e];
    }
    bf16x8 one, two;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = j0 + c * 8 + e < p.rank ? v[e] * scale : 0.0f;
      one[e] = (bf16)f;
      two[e] = (bf16)(__builtin_isfinite((float)one[e]) ? f - (float)one[e] : 0.0f);
    }
    bf16* const at = p.t + ((int64_t)(m0 + r) * padded + j0 + c * 8) * 2;
    store_vec(at, one);
    store_vec(at + 8, two);
  }
}

// Rows of whole dwords.  Bound: memory, x once.  Slabs of 128 of K of the rows and of the adapter go straight to a ring in LDS, 16
// lanes for 256 bytes of a row (to registers, in the layout of the operands, every lane fetches from a line of its own: 8192 x 4096,
// rank 64, 52 us), each of the four waves multiplies a quarter of a slab.
template <class T, int NR_, int MB_>
struct LowRing {
  static constexpr int NR = NR_, MB = MB_;
  static constexpr int ROWS = 16 * MB, RANKS = 16 * NR, WAVES = 4, BK = 128;
  static constexpr int LOADS = (ROWS + RANKS) / 4 / WAVES;  // of a wave for a slab, four rows each
  static constexpr int STAGE = (ROWS + RANKS) * BK;         // elements
  static constexpr int NS = 78 * 1024 / (STAGE * 2) < 6 ? 78 * 1024 / (STAGE * 2) : 6;  // (two workgroups a CU)
  static constexpr int PITCH = RANKS + 4;
  static constexpr int kLdsBytes = NS * STAGE * 2;
  static_assert((ROWS + RANKS) % (4 * WAVES) == 0 && WAVES * ROWS * PITCH * 4 <= kLdsBytes && kLdsBytes + ROWS * 4 <= 80 * 1024);
};
template <class T, class R>
__global__ void __launch_bounds__(R::WAVES * 64) low_ring_kernel(const LowParams p) {
  using Tr = ElemTraits<T>;
  using vec8 = typename Tr::vec8;
  constexpr int NR = R::NR, MB = R::MB, NS = R::NS;
  typedef __attribute__((address_space(3))) void lds_void;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  T* const smem = reinterpret_cast<T*>(smem_raw);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int m0 = p.first + blockIdx.x * R::ROWS, j0 = blockIdx.y * R::RANKS;
  const int padded = lora_chunks(p.rank) * 8;
  const int rows = p.M - m0 < R::ROWS ? p.M - m0 : R::ROWS, ranks = padded - j0 < R::RANKS ? padded - j0 : R::RANKS;
  LowTile l;
  __shared__ int of[R::ROWS];
  if (!low_begin<T, R::WAVES * 64>(p, l, of, m0, rows, j0, ranks, padded)) return;
  const int slabs = (p.K + R::BK - 1) / R::BK;
  const __amdgpu_buffer_rsrc_t rx = make_rsrc(reinterpret_cast<const T*>(p.x) + (int64_t)m0 * p.ldx, (uint32_t)(((rows - 1) * (uint32_t)p.ldx + (uint32_t)p.K) * 2u));
  // row r's piece c of a slab lies at place c ^ r of the row's 256 bytes: the 16 rows of a fragment are on different banks
  uint32_t off[R::LOADS];
  int at_k[R::LOADS];
#pragma unroll
  for (int i = 0; i < R::LOADS; ++i) {
    const int row = (wave + i * R::WAVES) * 4 + (lane >> 4);
    const bool of_x = row < R::ROWS;
    at_k[i] = ((lane & 15) ^ (row & 15)) * 8;
    off[i] = (uint32_t)(of_x ? row * (int)p.ldx : (row - R::ROWS) * p.K) * 2u + (uint32_t)at_k[i] * 2u;
  }
  for (int turn = 0;; ++turn) {
    const int id = l.first();
    if (id < 0) break;
    if (turn != (int)blockIdx.z) {
      l.drop(id);
      continue;
    }
    const int there = p.rank - j0 < R::RANKS ? p.rank - j0 : R::RANKS;
    const __amdgpu_buffer_rsrc_t ra = make_rsrc(reinterpret_cast<const T*>(p.a) + ((int64_t)id * p.rank + j0) * p.K, (uint32_t)(there > 0 ? there : 0) * (uint32_t)p.K * 2u);
    auto issue = [&](int kt) __attribute__((always_inline)) {
      T* const stage = smem + kt % NS * R::STAGE;
#pragma unroll
      for (int i = 0; i < R::LOADS; ++i) {
        const int j = wave + i * R::WAVES;
        const uint32_t o = at_k[i] + kt * R::BK < p.K ? off[i] + (uint32_t)(kt * R::BK * 2) : kOobOffset;
        if (j * 4 < R::ROWS)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (lds_void*)(stage + j * 512), 16, o, 0, 0, 0);
        else
          __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_void*)(stage + j * 512), 16, o, 0, 0, 0);
      }
    };
    f32x4 acc[MB][NR] = {};
    // LEFT: slabs behind this one that are on their way or to come, NS - 1 standing for any number from there on
    auto slab = [&](int kt, auto left_c) __attribute__((always_inline)) {
      constexpr int LEFT = decltype(left_c)::value;
      wait_vmcnt<(LEFT >= NS - 1 ? NS - 2 : LEFT) * R::LOADS>();
      __builtin_amdgcn_s_barrier();
      const T* const stage = smem + kt % NS * R::STAGE;
      const int c = wave * 4 + fq;
      u32x4 f[MB + NR];
#pragma unroll
      for (int b = 0; b < MB + NR; ++b) f[b] = *reinterpret_cast<const u32x4*>(stage + (b * 16 + fr) * R::BK + ((c ^ fr) << 3));
      if constexpr (LEFT >= NS - 1) issue(kt + NS - 1);
      if (LEFT == 0 && (p.K & 7) != 0) {
        // (the last piece of a row goes on in the next one)
        const int dwords = (p.K - kt * R::BK - c * 8) / 2;
#pragma unroll
        for (int b = 0; b < MB + NR; ++b)
#pragma unroll
          for (int d = 0; d < 4; ++d) f[b][d] = d < dwords ? f[b][d] : 0u;
      }
#pragma unroll
      for (int b = 0; b < MB; ++b)
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[b][r] = Tr::mfma16(__builtin_bit_cast(vec8, f[MB + r]), __builtin_bit_cast(vec8, f[b]), acc[b][r]);
    };
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
      if (s < slabs) issue(s);
    int kt = 0;
    for (; kt + NS - 1 < slabs; ++kt) slab(kt, std::integral_constant<int, NS - 1>{});
    static_for<0, NS - 1>([&](auto i) __attribute__((always_inline)) {
      constexpr int left = NS - 2 - decltype(i)::value;
      if (left < slabs) slab(slabs - 1 - left, std::integral_constant<int, left>{});
    });
    __syncthreads();
    // (the operands swapped: a lane has four neighbouring ranks of one row)
    float* const part = reinterpret_cast<float*>(smem_raw);
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int r = 0; r < NR; ++r)
        *reinterpret_cast<f32x4*>(part + (wave * R::ROWS + b * 16 + fr) * R::PITCH + r * 16 + fq * 4) = acc[b][r];
    __syncthreads();
    low_end<R::WAVES, R::PITCH>(p, part, of, id, m0, rows, j0, ranks, padded, R::ROWS);
    __syncthreads();
    l.drop(id);
  }
}

// Rows at any element, through registers: a step is 64 deep, each lane with 32 neighbouring bytes of a row for two matrix instructions
// (which k is which does not matter where both operands have it alike).
constexpr int kTileWaves = 8, kTileRows = 32;
template <class T, int NR>
__global__ void __launch_bounds__(kTileWaves * 64) low_tile_kernel(const LowParams p) {
  using Tr = ElemTraits<T>;
  using vec8 = typename Tr::vec8;
  constexpr int MB = kTileRows / 16, PITCH = NR * 16 + 4;
  __shared__ __attribute__((aligned(16))) float part[kTileWaves * kTileRows * PITCH];
  __shared__ int of[kTileRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int m0 = p.first + blockIdx.x * kTileRows, j0 = blockIdx.y * (NR * 16);
  const int padded = lora_chunks(p.rank) * 8;
  const int rows = p.M - m0 < kTileRows ? p.M - m0 : kTileRows, ranks = padded - j0 < NR * 16 ? padded - j0 : NR * 16;
  LowTile l;
  if (!low_begin<T, kTileWaves * 64>(p, l, of, m0, rows, j0, ranks, padded)) return;
  const T* xr[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    const int m = m0 + b * 16 + fr;
    xr[b] = reinterpret_cast<const T*>(p.x) + (int64_t)(m < p.M ? m : p.M - 1) * p.ldx + fq * 16;
  }
  const int steps = p.K / 64, per = (steps + kTileWaves - 1) / kTileWaves;
  const int s0 = wave * per < steps ? wave * per : steps, s1 = s0 + per < steps ? s0 + per : steps;
  for (;;) {
    const int id = l.first();
    if (id < 0) break;
    const T* ar[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int j = j0 + r * 16 + fr;
      ar[r] = reinterpret_cast<const T*>(p.a) + ((int64_t)id * p.rank + (j < p.rank ? j : p.rank - 1)) * p.K + fq * 16;
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
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int r = 0; r < NR; ++r)
        *reinterpret_cast<f32x4*>(part + (wave * kTileRows + b * 16 + fr) * PITCH + r * 16 + fq * 4) = acc[b][r];
    __syncthreads();
    low_end<kTileWaves, PITCH>(p, part, of, id, m0, rows, j0, ranks, padded, kTileRows);
    __syncthreads();
    l.drop(id);
  }
}

// tiles of `tile_rows` rows by `groups` groups of ranks, in as many launches as it takes
hipError_t launch_tiles(void (*kernel)(const LowParams), LowParams p, int tile_rows, int64_t groups, int turns, int threads, int lds, hipStream_t stream) {
  const int64_t tiles = ((int64_t)p.M + tile_rows - 1) / tile_rows, most = most_workgroups(threads) / (groups * turns);
  for (int64_t at = 0; at < tiles; at += most) {
    p.first = (int32_t)(at * tile_rows);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles - at < most ? tiles - at : most), (unsigned)groups, (unsigned)turns), dim3(threads), lds, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
template <class T, int NR, int MB>
hipError_t launch_ring(const LowParams& p, int64_t groups, hipStream_t stream) {
  using R = LowRing<T, NR, MB>;
  auto kernel = low_ring_kernel<T, R>;
  // LDS above 64 KiB has to be opted into once per device
  constexpr int kMaxDevices = 64;
  static std::once_flag once[kMaxDevices];
  static hipError_t errors[kMaxDevices];
  int dev = 0;
  const hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  std::call_once(once[dev % kMaxDevices], [&] {
    errors[dev % kMaxDevices] = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, R::kLdsBytes);
  });
  if (errors[dev % kMaxDevices] != hipSuccess) return errors[dev % kMaxDevices];
  return launch_tiles(kernel, p, R::ROWS, groups, kLoraFew, R::WAVES * 64, R::kLdsBytes, stream);
}
template <class T, int NR>
hipError_t launch_ring(const LowParams& p, int64_t groups, int cus, hipStream_t stream) {
  // 32 rows share an adapter's lines where that leaves a tile for every CU
  return (int64_t)p.M >= 32ll * cus ? launch_ring<T, NR, 2>(p, groups, stream) : launch_ring<T, NR, 1>(p, groups, stream);
}

template <class T>
hipError_t launch_low(LowParams p, hipStream_t stream) {
  const int padded = lora_chunks(p.rank) * 8;
  // A row by itself reads its whole adapter, from L2 mostly; a tile reads x once and an adapter once for its rows, and takes them one
  // by one where they have many adapters.  By themselves up to twice the waves that the chip holds at once, two ranks each then.  Of
  // rank 16, K = 4096, with one adapter / sixteen requests' rows in turn / 48 adapters at random: 1024 rows 15, 16 and 16 us by
  // themselves, 9 and 15 in tiles with the first two; 2048 rows 25, 25 and 24 by themselves, 12, 10 and 50 in tiles.
  const int64_t waves = (int64_t)p.M * padded;
  constexpr int64_t kAtOnce = 8192;
  if (waves <= 2 * kAtOnce) {
    const int ranks = waves <= kAtOnce ? 1 : 2, per = kRowThreads / 64 * ranks;
    hipLaunchKernelGGL((ranks == 1 ? low_rows_kernel<T, 1> : low_rows_kernel<T, 2>), dim3(p.M, (padded + per - 1) / per), dim3(kRowThreads), 0, stream, p);
    return hipGetLastError();
  }
  const int nr = padded > 32 ? 4 : (padded > 16 ? 2 : 1);
  const int64_t groups = (padded + nr * 16 - 1) / (nr * 16);
  const bool dwords = ((p.K | p.ldx) & 1) == 0 && ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.a)) & 3) == 0 &&
      p.ldx <= (1 << 24) && p.K <= (1 << 23);
  if (dwords) {
    const int cus = current_device_cus();
    return nr == 4 ? launch_ring<T, 4>(p, groups, cus, stream) : (nr == 2 ? launch_ring<T, 2>(p, groups, cus, stream) : launch_ring<T, 1>(p, groups, cus, stream));
  }
  auto kernel = nr == 4 ? low_tile_kernel<T, 4> : (nr == 2 ? low_tile_kernel<T, 2> : low_tile_kernel<T, 1>);
  return launch_tiles(kernel, p, kTileRows, groups, 1, kTileWaves * 64, 0, stream);
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
