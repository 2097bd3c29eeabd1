// Products of 8-bit integers whose rows lie at any byte (K, pitches or pointers that are no whole dwords), which the instances
// of gemm_tiles.inc do not take:  C[m, n] = scale_a[m] scale_b[n] sum_k A[m, k] B[n, k] (+ bias[n]).
//
// The slabs go through registers: 16 bytes of a row a lane, read at any address, the next slab's while one is multiplied; the
// last slab's pieces that K ends in are put together byte by byte, so that nothing past the end of a row is read.  Rows that
// are not there are the last one once more.  One barrier a slab, two LDS stages.
// What bounds it: the reads at odd addresses, two lines for most of them.
#include "gemm_int8_any.hpp"

#include "common.hpp"
#include "epilogue.hpp"

namespace aitamd {
namespace {

template <int BM_, int BN_>
struct Int8Tile {
  static constexpr int BM = BM_, BN = BN_, BK = 64;  // (bytes)
  static constexpr int NT = 256;                     // 2 x 2 waves
  static constexpr int MI = BM / 32, NI = BN / 32;   // 16 x 16 blocks of a wave's part
  static constexpr int PA = BM * 4 / NT, PB = BN * 4 / NT;  // pieces a lane loads
  static constexpr int STAGE = (BM + BN) * BK;
};

// piece c of row r in LDS: the 16 rows of a fragment on different banks
AITAMD_DEVICE int int8_place(int row, int c) { return row * 64 + ((c ^ ((row >> 1) & 3)) << 4); }

AITAMD_DEVICE u32x4 int8_piece(const int8_t* row, int k, int K) {
  u32x4 v = {};
  if (k + 16 <= K) {
    v = load_vec<u32x4>(row + k);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (k + j < K) v[j / 4] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j % 4));
  }
  return v;
}

template <class Out, class Tile, bool BIAS>
__global__ void __launch_bounds__(Tile::NT, 2) gemm_int8_any_kernel(const GemmParams p) {
  constexpr int MI = Tile::MI, NI = Tile::NI, PA = Tile::PA, PB = Tile::PB;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * Tile::STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, fr = lane & 15, fq = lane >> 4;
  int batch, tm, tn;
  map_tile(p, blockIdx.x, batch, tm, tn);
  const int m0 = tm * Tile::BM, n0 = tn * Tile::BN;

  const int8_t *a_row[PA], *b_row[PB];
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    const int m = m0 + (tid >> 2) + i * 64;
    a_row[i] = reinterpret_cast<const int8_t*>(p.a) + (int64_t)(m < p.M ? m : p.M - 1) * p.lda;
  }
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int n = n0 + (tid >> 2) + i * 64;
    b_row[i] = reinterpret_cast<const int8_t*>(p.b) + (int64_t)(n < p.N ? n : p.N - 1) * p.ldb;
  }
  u32x4 ra[PA], rb[PB];
  auto fetch = [&](int kt) {
    const int k = kt * Tile::BK + (tid & 3) * 16;
#pragma unroll
    for (int i = 0; i < PA; ++i) ra[i] = int8_piece(a_row[i], k, p.K);
#pragma unroll
    for (int i = 0; i < PB; ++i) rb[i] = int8_piece(b_row[i], k, p.K);
  };
  auto put = [&](int stage) {
    unsigned char* st = smem + stage * Tile::STAGE;
#pragma unroll
    for (int i = 0; i < PA; ++i) *reinterpret_cast<u32x4*>(st + int8_place((tid >> 2) + i * 64, tid & 3)) = ra[i];
#pragma unroll
    for (int i = 0; i < PB; ++i) *reinterpret_cast<u32x4*>(st + Tile::BM * 64 + int8_place((tid >> 2) + i * 64, tid & 3)) = rb[i];
  };
  i32x4 acc[MI][NI];
#pragma unroll
  for (int mi = 0; mi < MI; ++mi)
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = i32x4{};
  const int k_tiles = (p.K + Tile::BK - 1) / Tile::BK;
  if (k_tiles > 0) {
    fetch(0);
    put(0);
    __syncthreads();
  }
  for (int kt = 0; kt < k_tiles; ++kt) {
    // (the other stage's readers have passed the last barrier)
    const bool more = kt + 1 < k_tiles;
    if (more) fetch(kt + 1);
    const unsigned char* st = smem + (kt & 1) * Tile::STAGE;
    i32x4 af[MI], bf[NI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) af[mi] = *reinterpret_cast<const i32x4*>(st + int8_place(wm * (Tile::BM / 2) + mi * 16 + fr, fq));
#pragma unroll
    for (int ni = 0; ni < NI; ++ni)
      bf[ni] = *reinterpret_cast<const i32x4*>(st + Tile::BM * 64 + int8_place(wn * (Tile::BN / 2) + ni * 16 + fr, fq));
    // (operands swapped: a lane holds 4 consecutive columns of one row)
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[ni], af[mi], acc[mi][ni], 0, 0, 0);
    if (more) put((kt + 1) & 1);
    __syncthreads();
  }
  using Tr = ElemTraits<Out>;
  using Epi = Epilogue<BIAS ? kEpiBias : kEpiNone>;
  float one = 1.0f;
  asm volatile("" : "+s"(one));  // (opaque to the optimizer: see to_float_plus)
#pragma unroll
  for (int ni = 0; ni < NI; ++ni) {
    const int n = n0 + wn * (Tile::BN / 2) + ni * 16 + fq * 4;
    float scale_n[4];
    Out bias[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = n + j < p.N ? n + j : p.N - 1;
      scale_n[j] = p.scale_b[at];
      if constexpr (BIAS) bias[j] = reinterpret_cast<const Out*>(p.bias)[at];
    }
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
      const int m = m0 + wm * (Tile::BM / 2) + mi * 16 + fr;
      if (m >= p.M) continue;
      const float scale = p.scale_a[m];
      Out* c = reinterpret_cast<Out*>(p.c) + (int64_t)m * p.ldc + n;
      typename Tr::vec4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = epilogue1<Epi, Out>((float)acc[mi][ni][j] * (scale * scale_n[j]), bias[j], Out{}, Out{}, one);
      if (n + 4 <= p.N) {
        store_vec(c, o);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) c[j] = o[j];
      }
    }
  }
}

template <class Out, class Tile>
hipError_t launch(GemmParams p, hipStream_t stream) {
  set_tiles(p, Tile::BM, Tile::BN, 3, -1);
  const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
  if (total > 0x7fffffffll) return hipErrorInvalidValue;
  const auto kernel = p.bias != nullptr ? gemm_int8_any_kernel<Out, Tile, true> : gemm_int8_any_kernel<Out, Tile, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)total), dim3(Tile::NT), 0, stream, p);
  return hipGetLastError();
}

template <class Out>
hipError_t pick(const GemmParams& p, int cus, hipStream_t stream) {
  // 128 x 128 where that leaves a tile for every CU
  const int64_t tiles = (((int64_t)p.M + 127) / 128) * (((int64_t)p.N + 127) / 128);
  return tiles >= cus ? launch<Out, Int8Tile<128, 128>>(p, stream) : launch<Out, Int8Tile<64, 64>>(p, stream);
}

}  // namespace

hipError_t launch_gemm_int8_any(const GemmParams& p, bool bf16_out, int cus, hipStream_t stream) {
  return bf16_out ? pick<bf16>(p, cus, stream) : pick<f16>(p, cus, stream);
}

}  // namespace aitamd
