// Products of 8-bit integers whose rows lie at any byte (K, pitches or pointers that are no whole dwords), which the instances
// of gemm_tiles.inc do not take:  C[m, n] = scale_a[m] scale_b[n] sum_k A[m, k] B[n, k] (+ bias[n]).
//
// The slabs go through registers: 16 bytes of a row a lane, read at any address, the next slab's while one is multiplied; the
// piece that K ends in is the row's last 16 bytes, shifted, so that nothing past the end of a row is read.  Rows that
// are not there are the last one once more.  One barrier a slab, two LDS stages.
// What bounds it: the reads at odd addresses, half a microsecond a slab where a CU has one workgroup.  From a few slabs on it is
// faster to lay the rows out in scratch memory first (int8_align_kernel, one launch for both operands) and multiply those with the
// other instances; this kernel is for short rows, and for calls without scratch memory.
#include "gemm_int8_any.hpp"

#include "common.hpp"
#include "device.hpp"
#include "epilogue.hpp"

namespace aitamd {
namespace {

// D_: slabs on their way in registers
template <int BM_, int BN_, int BK_, int D_>
struct Int8Tile {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, D = D_;  // (BK in bytes)
  static constexpr int NT = 256;                     // 2 x 2 waves
  static constexpr int MI = BM / 32, NI = BN / 32;   // 16 x 16 blocks of a wave's part
  static constexpr int CPR = BK / 16;                // pieces of a row
  static constexpr int RPP = NT / CPR;               // rows that all lanes load at a time
  static constexpr int PA = BM / RPP, PB = BN / RPP; // pieces a lane loads
  static constexpr int STAGE = (BM + BN) * BK;
  // piece c of row r in LDS: the 16 rows of a fragment on different banks
  static constexpr __device__ int place(int row, int c) { return row * BK + ((c ^ (CPR == 4 ? (row >> 1) & 3 : row & (CPR - 1))) << 4); }
};

// The 16 bytes of a row from byte k on, those past its end as zeros: the last 16 of the row, shifted (rows shorter than that byte
// by byte).
AITAMD_DEVICE u32x4 int8_piece(const int8_t* row, int k, int K) {
  u32x4 v = {};
  if (K < 16) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (k + j < K) v[j / 4] |= (uint32_t)(uint8_t)row[k + j] << (8 * (j % 4));
    return v;
  }
  const int at = k + 16 <= K ? k : K - 16, by = k - at;  // (16 and more: nothing is left)
  v = load_vec<u32x4>(row + at);
  uint32_t t[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = __builtin_amdgcn_alignbyte(i < 3 ? v[i < 3 ? i + 1 : 0] : 0u, v[i], by & 3);
  const int dwords = by >> 2;
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = 0;
#pragma unroll
    for (int x = i; x < 4; ++x) w = x - i == dwords ? t[x] : w;
    o[i] = w;
  }
  return o;
}

template <class Out, class Tile, bool BIAS>
__global__ void __launch_bounds__(Tile::NT, 2) gemm_int8_any_kernel(const GemmParams p) {
  constexpr int MI = Tile::MI, NI = Tile::NI, PA = Tile::PA, PB = Tile::PB, D = Tile::D, CPR = Tile::CPR;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1, fr = lane & 15, fq = lane >> 4;
  int batch, tm, tn;
  map_tile(p, blockIdx.x, batch, tm, tn);
  const int m0 = tm * Tile::BM, n0 = tn * Tile::BN;
  const int l_row = tid / CPR, l_piece = tid % CPR;

  const int8_t *a_row[PA], *b_row[PB];
#pragma unroll
  for (int i = 0; i < PA; ++i) {
    const int m = m0 + l_row + i * Tile::RPP;
    a_row[i] = reinterpret_cast<const int8_t*>(p.a) + (int64_t)(m < p.M ? m : p.M - 1) * p.lda;
  }
#pragma unroll
  for (int i = 0; i < PB; ++i) {
    const int n = n0 + l_row + i * Tile::RPP;
    b_row[i] = reinterpret_cast<const int8_t*>(p.b) + (int64_t)(n < p.N ? n : p.N - 1) * p.ldb;
  }
  const int k_tiles = (p.K + Tile::BK - 1) / Tile::BK;
  u32x4 ra[D][PA], rb[D][PB];
  auto fetch = [&](int kt, auto d_c) {
    constexpr int d = decltype(d_c)::value;
    const int k = kt * Tile::BK + l_piece * 16;
    // (a slab that K does not end in: no branches; one past the end: zeros, which nobody multiplies)
    if ((kt + 1) * Tile::BK <= p.K) {
#pragma unroll
      for (int i = 0; i < PA; ++i) ra[d][i] = load_vec<u32x4>(a_row[i] + k);
#pragma unroll
      for (int i = 0; i < PB; ++i) rb[d][i] = load_vec<u32x4>(b_row[i] + k);
    } else if (kt < k_tiles) {
#pragma unroll
      for (int i = 0; i < PA; ++i) ra[d][i] = int8_piece(a_row[i], k, p.K);
#pragma unroll
      for (int i = 0; i < PB; ++i) rb[d][i] = int8_piece(b_row[i], k, p.K);
    }
  };
  auto put = [&](int stage, auto d_c) {
    constexpr int d = decltype(d_c)::value;
    unsigned char* st = smem + stage * Tile::STAGE;
#pragma unroll
    for (int i = 0; i < PA; ++i) *reinterpret_cast<u32x4*>(st + Tile::place(l_row + i * Tile::RPP, l_piece)) = ra[d][i];
#pragma unroll
    for (int i = 0; i < PB; ++i) *reinterpret_cast<u32x4*>(st + Tile::BM * Tile::BK + Tile::place(l_row + i * Tile::RPP, l_piece)) = rb[d][i];
  };
  i32x4 acc[MI][NI];
#pragma unroll
  for (int mi = 0; mi < MI; ++mi)
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = i32x4{};
  auto barrier = [&]() {  // this wave's LDS accesses are done; the loads on their way stay there
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // slab 0 in LDS, slabs 1 .. D on their way
  if (k_tiles > 0) {
    static_for<0, D>([&](auto d) { fetch(d, d); });
    put(0, std::integral_constant<int, 0>{});
    fetch(D, std::integral_constant<int, 0>{});
    barrier();
  }
  for (int kt0 = 0; kt0 < k_tiles; kt0 += D) {
    static_for<0, D>([&](auto u) {
      const int kt = kt0 + u;
      if (kt >= k_tiles) return;
      const unsigned char* st = smem + (kt & 1) * Tile::STAGE;
#pragma unroll
      for (int kk = 0; kk < Tile::BK / 64; ++kk) {
        i32x4 af[MI], bf[NI];
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) af[mi] = *reinterpret_cast<const i32x4*>(st + Tile::place(wm * (Tile::BM / 2) + mi * 16 + fr, kk * 4 + fq));
#pragma unroll
        for (int ni = 0; ni < NI; ++ni)
          bf[ni] = *reinterpret_cast<const i32x4*>(st + Tile::BM * Tile::BK + Tile::place(wn * (Tile::BN / 2) + ni * 16 + fr, kk * 4 + fq));
        // (operands swapped: a lane holds 4 consecutive columns of one row)
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bf[ni], af[mi], acc[mi][ni], 0, 0, 0);
      }
      // slab kt + 1 takes the stage of slab kt - 1, which every wave has left; its registers take slab kt + 1 + D
      constexpr std::integral_constant<int, (decltype(u)::value + 1) % D> nx{};
      if (kt + 1 < k_tiles) {
        put((kt + 1) & 1, nx);
        fetch(kt + 1 + D, nx);
      }
      barrier();
    });
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
  static_assert(2 * Tile::STAGE <= 64 * 1024, "no opt-in to more LDS");
  set_tiles(p, Tile::BM, Tile::BN, 3, -1);
  const int64_t total = (int64_t)p.tiles_m * p.tiles_n;
  if (total > most_workgroups(Tile::NT)) return hipErrorInvalidValue;
  const auto kernel = p.bias != nullptr ? gemm_int8_any_kernel<Out, Tile, true> : gemm_int8_any_kernel<Out, Tile, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)total), dim3(Tile::NT), 2 * Tile::STAGE, stream, p);
  return hipGetLastError();
}

template <class Out>
hipError_t pick(const GemmParams& p, int cus, hipStream_t stream) {
  // 128 x 128 where that leaves a tile for every CU
  const int64_t tiles = (((int64_t)p.M + 127) / 128) * (((int64_t)p.N + 127) / 128);
  return tiles >= cus ? launch<Out, Int8Tile<128, 128, 64, 2>>(p, stream) : launch<Out, Int8Tile<64, 64, 128, 2>>(p, stream);
}

// Rows of up to two matrices at any byte to rows of whole 16-byte pieces, zeros behind their end: a piece a lane
struct AlignParams {
  const int8_t* from[2];
  unsigned char* to[2];
  int64_t pitch[2], pieces[2];
  int32_t K;
  uint32_t per_row;
  Divisor by_row;
};
template <bool WIDE>  // more pieces than 31 bits count
__global__ void __launch_bounds__(256) int8_align_kernel(const AlignParams p) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.pieces[0] + p.pieces[1]; i += (int64_t)gridDim.x * 256) {
    const int x = i < p.pieces[0] ? 0 : 1;
    const int64_t at = x == 0 ? i : i - p.pieces[0];
    const int64_t row = WIDE ? at / p.per_row : quotient((int)at, p.by_row);
    const int piece = (int)(at - row * p.per_row);
    *reinterpret_cast<u32x4*>(p.to[x] + at * 16) = int8_piece(p.from[x] + row * p.pitch[x], piece * 16, p.K);
  }
}

}  // namespace

hipError_t launch_gemm_int8_any(const GemmParams& p, bool bf16_out, int cus, hipStream_t stream) {
  return bf16_out ? pick<bf16>(p, cus, stream) : pick<f16>(p, cus, stream);
}

hipError_t launch_int8_align(const int8_t* a, int64_t lda, int64_t M, void* to_a, const int8_t* b, int64_t ldb, int64_t N, void* to_b, int64_t K,
                             hipStream_t stream) {
  const int64_t per_row = (K + 15) / 16, pieces = (M + N) * per_row;
  const AlignParams p{{a, b}, {static_cast<unsigned char*>(to_a), static_cast<unsigned char*>(to_b)}, {lda, ldb}, {M * per_row, N * per_row},
                      (int32_t)K, (uint32_t)per_row, make_divisor(per_row)};
  const int64_t wgs = (pieces + 255) / 256;
  hipLaunchKernelGGL(pieces > 0x7fffffffll ? int8_align_kernel<true> : int8_align_kernel<false>, dim3((unsigned)(wgs < (1 << 20) ? wgs : 1 << 20)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace aitamd
