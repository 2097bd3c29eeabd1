// The low-rank part of a projection that many requests share: rows of one launch belong to different adapters,
//     y[m, n] = sum_k x[m, k] w[n, k] (+ bias[n]) + sum_j t[m, j] b[i(m)][n, j],   t[m, j] = scale[i(m)] sum_k x[m, k] a[i(m)][j, k].
// A launch ahead of the product's makes t (lora_api.hip); the product's tiles add t b to their accumulators behind the K loop, as
// if K went on, and round once.
//
// t lies in scratch memory in two bfloat16 numbers that add up to it (off by 2^-17 at most, and of the range of 32 bits, which
// one half of the other type or both do not have), the first of eight ranks and then the second of them.  bfloat16 adapters are
// multiplied with both; a half is the sum of two bfloat16 numbers too (8 of its 11 bits and the 3 behind them), so that halves are
// four products: exact, all of them.
//
// Per wave: the adapters of its rows one after the other, on matrix instructions, for all its rows at once; each row takes the
// products with its own.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "epilogue.hpp"
#include "gemm_kernel.hpp"

namespace aitamd {

// The workgroups of a shared tile that have its adapters and none of K, a power of two of them: one alone takes longer than K where every
// row has its own (64 x 6144 x 4096, 48 adapters at random, rank 16 / 64: 21.8 / 46 us with one workgroup, 18.6 / 36.8 so; with one
// adapter for all rows 18.2 / 18.9 and 18.1 / 20.1).
constexpr int kLoraMostParts = 4;
constexpr int lora_parts_of_tile(int rank) { return rank > 32 ? kLoraMostParts : 2; }

// a row's elements in scratch memory: chunks of eight ranks, two parts each
constexpr int lora_chunks(int rank) { return (rank + 7) / 8; }
AITAMD_DEVICE const bf16* lora_row(const GemmParams& p, int m) {
  return reinterpret_cast<const bf16*>(p.lora_t) + (int64_t)m * (lora_chunks(p.lora_rank) * 16);
}
// the adapter of row m, or -1 (-2: there is no such row)
AITAMD_DEVICE int lora_adapter(const GemmParams& p, int m) {
  if (m >= p.M) return -2;
  const int id = p.lora_of[m];
  return (uint32_t)id < (uint32_t)p.lora_n ? id : -1;
}
// the adapter's row of column n
template <class T>
AITAMD_DEVICE const T* lora_column(const GemmParams& p, int id, int n) {
  return reinterpret_cast<const T*>(p.lora_b) + ((int64_t)id * p.N + n) * p.lora_rank;
}
// eight numbers as the sums of two (an infinity or a NaN as itself and zero)
template <class T>
AITAMD_DEVICE void lora_parts(typename ElemTraits<T>::vec8 v, bf16x8& one, bf16x8& two) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = ElemTraits<T>::to_float(v[j]);
    one[j] = (bf16)f;
    two[j] = __builtin_isfinite(f) ? (bf16)(f - (float)one[j]) : (bf16)0.0f;
  }
}
// eight bfloat16 numbers: whether they all are; those that are, or (pass 1) the largest number for those that are not; the largest
// number with the sign of each
AITAMD_DEVICE bool lora_numbers(u32x4 v) {
  bool all = true;
#pragma unroll
  for (int d = 0; d < 4; ++d) all = all && (v[d] & 0x7f80u) != 0x7f80u && (v[d] & 0x7f800000u) != 0x7f800000u;
  return all;
}
AITAMD_DEVICE u32x4 lora_split(u32x4 v, int pass) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t none = ((v[d] & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((v[d] & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
    v[d] = pass == 0 ? v[d] & ~none : ((v[d] & 0x80008000u) | 0x7f7f7f7fu) & none;
  }
  return v;
}
AITAMD_DEVICE u32x4 lora_largest(u32x4 v) {
#pragma unroll
  for (int d = 0; d < 4; ++d) v[d] = (v[d] & 0x80008000u) | 0x7f7f7f7fu;
  return v;
}

// The part of a wave whose rows row0 + mi * MT + (lane % MT) meet columns col0 + ni * MT + (lane % MT).
template <class T, int MT, int MI, int NI>
struct LoraTile {
  // 16 x 16: a step's four quarters are both parts of t of two chunks (halves: both by both of one); 32 x 32: its two
  // halves are both parts of t of one chunk (halves: once with each of the adapter's)
  static constexpr bool kHalves = !std::is_same_v<T, bf16>;
  static constexpr int PER = MT == 16 && !kHalves ? 2 : 1;
  int of[MI];

  AITAMD_DEVICE void read(const GemmParams& p, int row0, int lane) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) of[mi] = lora_adapter(p, row0 + mi * MT + lane % MT);
  }
  // the first adapter of those left, or -1 (the same for all lanes)
  static AITAMD_DEVICE int first_of(const int (&left)[MI]) {
    int id = -1;
    static_for<0, MI>([&](auto i) __attribute__((always_inline)) {
      constexpr int mi = MI - 1 - decltype(i)::value;
      const uint64_t some = __builtin_amdgcn_ballot_w64(left[mi] >= 0);
      if (some != 0) id = __builtin_amdgcn_readlane(left[mi], __builtin_ctzll(some));
    });
    return id;
  }
  // the operands w of chunks c0 on, without what lies behind the last rank: the next column's first.  An odd rank shares its dword
  // with that (with the buffer's end, which takes whole dwords), and is read again by itself.
  template <int STEPS>
  static AITAMD_DEVICE void last_ranks(int rank, int c0, int half, __amdgpu_buffer_rsrc_t rb, uint32_t b_at, u32x4 (&w)[STEPS][NI]) {
    if (8 * (c0 + STEPS * PER) <= rank) return;
    const uint32_t b_pitch = (uint32_t)rank * 2u;
    static_for<0, STEPS>([&](auto s_c) __attribute__((always_inline)) {
      const int c = c0 + decltype(s_c)::value * PER + half, dwords = rank / 2 - 4 * c;
      static_for<0, NI>([&](auto ni) __attribute__((always_inline)) {
        const uint32_t at = b_at + (uint32_t)(decltype(ni)::value * MT) * b_pitch + (uint32_t)((rank - 1) * 2 - half * 16);
        const uint32_t last =
            (rank & 1) != 0 && 8 * c < rank ? (uint32_t)(uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rb, at, 0, 0) : 0u;
#pragma unroll
        for (int d = 0; d < 4; ++d) w[decltype(s_c)::value][ni][d] = d < dwords ? w[decltype(s_c)::value][ni][d] : (d == dwords ? last : 0u);
      });
    });
  }
  // The products of every row with each adapter, of which a row takes those with its own: acc[mi][ni], whose elements are all of row
  // lane % MT of block mi.  STEPS matrix instructions' worth of AHEAD adapters are on their way together: where each row has its own, the
  // time is that of the trips to memory.
  // Of the adapters in the order of their first rows, those whose numbers' bits `others` are `part_of`.
  template <int STEPS, int AHEAD, class Acc>
  AITAMD_DEVICE void add_own(const GemmParams& p, int row0, int col0, int lane, int part_of, int others, Acc (&acc)[MI][NI]) const {
    using Op = MfmaOp<bf16, MT>;
    const int fr = lane % MT, fq = lane / MT;
    const int rank = p.lora_rank, chunks = lora_chunks(rank);
    const int rows = p.M - row0 < MI * MT ? p.M - row0 : MI * MT, columns = p.N - col0 < NI * MT ? p.N - col0 : NI * MT;
    if (rows <= 0 || columns <= 0) return;
    const uint32_t t_pitch = (uint32_t)chunks * 32u, b_pitch = (uint32_t)rank * 2u;
    const __amdgpu_buffer_rsrc_t rt = make_rsrc(lora_row(p, row0), (uint32_t)rows * t_pitch);
    const int half = PER == 2 ? fq & 1 : 0;
    const int part = MT == 32 ? fq : (PER == 2 ? fq >> 1 : fq & 1);
    uint32_t t_at = (uint32_t)fr * t_pitch + (uint32_t)(half * 32 + part * 16), b_at = (uint32_t)fr * b_pitch + (uint32_t)(half * 16);
    // (opaque: what hangs on the tile alone would be computed ahead of the K loop, held over it and spilled)
    asm volatile("" : "+v"(t_at), "+v"(b_at));
    int left[MI];
#pragma unroll 1
    for (int c0 = 0; c0 < chunks; c0 += STEPS * PER) {
      u32x4 t[STEPS][MI];
      static_for<0, MI>([&](auto mi) __attribute__((always_inline)) {
        left[mi] = of[mi];
        static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
          const uint32_t tc = t_at + (uint32_t)(c0 + s * PER) * 32u + (uint32_t)(decltype(mi)::value * MT) * t_pitch;
          t[s][mi] = buffer_load_16B(rt, c0 + s * PER + half < chunks ? tc : kOobOffset);
        });
      });
      for (int number = 0;;) {
        int id[AHEAD];
        u32x4 w[AHEAD][STEPS][NI];
        static_for<0, AHEAD>([&](auto i) __attribute__((always_inline)) {
          do {
            id[i] = first_of(left);
            static_for<0, MI>([&](auto mi) __attribute__((always_inline)) { left[mi] = left[mi] == id[i] ? -1 : left[mi]; });
          } while (id[i] >= 0 && (number++ & others) != part_of);
          if (id[i] < 0) return;
          const __amdgpu_buffer_rsrc_t rb = make_rsrc(lora_column<T>(p, id[i], col0), (uint32_t)columns * b_pitch);
          static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
            const uint32_t bc = b_at + (uint32_t)(c0 + s * PER) * 16u;
            static_for<0, NI>([&](auto ni) __attribute__((always_inline)) {
              w[i][s][ni] = buffer_load_16B(rb, c0 + s * PER + half < chunks ? bc + (uint32_t)(decltype(ni)::value * MT) * b_pitch : kOobOffset);
            });
          });
        });
        static_for<0, AHEAD>([&](auto i) __attribute__((always_inline)) {
          if (id[i] < 0) return;
          if (8 * (c0 + STEPS * PER) > rank) {
            const __amdgpu_buffer_rsrc_t rb = make_rsrc(lora_column<T>(p, id[i], col0), (uint32_t)columns * b_pitch);
            last_ranks(rank, c0, half, rb, b_at, w[i]);
          }
          bf16x8 two[STEPS][NI];
          if constexpr (kHalves) {
            static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
              static_for<0, NI>([&](auto ni) __attribute__((always_inline)) {
                bf16x8 one;
                lora_parts<T>(__builtin_bit_cast(typename ElemTraits<T>::vec8, w[i][s][ni]), one, two[s][ni]);
                w[i][s][ni] = __builtin_bit_cast(u32x4, MT == 16 && (fq >> 1) ? two[s][ni] : one);
              });
            });
          }
          static_for<0, MI>([&](auto mi) __attribute__((always_inline)) {
            const bool own = of[mi] == id[i];
            if (__builtin_amdgcn_ballot_w64(own) == 0) return;
            static_for<0, NI>([&](auto ni) __attribute__((always_inline)) {
              Acc sum{};
              static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
                const bf16x8 a = __builtin_bit_cast(bf16x8, t[s][mi]);
                sum = Op::run(__builtin_bit_cast(bf16x8, w[i][s][ni]), a, sum);
                if constexpr (kHalves && MT == 32) sum = Op::run(two[s][ni], a, sum);
              });
#pragma unroll
              for (int e = 0; e < (int)(sizeof(Acc) / 4); ++e) acc[mi][ni][e] += own ? sum[e] : 0.0f;
            });
          });
        });
        if (id[AHEAD - 1] < 0) break;
      }
    }
  }
  // ... for accumulators that matrix instructions alone may touch: each adapter with the rows of the others set to zero.
  // multiply(b, a, mi, ni): accumulator (mi, ni) plus the product of the weight rows b and the rows a, both bf16x8.  Through
  // buffers that end with the rows and the columns: 32-bit offsets, and no branch around what is not there.
  template <int STEPS, class M>
  AITAMD_DEVICE void add(const GemmParams& p, int row0, int col0, int lane, M&& multiply) const {
    const int fr = lane % MT, fq = lane / MT;
    const int rank = p.lora_rank, chunks = lora_chunks(rank);
    const int rows = p.M - row0 < MI * MT ? p.M - row0 : MI * MT, columns = p.N - col0 < NI * MT ? p.N - col0 : NI * MT;
    if (rows <= 0 || columns <= 0) return;
    const uint32_t t_pitch = (uint32_t)chunks * 32u, b_pitch = (uint32_t)rank * 2u;
    const __amdgpu_buffer_rsrc_t rt = make_rsrc(lora_row(p, row0), (uint32_t)rows * t_pitch);
    const int half = PER == 2 ? fq & 1 : 0;
    const int part = MT == 32 ? fq : (PER == 2 ? fq >> 1 : fq & 1);
    uint32_t t_at = (uint32_t)fr * t_pitch + (uint32_t)(half * 32 + part * 16), b_at = (uint32_t)fr * b_pitch + (uint32_t)(half * 16);
    // (opaque: what hangs on the tile alone would be computed ahead of the K loop, held over it and spilled)
    asm volatile("" : "+v"(t_at), "+v"(b_at));
    int left[MI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) left[mi] = of[mi];
    for (;;) {
      const int id = first_of(left);
      if (id < 0) break;
      const __amdgpu_buffer_rsrc_t rb = make_rsrc(lora_column<T>(p, id, col0), (uint32_t)columns * b_pitch);
      // rows of others among the wave's
      bool mixed = false;
      static_for<0, MI>([&](auto mi) __attribute__((always_inline)) {
        mixed = mixed || __builtin_amdgcn_ballot_w64(of[mi] != id && of[mi] != -2) != 0;
      });
      for (int c0 = 0; c0 < chunks; c0 += STEPS * PER) {
        // Numbers that are none, times the zeros of other requests' rows, would reach them: where a wave meets some, the product is
        // taken without them first, then again with the largest number in their places and zeros in the others', times the
        // largest: an infinity where it belongs and zero elsewhere.
        bool again = false;
        for (int pass = 0; pass < 2; ++pass) {
          u32x4 w[STEPS][NI], t[STEPS][MI];
          static_for<0, STEPS>([&](auto s_c) __attribute__((always_inline)) {
            constexpr int s = decltype(s_c)::value;
            const bool on = c0 + s * PER + half < chunks;
            const uint32_t tc = t_at + (uint32_t)(c0 + s * PER) * 32u, bc = b_at + (uint32_t)(c0 + s * PER) * 16u;
            static_for<0, NI>([&](auto ni) __attribute__((always_inline)) {
              w[s][ni] = buffer_load_16B(rb, on ? bc + (uint32_t)(decltype(ni)::value * MT) * b_pitch : kOobOffset);
            });
            static_for<0, MI>([&](auto mi) __attribute__((always_inline)) {
              t[s][mi] = buffer_load_16B(rt, on && left[mi] == id ? tc + (uint32_t)(decltype(mi)::value * MT) * t_pitch : kOobOffset);
            });
          });
          last_ranks(rank, c0, half, rb, b_at, w);
          bf16x8 two[STEPS][NI];
          if constexpr (kHalves) {
            static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
              static_for<0, NI>([&](auto ni) __attribute__((always_inline)) {
                bf16x8 one;
                lora_parts<T>(__builtin_bit_cast(typename ElemTraits<T>::vec8, w[s][ni]), one, two[s][ni]);
                w[s][ni] = __builtin_bit_cast(u32x4, MT == 16 && (fq >> 1) ? two[s][ni] : one);
              });
            });
          }
          if (mixed) {
            if (pass == 0) {
              bool numbers = true;
              static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
                static_for<0, NI>([&](auto ni) __attribute__((always_inline)) { numbers = numbers && lora_numbers(w[s][ni]); });
              });
              again = __builtin_amdgcn_ballot_w64(!numbers) != 0;
            }
            if (again) {
              static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
                static_for<0, NI>([&](auto ni) __attribute__((always_inline)) { w[s][ni] = lora_split(w[s][ni], pass); });
                if (pass == 1) {
                  const bool on = c0 + decltype(s)::value * PER + half < chunks;
                  static_for<0, MI>([&](auto mi) __attribute__((always_inline)) { t[s][mi] = on && left[mi] == id ? lora_largest(t[s][mi]) : u32x4{}; });
                }
              });
            }
          }
          static_for<0, MI>([&](auto mi) __attribute__((always_inline)) {
            if (__builtin_amdgcn_ballot_w64(left[mi] == id) == 0) return;
            static_for<0, STEPS>([&](auto s) __attribute__((always_inline)) {
              const bf16x8 a = __builtin_bit_cast(bf16x8, t[s][mi]);
              static_for<0, NI>([&](auto ni) __attribute__((always_inline)) { multiply(__builtin_bit_cast(bf16x8, w[s][ni]), a, mi, ni); });
              if constexpr (kHalves && MT == 32) {
                if (pass == 0)
                  static_for<0, NI>([&](auto ni) __attribute__((always_inline)) { multiply(two[s][ni], a, mi, ni); });
              }
            });
          });
          if (!again) break;
        }
      }
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) left[mi] = left[mi] == id ? -1 : left[mi];
    }
  }
};

// t of eight ranks
AITAMD_DEVICE void lora_sum(const bf16* t, int c, float (&f)[8]) {
  const bf16x8 one = load_vec<bf16x8>(t + c * 16), two = load_vec<bf16x8>(t + c * 16 + 8);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (float)one[j] + (float)two[j];
}
// column n of row m by itself: the sum v and its adapter's
template <class T>
AITAMD_DEVICE float lora_add(float v, const GemmParams& p, int m, int n) {
  using Tr = ElemTraits<T>;
  const int id = lora_adapter(p, m);
  if (id < 0) return v;
  const int rank = p.lora_rank, whole = rank / 8;
  const bf16* const t = lora_row(p, m);
  const T* const row = lora_column<T>(p, id, n);
  float f[8];
  for (int c = 0; c < whole; ++c) {
    const auto w = load_vec<typename Tr::vec8>(row + c * 8);
    lora_sum(t, c, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) v = __builtin_fmaf(f[e], Tr::to_float(w[e]), v);
  }
#pragma unroll 1
  for (int e = whole * 8; e < rank; ++e)
    v = __builtin_fmaf((float)t[whole * 16 + e % 8] + (float)t[whole * 16 + 8 + e % 8], Tr::to_float(row[e]), v);
  return v;
}

}  // namespace aitamd
