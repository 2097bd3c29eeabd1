// Rotation of a head's dims by its token's position: pair i (dims i and n + i, or 2 i and 2 i + 1 where neighbours are
// paired) turns by position * freqs[i],
//     (x1, x2) -> scale * (x1 cos - x2 sin, x2 cos + x1 sin),
// and dims from 2 n on are handed through.  The inverse rotation, which is also the gradient's, has the sine's sign changed.
//
// The angle is taken in 64 bits, as a fraction of a turn: in 32, position 10^6 would be off by 0.06 rad.  What is left
// after whole turns are taken off is at most half a turn and goes on in 32 bits (off by 2^-25 of a turn).  The sines of a
// workgroup's tokens are taken once, into LDS, for all of their heads.
#pragma once

#include "common.hpp"

namespace aitamd {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryTable = 2048;      // (cosine, sine) entries of a workgroup: 16 KiB
constexpr int64_t kRotaryMaxDim = 1024; // of a head
constexpr int kRotaryMaxTokens = 64;    // of a workgroup

// Entries [0, tokens * n) of `table`: token t's pair i at t * n + i; position(t) gives the token's position.
template <class P>
AITAMD_DEVICE void fill_rotary_table(float2* table, const float* freqs, int n, Divisor by_n, int tokens, float scale, float sine_sign,
                                     P&& position) {
  for (int i = threadIdx.x; i < tokens * n; i += kRotaryThreads) {
    const int t = quotient(i, by_n), pair = i - t * n;
    double turns = (double)position(t) * ((double)freqs[pair] * 0.15915494309189533577);
    turns -= __builtin_rint(turns);
    float s, c;
    sincospif((float)(2.0 * turns), &s, &c);
    table[i] = make_float2(c * scale, s * (scale * sine_sign));
  }
}

// What a lane handles of a head at once, a piece: VEC pairs of halves (VEC elements each), or VEC / 2 pairs of neighbours; behind
// the rotated dims VEC elements.  VEC = 1: one pair, behind them one element.
constexpr int rotary_pieces(int n, int head_dim, bool interleaved, int vec) {
  return vec > 1 ? (interleaved ? 2 * n / vec : n / vec) + (head_dim - 2 * n) / vec : n + head_dim - 2 * n;
}
// The widest pieces that heads of `head_dim` with n pairs divide into (at any alignment: see load_vec)
inline int rotary_vec(int64_t n, int64_t head_dim, bool interleaved) {
  for (int vec = 8; vec > 1; vec /= 2)
    if (head_dim % vec == 0 && (interleaved ? (2 * n) % vec == 0 : n % vec == 0) && (head_dim - 2 * n) % vec == 0) return vec;
  return 1;
}

template <class T, int N>
struct RotaryVec {
  typedef T type __attribute__((ext_vector_type(N)));
};
// One piece on its way: where it comes from and goes to, its elements, its pairs' sines (null: handed through)
template <class T, int VEC, bool INTERLEAVED>
struct RotaryPiece {
  using Tr = ElemTraits<T>;
  using vec = typename RotaryVec<T, VEC>::type;
  T *y1, *y2;
  const float2* table;
  vec v1, v2;
  // piece `c` of the head at `x`, with the token's table, to `y` (which may be `x`)
  AITAMD_DEVICE void load(const T* x, T* y, int c, int n, const float2* of_token) {
    const int turned = VEC == 1 ? n : (INTERLEAVED ? 2 * n / VEC : n / VEC);
    int i1, i2;
    if (c >= turned) {
      i1 = 2 * n + (c - turned) * VEC;
      i2 = i1;
      table = nullptr;
    } else {
      // (VEC = 1: neighbours are two elements of their own)
      i1 = INTERLEAVED && VEC == 1 ? 2 * c : c * VEC;
      i2 = INTERLEAVED ? i1 + 1 : n + i1;
      table = of_token + (INTERLEAVED && VEC > 1 ? c * (VEC / 2) : c * VEC);
    }
    y1 = y + i1;
    y2 = y + i2;
    v1 = load_vec<vec>(x + i1);
    if constexpr (!INTERLEAVED || VEC == 1) v2 = load_vec<vec>(x + i2);
  }
  AITAMD_DEVICE void store() {
    if (table != nullptr) {
      if constexpr (INTERLEAVED && VEC > 1) {
#pragma unroll
        for (int j = 0; j < VEC / 2; ++j) {
          const float2 w = table[j];
          const float a = Tr::to_float(v1[2 * j]), b = Tr::to_float(v1[2 * j + 1]);
          v1[2 * j] = Tr::from_float(a * w.x - b * w.y);
          v1[2 * j + 1] = Tr::from_float(b * w.x + a * w.y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 w = table[j];
          const float a = Tr::to_float(v1[j]), b = Tr::to_float(v2[j]);
          v1[j] = Tr::from_float(a * w.x - b * w.y);
          v2[j] = Tr::from_float(b * w.x + a * w.y);
        }
        store_vec(y2, v2);
      }
    }
    store_vec(y1, v1);
  }
};

// Pieces of a lane on their way together (16384 x 32 x 128, 64 dims of neighbours: 46.9 us with one, 40.8 with two)
constexpr int kRotaryAhead = 2;

// Tokens of a workgroup: about four pieces for each lane where there are tokens enough for every CU, within the table
inline int rotary_tokens(int64_t tokens, int64_t pieces_per_token, int64_t n, int cus) {
  int64_t t = 4 * kRotaryThreads / (pieces_per_token > 0 ? pieces_per_token : 1);
  const int64_t fill = (tokens + 2 * cus - 1) / (2 * cus);
  if (t > fill) t = fill;
  if (n > 0 && t > kRotaryTable / n) t = kRotaryTable / n;
  if (t > kRotaryMaxTokens) t = kRotaryMaxTokens;
  return t < 1 ? 1 : (int)t;
}

}  // namespace aitamd
