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

// What a lane handles of a head at once: VEC = 8: eight pairs of halves 16 bytes each (HALVES), or four pairs of neighbours;
// behind the rotated dims 8 elements.  VEC = 1: one pair, behind them one element.
constexpr int rotary_pieces(int n, int head_dim, bool interleaved, int vec) {
  return vec == 8 ? (interleaved ? n / 4 : n / 8) + (head_dim - 2 * n) / 8 : n + head_dim - 2 * n;
}

// Piece `c` of the head at `x`, rotated by the token's table, to `y` (which may be `x`)
template <class T, int VEC, bool INTERLEAVED>
AITAMD_DEVICE void rotate_piece(const T* x, T* y, int c, int n, const float2* table) {
  using Tr = ElemTraits<T>;
  using vec8 = typename Tr::vec8;
  if constexpr (VEC == 8) {
    const int turned = INTERLEAVED ? n / 4 : n / 8;
    if (c >= turned) {
      const int at = 2 * n + (c - turned) * 8;
      store_vec(y + at, load_vec<vec8>(x + at));
    } else if constexpr (INTERLEAVED) {
      const vec8 v = load_vec<vec8>(x + c * 8);
      vec8 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 w = table[c * 4 + j];
        const float a = Tr::to_float(v[2 * j]), b = Tr::to_float(v[2 * j + 1]);
        o[2 * j] = Tr::from_float(a * w.x - b * w.y);
        o[2 * j + 1] = Tr::from_float(b * w.x + a * w.y);
      }
      store_vec(y + c * 8, o);
    } else {
      const vec8 v1 = load_vec<vec8>(x + c * 8), v2 = load_vec<vec8>(x + n + c * 8);
      vec8 o1, o2;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 w = table[c * 8 + j];
        const float a = Tr::to_float(v1[j]), b = Tr::to_float(v2[j]);
        o1[j] = Tr::from_float(a * w.x - b * w.y);
        o2[j] = Tr::from_float(b * w.x + a * w.y);
      }
      store_vec(y + c * 8, o1);
      store_vec(y + n + c * 8, o2);
    }
  } else {
    if (c >= n) {
      y[n + c] = x[n + c];
    } else {
      const int i1 = INTERLEAVED ? 2 * c : c, i2 = INTERLEAVED ? 2 * c + 1 : n + c;
      const float2 w = table[c];
      const float a = Tr::to_float(x[i1]), b = Tr::to_float(x[i2]);
      y[i1] = Tr::from_float(a * w.x - b * w.y);
      y[i2] = Tr::from_float(b * w.x + a * w.y);
    }
  }
}

// Whether heads of `head_dim` with n pairs go 8 elements at a time (at any alignment: see load_vec)
inline bool rotary_wide(int64_t n, int64_t head_dim, bool interleaved) {
  return head_dim % 8 == 0 && (interleaved ? (2 * n) % 8 == 0 : n % 8 == 0);
}

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
