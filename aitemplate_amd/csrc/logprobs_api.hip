// C ABI launcher of aitamd_token_logprobs: of rows of logits the log probabilities and ranks of given tokens, the entropies and the
// most probable tokens, in one pass over the logits.
//
// With c = scale log2(e) and m the largest x seen so far, a thread keeps s = sum 2^d and u = sum 2^d d of its elements, d = c x - R with
// R = c m rounded (any number next to it would do: it comes off again), both in 32 bits; a larger m multiplies s by f = 2^(R - R') and
// makes u f (u + s (R - R')).  Joined over a row,
//     log p(t) = scale (x_t - m) + ln 2 (c m - R) - ln s,     entropy = ln s - ln 2 u / s.
// Bound: memory; the vector instructions, ten an element (the exponential as four of them), are next to it for 2-byte logits.  Few rows:
// several workgroups a row, joined by a second launch.
//
// The most probable: 64-bit keys (value, then the lower token), all different.  A workgroup keeps those that may be among them in
// LDS: what reaches a bound is put behind the others with one atomic addition each, so their order varies from run to run, and the
// outcome does not.  The first round's bound is next to the `top`-th largest of its lanes' largest (with the least of the waves'
// shares of them for one, some five times as many reach it: 4096 x 32768 in fp16 with 20 alternatives 157 us with that bound to the
// end, 104 with a selection behind every round); whenever as many again have come, the best `top` are picked and the last of them is
// the bound from there on.  Where they do not fit (ascending rows, many equal ones), the round is done again with the exact
// bound that at most `top` threads reach.
#include "../../include/aitemplate_amd_kernels.h"
#include "common.hpp"
#include "device.hpp"
#include "errors.hpp"

namespace aitamd {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kEach = 16;                       // elements of a thread in a round
constexpr int kRound = kThreads * kEach;
constexpr int kMostTop = 64;
constexpr int kKeys = 2048;                     // candidates in LDS
static_assert(kWaves * (kMostTop / kWaves + 2) <= 128, "two of a lane");
constexpr int kMostSplits = kKeys / kMostTop;
static_assert(kMostTop + kMostTop * kEach <= kKeys, "a round done again fits behind those kept");

struct LogprobParams {
  const void *logits, *tokens;
  float *logprob, *entropy, *top_logprob;
  int32_t *rank, *top_token;
  unsigned char* parts;  // of (row, split): PartHead, then `top` keys
  int64_t ld;
  int32_t rows, V, top, splits, per_split, tokens_64, part_bytes, first;
  float scale;
};
struct PartHead {
  float m, s, u;
  int32_t ahead;
};

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

AITAMD_DEVICE float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The first element that a piece of it would not be whole for is read one by one.
template <class T>
struct Logits {
  static constexpr int VEC = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(VEC)));
};

// larger for a larger number; NaN the least
AITAMD_DEVICE uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? 0u : ((int32_t)b < 0 ? ~b : b | 0x80000000u);
}
AITAMD_DEVICE float unordered(uint32_t o) { return __uint_as_float((int32_t)o < 0 ? o & 0x7fffffffu : ~o); }
AITAMD_DEVICE uint64_t key_of(float x, int token) { return (uint64_t)ordered(x) << 32 | (uint32_t)~token; }

// the largest number of a piece (-inf where there is none)
template <class T>
AITAMD_DEVICE float largest_of(typename Logits<T>::vec v) {
  if constexpr (std::is_same_v<T, f16>) {
    // (two at a time)
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(f16x2{v[0], v[1]}, f16x2{v[2], v[3]}),
                                              __builtin_elementwise_max(f16x2{v[4], v[5]}, f16x2{v[6], v[7]}));
    return fmaxf(fmaxf((float)m[0], (float)m[1]), -__builtin_inff());
  } else {
    float m = (float)v[0];
#pragma unroll
    for (int e = 1; e < Logits<T>::VEC; ++e) m = fmaxf(m, (float)v[e]);
    return fmaxf(m, -__builtin_inff());
  }
}
// v joined with that of the lane which a step of a reduction along the wave gives (none: `none`)
template <int CTRL>
AITAMD_DEVICE float lane_step(float v, float none) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, 0xf, 0xf, false));
}
// over the 64 lanes, for all of them: neighbours in rows of 16 (row_shr 1, 2, 4, 8), then rows (row_bcast 15, 31)
template <class F>
AITAMD_DEVICE float wave_reduce(float v, float none, F&& f) {
  v = f(v, lane_step<0x111>(v, none));
  v = f(v, lane_step<0x112>(v, none));
  v = f(v, lane_step<0x114>(v, none));
  v = f(v, lane_step<0x118>(v, none));
  v = f(v, lane_step<0x142>(v, none));
  v = f(v, lane_step<0x143>(v, none));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
AITAMD_DEVICE float wave_max(float v) {
  return wave_reduce(v, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); });
}
AITAMD_DEVICE float wave_sum(float v) {
  return wave_reduce(v, 0.0f, [](float a, float b) { return a + b; });
}

// The `keep` largest of n keys, in order, zeros behind the last: every key counts those above it (they are all different, but for
// zeros, which are none), several neighbouring lanes the keys of one where there are fewer than threads.  All threads; there is room
// for 8 keys more (or for THREADS + 8 in all), which are overwritten, and `out` does not overlap them.
template <int THREADS>
AITAMD_DEVICE void largest(uint64_t* keys, int n, uint64_t* out, int keep) {
  int shift = 0;
  while (shift < 6 && n << (shift + 1) <= THREADS) ++shift;
  const int parts = 1 << shift, part = threadIdx.x & (parts - 1);
  for (int i = threadIdx.x; i < keep; i += THREADS) out[i] = 0;
  for (int i = threadIdx.x; i < 8 * parts; i += THREADS) keys[n + i] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n; i0 += THREADS >> shift) {
    const int i = i0 + (threadIdx.x >> shift);
    const uint64_t mine = i < n ? keys[i] : ~0ull;
    int above = 0;
    // (eight at a time: one by one, every read is waited for)
    for (int j = part; j < n; j += 8 * parts) {
#pragma unroll
      for (int e = 0; e < 8; ++e) above += keys[j + e * parts] > mine ? 1 : 0;
    }
    for (int d = 1; d < parts; d <<= 1) above += __shfl_xor(above, d);
    if (i < n && mine != 0 && part == 0 && above < keep) out[above] = mine;
  }
}

// Numbers next to the lowest of the type (a mask's) times c may leave the range: they go by their differences.
AITAMD_DEVICE bool in_range(float m, float c) { return fabsf(m * c) < 1e38f; }
// From one R to another, at least -1000 (2^-1000 is 0)
AITAMD_DEVICE float step_down(float m, float to, float c) {
  return fmaxf(in_range(m, c) && in_range(to, c) ? m * c - to * c : (m - to) * c, -1000.0f);
}
AITAMD_DEVICE void join(float& m, float& s, float& u, float m2, float s2, float u2, float c) {
  const float to = fmaxf(m, m2);
  const float d1 = step_down(m, to, c), d2 = step_down(m2, to, c);
  const float f1 = exp2_fast(d1), f2 = exp2_fast(d2);
  u = f1 * (u + s * d1) + f2 * (u2 + s2 * d2);
  s = s * f1 + s2 * f2;
  m = to;
}

AITAMD_DEVICE int token_of(const LogprobParams& p, int row) {
  const int64_t t = p.tokens_64 ? reinterpret_cast<const int64_t*>(p.tokens)[row] : reinterpret_cast<const int32_t*>(p.tokens)[row];
  return t >= 0 && t < p.V ? (int)t : -1;
}

// What a row's threads have found, to the results (by one wave)
template <class T>
AITAMD_DEVICE void finish(const LogprobParams& p, int row, float m, float s, float u, int ahead, const uint64_t* best) {
  const int lane = threadIdx.x & 63;
  // (the sum is of 2^(c x - R), and R not quite c m)
  const float c = p.scale * kLog2e, log_s = logf(s) - (in_range(m, c) ? kLn2 * __builtin_fmaf(m, c, -(m * c)) : 0.0f);
  if (lane == 0) {
    const int token = token_of(p, row);
    float lp = 0.0f;
    if (token >= 0) {
      const float x = (float)reinterpret_cast<const T*>(p.logits)[row * p.ld + token];
      lp = s == 0.0f ? -__builtin_inff() : (x - m) * p.scale - log_s;
    }
    p.logprob[row] = lp;
    p.entropy[row] = s == 0.0f ? 0.0f : logf(s) - kLn2 * (u / s);
    p.rank[row] = token >= 0 ? ahead : -1;
  }
  if (lane < p.top) {
    const uint64_t key = best[lane];
    const float x = unordered((uint32_t)(key >> 32));
    p.top_token[(int64_t)row * p.top + lane] = key >> 32 == 0 ? -1 : (int32_t)~(uint32_t)key;
    p.top_logprob[(int64_t)row * p.top + lane] = key >> 32 == 0 ? __builtin_nanf("") : (s == 0.0f ? -__builtin_inff() : (x - m) * p.scale - log_s);
  }
}

// (LDS alone is waited for: the next round's logits are on their way)
AITAMD_DEVICE void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 8 : 6) logprob_kernel(const LogprobParams p) {
  constexpr int VEC = Logits<T>::VEC, PIECES = kEach / VEC;
  using vec = typename Logits<T>::vec;
  __shared__ uint64_t keys[TOP ? kKeys + 8 : 1], best[TOP ? kThreads : 1];
  __shared__ float lane_best[kWaves * (kMostTop / kWaves + 2)];
  __shared__ PartHead heads[kWaves];
  __shared__ int added[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int item = p.first + blockIdx.x, row = item / p.splits, split = item - row * p.splits;
  const int v0 = split * p.per_split, v1 = p.V - v0 < p.per_split ? p.V : v0 + p.per_split;
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.ld;
  const float c = p.scale * kLog2e;
  vec next[PIECES];
  const int rounds = (v1 - v0 + kRound - 1) / kRound;
  auto piece_at = [&](int round, int i) { return v0 + round * kRound + (i * kThreads + tid) * VEC; };
  // (a branch for the whole workgroup: one for each piece would be waited at)
  auto load = [&](int round, vec (&v)[PIECES]) __attribute__((always_inline)) {
    if (v0 + (round + 1) * kRound <= v1) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) v[i] = load_vec<vec>(x + piece_at(round, i));
    } else {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int at = piece_at(round, i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = (T)-__builtin_inff();
        if (at + VEC <= v1) {
          v[i] = load_vec<vec>(x + at);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e)
            if (at + e < v1) v[i][e] = x[at + e];
        }
      }
    }
  };
  load(0, next);
  const int token = token_of(p, row);
  const float given = token >= 0 ? (float)x[token] : __builtin_inff();
  // (what of the elements in front of the token is not at most the number below its logit is at least as large)
  float below = given;
  if (given == -__builtin_inff())
    below = __builtin_nanf("");
  else if (token >= 0)
    below = given == 0.0f ? -__uint_as_float(1u) : __uint_as_float(__float_as_uint(given) + (given > 0.0f ? -1 : 1));

  float m = -3.402823466e38f, s = 0.0f, u = 0.0f;
  int ahead = 0;
  // the bound of what may be among the most probable, by value and by key; candidates so far
  float bound = -__builtin_inff();
  uint64_t bound_key = 0;
  int kept = 0;
  if (TOP && tid < 3) added[tid] = 0;
  if constexpr (TOP) barrier();

  for (int r = 0; r < rounds; ++r) {
    vec v[PIECES];
    float most[PIECES], here = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      v[i] = next[i];
      most[i] = largest_of<T>(v[i]);
      here = fmaxf(here, most[i]);
    }
    if (r + 1 < rounds) load(r + 1, next);
    if (here > m) {
      const float d = step_down(m, here, c), f = exp2_fast(d);
      u = f * (u + s * d);
      s *= f;
      m = here;
    }
    auto sum = [&](auto by_product) __attribute__((always_inline)) {
      const float R = m * c;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const float than = piece_at(r, i) + VEC <= token ? below : given;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xe = (float)v[i][e];
          const float d = decltype(by_product)::value ? __builtin_fmaf(xe, c, -R) : (xe - m) * c;
          const float w = exp2_fast(d);
          s += w;
          u = __builtin_fmaf(w, fmaxf(d, -1000.0f), u);
          ahead += __builtin_popcountll(__builtin_amdgcn_ballot_w64(!(xe <= than)));
        }
      }
    };
    if (__builtin_amdgcn_ballot_w64(!in_range(m, c)) == 0)
      sum(std::true_type{});
    else
      sum(std::false_type{});
    if constexpr (TOP) {
      if (r == 0) {
        // The largest of every wave's lanes, a few more each than make `top` together: the `top`-th of them all, found by halving to
        // 20 bits, is a bound that `top` elements reach and not many more.
        const int g = (p.top + kWaves - 1) / kWaves + 2;
        float left = here;
        for (int i = 0; i < g; ++i) {
          const float top_one = wave_max(left);
          const uint64_t who = __builtin_amdgcn_ballot_w64(left == top_one);
          if (who != 0 && lane == __builtin_ctzll(who)) left = -__builtin_inff();
          if (lane == 0) lane_best[wave * g + i] = top_one;
        }
        barrier();
        const uint32_t one = lane < kWaves * g ? ordered(lane_best[lane]) : 0u;
        const uint32_t two = lane + 64 < kWaves * g ? ordered(lane_best[lane + 64]) : 0u;
        uint32_t at_least = 0;
        for (int bit = 31; bit >= 12; --bit) {
          const uint32_t more = at_least | 1u << bit;
          const int reach = __builtin_popcountll(__builtin_amdgcn_ballot_w64(one >= more)) + __builtin_popcountll(__builtin_amdgcn_ballot_w64(two >= more));
          if (reach >= p.top) at_least = more;
        }
        if (at_least > ordered(-__builtin_inff())) bound = unordered(at_least);
      }
      int* const count = &added[r % 3];
      if (tid == 0) added[(r + 1) % 3] = 0;
      auto put = [&](float xe, int t, uint64_t least) __attribute__((always_inline)) {
        const uint64_t key = key_of(xe, t);
        if (t < v1 && key >= least) {
          const int place = kept + atomicAdd(count, 1);
          if (place < kKeys) keys[place] = key;
        }
      };
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        if (most[i] >= bound) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float xe = (float)v[i][e];
            if (xe >= bound) put(xe, piece_at(r, i) + e, bound_key);
          }
        }
      }
      barrier();
      const int found = kept + *count;
      if (found > kKeys) {
        // (the elements from memory once more: rarely needed, not to be held in registers for it)
        auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll 1
          for (int i = 0; i < PIECES; ++i)
#pragma unroll 1
            for (int e = 0; e < VEC; ++e) {
              const int t = piece_at(r, i) + e;
              if (t < v1) f((float)x[t], t);
            }
        };
        // the largest of those from the rounds before (at their places still), then of every thread its largest
        uint64_t mine = 0;
        each([&](float xe, int t) {
          const uint64_t key = key_of(xe, t);
          mine = key > mine ? key : mine;
        });
        barrier();
        if (tid == 0) *count = 0;
        largest<kThreads>(keys, kept, best, p.top);
        barrier();
        if (kept > p.top) kept = p.top;
        if (tid < kept) keys[tid] = best[tid];
        keys[kMostTop + tid] = mine;
        barrier();
        largest<kThreads>(keys + kMostTop, kThreads, best, p.top);
        barrier();
        const uint64_t least = best[p.top - 1] > bound_key ? best[p.top - 1] : bound_key;
        each([&](float xe, int t) {
          if (xe == xe) put(xe, t, least);
        });
        barrier();
        kept += *count;
      } else {
        kept = found;
      }
      if (kept > p.top && (found > kKeys || (kept >= 2 * p.top + 32 && r + 1 < rounds))) {
        // the best of them, and a bound for the rounds to come (paid for by as many that have come)
        largest<kThreads>(keys, kept, best, p.top);
        barrier();
        kept = p.top;
        bound_key = best[p.top - 1];
        bound = unordered((uint32_t)(bound_key >> 32));
        if (tid < kept) keys[tid] = best[tid];
      }
    }
  }
  // the token's own piece: equal ones in front of it
  const bool here_too = token >= v0 && token < v1;
  if (here_too && tid == 0) {
    const int from = v0 + (token - v0) / VEC * VEC;
    int equal = 0;
    for (int t = from; t < token; ++t) equal += (float)x[t] == given ? 1 : 0;
    ahead += equal;
  }
  // the workgroup's sums
  float to = wave_max(m);
  {
    const float d = step_down(m, to, c), f = exp2_fast(d);
    u = wave_sum(f * (u + s * d));
    s = wave_sum(s * f);
  }
  if (lane == 0) heads[wave] = {to, s, u, ahead};
  barrier();
  if constexpr (TOP) {
    largest<kThreads>(keys, kept, best, p.top);
    barrier();
  }
  if (wave != 0) return;
  PartHead all = heads[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    const PartHead h = heads[w];
    join(all.m, all.s, all.u, h.m, h.s, h.u, c);
    all.ahead += h.ahead;
  }
  if (p.splits == 1) {
    finish<T>(p, row, all.m, all.s, all.u, all.ahead, best);
  } else {
    unsigned char* const part = p.parts + (int64_t)item * p.part_bytes;
    if (lane == 0) *reinterpret_cast<PartHead*>(part) = all;
    if (TOP && lane < p.top) reinterpret_cast<uint64_t*>(part + sizeof(PartHead))[lane] = best[lane];
  }
}

constexpr int kJoinThreads = 512;
template <class T>
__global__ void __launch_bounds__(kJoinThreads) logprob_join_kernel(const LogprobParams p) {
  __shared__ uint64_t keys[kKeys], some[kKeys + 8], best[kMostTop];
  __shared__ int count;
  const int tid = threadIdx.x, row = p.first + blockIdx.x;
  const unsigned char* const part = p.parts + (int64_t)row * p.splits * p.part_bytes;
  const float c = p.scale * kLog2e;
  for (int i = tid; i < p.splits * p.top; i += kJoinThreads) {
    const int w = i / p.top;
    keys[i] = reinterpret_cast<const uint64_t*>(part + (int64_t)w * p.part_bytes + sizeof(PartHead))[i - w * p.top];
  }
  if (tid == 0) count = 0;
  PartHead all{-3.402823466e38f, 0.0f, 0.0f, 0};
  if (tid < 64) {
    if (tid < p.splits) all = *reinterpret_cast<const PartHead*>(part + (int64_t)tid * p.part_bytes);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const PartHead other{__shfl_xor(all.m, d), __shfl_xor(all.s, d), __shfl_xor(all.u, d), __shfl_xor(all.ahead, d)};
      join(all.m, all.s, all.u, other.m, other.s, other.u, c);
      all.ahead += other.ahead;
    }
  }
  __syncthreads();
  if (p.top > 0) {
    // every part's keys are in order: `top` of all of them reach the least of the parts' g-th ones
    const int n = p.splits * p.top, g = (p.top + p.splits - 1) / p.splits;
    uint64_t bound = keys[g - 1];
    for (int w = 1; w < p.splits; ++w) bound = keys[w * p.top + g - 1] < bound ? keys[w * p.top + g - 1] : bound;
    for (int i = tid; i < n; i += kJoinThreads)
      if (keys[i] >= bound) some[atomicAdd(&count, 1)] = keys[i];
    __syncthreads();
    largest<kJoinThreads>(some, count, best, p.top);
    __syncthreads();
  }
  if (tid < 64) finish<T>(p, row, all.m, all.s, all.u, all.ahead, best);
}

// Workgroups of a row: as many as fill the chip with two each, of a round at least; one where its rounds cost no more than the second
// launch (1 x 32000 fp32, four rounds: 11.3 us by one, 7.6 and 4.4 by four and the join; another round is one more)
int logprob_splits(int64_t rows, int64_t V, int cus) {
  const int64_t rounds = (V + kRound - 1) / kRound;
  int64_t s = rows > 0 && rounds > 4 ? 2ll * cus / rows : 1;
  if (s > rounds) s = rounds;
  if (s > kMostSplits) s = kMostSplits;
  return (int)(s < 1 ? 1 : s);
}
int64_t part_bytes(int64_t top) { return ((int64_t)sizeof(PartHead) + top * 8 + 15) / 16 * 16; }

template <class T>
hipError_t launch(LogprobParams p, hipStream_t stream) {
  auto kernel = p.top > 0 ? logprob_kernel<T, true> : logprob_kernel<T, false>;
  const int64_t items = (int64_t)p.rows * p.splits, most = most_workgroups(kThreads);
  for (int64_t at = 0; at < items; at += most) {
    p.first = (int32_t)at;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(items - at < most ? items - at : most)), dim3(kThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.splits > 1) {
    p.first = 0;
    hipLaunchKernelGGL(logprob_join_kernel<T>, dim3((unsigned)p.rows), dim3(kJoinThreads), 0, stream, p);
    return hipGetLastError();
  }
  return hipSuccess;
}

}  // namespace
}  // namespace aitamd

using namespace aitamd;

extern "C" int64_t aitamd_token_logprobs_workspace_bytes(int64_t rows, int64_t vocabulary, int64_t top) {
  if (rows <= 0 || vocabulary <= 0 || top < 0 || top > kMostTop) return 0;
  const int s = logprob_splits(rows, vocabulary, current_device_cus());
  return s > 1 ? rows * s * part_bytes(top) : 0;
}

extern "C" int aitamd_token_logprobs(int dtype, const void* logits, const void* tokens, int tokens_64, float* logprob, float* entropy,
                                     int32_t* rank, float* top_logprob, int32_t* top_token, int64_t rows, int64_t vocabulary, int64_t ld,
                                     int64_t top, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "aitamd_token_logprobs";
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16 && dtype != AITAMD_F32) return fail("%s: bad dtype %d", who, dtype);
  if (rows < 0 || vocabulary < 0) return fail("%s: negative dimension", who);
  if (top < 0 || top > kMostTop || top > vocabulary)
    return fail("%s: top %lld: up to %d, and not more than there are tokens (%lld)", who, (long long)top, kMostTop, (long long)vocabulary);
  // (its product with log2(e) is finite too)
  if (!(scale > 0.0f) || !__builtin_isfinite(scale * kLog2e)) return fail("%s: scale %g is no positive number of the range", who, (double)scale);
  if (rows > 0x7fffffffll / kMostSplits || vocabulary > 0x7fffffffll - 2 * kRound) return fail("%s: dimension too large", who);
  if (rows == 0) return 0;
  if (vocabulary == 0) return fail("%s: no tokens", who);
  if (ld < vocabulary && rows > 1) return fail("%s: row pitch smaller than the row", who);
  if (!logits || !tokens || !logprob || !entropy || !rank || (top > 0 && (!top_logprob || !top_token))) return fail("%s: null pointer", who);
  if ((reinterpret_cast<uintptr_t>(logits) & (dtype == AITAMD_F32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(tokens) & (tokens_64 ? 7 : 3)))
    return fail("%s: logits and tokens have to be aligned to their elements", who);
  LogprobParams p{};
  p.logits = logits, p.tokens = tokens, p.tokens_64 = tokens_64;
  p.logprob = logprob, p.entropy = entropy, p.rank = rank, p.top_logprob = top_logprob, p.top_token = top_token;
  p.rows = (int32_t)rows, p.V = (int32_t)vocabulary, p.ld = ld, p.top = (int32_t)top, p.scale = scale;
  p.splits = logprob_splits(rows, vocabulary, current_device_cus());
  p.part_bytes = (int32_t)part_bytes(top);
  if (p.splits > 1) {
    const int64_t need = rows * p.splits * part_bytes(top);
    if (!workspace || workspace_bytes < need)
      return fail("%s: a workspace of %lld bytes is wanted, got %lld", who, (long long)need, workspace ? (long long)workspace_bytes : 0ll);
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail("%s: the workspace must be 16-byte aligned", who);
    p.parts = static_cast<unsigned char*>(workspace);
  }
  // (whole pieces, so that only a row's last one may be cut)
  p.per_split = (int32_t)(((vocabulary + p.splits - 1) / p.splits + 7) / 8 * 8);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F32 ? launch<float>(p, s) : (dtype == AITAMD_F16 ? launch<f16>(p, s) : launch<bf16>(p, s));
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return 0;
}
