// C ABI launchers of aitamd_qk_norm_rotary and aitamd_paged_kv_append_norm.
//
// A head x of D numbers becomes x r w with r = 1 / sqrt(sum x^2 / D + eps), then its pairs turn by the token's position
// (rotary.hpp): all in 32 bits, rounded once.  A head's pieces lie on neighbouring lanes of a wave, one each (a power of two of
// lanes for a head, up to the wave; of longer heads several each), which sum their squares among themselves and go on with
// what they have in registers.  A workgroup goes through its tokens' queries, then their keys (and values), so that a lane's weights
// are read once for all heads.
// Bound: memory, 4 bytes an element, as the rotation alone.  16384 x 20 x 256 in fp16, 335 MB: 69 us with half of each head turned
// (neighbours; 72 halves), 4.9 TB/s, a copy's rate; with all of it turned, twice the sines, 82.  16384 x 40 x 128 in bf16 71.
#include "../../include/aitemplate_amd_kernels.h"
#include "device.hpp"
#include "errors.hpp"
#include "paged.hpp"
#include "rotary.hpp"

namespace aitamd {
namespace {

// What a lane handles of a head at once: two vectors of VEC elements, whichever of them are turned and with whichever partners, so that
// a lane's work is the same (with one vector where neighbours are paired or none are, 16384 x 20 x 256 in fp16, half of it turned: 85 us,
// halves paired 120).  Pairs of halves: i1 .. and its partners i2 ..; pairs of neighbours, and what is not turned: neighbouring vectors,
// of which a head's last may be without a second.  VEC = 1: a pair, or two elements.
template <class T, int VEC, bool INTERLEAVED>
struct NormPiece {
  using Tr = ElemTraits<T>;
  using vec = typename RotaryVec<T, VEC>::type;
  static constexpr bool kPartners = !INTERLEAVED || VEC == 1;  // the second vector's are the first one's partners
  int i1, i2;       // i2 < 0: none
  int pair, pair2;  // the first pair of each (kPartners: of both), -1 behind the rotated dims
  vec v1, v2;

  AITAMD_DEVICE void place(int c, int n, int dim) {
    if constexpr (kPartners) {
      const int turned = n / VEC;
      pair = pair2 = c < turned ? c * VEC : -1;
      i1 = c < turned ? (INTERLEAVED ? 2 * c : c * VEC) : 2 * n + (c - turned) * 2 * VEC;
      i2 = c < turned && !INTERLEAVED ? n + i1 : i1 + VEC;
    } else {
      i1 = c * 2 * VEC;
      i2 = i1 + VEC;
      pair = i1 < 2 * n ? i1 / 2 : -1;
      pair2 = i2 < 2 * n ? i2 / 2 : -1;
    }
    if (i2 >= dim) i2 = -1;
  }
  AITAMD_DEVICE void load(const T* x) {
    v1 = load_vec<vec>(x + i1);
    v2 = vec{};
    if (i2 >= 0) v2 = load_vec<vec>(x + i2);
  }
  // the sum of squares, in 32 or 64 bits
  template <class S>
  AITAMD_DEVICE S squares() const {
    S s = 0;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const S a = (S)Tr::to_float(v1[j]), b = (S)Tr::to_float(v2[j]);
      s += a * a;
      s += b * b;
    }
    return s;
  }
  // as it is
  AITAMD_DEVICE void copy(T* y) const {
    store_vec(y + i1, v1);
    if (i2 >= 0) store_vec(y + i2, v2);
  }
  // the weights of the same elements
  AITAMD_DEVICE void weigh(const T* weight, vec& w1, vec& w2) const {
    w1 = w2 = load_vec<vec>(weight + i1);
    if (i2 >= 0) w2 = load_vec<vec>(weight + i2);
  }
  // times ra, times rb and the weights (NORM), turned
  template <bool NORM>
  AITAMD_DEVICE void store(T* y, vec w1, vec w2, float ra, float rb, const float2* table) const {
    auto times = [&](vec v, vec w, float (&f)[VEC]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        f[j] = Tr::to_float(v[j]);
        if constexpr (NORM) f[j] = f[j] * ra * (rb * Tr::to_float(w[j]));
      }
    };
    if constexpr (kPartners) {
      float a[VEC], b[VEC];
      vec o1, o2;
      times(v1, w1, a);
      times(v2, w2, b);
      if (pair >= 0) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float2 t = table[pair + j];
          const float turned = a[j] * t.x - b[j] * t.y;
          b[j] = b[j] * t.x + a[j] * t.y;
          a[j] = turned;
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        o1[j] = Tr::from_float(a[j]);
        o2[j] = Tr::from_float(b[j]);
      }
      store_vec(y + i1, o1);
      if (i2 >= 0) store_vec(y + i2, o2);
    } else {
      auto put = [&](vec v, vec w, int at, int of) __attribute__((always_inline)) {
        float a[VEC];
        vec o;
        times(v, w, a);
        if (of >= 0) {
#pragma unroll
          for (int j = 0; j < VEC; j += 2) {
            const float2 t = table[of + j / 2];
            const float turned = a[j] * t.x - a[j + 1] * t.y;
            a[j + 1] = a[j + 1] * t.x + a[j] * t.y;
            a[j] = turned;
          }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = Tr::from_float(a[j]);
        store_vec(y + at, o);
      };
      put(v1, w1, i1, pair);
      if (i2 >= 0) put(v2, w2, i2, pair2);
    }
  }
};
// the pieces of a head
constexpr int norm_pieces(int n, int head_dim, bool interleaved, int vec) {
  return interleaved && vec > 1 ? (head_dim + 2 * vec - 1) / (2 * vec) : n / vec + (head_dim - 2 * n + 2 * vec - 1) / (2 * vec);
}

// The sum over 1 << shift neighbouring lanes, in all of them: quads and rows of 16 by moves along the row (mirrored once their halves
// are even), then rows and halves of the wave exchanged.  (Through LDS, a trip for each step: 16384 x 20 x 256 100 us.)
template <int CTRL>
AITAMD_DEVICE float lane_move(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
AITAMD_DEVICE float lanes_sum(float v, int shift) {
  if (shift > 0) v += lane_move<0xb1>(v);   // quad_perm 1 0 3 2
  if (shift > 1) v += lane_move<0x4e>(v);   // quad_perm 2 3 0 1
  if (shift > 2) v += lane_move<0x141>(v);  // row_half_mirror
  if (shift > 3) v += lane_move<0x140>(v);  // row_mirror
  if (shift > 4) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (shift > 5) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}
AITAMD_DEVICE double lanes_sum(double v, int shift) {
  for (int d = 1; d < 1 << shift; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// 1 / sqrt(sum / dim + eps) as ra * rb.  Where the sum leaves the range of 32 bits (numbers above 2^57 or so; below 2^-50 without an
// eps), `again` gives it in 64.
template <class F>
AITAMD_DEVICE void inverse_length(float sum, float by_dim, float eps, float& ra, float& rb, F&& again) {
  const float mean = __builtin_fmaf(sum, by_dim, eps);
  const bool fits = mean > 1e-30f && mean < 1e30f;
  ra = rsqrtf(mean);
  rb = 1.0f;
  if (__builtin_amdgcn_ballot_w64(!fits) != 0) {
    const double exact = again() * (double)by_dim + (double)eps;
    if (!fits) {
      // (a NaN is neither; an infinity makes zeros, and NaN of itself)
      const double r = exact == 0.0 ? 0.0 : 1.0 / sqrt(exact);
      const double half = sqrt(r);
      ra = (float)half;
      rb = (float)half;
    }
  }
}

enum HeadKind : int { kNorm = 0, kTurnOnly = 1, kCopy = 2 };
template <class T>
struct Head {
  const T* x;  // null: nothing to do
  T* y;
  const float2* table;
};

struct Lanes {
  int32_t per_head, shift, pieces, n, dim;  // lanes of a head (1 << shift), its pieces, its pairs, its elements
  float by_dim, eps;
};

// Heads 0 .. count - 1 of one kind, AHEAD of a lane's on their way together.  head(i, h) is the same for all lanes of a head;
// weight(i): its weights (the same for all with weight_head = 0).
template <class T, int VEC, bool INTERLEAVED, int KIND, int AHEAD, class F, class W>
AITAMD_DEVICE void heads_of_workgroup(const Lanes& l, int count, bool one_weight, F&& head, W&& weight) {
  using Piece = NormPiece<T, VEC, INTERLEAVED>;
  const int lane = threadIdx.x & (l.per_head - 1), mine = threadIdx.x >> l.shift, at_once = kRotaryThreads >> l.shift;
  const bool one_each = l.pieces <= l.per_head;
  typename Piece::vec w1 = {}, w2 = {};
  if (KIND == kNorm && one_weight && count > 0 && lane < l.pieces) {
    Piece at;
    at.place(lane, l.n, l.dim);
    at.weigh(weight(0), w1, w2);
  }
  // (whole waves stay together: their lanes exchange sums)
  for (int first = 0; first < count; first += AHEAD * at_once) {
    Head<T> h[AHEAD];
    Piece piece[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const int i = first + mine + a * at_once;
      h[a].x = nullptr;
      if (i < count && lane < l.pieces) head(i, h[a]);
      piece[a].place(lane, l.n, l.dim);
      if (h[a].x != nullptr) piece[a].load(h[a].x);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      const bool on = h[a].x != nullptr;
      float ra = 1.0f, rb = 1.0f;
      if constexpr (KIND == kNorm) {
        float sum = on ? piece[a].template squares<float>() : 0.0f;
        if (!one_each && on) {
          for (int c = lane + l.per_head; c < l.pieces; c += l.per_head) {
            Piece more;
            more.place(c, l.n, l.dim);
            more.load(h[a].x);
            sum += more.template squares<float>();
          }
        }
        sum = lanes_sum(sum, l.shift);
        // (of lanes without a head: of a sum that fits)
        inverse_length(on ? sum : 1.0f / l.by_dim, l.by_dim, l.eps, ra, rb, [&]() {
          double s = 0.0;
          for (int c = lane; on && c < l.pieces; c += l.per_head) {
            Piece again;
            again.place(c, l.n, l.dim);
            again.load(h[a].x);
            s += again.template squares<double>();
          }
          return lanes_sum(s, l.shift);
        });
      }
      if (!on) continue;
      const T* w = KIND == kNorm && !(one_weight && one_each) ? weight(first + mine + a * at_once) : nullptr;
      auto put = [&](const Piece& q) __attribute__((always_inline)) {
        if constexpr (KIND == kCopy) {
          q.copy(h[a].y);
        } else {
          if (w != nullptr) q.weigh(w, w1, w2);
          q.template store<KIND == kNorm>(h[a].y, w1, w2, ra, rb, h[a].table);
        }
      };
      put(piece[a]);
      if (!one_each) {
        for (int c = lane + l.per_head; c < l.pieces; c += l.per_head) {
          Piece more;
          more.place(c, l.n, l.dim);
          more.load(h[a].x);
          put(more);
        }
      }
    }
  }
}

struct HeadsParams {
  const void* x;
  void* out;
  const void* weight;
  int64_t x_batch, x_seq, x_head, out_batch, out_seq, out_head, weight_head;
};
struct NormParams {
  HeadsParams q, k;
  const void* positions;
  const float* freqs;
  int64_t pos_batch, pos_seq;
  int32_t tokens, heads, kv_heads, seq, first, per_wg, positions_64;
  float scale;
  Lanes lanes;
  Divisor by_n, by_seq, by_heads, by_kv_heads;
};

constexpr int kNormAhead = 2;
// Waves of a SIMD that the registers are shared out to, hardly any of them spilled (the widest pieces with four instead of five: a step
// of eight prompts into the cache 54.8 us for 50.0)
constexpr int norm_waves(int vec) { return vec < 8 ? 6 : 5; }

template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, norm_waves(VEC)) norm_rotary_kernel(const NormParams p) {
  __shared__ float2 table[kRotaryTable];
  const int t0 = p.first + blockIdx.x * p.per_wg;
  const int tokens = p.tokens - t0 < p.per_wg ? p.tokens - t0 : p.per_wg;
  fill_rotary_table(table, p.freqs, p.lanes.n, p.by_n, tokens, p.scale, 1.0f, [&](int t) -> int64_t {
    const int b = quotient(t0 + t, p.by_seq);
    const int64_t at = b * p.pos_batch + (t0 + t - b * p.seq) * p.pos_seq;
    return p.positions_64 ? reinterpret_cast<const int64_t*>(p.positions)[at] : reinterpret_cast<const int32_t*>(p.positions)[at];
  });
  __syncthreads();
  auto all = [&](const HeadsParams& h, int heads, Divisor by) __attribute__((always_inline)) {
    if (heads == 0) return;
    auto head = [&](int i, Head<T>& r) __attribute__((always_inline)) {
      const int t = quotient(i, by), head = i - t * heads;
      const int b = quotient(t0 + t, p.by_seq), s = t0 + t - b * p.seq;
      r.x = reinterpret_cast<const T*>(h.x) + b * h.x_batch + s * h.x_seq + head * h.x_head;
      r.y = reinterpret_cast<T*>(h.out) + b * h.out_batch + s * h.out_seq + head * h.out_head;
      r.table = table + t * p.lanes.n;
    };
    auto weight = [&](int i) { return reinterpret_cast<const T*>(h.weight) + (i - quotient(i, by) * heads) * h.weight_head; };
    if (h.weight != nullptr)
      heads_of_workgroup<T, VEC, INTERLEAVED, kNorm, kNormAhead>(p.lanes, tokens * heads, h.weight_head == 0, head, weight);
    else
      heads_of_workgroup<T, VEC, INTERLEAVED, kTurnOnly, kNormAhead>(p.lanes, tokens * heads, true, head, weight);
  };
  // (the arguments of the one operand and then of the other: of both at once there are more than scalar registers)
  all(p.q, p.heads, p.by_heads);
  const NormParams& q = arguments_anew<NormParams>();
  all(q.k, q.kv_heads, q.by_kv_heads);
}

struct AppendNormParams {
  PagedCache cache;
  const void *q, *k, *v, *q_weight, *k_weight;
  void* q_out;
  const float* freqs;
  int64_t q_token, q_head, q_out_token, q_out_head, k_token, k_head, v_token, v_head, q_weight_head, k_weight_head, first_position;
  int32_t heads, first, per_wg;
  float scale;
  Lanes lanes;
  Divisor by_n, by_heads, by_kv_heads;
};

constexpr int kAppendNormAhead = 2;

// One launch for a layer's new tokens, as append_kernel (rotary_api.hip)
template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, norm_waves(VEC)) append_norm_kernel(const AppendNormParams p) {
  __shared__ float2 table[kRotaryTable];
  __shared__ int64_t slot[kRotaryMaxTokens];  // among the sequence's own tokens
  __shared__ int32_t page[kRotaryMaxTokens];  // -1: nowhere to go
  __shared__ int32_t in_page[kRotaryMaxTokens];
  __shared__ bool live[kRotaryMaxTokens];
  const PagedCache& c = p.cache;
  const int t0 = p.first + blockIdx.x * p.per_wg;
  const int tokens = c.tokens - t0 < p.per_wg ? c.tokens - t0 : p.per_wg;
  const int s0 = c.offsets != nullptr ? sequence_of_row(c, t0) : t0;  // (every wave for itself)
  if ((int)threadIdx.x < tokens) {
    const int t = threadIdx.x, row = t0 + t;
    int s = c.offsets != nullptr ? s0 : row;
    int first = row;
    if (c.offsets != nullptr) {
      while (s < c.batch && c.offsets[s + 1] <= row) ++s;
      first = s < c.batch ? c.offsets[s] : 0;
    }
    const bool in = s < c.batch && row >= first;
    live[t] = in;
    const int64_t at = in ? (int64_t)c.lengths[s] + (row - first) : -1;
    slot[t] = at;
    int pg = -1, within = 0;
    if (at >= 0 && at < c.most_keys) {
      const int which = quotient((int)at, c.by_page);
      within = (int)at - which * c.page_size;
      pg = c.table[s * c.table_pitch + which];
      if (pg >= c.pages) pg = -1;
    }
    page[t] = pg;
    in_page[t] = within;
  }
  __syncthreads();
  if (p.lanes.n > 0) {
    fill_rotary_table(table, p.freqs, p.lanes.n, p.by_n, tokens, p.scale, 1.0f, [&](int t) { return p.first_position + slot[t]; });
    __syncthreads();
  }
  auto all = [&](const T* weights, int64_t weight_head, int heads, Divisor by, auto&& head) __attribute__((always_inline)) {
    if (heads == 0) return;
    auto weight = [&](int i) { return weights + (i - quotient(i, by) * heads) * weight_head; };
    if (weights != nullptr)
      heads_of_workgroup<T, VEC, INTERLEAVED, kNorm, kAppendNormAhead>(p.lanes, tokens * heads, weight_head == 0, head, weight);
    else
      heads_of_workgroup<T, VEC, INTERLEAVED, kTurnOnly, kAppendNormAhead>(p.lanes, tokens * heads, true, head, weight);
  };
  all(reinterpret_cast<const T*>(p.q_weight), p.q_weight_head, p.heads, p.by_heads, [&](int i, Head<T>& r) __attribute__((always_inline)) {
    const int t = quotient(i, p.by_heads), head = i - t * p.heads;
    if (!live[t]) return;
    r.x = reinterpret_cast<const T*>(p.q) + (int64_t)(t0 + t) * p.q_token + head * p.q_head;
    r.y = reinterpret_cast<T*>(p.q_out) + (int64_t)(t0 + t) * p.q_out_token + head * p.q_out_head;
    r.table = table + t * p.lanes.n;
  });
  // (the arguments of the one operand and then of the other: of both at once there are more than scalar registers)
  const AppendNormParams& p2 = arguments_anew<AppendNormParams>();
  all(reinterpret_cast<const T*>(p2.k_weight), p2.k_weight_head, p2.cache.kv_heads, p2.by_kv_heads, [&](int i, Head<T>& r) __attribute__((always_inline)) {
    const int t = quotient(i, p2.by_kv_heads), head = i - t * p2.cache.kv_heads;
    if (!live[t] || page[t] < 0) return;
    r.x = reinterpret_cast<const T*>(p2.k) + (int64_t)(t0 + t) * p2.k_token + head * p2.k_head;
    r.y = reinterpret_cast<T*>(p2.cache.k) + page[t] * p2.cache.k_page + in_page[t] * p2.cache.k_slot + head * p2.cache.k_head;
    r.table = table + t * p2.lanes.n;
  });
  const AppendNormParams& p3 = arguments_anew<AppendNormParams>();
  auto value = [&](int i, Head<T>& r) __attribute__((always_inline)) {
    const int t = quotient(i, p3.by_kv_heads), head = i - t * p3.cache.kv_heads;
    if (!live[t] || page[t] < 0) return;
    r.x = reinterpret_cast<const T*>(p3.v) + (int64_t)(t0 + t) * p3.v_token + head * p3.v_head;
    r.y = reinterpret_cast<T*>(p3.cache.v) + page[t] * p3.cache.v_page + in_page[t] * p3.cache.v_slot + head * p3.cache.v_head;
    r.table = table;
  };
  heads_of_workgroup<T, VEC, INTERLEAVED, kCopy, kAppendNormAhead>(p3.lanes, tokens * p3.cache.kv_heads, true, value, [](int) -> const T* { return nullptr; });
}

template <class P>
hipError_t launch_wgs(void (*kernel)(P), P p, int64_t tokens, hipStream_t stream) {
  const int64_t wgs = (tokens + p.per_wg - 1) / p.per_wg, most = most_workgroups(kRotaryThreads);
  for (int64_t wg = 0; wg < wgs; wg += most) {
    p.first = (int32_t)(wg * p.per_wg);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(wgs - wg < most ? wgs - wg : most)), dim3(kRotaryThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
#define AITAMD_BY_VEC(KERNEL)                                                         \
  (interleaved ? (vec == 8     ? KERNEL<T, 8, true>                                   \
                      : vec == 4 ? KERNEL<T, 4, true>                                 \
                      : vec == 2 ? KERNEL<T, 2, true>                                 \
                                 : KERNEL<T, 1, true>)                                \
               : (vec == 8     ? KERNEL<T, 8, false>                                  \
                      : vec == 4 ? KERNEL<T, 4, false>                                \
                      : vec == 2 ? KERNEL<T, 2, false>                                \
                                 : KERNEL<T, 1, false>))
template <class T>
hipError_t launch_norm(const NormParams& p, int vec, bool interleaved, hipStream_t stream) {
  return launch_wgs(AITAMD_BY_VEC(norm_rotary_kernel), p, p.tokens, stream);
}
template <class T>
hipError_t launch_append(const AppendNormParams& p, int vec, bool interleaved, hipStream_t stream) {
  return launch_wgs(AITAMD_BY_VEC(append_norm_kernel), p, p.cache.tokens, stream);
}
#undef AITAMD_BY_VEC

int check_norm(const char* who, int64_t head_dim, int64_t rotated, const float* freqs, float eps) {
  if (head_dim > kRotaryMaxDim) return fail("%s: head_dim %lld is beyond %lld", who, (long long)head_dim, (long long)kRotaryMaxDim);
  if (rotated < 0 || rotated % 2 != 0 || rotated > head_dim)
    return fail("%s: %lld rotated dims: an even number up to head_dim %lld is wanted", who, (long long)rotated, (long long)head_dim);
  if (rotated > 0 && !freqs) return fail("%s: null pointer (freqs)", who);
  if (!(eps >= 0.0f) || !__builtin_isfinite(eps)) return fail("%s: eps %g is no number of at least 0", who, (double)eps);
  return 0;
}
// Lanes of a head: as many as it has pieces, rounded up to a power of two, up to a wave
Lanes head_lanes(int64_t n, int64_t head_dim, bool interleaved, int vec, float eps) {
  Lanes l{};
  l.n = (int32_t)n;
  l.dim = (int32_t)head_dim;
  l.pieces = norm_pieces((int)n, (int)head_dim, interleaved, vec);
  while ((1 << l.shift) < l.pieces && l.shift < 6) ++l.shift;
  l.per_head = 1 << l.shift;
  l.by_dim = 1.0f / (float)head_dim;
  l.eps = eps;
  return l;
}

}  // namespace
}  // namespace aitamd

using namespace aitamd;

extern "C" int aitamd_qk_norm_rotary(int dtype, const aitamd_heads* q, const aitamd_heads* k, const void* positions, int positions_64,
                                     const float* freqs, int64_t batch, int64_t seq, int64_t head_dim, int64_t rotated, int64_t pos_batch,
                                     int64_t pos_seq, float eps, float scale, int interleaved, void* stream) {
  const char* who = "aitamd_qk_norm_rotary";
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  if (batch < 0 || seq < 0 || head_dim < 0 || (q && q->heads < 0) || (k && k->heads < 0)) return fail("%s: negative dimension", who);
  if (check_norm(who, head_dim, rotated, freqs, eps)) return 1;
  const int64_t heads = q ? q->heads : 0, kv_heads = k ? k->heads : 0;
  if (batch == 0 || seq == 0 || heads + kv_heads == 0 || head_dim == 0) return 0;
  if ((heads > 0 && (!q->x || !q->out)) || (kv_heads > 0 && (!k->x || !k->out)) || (rotated > 0 && !positions)) return fail("%s: null pointer", who);
  const int64_t n = rotated / 2;
  const int vec = rotary_vec(n, head_dim, interleaved != 0);
  NormParams p{};
  p.lanes = head_lanes(n, head_dim, interleaved != 0, vec, eps);
  if (batch > 0x7fffffffll / seq || heads > 0x7fffffffll || kv_heads > 0x7fffffffll ||
      heads + kv_heads > 0x3fffffffll / kRotaryMaxTokens / p.lanes.per_head)
    return fail("%s: dimension too large", who);
  auto fill = [](const aitamd_heads* a) {
    HeadsParams h{};
    if (a) h = {a->x, a->out, a->weight, a->batch_stride, a->seq_stride, a->head_stride, a->out_batch_stride, a->out_seq_stride, a->out_head_stride,
                a->weight_head_stride};
    return h;
  };
  p.q = fill(q), p.k = fill(k);
  p.positions = positions, p.positions_64 = positions_64;
  p.freqs = freqs;
  p.pos_batch = pos_batch, p.pos_seq = pos_seq;
  p.tokens = (int32_t)(batch * seq), p.heads = (int32_t)heads, p.kv_heads = (int32_t)kv_heads, p.seq = (int32_t)seq;
  p.per_wg = rotary_tokens(batch * seq, (heads + kv_heads) * p.lanes.per_head, n, current_device_cus());
  p.scale = scale;
  p.by_n = make_divisor(n > 0 ? n : 1);
  p.by_seq = make_divisor(seq);
  p.by_heads = make_divisor(heads > 0 ? heads : 1);
  p.by_kv_heads = make_divisor(kv_heads > 0 ? kv_heads : 1);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F16 ? launch_norm<f16>(p, vec, interleaved != 0, s) : launch_norm<bf16>(p, vec, interleaved != 0, s);
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return 0;
}

extern "C" int aitamd_paged_kv_append_norm(int dtype, const aitamd_paged_cache* cache, const void* k, int64_t k_token, int64_t k_head,
                                           const void* v, int64_t v_token, int64_t v_head, const void* q, int64_t q_token, int64_t q_head,
                                           void* q_out, int64_t q_out_token, int64_t q_out_head, int64_t heads, const void* q_weight,
                                           int64_t q_weight_head, const void* k_weight, int64_t k_weight_head, float eps, const float* freqs,
                                           int64_t rotated, int64_t first_position, float scale, int interleaved, void* stream) {
  if (!q_weight && !k_weight)
    return aitamd_paged_kv_append(dtype, cache, k, k_token, k_head, v, v_token, v_head, q, q_token, q_head, q_out, q_out_token, q_out_head, heads,
                                  freqs, rotated, first_position, scale, interleaved, stream);
  const char* who = "aitamd_paged_kv_append_norm";
  AppendNormParams p{};
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  if (paged_cache(who, cache, 1, &p.cache)) return 1;
  const int64_t head_dim = cache->head_dim, kv_heads = cache->kv_heads, tokens = cache->tokens;
  if (check_norm(who, head_dim, rotated, freqs, eps)) return 1;
  if (heads < 0) return fail("%s: negative dimension", who);
  if (!q) heads = 0;
  if (tokens == 0 || (kv_heads == 0 && heads == 0) || cache->batch == 0 || head_dim == 0) return 0;
  if (kv_heads > 0 && (!k || !v || !cache->k || !cache->v)) return fail("%s: null pointer", who);
  if (heads > 0 && !q_out) return fail("%s: null pointer (q_out)", who);
  const int64_t n = rotated / 2;
  const int vec = rotary_vec(n, head_dim, interleaved != 0);
  p.lanes = head_lanes(n, head_dim, interleaved != 0, vec, eps);
  if (heads > 0x7fffff || kv_heads > 0x7fffff || heads + 2 * kv_heads > 0x3fffffffll / kRotaryMaxTokens / p.lanes.per_head)
    return fail("%s: dimension too large", who);
  p.q = q, p.k = k, p.v = v;
  p.q_weight = q_weight, p.k_weight = k_weight;
  p.q_weight_head = q_weight_head, p.k_weight_head = k_weight_head;
  p.q_out = q_out;
  p.freqs = freqs;
  p.heads = (int32_t)heads;
  p.per_wg = rotary_tokens(tokens, (heads + 2 * kv_heads) * p.lanes.per_head, n, current_device_cus());
  p.q_token = q_token, p.q_head = q_head, p.q_out_token = q_out_token, p.q_out_head = q_out_head;
  p.k_token = k_token, p.k_head = k_head, p.v_token = v_token, p.v_head = v_head;
  p.first_position = first_position;
  p.scale = scale;
  p.by_n = make_divisor(n > 0 ? n : 1);
  p.by_heads = make_divisor(heads > 0 ? heads : 1);
  p.by_kv_heads = make_divisor(kv_heads > 0 ? kv_heads : 1);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F16 ? launch_append<f16>(p, vec, interleaved != 0, s) : launch_append<bf16>(p, vec, interleaved != 0, s);
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return 0;
}
