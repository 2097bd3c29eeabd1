// C ABI launchers of aitamd_rotary_embedding and aitamd_paged_kv_append.
#include "../../include/aitemplate_amd_kernels.h"
#include "device.hpp"
#include "errors.hpp"
#include "paged.hpp"
#include "rotary.hpp"

namespace aitamd {
namespace {

struct RotaryParams {
  const void* x;
  void* out;
  const void* positions;
  const float* freqs;
  int32_t tokens, heads, n, seq;
  int32_t first, per_wg, pieces, positions_64;  // first: the launch's first token
  int64_t x_batch, x_seq, x_head, out_batch, out_seq, out_head, pos_batch, pos_seq;
  float scale, sine_sign;
  Divisor by_n, by_seq, by_pieces, by_heads;
};

// Bound: memory, 4 bytes an element; a workgroup takes a few whole tokens, so that their sines are taken once.
template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryParams p) {
  __shared__ float2 table[kRotaryTable];
  const int t0 = p.first + blockIdx.x * p.per_wg;
  const int tokens = p.tokens - t0 < p.per_wg ? p.tokens - t0 : p.per_wg;
  fill_rotary_table(table, p.freqs, p.n, p.by_n, tokens, p.scale, p.sine_sign, [&](int t) -> int64_t {
    const int b = quotient(t0 + t, p.by_seq);
    const int64_t at = b * p.pos_batch + (t0 + t - b * p.seq) * p.pos_seq;
    return p.positions_64 ? reinterpret_cast<const int64_t*>(p.positions)[at] : reinterpret_cast<const int32_t*>(p.positions)[at];
  });
  __syncthreads();
  const int items = tokens * p.heads * p.pieces;
  for (int i0 = threadIdx.x; i0 < items; i0 += kRotaryAhead * kRotaryThreads) {
    RotaryPiece<T, VEC, INTERLEAVED> piece[kRotaryAhead];
#pragma unroll
    for (int a = 0; a < kRotaryAhead; ++a) {
      const int i = i0 + a * kRotaryThreads;
      if (i >= items) continue;
      const int th = quotient(i, p.by_pieces), c = i - th * p.pieces;
      const int t = quotient(th, p.by_heads), head = th - t * p.heads;
      const int b = quotient(t0 + t, p.by_seq), s = t0 + t - b * p.seq;
      piece[a].load(reinterpret_cast<const T*>(p.x) + b * p.x_batch + s * p.x_seq + head * p.x_head,
                    reinterpret_cast<T*>(p.out) + b * p.out_batch + s * p.out_seq + head * p.out_head, c, p.n, table + t * p.n);
    }
#pragma unroll
    for (int a = 0; a < kRotaryAhead; ++a)
      if (i0 + a * kRotaryThreads < items) piece[a].store();
  }
}

// p.per_wg tokens a workgroup, in as many launches as it takes
template <class P>
hipError_t launch_tokens(void (*kernel)(P), P p, int64_t tokens, hipStream_t stream) {
  const int64_t wgs = (tokens + p.per_wg - 1) / p.per_wg, most = most_workgroups(kRotaryThreads);
  for (int64_t wg = 0; wg < wgs; wg += most) {
    p.first = (int32_t)(wg * p.per_wg);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(wgs - wg < most ? wgs - wg : most)), dim3(kRotaryThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <class T, int VEC>
hipError_t launch_rotary(const RotaryParams& p, bool interleaved, hipStream_t stream) {
  return launch_tokens(interleaved ? rotary_kernel<T, VEC, true> : rotary_kernel<T, VEC, false>, p, p.tokens, stream);
}
template <class T>
hipError_t launch_rotary(const RotaryParams& p, int vec, bool interleaved, hipStream_t stream) {
  return vec == 8 ? launch_rotary<T, 8>(p, interleaved, stream)
      : vec == 4  ? launch_rotary<T, 4>(p, interleaved, stream)
      : vec == 2  ? launch_rotary<T, 2>(p, interleaved, stream)
                  : launch_rotary<T, 1>(p, interleaved, stream);
}

// (two: 50.0 us for eight prompts of 517 to 2048 tokens, 32 + 2 x 8 heads of 128 dims; one: 48.8.  The loops over them stay: of the
// same work written for one alone, three ways, the compiler makes code that takes 0.8 % longer)
constexpr int kAppendAhead = 1;

struct AppendParams {
  PagedCache cache;
  const void *q, *k, *v;
  void* q_out;
  const float* freqs;
  int32_t heads, n, first, per_wg, pieces, pieces_v, per_token;
  int64_t q_token, q_head, q_out_token, q_out_head, k_token, k_head, v_token, v_head, first_position;
  float scale;
  Divisor by_n, by_token, by_pieces, by_pieces_v;
};

// One launch for a layer's new tokens: queries rotated, keys rotated into their pages, values into theirs.
// Bound: memory, as the rotation alone.
template <class T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads) append_kernel(const AppendParams p) {
  __shared__ float2 table[kRotaryTable];
  __shared__ int64_t slot[kRotaryMaxTokens];     // among the sequence's own tokens
  __shared__ int32_t page[kRotaryMaxTokens];     // -1: nowhere to go
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
  if (p.n > 0) {
    fill_rotary_table(table, p.freqs, p.n, p.by_n, tokens, p.scale, 1.0f, [&](int t) { return p.first_position + slot[t]; });
    __syncthreads();
  }
  const int q_items = p.heads * p.pieces, k_items = q_items + c.kv_heads * p.pieces, items = tokens * p.per_token;
  for (int i0 = threadIdx.x; i0 < items; i0 += kAppendAhead * kRotaryThreads) {
    RotaryPiece<T, VEC, INTERLEAVED> piece[kAppendAhead];
    bool on[kAppendAhead];
#pragma unroll
    for (int a = 0; a < kAppendAhead; ++a) {
      const int i = i0 + a * kRotaryThreads;
      const int t = i < items ? quotient(i, p.by_token) : 0, item = i - t * p.per_token;
      on[a] = i < items && live[t] && (item < q_items || page[t] >= 0);
      if (!on[a]) continue;
      const int64_t row = t0 + t;
      // where the item's head lies and goes to, and which of its pieces it is
      const bool is_v = item >= k_items;
      const int of = item < q_items ? item : (is_v ? item - k_items : item - q_items);
      const int head = quotient(of, is_v ? p.by_pieces_v : p.by_pieces), at = of - head * (is_v ? p.pieces_v : p.pieces);
      const T* x;
      T* y;
      if (item < q_items) {
        x = reinterpret_cast<const T*>(p.q) + row * p.q_token + head * p.q_head;
        y = reinterpret_cast<T*>(p.q_out) + row * p.q_out_token + head * p.q_out_head;
      } else if (!is_v) {
        x = reinterpret_cast<const T*>(p.k) + row * p.k_token + head * p.k_head;
        y = reinterpret_cast<T*>(c.k) + page[t] * c.k_page + in_page[t] * c.k_slot + head * c.k_head;
      } else {
        x = reinterpret_cast<const T*>(p.v) + row * p.v_token + head * p.v_head;
        y = reinterpret_cast<T*>(c.v) + page[t] * c.v_page + in_page[t] * c.v_slot + head * c.v_head;
      }
      piece[a].load(x, y, at, is_v ? 0 : p.n, table + t * p.n);
    }
#pragma unroll
    for (int a = 0; a < kAppendAhead; ++a)
      if (on[a]) piece[a].store();
  }
}

template <class T, int VEC>
hipError_t launch_append(const AppendParams& p, bool interleaved, hipStream_t stream) {
  return launch_tokens(interleaved ? append_kernel<T, VEC, true> : append_kernel<T, VEC, false>, p, p.cache.tokens, stream);
}
template <class T>
hipError_t launch_append(const AppendParams& p, int vec, bool interleaved, hipStream_t stream) {
  return vec == 8 ? launch_append<T, 8>(p, interleaved, stream)
      : vec == 4  ? launch_append<T, 4>(p, interleaved, stream)
      : vec == 2  ? launch_append<T, 2>(p, interleaved, stream)
                  : launch_append<T, 1>(p, interleaved, stream);
}

int check_rotation(const char* who, int64_t head_dim, int64_t rotated, const float* freqs) {
  if (head_dim > kRotaryMaxDim) return fail("%s: head_dim %lld is beyond %lld", who, (long long)head_dim, (long long)kRotaryMaxDim);
  if (rotated < 0 || rotated % 2 != 0 || rotated > head_dim)
    return fail("%s: %lld rotated dims: an even number up to head_dim %lld is wanted", who, (long long)rotated, (long long)head_dim);
  if (rotated > 0 && !freqs) return fail("%s: null pointer (freqs)", who);
  return 0;
}

}  // namespace
}  // namespace aitamd

using namespace aitamd;

extern "C" int aitamd_rotary_embedding(int dtype, const void* x, void* out, const void* positions, int positions_64, const float* freqs,
                                       int64_t batch, int64_t seq, int64_t heads, int64_t head_dim, int64_t rotated, int64_t x_batch,
                                       int64_t x_seq, int64_t x_head, int64_t out_batch, int64_t out_seq, int64_t out_head,
                                       int64_t pos_batch, int64_t pos_seq, float scale, int interleaved, int inverse, void* stream) {
  const char* who = "aitamd_rotary_embedding";
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  if (batch < 0 || seq < 0 || heads < 0 || head_dim < 0) return fail("%s: negative dimension", who);
  if (check_rotation(who, head_dim, rotated, freqs)) return 1;
  if (batch == 0 || seq == 0 || heads == 0 || head_dim == 0) return 0;
  if (!x || !out || (rotated > 0 && !positions)) return fail("%s: null pointer", who);
  const int64_t n = rotated / 2;
  const int vec = rotary_vec(n, head_dim, interleaved != 0);
  const int64_t pieces = rotary_pieces((int)n, (int)head_dim, interleaved != 0, vec);
  if (batch > 0x7fffffffll / seq || heads > 0x7fffffffll / kRotaryMaxTokens / pieces) return fail("%s: dimension too large", who);
  RotaryParams p{};
  p.x = x;
  p.out = out;
  p.positions = positions;
  p.freqs = freqs;
  p.tokens = (int32_t)(batch * seq);
  p.heads = (int32_t)heads;
  p.n = (int32_t)n;
  p.seq = (int32_t)seq;
  p.per_wg = rotary_tokens(batch * seq, heads * pieces, n, current_device_cus());
  p.pieces = (int32_t)pieces;
  p.positions_64 = positions_64;
  p.x_batch = x_batch, p.x_seq = x_seq, p.x_head = x_head;
  p.out_batch = out_batch, p.out_seq = out_seq, p.out_head = out_head;
  p.pos_batch = pos_batch, p.pos_seq = pos_seq;
  p.scale = scale;
  p.sine_sign = inverse ? -1.0f : 1.0f;
  p.by_n = make_divisor(n > 0 ? n : 1);
  p.by_seq = make_divisor(seq);
  p.by_pieces = make_divisor(pieces);
  p.by_heads = make_divisor(heads);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F16 ? launch_rotary<f16>(p, vec, interleaved != 0, s) : launch_rotary<bf16>(p, vec, interleaved != 0, s);
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return 0;
}

extern "C" int aitamd_paged_kv_append(int dtype, const aitamd_paged_cache* cache, const void* k, int64_t k_token, int64_t k_head,
                                      const void* v, int64_t v_token, int64_t v_head, const void* q, int64_t q_token, int64_t q_head,
                                      void* q_out, int64_t q_out_token, int64_t q_out_head, int64_t heads, const float* freqs,
                                      int64_t rotated, int64_t first_position, float scale, int interleaved, void* stream) {
  const char* who = "aitamd_paged_kv_append";
  AppendParams p{};
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  if (paged_cache(who, cache, 1, &p.cache)) return 1;
  const int64_t head_dim = cache->head_dim, kv_heads = cache->kv_heads, tokens = cache->tokens;
  if (check_rotation(who, head_dim, rotated, freqs)) return 1;
  if (heads < 0) return fail("%s: negative dimension", who);
  if (!q) heads = 0;
  if (tokens == 0 || (kv_heads == 0 && heads == 0) || cache->batch == 0 || head_dim == 0) return 0;
  if (kv_heads > 0 && (!k || !v || !cache->k || !cache->v)) return fail("%s: null pointer", who);
  if (heads > 0 && !q_out) return fail("%s: null pointer (q_out)", who);
  const int64_t n = rotated / 2;
  const int vec = rotary_vec(n, head_dim, interleaved != 0);
  const int64_t pieces = rotary_pieces((int)n, (int)head_dim, interleaved != 0, vec);
  const int64_t pieces_v = head_dim / vec;
  if (heads > 0x7fffff || kv_heads > 0x7fffff || (heads + kv_heads) * pieces + kv_heads * pieces_v > 0x7fffffffll / kRotaryMaxTokens)
    return fail("%s: dimension too large", who);
  p.q = q, p.k = k, p.v = v;
  p.q_out = q_out;
  p.freqs = freqs;
  p.heads = (int32_t)heads;
  p.n = (int32_t)n;
  p.pieces = (int32_t)pieces;
  p.pieces_v = (int32_t)pieces_v;
  p.per_token = (int32_t)((heads + kv_heads) * pieces + kv_heads * pieces_v);
  p.per_wg = rotary_tokens(tokens, p.per_token, n, current_device_cus());
  p.q_token = q_token, p.q_head = q_head, p.q_out_token = q_out_token, p.q_out_head = q_out_head;
  p.k_token = k_token, p.k_head = k_head, p.v_token = v_token, p.v_head = v_head;
  p.first_position = first_position;
  p.scale = scale;
  p.by_n = make_divisor(n > 0 ? n : 1);
  p.by_token = make_divisor(p.per_token);
  p.by_pieces = make_divisor(pieces);
  p.by_pieces_v = make_divisor(pieces_v);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F16 ? launch_append<f16>(p, vec, interleaved != 0, s) : launch_append<bf16>(p, vec, interleaved != 0, s);
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return 0;
}
