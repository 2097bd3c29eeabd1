// C ABI launcher of aitamd_prefix_attention.
#include <mutex>

#include "../../include/aitemplate_amd_kernels.h"
#include "device.hpp"
#include "errors.hpp"
#include "paged.hpp"
#include "prefix_attention.hpp"

namespace aitamd {
namespace {

constexpr int kMaxDevices = 64;

template <int HD>
struct Tiles {
  using Many = PagedTile<HD, 4, 1, 2, HD <= 128 ? 2 : 1>;  // 128 rows
  using Few = PagedTile<HD, 1, 4, 1, HD <= 128 ? 2 : 1>;   // 32
};

// How a call is dealt to workgroups (the same for every head dim: the tiles have the same rows and about the same keys)
struct Plan {
  bool each;            // tiles of one sequence's rows over prefix and own keys; otherwise the prefix for all rows together
  bool many;            // tiles of 128 rows (not each: the prefix's), otherwise 32
  int64_t row_tiles;    // of all sequences at most (each), of the prefix
  int64_t own_tiles;    // not each: row tiles of all sequences at most
  int64_t prefix_slots, own_slots;
  int64_t slots() const { return prefix_slots + own_slots; }
};

// parts that `items` workgroups' keys are split into: about `wgs` workgroups in all, of at least `least` keys each
int64_t parts(int64_t items, int64_t keys, int64_t least, int64_t wgs) {
  int64_t n = wgs / (items > 0 ? items : 1);
  if (n > keys / least) n = keys / least;
  return n < 1 ? 1 : (n > kMostSlots / 2 ? kMostSlots / 2 : n);
}

Plan make_plan(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t prefix, int64_t most_keys, int64_t head_dim, bool ragged,
               int cus) {
  const int64_t group = heads / kv_heads, rows = tokens * group;
  Plan n{};
  n.many = ragged && rows > 32 * batch;
  n.each = n.many || batch == 1;
  const int64_t tile = n.many ? 128 : 32;
  // (every sequence has one tile that is not full at most)
  const int64_t at_most = ragged ? rows / tile + batch : batch * ((group + tile - 1) / tile);
  if (n.each) {
    n.row_tiles = at_most;
    const int64_t keys = prefix + most_keys;
    // (four tiles of 128 keys one after the other take as long as one and the join)
    n.own_slots = !n.many && keys <= 512 ? 1 : parts((rows > tile ? rows / tile : 1) * kv_heads, keys, 256, 2 * cus);
  } else {
    // Two workgroups fit a CU.  The prefix's workgroups, bound by their matrix instructions, come first and should last as long as
    // what is beside them, the sequences' own keys, which memory bounds: of that only what the table has room for is known, and
    // half of it taken.  One a CU at most (each leaves its rows' parts to the join), half as many at least.  us with 128 / 192 /
    // 256 / 512 of them: 64 sequences behind 8192 keys with 516 of their own on average 46.6 / 47.7 / 49.5 / 61.0, with one 35 / 29 /
    // 28 / 33, 32 sequences 32.6 / 32.5 / 34.0, 64 behind 32768 keys with one of their own 108 / 78 / 64 / 63.
    n.many = rows > 32;
    n.own_tiles = at_most;
    n.row_tiles = n.many ? (rows + 127) / 128 : 1;
    const double tiles = (double)(n.row_tiles * kv_heads) * (double)prefix / 64.0, tile_us = 1.4 * (double)(64 + head_dim) / 192.0;
    const double own_us = (double)(batch * kv_heads * head_dim) * (double)most_keys * 2.0 / 4.5e6;
    const double wgs = own_us * cus > tiles * tile_us ? tiles * tile_us / own_us : cus;
    n.prefix_slots = prefix > 0 ? parts(n.row_tiles * kv_heads, prefix, 256, wgs > cus / 2 ? (int64_t)wgs : cus / 2) : 0;
    n.own_slots = parts(at_most * kv_heads, most_keys, 256, 2 * cus);
  }
  return n;
}

struct LdsOptIn {
  std::once_flag once[kMaxDevices];
  hipError_t err[kMaxDevices];
  hipError_t operator()(const void* kernel, int bytes) {
    int dev = 0;
    const hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    dev %= kMaxDevices;
    std::call_once(once[dev], [&] { err[dev] = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes); });
    return err[dev];
  }
};

template <class T, int HD>
hipError_t launch_attention(PrefixParams& p, const Plan& plan, int64_t wgs, hipStream_t stream) {
  using Many = typename Tiles<HD>::Many;
  using Few = typename Tiles<HD>::Few;
  auto go = [&](auto kernel, int threads, int lds, LdsOptIn& opt_in) {
    const hipError_t e = opt_in(reinterpret_cast<const void*>(kernel), lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(threads), lds, stream, p);
    return hipGetLastError();
  };
  constexpr int kLds = Many::kLdsBytes > Few::kLdsBytes ? Many::kLdsBytes : Few::kLdsBytes;
  static LdsOptIn opt_in[4];
  if (plan.each)
    return plan.many ? go(prefix_prompt_kernel<T, Many>, Many::NT, Many::kLdsBytes, opt_in[0])
                     : go(prefix_prompt_kernel<T, Few>, Few::NT, Few::kLdsBytes, opt_in[1]);
  return plan.many ? go(prefix_decode_kernel<T, Many, Few>, Many::NT, kLds, opt_in[2])
                   : go(prefix_decode_kernel<T, Few, Few>, Few::NT, Few::kLdsBytes, opt_in[3]);
}

template <class T>
hipError_t launch_all(PrefixParams& p, const Plan& plan, int64_t wgs, hipStream_t stream) {
  const int d = p.head_dim;
  hipError_t e = d <= 64 ? launch_attention<T, 64>(p, plan, wgs, stream)
      : d <= 96          ? launch_attention<T, 96>(p, plan, wgs, stream)
      : d <= 128         ? launch_attention<T, 128>(p, plan, wgs, stream)
                         : launch_attention<T, 256>(p, plan, wgs, stream);
  if (e != hipSuccess || plan.slots() == 1) return e;
  const unsigned rows = (unsigned)(p.cache.tokens * p.heads);
  const auto join = d <= 64 ? prefix_join_kernel<T, 16> : (d <= 128 ? prefix_join_kernel<T, 32> : prefix_join_kernel<T, 64>);
  hipLaunchKernelGGL(join, dim3(rows), dim3(256), 0, stream, p, (int)plan.slots(), make_divisor(p.heads));
  return hipGetLastError();
}

// the sizes that both entry points take
int check_sizes(const char* who, const aitamd_paged_cache* cache, int64_t heads, int64_t prefix_length, PagedCache* c) {
  if (paged_cache(who, cache, 16, c)) return 1;
  if (heads < 0 || prefix_length < 0) return fail("%s: negative dimension", who);
  if (cache->kv_heads == 0 ? heads != 0 : heads % cache->kv_heads != 0)
    return fail("%s: %lld query heads are not a multiple of %lld key heads", who, (long long)heads, (long long)cache->kv_heads);
  if (cache->head_dim > 256 || cache->head_dim % 8 != 0)
    return fail("%s: head_dim %lld: a multiple of 8 up to 256 is wanted", who, (long long)cache->head_dim);
  if (heads > 0 && (cache->tokens > 0x3fffffffll / heads || cache->batch > 0x3fffffffll / heads)) return fail("%s: dimension too large", who);
  if (prefix_length > 0x3fffffffll || c->most_keys > 0x3fffffff) return fail("%s: too many keys", who);
  return 0;
}

int64_t workspace_of(const Plan& plan, int64_t tokens, int64_t heads, int64_t head_dim) {
  if (plan.slots() <= 1) return 0;
  const int64_t rows = plan.slots() * tokens * heads;
  return rows * head_dim * 4 + rows * 8;
}

}  // namespace
}  // namespace aitamd

using namespace aitamd;

extern "C" int64_t aitamd_prefix_attention_workspace_bytes(const aitamd_paged_cache* cache, int64_t heads, int64_t prefix_length) {
  const char* who = "aitamd_prefix_attention_workspace_bytes";
  PagedCache c{};
  if (check_sizes(who, cache, heads, prefix_length, &c)) return -1;
  if (cache->tokens == 0 || heads == 0 || cache->batch == 0 || cache->head_dim == 0) return 0;
  const Plan plan = make_plan(cache->tokens, cache->batch, heads, cache->kv_heads, prefix_length, c.most_keys, cache->head_dim,
                              cache->offsets != nullptr, current_device_cus());
  return workspace_of(plan, cache->tokens, heads, cache->head_dim);
}

extern "C" int aitamd_prefix_attention(int dtype, const aitamd_paged_cache* cache, const void* q, int64_t q_token, int64_t q_head, void* out,
                                       int64_t out_token, int64_t out_head, int64_t heads, const int32_t* prefix_table,
                                       int64_t prefix_pages, int64_t prefix_length, float scale, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  const char* who = "aitamd_prefix_attention";
  if (dtype != AITAMD_F16 && dtype != AITAMD_BF16) return fail("%s: bad dtype %d", who, dtype);
  PrefixParams p{};
  if (check_sizes(who, cache, heads, prefix_length, &p.cache)) return 1;
  const int64_t tokens = cache->tokens, batch = cache->batch, kv_heads = cache->kv_heads, head_dim = cache->head_dim;
  if (tokens == 0 || heads == 0 || batch == 0 || head_dim == 0) return 0;
  if (!q || !out || !cache->k || !cache->v || (prefix_length > 0 && !prefix_table)) return fail("%s: null pointer", who);
  if (prefix_pages < 0 || prefix_length > prefix_pages * cache->page_size)
    return fail("%s: a prefix of %lld keys does not lie in %lld pages of %lld", who, (long long)prefix_length, (long long)prefix_pages,
                (long long)cache->page_size);
  if (reinterpret_cast<uintptr_t>(prefix_table) & 3) return fail("%s: the prefix's table has to be 4-byte aligned", who);
  // 16-byte loads, and 16 keys of a page within 32-bit offsets, one after the other
  if ((reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v)) & 15)
    return fail("%s: the cache has to be 16-byte aligned", who);
  const int64_t strides[6] = {cache->k_page_stride, cache->k_slot_stride, cache->k_head_stride,
                              cache->v_page_stride, cache->v_slot_stride, cache->v_head_stride};
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 8 != 0) return fail("%s: the cache's strides have to be multiples of 8 elements", who);
  for (int i = 1; i < 6; i += 3)
    if (strides[i] < head_dim || strides[i] > (1 << 24))
      return fail("%s: a token's stride of %lld in the cache: head_dim = %lld to 2^24 is wanted", who, (long long)strides[i], (long long)head_dim);
  // ... pages apart by less than 2^32 of those 16 bytes, and within one of them by less than 2 GiB
  for (int i = 0; i < 6; i += 3)
    if (strides[i] < 0 || strides[i] / 8 > 0xffffffffll) return fail("%s: a page's stride of %lld in the cache is too large", who, (long long)strides[i]);
  for (int i = 1; i < 6; i += 3)
    if (strides[i] * cache->page_size * 2 > 0x7fffffffll) return fail("%s: pages of %lld tokens %lld elements apart are too large", who,
                                                                    (long long)cache->page_size, (long long)strides[i]);
  p.scale_log2e = scale * 1.4426950408889634f;
  if (!__builtin_isfinite(p.scale_log2e)) return fail("%s: a scale of %g", who, (double)scale);
  const Plan plan = make_plan(tokens, batch, heads, kv_heads, prefix_length, p.cache.most_keys, head_dim, cache->offsets != nullptr,
                              current_device_cus());
  const int64_t need = workspace_of(plan, tokens, heads, head_dim);
  if (need > 0) {
    if (!workspace || workspace_bytes < need)
      return fail("%s: %lld bytes of workspace are wanted, got %lld", who, (long long)need, (long long)(workspace ? workspace_bytes : 0));
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail("%s: the workspace has to be 16-byte aligned", who);
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + plan.slots() * tokens * heads * head_dim);
  }
  p.q = q;
  p.out = out;
  p.prefix_table = prefix_table;
  p.q_token = q_token, p.q_head = q_head, p.out_token = out_token, p.out_head = out_head;
  p.heads = (int32_t)heads;
  p.group = (int32_t)(heads / kv_heads);
  p.head_dim = (int32_t)head_dim;
  p.prefix = (int32_t)prefix_length;
  p.row_tiles = (int32_t)plan.row_tiles;
  p.prefix_slots = (int32_t)plan.prefix_slots;
  p.own_slots = (int32_t)plan.own_slots;
  p.by_group = make_divisor(p.group);
  p.by_row_tiles = make_divisor(plan.row_tiles > 0 ? plan.row_tiles : 1);
  p.by_own_slots = make_divisor(plan.own_slots);
  p.by_kv_heads = make_divisor(kv_heads);
  int64_t wgs;
  if (plan.each) {
    wgs = (plan.row_tiles * kv_heads * plan.own_slots + kNumXcd - 1) / kNumXcd * kNumXcd;
  } else {
    p.prefix_wgs = (int32_t)((plan.prefix_slots * kv_heads + kNumXcd - 1) / kNumXcd * kNumXcd * plan.row_tiles);
    wgs = p.prefix_wgs + plan.own_tiles * kv_heads * plan.own_slots;
  }
  if (wgs > most_workgroups(256) || (plan.slots() > 1 && tokens * heads > most_workgroups(256))) return fail("%s: dimension too large", who);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hipError_t e = dtype == AITAMD_F16 ? launch_all<f16>(p, plan, wgs, s) : launch_all<bf16>(p, plan, wgs, s);
  if (e != hipSuccess) return fail("%s: launch failed: %s", who, hipGetErrorString(e));
  return 0;
}
