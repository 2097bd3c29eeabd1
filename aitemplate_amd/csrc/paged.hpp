// A cache of keys and values in pages, as the kernels take it (the C ABI's aitamd_paged_cache, checked).
#pragma once

#include "../../include/aitemplate_amd_kernels.h"
#include "common.hpp"
#include "errors.hpp"

namespace aitamd {

struct PagedCache {
  void *k, *v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;  // strides, in elements
  const int32_t *table, *lengths, *offsets;
  int64_t table_pitch;
  int32_t pages, page_size, kv_heads, batch, tokens;
  int32_t most_keys;  // that a row of the table has room for
  Divisor by_page;
};

// The sequence that holds row `row`: how many of offsets[1 .. batch] are at most `row` (batch: none holds it).  All 64 lanes
// together; every step takes a 64th of what is left, so up to 64 sequences are one trip to memory.
AITAMD_DEVICE int sequence_of_row(const PagedCache& c, int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, left = c.batch;
  while (left > 0) {
    const int step = (int)(((uint32_t)left + 63u) / 64u);
    const bool in = lane * step < left;
    const int last = lane * step + step - 1 < left - 1 ? lane * step + step - 1 : left - 1;
    const int at_most = in ? (c.offsets[1 + lo + last] <= row ? 1 : 0) : 0;
    const int whole = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at_most != 0)) * step;
    if (whole >= left) return lo + left;
    lo += whole;
    left = step == 1 ? 0 : (left - whole < step ? left - whole : step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// page_multiple: what the page size has to be a multiple of
inline int paged_cache(const char* who, const aitamd_paged_cache* a, int64_t page_multiple, PagedCache* c) {
  if (!a) return fail("%s: null pointer (cache)", who);
  if (a->pages < 0 || a->kv_heads < 0 || a->head_dim < 0 || a->max_pages < 0 || a->batch < 0 || a->tokens < 0)
    return fail("%s: negative dimension", who);
  if (a->page_size <= 0 || a->page_size % page_multiple != 0)
    return fail("%s: page_size %lld: a positive multiple of %lld is wanted", who, (long long)a->page_size, (long long)page_multiple);
  if (a->pages > 0x7fffffffll || a->page_size > 0x7fffffffll || a->kv_heads > 0x7fffffffll || a->batch >= 0x7fffffffll ||
      a->tokens > 0x7fffffffll || a->max_pages > 0x7fffffffll / a->page_size)
    return fail("%s: dimension too large", who);
  if (!a->offsets && a->tokens != a->batch)
    return fail("%s: without offsets every sequence has one row: %lld rows, %lld sequences", who, (long long)a->tokens, (long long)a->batch);
  if (a->batch > 0 && a->tokens > 0 && (!a->lengths || (a->max_pages > 0 && !a->table))) return fail("%s: null pointer (table, lengths)", who);
  if ((reinterpret_cast<uintptr_t>(a->table) | reinterpret_cast<uintptr_t>(a->lengths) | reinterpret_cast<uintptr_t>(a->offsets)) & 3)
    return fail("%s: table, lengths and offsets have to be 4-byte aligned", who);
  c->k = a->k, c->v = a->v;
  c->k_page = a->k_page_stride, c->k_slot = a->k_slot_stride, c->k_head = a->k_head_stride;
  c->v_page = a->v_page_stride, c->v_slot = a->v_slot_stride, c->v_head = a->v_head_stride;
  c->table = a->table, c->lengths = a->lengths, c->offsets = a->offsets;
  c->table_pitch = a->table_pitch;
  c->pages = (int32_t)a->pages;
  c->page_size = (int32_t)a->page_size;
  c->kv_heads = (int32_t)a->kv_heads;
  c->batch = (int32_t)a->batch;
  c->tokens = (int32_t)a->tokens;
  c->most_keys = (int32_t)(a->max_pages * a->page_size);
  c->by_page = make_divisor(a->page_size);
  return 0;
}

}  // namespace aitamd
