// Attention of a batch's new rows over a paged cache: each row sees a prefix that the whole batch shares and its own
// sequence's pages up to itself,
//     out[r] = sum_n exp(c s[r, n]) v[n] / sum_n exp(c s[r, n]),   s[r, n] = q[r] . k[n],
// taken in one pass over the keys with the running maximum m and sum l of each row.  Parts of the keys that different
// workgroups take leave (m, l, sum exp(c (s - m)) v) each and are joined afterwards: with M the largest m,
// the weights are exp(c (m - M)).
//
// A wave owns 32 rows (a row is one query head of one token; the query heads of a key head are neighbours) and takes the
// scores in transposed form, S^T = K Q^T, whose accumulator layout is that of the second product's operand, O^T += V^T P^T:
// the probabilities never leave the registers.  WR waves stand side by side over rows and share every tile of keys; WK waves
// take 32 keys of a tile each, for themselves, and join at the end.
//
// Bound, 128 rows of 96 dims: a tile of 64 keys is 768 cycles of each SIMD's matrix unit, 0.32 us, and as many of vector
// instructions.  A workgroup alone on its CU takes 1.4 us for it, one after the other with the reads of LDS and the scalars between
// them; of two workgroups on a CU the one's matrix instructions run beside the other's vector instructions in part, 0.83 us a tile
// (128 dims: 1.6 and 1.1): 960 TFLOP/s for 32 heads of 2048 rows over a prefix of 9984 keys, 1040 with 128 dims.  It is neither the
// reads of K from LDS nor the latency of the loads: some 10 000 keys, the rows' own among them, at 890 and 975 TFLOP/s, with the next
// tile's K read into registers between the second product's steps at 902 and 950, no faster with a third stage for K.
//
// Keys and values go from their pages straight to LDS: 16 consecutive keys lie in one page (page sizes are multiples of
// 16), so the page is one scalar per 16 keys and the bounds of its buffer descriptor cut off what is past the last key:
// what lies there may be anything, and is not read.
#pragma once

#include "attention_kernel.hpp"
#include "paged.hpp"

namespace aitamd {

// The weights exp(c (s - m)) are rounded to the type's 16 bits for the second product, by half a step at most (2^-11 relative in fp16,
// 2^-8 in bf16), and their sum is taken of the rounded ones: a result moves by as much of the weighted mean of |v|.  As sums of two
// 16-bit numbers they would take the second product, half of the matrix instructions, twice.  Error of three timed cases against
// 64 bits (norm, relative): 2.9e-4 in fp16 and 2.3e-3 in bf16, of which rounding the result alone is 2.1e-4 and 1.7e-3.
//
// fp16 also ends at 2^-25 below and at 2^16 above.  What is below is lost, however many keys it is of: with the reference point's
// weight at 1, 2^17 keys of 2^-25.5 of the largest weight each, 0.3 % of the result, were none.  So weights in fp16 are held
// 2^kRaiseLog2 times as large (the sum too: it cancels), and the full form leaves the reference point 2^kLazyLog2 below a row's
// maximum at most, 2^15 together.  What is lost is below 2^-33 of the largest weight, n such keys n 2^-33: 2^-13 of it for 10^6
// keys.  More would leave the fast form less room for maxima that grow: four prompts of 512 rows behind 2000 keys, 64 dims, scores
// with a deviation of 1, 2, 4 and 8: 78.4, 77.9, 77.9, 86.1 us at 1, 78.4, 78.2, 89.4, 94.0 at 2^8, 78.1, 84.2, 92.1, 96.0 at 2^11.
// bf16 has the range of 32 bits.
template <class T>
struct Weights {
  static constexpr float kRaiseLog2 = 8.0f, kLazyLog2 = 7.0f;
  // Row sums up to which the fast form stands: a weight out of range is an infinity and shows in any finite bound; 2^30 keys of up
  // to 2^16 do not trip it, and their products with values stay far below the largest float.
  static constexpr float kMaxSum = 0x1p47f;
};
template <>
struct Weights<bf16> {
  static constexpr float kRaiseLog2 = 0.0f, kLazyLog2 = 8.0f, kMaxSum = kMaxRowSum;
};

struct PrefixParams {
  PagedCache cache;
  const void* q;
  void* out;
  float* part_o;   // [slot, token, head, head_dim]
  float2* part_ml; // [slot, token, head]: c * m and l (l, as part_o, 2^kRaiseLog2 times as large: see Weights)
  const int32_t* prefix_table;
  int64_t q_token, q_head, out_token, out_head;
  int32_t heads, group, head_dim, prefix;
  int32_t row_tiles, prefix_slots, own_slots, prefix_wgs;
  float scale_log2e;
  Divisor by_group, by_row_tiles, by_own_slots, by_kv_heads;
};

// HD: head dims, padded; a row takes the next power of two in LDS.  WR > 1: waves side by side over rows, the second product a
// tile behind the first (K(t) and V(t - 1) are multiplied while K(t + 1) and V(t + 1) land: two stages for K, three for V).
// WK > 1: over keys, a wave loads a tile, waits and multiplies; the CU's other waves have theirs on the way meanwhile.
template <int HD_, int WR_, int WK_, int KB_, int OCC_>
struct PagedTile {
  static constexpr int HD = HD_, WR = WR_, WK = WK_, KB = KB_, OCC = OCC_;
  static constexpr int KP = HD <= 64 ? 64 : (HD <= 128 ? 128 : 256);
  static constexpr int KS = HD / 16, OT = HD / 32;
  static constexpr int NW = WR * WK, NT = 64 * NW;
  static constexpr int ROWS = 32 * WR;
  static constexpr int BN = 32 * KB * WK;     // keys of a tile
  static constexpr int KPW = BN / NW;         // keys a wave loads
  static constexpr int GROUPS = KPW / 16;
  static constexpr int CHUNKS = KP / 8;       // 16-byte pieces of a row in LDS
  static constexpr int RPL = 64 / CHUNKS;     // rows of a wave-load
  static constexpr int LPG = 16 / RPL;        // wave-loads of 16 keys
  static constexpr bool PIPED = WR > 1;
  static constexpr int NK = PIPED ? 2 : 1, NV = PIPED ? 3 : 1;
  static constexpr int STAGE = BN * KP;       // elements
  static constexpr int kRing = (NK + NV) * STAGE * 2;
  static constexpr int kMerge = WK > 1 ? WK * (16 * OT + 2) * 64 * 4 : 0;
  static constexpr int kLdsBytes = kRing > kMerge ? kRing : kMerge;
  // 16-byte piece c of row r lies at piece c ^ swizzle(r).  K: 32 rows' piece at a time; V: see AttnTile::v_swz.
  static constexpr int k_swz(int row) { return CHUNKS == 8 ? (row / 2) % 8 : row % 16; }
  static constexpr int v_swz(int row) { return CHUNKS == 8 ? 4 * ((row / 2) % 2) : 4 * (row % 4); }
  static_assert(WK == 1 || (WR == 1 && KPW == 32 * KB), "waves side by side over keys load what they multiply");
  static_assert(KPW % 16 == 0, "a wave loads whole groups of 16 keys");
  static_assert(kLdsBytes <= 160 * 1024, "LDS budget");
};

// What one workgroup does: rows [row0, rows) of the `rows` that start at token `token0`, for key head `kv_head`, over tiles
// [t_lo, t_hi): the first `prefix_tiles` of all are the prefix's, the others the sequence's own (`own_keys` of them, of which the
// rows of the j-th token see seen + j).
struct PagedWork {
  const int32_t* table;
  int kv_head, token0, row0, rows, t_lo, t_hi, prefix_tiles, own_keys, seen, slot;
};

// 16 bytes a lane from memory to LDS: lane l's to dst + 16 l.  (The host pass does not know the builtin, and gives up a function
// template that holds it where two kernels call it.)
AITAMD_DEVICE void load_to_lds(__amdgpu_buffer_rsrc_t r, void* dst, uint32_t off) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef __attribute__((address_space(3))) void lds_void;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 16, off, 0, 0, 0);
#endif
}

template <class T, class Tile>
AITAMD_DEVICE void attend(const PrefixParams& p, const PagedWork& w, unsigned char* smem_raw) {
  using Tr = ElemTraits<T>;
  using W = Weights<T>;
  using vec8 = typename Tr::vec8;
  using vec4 = typename Tr::vec4;
  typedef __attribute__((address_space(3))) const T lds_T;
  typedef __attribute__((address_space(3))) const vec8 lds_vec8;
  constexpr int KP = Tile::KP, KS = Tile::KS, OT = Tile::OT, KB = Tile::KB, WR = Tile::WR, WK = Tile::WK, BN = Tile::BN;
  constexpr int V_LOADS = Tile::GROUPS * Tile::LPG;  // of a wave and a tile
  T* const sK = reinterpret_cast<T*>(smem_raw);
  T* const sV = sK + Tile::NK * Tile::STAGE;
  const PagedCache& c = p.cache;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = WK == 1 ? wave : 0, wk = WK == 1 ? 0 : wave;
  const int r32 = lane & 31, h = lane >> 5;

  // lane offsets of the loads of 16 keys
  uint32_t k_off[Tile::LPG], v_off[Tile::LPG];
#pragma unroll
  for (int i = 0; i < Tile::LPG; ++i) {
    const int row = i * Tile::RPL + lane / Tile::CHUNKS, slot = lane % Tile::CHUNKS;
    const int kc = slot ^ Tile::k_swz(row), vc = slot ^ Tile::v_swz(row);
    k_off[i] = kc * 8 < p.head_dim ? (uint32_t)row * (uint32_t)(c.k_slot * 2) + (uint32_t)kc * 16u : kOobOffset;
    v_off[i] = vc * 8 < p.head_dim ? (uint32_t)row * (uint32_t)(c.v_slot * 2) + (uint32_t)vc * 16u : kOobOffset;
  }
  // The tile that is to be loaded next, of this wave's 16 keys at a time: their page, where in it they begin and how many
  // there are.  All scalars, prepared a tile ahead: the page is a trip to memory.
  typedef const __attribute__((address_space(4))) int32_t* scalar_ptr;
  int next_t = w.t_lo, next_key, next_keys;
  scalar_ptr next_table;
  auto enter = [&](bool shared) {  // the prefix's tiles, or the sequence's own
    next_key = (next_t - (shared ? 0 : w.prefix_tiles)) * BN + wave * Tile::KPW;
    next_keys = shared ? p.prefix : w.own_keys;
    next_table = (scalar_ptr) reinterpret_cast<uintptr_t>(shared ? p.prefix_table : w.table);
  };
  enter(next_t < w.prefix_tiles);
  int page[Tile::GROUPS], within[Tile::GROUPS], rows[Tile::GROUPS];
  auto prepare = [&]() {
    if (next_t >= w.t_hi) return;
    if (next_t == w.prefix_tiles) enter(false);
#pragma unroll
    for (int g = 0; g < Tile::GROUPS; ++g) {
      const int key = next_key + g * 16, left = next_keys - key;
      const int at = left > 0 ? key : 0, which = quotient(at, c.by_page);
      page[g] = next_table[which];
      within[g] = at - which * c.page_size;
      rows[g] = left > 0 ? (left < 16 ? left : 16) : 0;
    }
    next_key += BN;
    ++next_t;
  };
  const char* const k_base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(c.k) + w.kv_head * c.k_head);
  const char* const v_base = reinterpret_cast<const char*>(reinterpret_cast<const T*>(c.v) + w.kv_head * c.v_head);
  const uint32_t k_page16 = (uint32_t)(c.k_page / 8), v_page16 = (uint32_t)(c.v_page / 8);  // in 16-byte units
  const uint32_t k_slot = (uint32_t)(c.k_slot * 2), v_slot = (uint32_t)(c.v_slot * 2);      // in bytes
  const uint32_t row_bytes = (uint32_t)p.head_dim * 2u;
  // the prepared tile into stage k_in, v_in (offsets in elements)
  int k_in = 0, v_in = 0;
  auto issue = [&]() {
    T* const dk = sK + k_in + wave * Tile::KPW * KP;
    T* const dv = sV + v_in + wave * Tile::KPW * KP;
    __amdgpu_buffer_rsrc_t rv[Tile::GROUPS];
#pragma unroll
    for (int g = 0; g < Tile::GROUPS; ++g) {
      // (a page that is none: nothing in bounds, so zeros)
      const uint32_t pg = (uint32_t)__builtin_amdgcn_readfirstlane(page[g]);
      const uint32_t n = (uint32_t)__builtin_amdgcn_readfirstlane(pg < (uint32_t)c.pages ? rows[g] : 0);
      const uint32_t in = (uint32_t)__builtin_amdgcn_readfirstlane(within[g]);
      const __amdgpu_buffer_rsrc_t rk = make_rsrc(k_base + (((uint64_t)pg * k_page16) << 4) + in * k_slot, n > 0 ? (n - 1) * k_slot + row_bytes : 0u);
      rv[g] = make_rsrc(v_base + (((uint64_t)pg * v_page16) << 4) + in * v_slot, n > 0 ? (n - 1) * v_slot + row_bytes : 0u);
#pragma unroll
      for (int i = 0; i < Tile::LPG; ++i) load_to_lds(rk, dk + g * 16 * KP + i * 512, k_off[i]);
    }
    // (behind all of K: a wait for the last V_LOADS leaves them out)
#pragma unroll
    for (int g = 0; g < Tile::GROUPS; ++g)
#pragma unroll
      for (int i = 0; i < Tile::LPG; ++i) load_to_lds(rv[g], dv + g * 16 * KP + i * 512, v_off[i]);
    k_in = k_in == (Tile::NK - 1) * Tile::STAGE ? 0 : k_in + Tile::STAGE;
    v_in = v_in == (Tile::NV - 1) * Tile::STAGE ? 0 : v_in + Tile::STAGE;
  };

  // Q fragments (B operand of S^T = K Q^T): lane (row = r32, k = 16 ks + 8 h + j)
  const int row = w.row0 + wr * 32 + r32;
  const int ahead = quotient(row, p.by_group);                   // the row's token, from token0
  const int head = w.kv_head * p.group + row - ahead * p.group;
  const int64_t token = w.token0 + ahead;
  const bool live = row < w.rows;
  const uint32_t flip = p.scale_log2e < 0.0f ? 0x80008000u : 0u;  // a negative scale changes sides: (-Q) K^T, exact
  const float cs = fmaxf(__builtin_fabsf(p.scale_log2e), 1e-37f); // (a scale of zero counts as one that makes every score the same)
  vec8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int k0 = ks * 16 + h * 8;
    u32x4 raw = {};
    if (live && k0 < p.head_dim) raw = load_vec<u32x4>(reinterpret_cast<const T*>(p.q) + token * p.q_token + head * p.q_head + k0);
#pragma unroll
    for (int d = 0; d < 4; ++d) raw[d] ^= flip;
    qf[ks] = __builtin_bit_cast(vec8, raw);
  }
  // own keys that this row sees
  int seen = w.seen + ahead;
  seen = seen < w.own_keys ? seen : w.own_keys;
  // ... that every row of the wave does, and that some row does (rows are in order)
  const int every = __builtin_amdgcn_readfirstlane(seen), some_own = __builtin_amdgcn_readlane(seen, 31);

  // LDS offsets of the fragment reads
  int k_rd[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) k_rd[ks] = (wk * 32 * KB + r32) * KP + ((2 * ks + h) ^ Tile::k_swz(r32)) * 8;
  const int tr_row = (lane & 15) >> 2;
  const int tr_col = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  int v_rd[OT];
#pragma unroll
  for (int ot = 0; ot < OT; ++ot)
    v_rd[ot] = (wk * 32 * KB + h * 4 + tr_row) * KP + ((ot * 32) ^ (Tile::v_swz(tr_row) * 8)) + tr_col;

  f32x16 oacc[OT];
#pragma unroll
  for (int ot = 0; ot < OT; ++ot) oacc[ot] = f32x16{};
  float m_run = -INFINITY, l_run = 0.0f;

  vec8 pf[2 * KB];  // P^T fragments (of the tile whose second product is due)

  auto read_v = [&](lds_T* base, int i, int ot) {
    const vec4 lo = AttnVec<T>::tr_read(base + v_rd[ot] + i * 16 * KP);
    const vec4 hi = AttnVec<T>::tr_read(base + v_rd[ot] + (i * 16 + 8) * KP);
    return join_halves<T>(lo, hi);
  };
  auto second_product = [&](lds_T* base) {
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i)
#pragma unroll
      for (int ot = 0; ot < OT; ++ot) oacc[ot] = Tr::mfma32(read_v(base, i, ot), pf[i], oacc[ot]);
  };
  auto scores = [&](const T* st, f32x16* s) {
    lds_T* kb_ptr = (lds_T*)st;
    // (all reads first: left to itself the compiler fetches a pair and waits for it in front of every second product)
    vec8 kf[KB][KS];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[kb][ks] = *(lds_vec8*)(kb_ptr + kb * 32 * KP + k_rd[ks]);
    __builtin_amdgcn_sched_barrier(0x6);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[kb] = Tr::mfma32(kf[kb][ks], qf[ks], ks == 0 ? f32x16{} : s[kb]);
  };
  // Probabilities of a tile in the full form: masks, the row's maximum, a moved reference point, rescaled accumulators.
  // first: this wave's first key; limit: keys the row sees; whole: every row sees all of the tile's
  auto full_form = [&](f32x16* s, int first, int limit, bool whole) {
    if (!whole) {
      const int left = limit - first - h * 4;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (kb * 32 + (e >> 2) * 8 + (e & 3) >= left) s[kb][e] = -INFINITY;
    }
    float most = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) most = fmaxf(most, s[kb][e]);
    most = max_across_halves(most);
    // The reference point moves only when the row maximum has grown by more than kLazyLog2 binary orders since it was last
    // taken: until then P is 2^kLazyLog2 times what it is at the reference point at most, harmless in fp32 sums and in P.
    const float m_cand = fmaxf(m_run, most);
    const float drift = (m_run - m_cand) * cs;  // <= 0; -inf (or NaN for inf - inf) on the first live tile
    const bool move = !(drift >= -W::kLazyLog2);
    const float m_new = move ? m_cand : m_run;
    const float m_safe = __builtin_isinf(m_new) ? 0.0f : m_new;  // every key so far masked
    const float alpha = !move ? 1.0f : (__builtin_isinf(m_run) ? 0.0f : __builtin_amdgcn_exp2f(drift));
    const float mc = W::kRaiseLog2 - m_safe * cs;
    l_run *= alpha;
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        pf[i][j] = Tr::from_float(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][(i & 1) * 8 + j], cs, mc)));
      l_run = add_elements(pf[i], l_run);
    }
    m_run = m_new;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
      for (int ot = 0; ot < OT; ++ot)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[ot][e] *= alpha;
    }
  };

  prepare();
  if constexpr (Tile::PIPED) {
    bool due = false;     // (wave-uniform) pf holds a tile's probabilities
    bool ref_ok = false;  // (wave-uniform) every row of the wave has a finite reference point
    int k_at = 0, v_at = 0;  // stages of K(t) and V(t - 1)
    if (w.t_lo < w.t_hi) {
      issue();
      prepare();
    }
    int first = (w.t_lo < w.prefix_tiles ? w.t_lo : w.t_lo - w.prefix_tiles) * BN;  // the tile's first key
    for (int t = w.t_lo; t < w.t_hi; ++t, first += BN) {
      // K(t) and V(t - 1) have landed once only V(t) is out; past the barrier everybody's have, and nobody reads the stages of
      // K(t - 1) and V(t - 2) any more
      attn_wait_vmcnt<V_LOADS>();
      __builtin_amdgcn_s_barrier();
      if (t + 1 < w.t_hi) {
        issue();
        prepare();
      }
      const bool shared = t < w.prefix_tiles;
      if (t == w.prefix_tiles) first = 0;
      lds_T* const vb = (lds_T*)(sV + v_at);
      // (the last tiles may hold nothing that this wave's rows see: masked like any other.  us, eight ragged prompts, with a branch
      // around all of this / so: head dim 64 63.7 / 62.9, 80 82.4 / 79.3, 128 94.4 / 95.3, 256 251 / 252)
      f32x16 s[KB];
      scores(sK + k_at, s);
      const bool whole = first + 32 * KB <= (shared ? p.prefix : every);
      bool full = !ref_ok || !whole;
      if (!full) {
        // The probabilities against the reference point the row has (exact whatever it is, as long as nothing leaves its range),
        // between the matrix instructions of the tile before.
        const float l_before = l_run, mc = W::kRaiseLog2 - m_run * cs;
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i) {
#pragma unroll
          for (int ot = 0; ot < OT; ++ot) oacc[ot] = Tr::mfma32(read_v(vb, i, ot), pf[i], oacc[ot]);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            pf[i][j] = Tr::from_float(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][(i & 1) * 8 + j], cs, mc)));
          l_run = add_elements(pf[i], l_run);
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(l_run <= W::kMaxSum)) != 0, 0)) {
          l_run = l_before;  // (NaN, or a maximum far above the reference point: again, in the full form)
          full = true;
          due = false;
        }
      }
      if (full) {
        if (due) second_product(vb);
        due = first < (shared ? p.prefix : some_own);
        full_form(s, first, shared ? p.prefix : seen, whole);
        ref_ok = __builtin_amdgcn_ballot_w64(__builtin_isinf(m_run)) == 0;
      }
      k_at = k_at == (Tile::NK - 1) * Tile::STAGE ? 0 : k_at + Tile::STAGE;
      if (t > w.t_lo) v_at = v_at == (Tile::NV - 1) * Tile::STAGE ? 0 : v_at + Tile::STAGE;  // (V(t): behind V(t - 1)'s, which for the first is none)
    }
    attn_wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    if (due) second_product((lds_T*)(sV + v_at));
  } else {
    for (int t = w.t_lo; t < w.t_hi; ++t) {
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave has read the last tile
      issue();
      prepare();
      const bool shared = t < w.prefix_tiles;
      const int first = (shared ? t : t - w.prefix_tiles) * BN + wk * 32 * KB;  // this wave's first key
      const bool there = first < (shared ? p.prefix : some_own);
      attn_wait_vmcnt<V_LOADS>();
      f32x16 s[KB];
      if (there) scores(sK, s);
      attn_wait_vmcnt<0>();
      if (!there) continue;
      full_form(s, first, shared ? p.prefix : seen, first + 32 * KB <= (shared ? p.prefix : every));
      second_product((lds_T*)sV);
    }
  }
  l_run = sum_across_halves(l_run);

  // ---- waves side by side over keys: each takes some of the dims of all
  if constexpr (WK > 1) {
    __syncthreads();
    constexpr int NVAL = 16 * OT + 2;
    float* const xch = reinterpret_cast<float*>(smem_raw) + lane;
#pragma unroll
    for (int ot = 0; ot < OT; ++ot)
#pragma unroll
      for (int e = 0; e < 16; ++e) xch[(wk * NVAL + ot * 16 + e) * 64] = oacc[ot][e];
    xch[(wk * NVAL + NVAL - 2) * 64] = m_run;
    xch[(wk * NVAL + NVAL - 1) * 64] = l_run;
    __syncthreads();
    float m[WK], m_all = -INFINITY;
#pragma unroll
    for (int i = 0; i < WK; ++i) {
      m[i] = xch[(i * NVAL + NVAL - 2) * 64];
      m_all = fmaxf(m_all, m[i]);
    }
    m_run = m_all;
    l_run = 0.0f;
#pragma unroll
    for (int i = 0; i < WK; ++i) {
      m[i] = __builtin_isinf(m[i]) ? 0.0f : __builtin_amdgcn_exp2f((m[i] - m_all) * cs);
      l_run += m[i] * xch[(i * NVAL + NVAL - 1) * 64];
    }
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
      if (ot % WK != wk) continue;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < WK; ++i) sum += m[i] * xch[(i * NVAL + ot * 16 + e) * 64];
        oacc[ot][e] = sum;
      }
    }
  }
  if (!live) return;
  // ---- store: the result, or this part of it (its arguments fetched here and not held over the loop)
  const PrefixParams& a = arguments_anew<PrefixParams>();
  if (a.part_o == nullptr) {
    const float inv = l_run > 0.0f ? 1.0f / l_run : (l_run == 0.0f ? 0.0f : l_run);  // (NaN stays)
    T* const o = reinterpret_cast<T*>(a.out) + token * a.out_token + head * a.out_head;
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
      if (ot % WK != wk) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = ot * 32 + g * 8 + h * 4;
        vec4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = Tr::from_float(oacc[ot][g * 4 + j] * inv);
        if (d < a.head_dim) store_vec(o + d, v);
      }
    }
  } else {
    const int64_t at = ((int64_t)w.slot * a.cache.tokens + token) * a.heads + head;
    if (wk == 0 && h == 0) a.part_ml[at] = make_float2(l_run == 0.0f ? -INFINITY : m_run * cs, l_run);
    float* const o = a.part_o + at * a.head_dim;
#pragma unroll
    for (int ot = 0; ot < OT; ++ot) {
      if (ot % WK != wk) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = ot * 32 + g * 8 + h * 4;
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = oacc[ot][g * 4 + j];
        if (d < a.head_dim) *reinterpret_cast<f32x4*>(o + d) = v;
      }
    }
  }
}

// Rows of tokens [first, last) of sequence `s`, within the buffers whatever the offsets are
AITAMD_DEVICE void rows_of(const PagedCache& c, int s, int& first, int& last) {
  if (c.offsets == nullptr) {
    first = s;
    last = s + 1;
    return;
  }
  first = c.offsets[s];
  last = c.offsets[s + 1];
  first = first < 0 ? 0 : (first < c.tokens ? first : c.tokens);
  last = last < first ? first : (last < c.tokens ? last : c.tokens);
}

// Keys of its own that a sequence's first new row sees, and how many its last one does
AITAMD_DEVICE void keys_of_sequence(const PagedCache& c, int s, int count, int& seen, int& keys) {
  // (lengths below zero: a sequence that is not there; its rows see no key of their own until they are counted up)
  const int len = c.lengths[s];
  seen = len >= c.most_keys ? c.most_keys : len + 1;
  const int64_t all = (int64_t)len + count;
  keys = all <= 0 ? 0 : (all < c.most_keys ? (int)all : c.most_keys);
}

// [lo, hi) of `tiles` that part `i` of `parts` takes
AITAMD_DEVICE void part_of(int tiles, int i, int parts, int& lo, int& hi) {
  lo = (int)((int64_t)tiles * i / parts);
  hi = (int)((int64_t)tiles * (i + 1) / parts);
}

// The sequence that the `tile`-th row tile of all sequences belongs to (-1: there are fewer), and which of its tiles that is:
// 64 sequences at a time, their tiles added up.
AITAMD_DEVICE int sequence_of_tile(const PrefixParams& p, int tile_rows, int& tile) {
  const PagedCache& c = p.cache;
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base < c.batch; base += 64) {
    int mine = 0;
    if (base + lane < c.batch) {
      int first, last;
      rows_of(c, base + lane, first, last);
      mine = ((last - first) * p.group + tile_rows - 1) / tile_rows;
    }
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = __shfl_up(upto, d);
      if (lane >= d) upto += other;
    }
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before + upto <= tile));
    if (n < 64) {
      // (lanes past the last sequence have no tiles, so lane n is a sequence)
      tile = __builtin_amdgcn_readfirstlane(tile - before - (n > 0 ? __shfl(upto, n - 1) : 0));
      return __builtin_amdgcn_readfirstlane(base + n);
    }
    before += __shfl(upto, 63);
  }
  return -1;
}

// Few rows a sequence (decoding).  The first workgroups take the prefix, for the rows of all sequences together; the others
// one sequence's own keys each.
template <class T, class Shared, class Own>
__global__ void __launch_bounds__(Shared::NT, Shared::OCC) prefix_decode_kernel(const PrefixParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  static_assert(Shared::NT == Own::NT, "one workgroup size");
  const PagedCache& c = p.cache;
  PagedWork w{};
  if ((int)blockIdx.x < p.prefix_wgs) {
    // consecutive workgroups go to the 8 XCDs in turn: the row tiles of one (head, part) follow each other on one of them
    const int id = blockIdx.x, xcd = id % kNumXcd, local = id / kNumXcd;
    const int nth = quotient(local, p.by_row_tiles), tile = local - nth * p.row_tiles;
    const int pair = nth * kNumXcd + xcd;
    const int part = quotient(pair, p.by_kv_heads);
    w.kv_head = pair - part * c.kv_heads;
    if (part >= p.prefix_slots) return;
    int tokens = c.tokens;
    if (c.offsets != nullptr) {
      const int last = c.offsets[c.batch];
      tokens = last < 0 ? 0 : (last < tokens ? last : tokens);
    }
    w.rows = tokens * p.group;
    w.row0 = tile * Shared::ROWS;
    if (w.row0 >= w.rows) return;
    w.prefix_tiles = (p.prefix + Shared::BN - 1) / Shared::BN;
    part_of(w.prefix_tiles, part, p.prefix_slots, w.t_lo, w.t_hi);
    w.slot = part;
    attend<T, Shared>(p, w, smem_raw);
  } else {
    const int id = blockIdx.x - p.prefix_wgs;
    const int pair = quotient(id, p.by_own_slots), part = id - pair * p.own_slots;
    int s = quotient(pair, p.by_kv_heads);
    w.kv_head = pair - s * c.kv_heads;
    int first, last, tile = 0;
    if (c.offsets != nullptr || p.group > Own::ROWS) {
      tile = s;
      s = sequence_of_tile(p, Own::ROWS, tile);
      if (s < 0) return;
    }
    rows_of(c, s, first, last);
    w.token0 = first;
    w.rows = (last - first) * p.group;
    w.row0 = tile * Own::ROWS;
    if (w.row0 >= w.rows) return;
    keys_of_sequence(c, s, last - first, w.seen, w.own_keys);
    w.table = c.table + s * c.table_pitch;
    part_of((w.own_keys + Own::BN - 1) / Own::BN, part, p.own_slots, w.t_lo, w.t_hi);
    w.slot = p.prefix_slots + part;
    attend<T, Own>(p, w, smem_raw);
  }
}

// Many rows a sequence (prompts, pieces of them), or one sequence alone.  A workgroup takes a tile of one sequence's rows over the
// prefix and then over the sequence's own keys.
template <class T, class Tile>
__global__ void __launch_bounds__(Tile::NT, Tile::OCC) prefix_prompt_kernel(const PrefixParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem_raw[];
  const PagedCache& c = p.cache;
  // an XCD takes a run of (key head, part) pairs' row tiles, so that the keys they share come to one L2
  const int per_xcd = gridDim.x / kNumXcd;
  const int id = (int)(blockIdx.x % kNumXcd) * per_xcd + (int)(blockIdx.x / kNumXcd);
  const int pair = quotient(id, p.by_row_tiles);
  int tile = id - pair * p.row_tiles, first, last;
  const int part = quotient(pair, p.by_kv_heads);
  if (part >= p.own_slots) return;
  int s = 0;
  if (c.batch > 1) {
    s = sequence_of_tile(p, Tile::ROWS, tile);
    if (s < 0) return;
  }
  PagedWork w{};
  rows_of(c, s, first, last);
  w.kv_head = pair - part * c.kv_heads;
  w.token0 = first;
  w.rows = (last - first) * p.group;
  w.row0 = tile * Tile::ROWS;
  if (w.row0 >= w.rows) return;
  keys_of_sequence(c, s, last - first, w.seen, w.own_keys);
  // (no further than the tile's last row sees)
  const int last_row = w.row0 + Tile::ROWS < w.rows ? w.row0 + Tile::ROWS - 1 : w.rows - 1;
  const int last_seen = w.seen + quotient(last_row, p.by_group);
  w.own_keys = last_seen < 0 ? 0 : (last_seen < w.own_keys ? last_seen : w.own_keys);
  w.table = c.table + s * c.table_pitch;
  w.prefix_tiles = (p.prefix + Tile::BN - 1) / Tile::BN;
  part_of(w.prefix_tiles + (w.own_keys + Tile::BN - 1) / Tile::BN, part, p.own_slots, w.t_lo, w.t_hi);
  w.slot = part;
  attend<T, Tile>(p, w, smem_raw);
}

// The parts of a row joined.  A workgroup takes one row: LANES lanes of 4 dims each, and 256 / LANES groups of those that take
// every so manieth part; the parts' weights are computed once, by as many lanes.  Bound: latency, of three trips to memory (offsets,
// (m, l), parts) one after the other.  64 x 32 rows of 33 parts of 128 dims: 28 us with one lane going through a row's parts, 6 so (of 17).
constexpr int kMostSlots = 128;
template <class T, int LANES>
__global__ void __launch_bounds__(256) prefix_join_kernel(const PrefixParams p, int slots, Divisor by_heads) {
  constexpr int GROUPS = 256 / LANES;
  __shared__ float weight[kMostSlots];
  __shared__ float sums[4];
  __shared__ __attribute__((aligned(16))) f32x4 part[GROUPS][LANES];
  const int row = blockIdx.x, token = quotient(row, by_heads), head = row - token * p.heads;
  const int64_t rows = (int64_t)p.cache.tokens * p.heads;
  const int tid = threadIdx.x, lane = tid % LANES, group = tid / LANES, d = lane * 4;
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (tid < slots) ml = p.part_ml[tid * rows + row];
  if (p.cache.offsets != nullptr && (token < p.cache.offsets[0] || token >= p.cache.offsets[p.cache.batch])) return;
  // (the first two waves hold all parts)
  float most = ml.x;
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) most = fmaxf(most, __shfl_xor(most, s));
  if ((tid & 63) == 0 && tid < kMostSlots) sums[tid >> 6] = most;
  __syncthreads();
  most = fmaxf(sums[0], sums[1]);
  // (no key: no weight, whatever lies in its place)
  const float w = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - most);
  if (tid < kMostSlots) weight[tid] = w;
  float sum = ml.y == 0.0f ? 0.0f : ml.y * w;
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) sum += __shfl_xor(sum, s);
  if ((tid & 63) == 0 && tid < kMostSlots) sums[2 + (tid >> 6)] = sum;
  __syncthreads();
  sum = sums[2] + sums[3];
  f32x4 o = {};
  if (d < p.head_dim) {
    const float* at = p.part_o + (int64_t)row * p.head_dim + d;
    const int64_t step = rows * p.head_dim;
#pragma unroll 4
    for (int s = group; s < slots; s += GROUPS) {
      const float by = weight[s];
      const f32x4 v = *reinterpret_cast<const f32x4*>(at + s * step);
      // (a part without keys is not written)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += by == 0.0f ? 0.0f : v[j] * by;
    }
  }
  part[group][lane] = o;
  __syncthreads();
  if (group != 0 || d >= p.head_dim) return;
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) o += part[g][lane];
  const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
  typename ElemTraits<T>::vec4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = ElemTraits<T>::from_float(o[j] * inv);
  store_vec(reinterpret_cast<T*>(p.out) + token * p.out_token + head * p.out_head + d, y);
}

}  // namespace aitamd
