// Causal attention of the new rows of a batch over a paged cache.
//
//   o[t, h] = sum_j p_j v[j, h / g],  p = softmax_j(scale q[t, h] . k[j, h / g]),  j <= len - n + (t - first row)
// for every sequence of the batch: n new rows (one when it decodes, a chunk when a prompt comes in), len tokens in the cache
// with the new ones, g = q heads a kv head.  A row that sees no key is zero.
//
// The g query heads of a kv head read the same keys, so they are rows of one tile: row p of a sequence's tiles is token p / g,
// head p % g.  Both products run on the matrix cores with the keys' product transposed, S^T = K Q^T: a lane then
// holds one query row and some keys of it, the softmax's maximum and sum cross lanes once or twice, and the probabilities lie in
// the registers as the next product, O^T = V^T P^T, reads them (the keys of a step may come in any order, as long as P and V
// agree).  V is read from LDS through the transposing load.  One pass over the keys with the running maximum and sum; statistics
// and accumulators in float.  The probabilities are rounded to the element type for the second product: relative errors of half
// a step each, of random sign, so about as much as the rounding of the result itself.  Their sum is taken of the rounded ones: what the errors
// have in common leaves the result alone, and values that are all alike come back.
//
// Sequences of up to 16 tile rows (decoding) are bound by HBM: the four waves of a workgroup take 32 keys in turn, K straight to
// registers, V through a part of LDS of the wave's own, no barrier until the end.  256 single tokens over up to 4095, 8 kv heads of 128:
// 2.13 GB in 362 to 382 us by the card, 5.6 to 5.9 TB/s (a plain copy reaches 4.9); three over 131000 5.6 to 5.8 TB/s.  (Three or four workgroups
// a CU, with fewer registers: 433 and 688 us.)  Others take 128 tile rows a workgroup, 32 a wave, over K and V tiles of 64 keys that the
// four waves share: 2048 rows of 32 heads over 14336 tokens 500 to 535 us by the card, 0.96 to 1.03 PFLOP/s (a library's matrix product of 8192
// a side 1.17); the matrix cores are busy half of the time at the 1.9 GHz that the card's power leaves them, and LDS a quarter of it,
// without conflicts.  A long axis is cut into parts where there are few tiles (the plan decides, by the batch's total of keys); the
// parts' results are joined by a second launch, in order.
//
// Keys of pages that the pool does not hold, and mostly keys past a sequence's end, read as zeros from a constant and get no weight.
// Keys of later rows of a chunk, and the other places of a last page, are in the cache; their weight is zero, but zero times an infinity or NaN is
// not, so the tiles that some rows see in part look whether their V has such a value and then add key by key to the rows that see it.
#pragma once
#include <type_traits>

#include "smlm_common.hpp"
#include "wave_scan.hpp"

namespace smlm {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if (DT == SMLM_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Tile rows of a sequence up to which it takes the few-row path: one operand's.  (Two operands, 32 rows, with the join: 64 chunks of eight
// rows, four heads a kv head, over up to 4000 tokens 133 us, on the other path 119, 16 over 2000 43 and 31, four over 30000 123 and 95; with
// heads of 64 73 and 76.)
constexpr int kAttnSmallRows = 16;
constexpr int kAttnBigRows = 128;    // tile rows of a workgroup of the other
constexpr int kAttnSlots = 512;      // workgroups on the card at a time: two a CU
// Workgroups over the card that tiles are cut for, at most: four turns of it even out sequences of uneven lengths, more cost more in
// joins.  (1024, 2048, 4096 for few rows, with the join: 256 single tokens over up to 4095 tokens 394, 386, 387 us, three over up to 131000 251,
// 259, 267, 64 chunks of four rows 118, 121, 137, eight prompts of 512 rows and 128 single tokens 282, 291, 317.)
constexpr int kAttnSmallItems = 2048, kAttnBigItems = 1024;
// Keys of a part, at least: two turns of the four waves.  (128, 256, 512: a token over 2000 tokens 6.7, 8.2, 10.8 us, four over 4000
// 19.3, 15.9, 15.6, 32 over up to 1500 with the join 34, 30, 28.)
constexpr int kAttnMinKeys = 256;
// Items with few rows for each of the others, in turns.  (None, 1, 2, 3, 4: eight prompts of 512 rows over up to 1500 tokens and 128 single tokens over
// up to 4000 282, 282, 260, 297, 272 us, sixteen of 1024 from nothing and 40 single tokens 294, 325, 287, 340, 291, four of 512 and 64 with a kv
// head a query head 240, 228, 229, 227, 227.  One and three are the bad ones, as if a CU got its second workgroup 32 items, its XCD's CUs, after the
// first: with turns of two or four items it is then of the same kind.)
constexpr int kAttnPer = 2;
// Parts of a few-row tile from which the threads of a join share them out.  (85 parts: 30 us one after the other, 7 so; 8 parts 5.8 and 5.0.)
constexpr int kAttnManyParts = 8;

struct AttnItem {   // a tile of a sequence and a part of its keys
  int row0, n, len, trow;  // the sequence: first row, rows, tokens, row of the page table
  int first;               // first tile row
  int kb, ke;              // keys
  int part;                // where its part of the result goes, or -1: it is the whole
};
struct AttnJoin {   // rows of a tile whose keys were cut
  int row0, first;         // the sequence's first row, the tile's first row
  int big;                 // a tile of many rows
  int part, parts;         // its parts
  int from, step, rows;    // its rows from, from + step, ... below rows (eight at each, or one where the parts are many)
};
struct AttnPlanView {
  int* hdr;          // [16]: 0 items, 1 joins, what the plan is for: 2 tokens that a row of the table holds, 3 T, 4 S, 5 g, 6 kv heads, 7 R
  int* start;        // [4][S + 1] running sums by sequence: items with few rows, other items, joins, parts
  AttnItem* items;
  AttnJoin* joins;
};

inline int attn_tiles_max(int T, int S, int g) { return (int)((int64_t)T * g / kAttnBigRows) + S; }
inline int attn_items_max(int T, int S, int g, int Hkv) { return attn_tiles_max(T, S, g) + (kAttnSmallItems + kAttnBigItems) / Hkv + 2; }
// (a tile's rows are joined by at most rows / 8 workgroups, or by eight where its parts are eight and more)
inline int attn_joins_max(int T, int S, int g, int Hkv) {
  const int64_t cut = (4 * kAttnSmallItems + 16 * kAttnBigItems) / Hkv + 16, tiles = (int64_t)attn_tiles_max(T, S, g) * 16;
  return (int)(cut < tiles ? cut : tiles);
}
// (a tile of x times the cut's keys has round(x) parts, which is more than one from x = 1.5 on: at most 4 x / 3)
// Parts of few-row tiles and of others, for sequences of at most `most` tokens; no more than the tiles there can be have at kAttnMinKeys.
inline int attn_parts_max(int Hkv, int items, int64_t tiles, int most) {
  const int64_t cut = 4 * (int64_t)(items / Hkv + 1) / 3 + 1, all = most > kAttnMinKeys ? tiles * (most / kAttnMinKeys + 1) : 0;
  return (int)(cut < all ? cut : all);
}
inline int attn_parts_small(int S, int Hkv, int most) { return attn_parts_max(Hkv, kAttnSmallItems, S, most); }
inline int attn_parts_big(int T, int S, int g, int Hkv, int most) {
  const int64_t rows = (int64_t)T * g, seqs = rows / (kAttnSmallRows + 1);  // (sequences of more rows than a few)
  return attn_parts_max(Hkv, kAttnBigItems, rows / kAttnBigRows + (seqs < S ? seqs : S), most);
}
inline size_t attn_plan_carve(void* base, int T, int S, int g, int Hkv, AttnPlanView* pv) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return base ? reinterpret_cast<char*>(base) + o : nullptr;
  };
  AttnPlanView v;
  v.hdr = reinterpret_cast<int*>(take(64));
  v.start = reinterpret_cast<int*>(take((size_t)4 * (S + 1) * 4));
  v.items = reinterpret_cast<AttnItem*>(take((size_t)attn_items_max(T, S, g, Hkv) * sizeof(AttnItem)));
  v.joins = reinterpret_cast<AttnJoin*>(take((size_t)attn_joins_max(T, S, g, Hkv) * sizeof(AttnJoin)));
  if (pv) *pv = v;
  return off;
}

// ---- the plan ---------------------------------------------------------------------------------------------
struct AttnPlanArgs {
  AttnPlanView plan;
  const int *q_indptr, *kv_len, *requests;  // [S + 1], [S], [S] rows of the page table (null: s)
  int T, S, g, Hkv, R;
  int most;                                 // tokens that a row of the table holds
  int items_max, joins_max, parts_small_max, parts_big_max;
};

struct AttnSeq {
  int row0, n, len, trow, tile, tiles;
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnPlanArgs& a, int s) {
  AttnSeq q;
  const int r0 = a.q_indptr[s], r1 = a.q_indptr[s + 1];
  q.row0 = r0 < 0 ? 0 : (r0 > a.T ? a.T : r0);
  const int e = r1 > a.T ? a.T : r1;
  q.n = e > q.row0 ? e - q.row0 : 0;
  q.trow = a.requests ? a.requests[s] : s;
  q.len = a.kv_len[s];
  if (q.trow < 0 || q.trow >= a.R || q.len < 0) q.trow = 0, q.len = 0;
  if (q.len > a.most) q.len = a.most;
  const int rows = q.n * a.g;
  q.tile = rows <= kAttnSmallRows ? kAttnSmallRows : kAttnBigRows;
  q.tiles = (rows + q.tile - 1) / q.tile;
  return q;
}

constexpr int kAttnPlanThreads = 1024;

// workgroups that share the join of one of a sequence's tiles
__device__ __forceinline__ int attn_shares(const AttnSeq& q, int parts, int g) {
  const int rows = min(q.tile, q.n * g);
  return q.tile == kAttnSmallRows && parts >= kAttnManyParts ? min(8, rows) : (rows + 7) / 8;
}

constexpr int kAttnPlanLds = kAttnPlanThreads;  // up to here the sequences stay in LDS: every read of memory is most of a microsecond

// The number of parts that a tile of the card's average length is cut into, for n tiles (times kv heads): as many as leave the
// card's places for workgroups fullest, if that is worth the parts' traffic.  (Cutting 512 tiles, which just fill the card, in two:
// 2048 rows over 14336 tokens 502 -> 509 us and 17 for the join.  Up to 16, 32 and 64 parts: eight tiles over 100000 tokens 132, 89, 92 with the join.)
__device__ __forceinline__ int attn_parts(int n) {
  if (n >= kAttnBigItems) return 1;
  constexpr int kParts[9] = {1, 2, 3, 4, 6, 8, 12, 16, 32};
  int best = 1;
  float cost = 1e30f;
#pragma unroll
  for (int i = 0; i < 9; ++i) {
    const float c = (float)((n * kParts[i] + kAttnSlots - 1) / kAttnSlots) * (i ? 1.1f / (float)kParts[i] : 1.0f);
    if (c < cost * 0.97f) cost = c, best = kParts[i];
  }
  return best;
}

// One workgroup.  The sequences' tiles are cut into parts of about `cut` keys, by the sequences' lengths; the cuts follow from the batch's
// totals, so that the numbers of items and parts have bounds that the host knows, as long as no two sequences share a row: the plan of
// a q_indptr that decreases holds nothing, and a call with it does nothing.
__global__ __launch_bounds__(kAttnPlanThreads) void attn_plan_kernel(AttnPlanArgs a) {
  __shared__ int wave_tot[16][5];
  __shared__ float red[3][16];
  __shared__ int first_s[2][kAttnPlanLds + 1], join_s[kAttnPlanLds], part_s[kAttnPlanLds];
  __shared__ AttnSeq seq_s[kAttnPlanLds];
  __shared__ int bin_s[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, threads = (int)blockDim.x, waves = threads >> 6;
  const bool local = a.S <= kAttnPlanLds;
  float keys[2] = {0.0f, 0.0f};  // of the few-row tiles, of the others (only the cuts hang on them: a float will do)
  float n_big_f = 0.0f;          // tiles of the others; infinite where q_indptr decreases
  for (int s = tid; s < a.S; s += threads) {
    const AttnSeq q = attn_seq(a, s);
    const bool small = q.tile == kAttnSmallRows;
    keys[0] += small ? (float)q.tiles * (float)q.len : 0.0f;
    keys[1] += small ? 0.0f : (float)q.tiles * (float)q.len;
    n_big_f += a.q_indptr[s + 1] < a.q_indptr[s] ? INFINITY : (small ? 0.0f : (float)q.tiles);
    if (local) seq_s[s] = q;
  }
  keys[0] = wave_total(keys[0]), keys[1] = wave_total(keys[1]), n_big_f = wave_total(n_big_f);
  if (lane == 0) red[0][wave] = keys[0], red[1][wave] = keys[1], red[2][wave] = n_big_f;
  __syncthreads();
  keys[0] = keys[1] = n_big_f = 0.0f;
  for (int w = 0; w < waves; ++w) keys[0] += red[0][w], keys[1] += red[1][w], n_big_f += red[2][w];
  const int n_big = (int)fminf(n_big_f, 1.0e9f);
  // keys of a part: total / items, and a little more than the rounding of a float may take
  auto cut_of = [&](float total, int items) {
    const float c = total * (float)a.Hkv / (float)(items > 0 ? items : 1) * 1.0001f + 1.0f;
    return (int)fminf(fmaxf(c, (float)kAttnMinKeys), 1.0e9f);
  };
  const int heads_big = n_big < kAttnBigItems ? n_big * a.Hkv : kAttnBigItems;  // (no more is asked of it)
  const int want = heads_big < kAttnBigItems ? heads_big * attn_parts(heads_big) : kAttnBigItems;
  const int cut_small = cut_of(keys[0], kAttnSmallItems), cut_big = cut_of(keys[1], want < kAttnBigItems ? want : kAttnBigItems);
  int at[5] = {0, 0, 0, 0, 0};  // items with few rows, other items, joins, parts of the ones, of the others
  int* start = a.plan.start;
  for (int base = 0; base < a.S; base += threads) {
    const int s = base + tid;
    int n[5] = {0, 0, 0, 0, 0}, v[5];
    bool small = true;
    if (s < a.S) {
      const AttnSeq q = local ? seq_s[s] : attn_seq(a, s);
      small = q.tile == kAttnSmallRows;
      const uint32_t cut = (uint32_t)(small ? cut_small : cut_big), ns = max(1u, ((uint32_t)q.len + cut / 2) / cut);
      const int items = q.tiles * (int)ns, parts = ns > 1 ? items : 0;
      n[0] = small ? items : 0, n[1] = small ? 0 : items;
      n[2] = ns > 1 ? q.tiles * attn_shares(q, (int)ns, a.g) : 0;
      n[3] = small ? parts : 0, n[4] = small ? 0 : parts;
    }
    __syncthreads();  // the last turn's sums have been read
#pragma unroll
    for (int i = 0; i < 5; ++i) {
      v[i] = wave_scan(n[i]);
      if (lane == 63) wave_tot[wave][i] = v[i];
    }
    __syncthreads();
    int all[5] = {0, 0, 0, 0, 0};
    for (int w = 0; w < waves; ++w) {
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const int t = wave_tot[w][i];
        if (w < wave) v[i] += t;
        all[i] += t;
      }
    }
    if (s < a.S) {
      const int join = at[2] + v[2] - n[2], part = small ? at[3] + v[3] - n[3] : at[4] + v[4] - n[4];
      if (local) {
        first_s[0][s + 1] = at[0] + v[0], first_s[1][s + 1] = at[1] + v[1];
        join_s[s] = join, part_s[s] = part;
      } else {
        start[s + 1] = at[0] + v[0], start[(a.S + 1) + s + 1] = at[1] + v[1];
        start[2 * (a.S + 1) + s] = join, start[3 * (a.S + 1) + s] = part;
      }
    }
#pragma unroll
    for (int i = 0; i < 5; ++i) at[i] += all[i];
  }
  const bool fits = n_big_f != INFINITY && at[0] + at[1] <= a.items_max && at[2] <= a.joins_max && at[3] <= a.parts_small_max &&
                    at[4] <= a.parts_big_max;
  const int items = fits ? at[0] + at[1] : 0;
  if (tid == 0) {
    first_s[0][0] = first_s[1][0] = start[0] = start[a.S + 1] = 0;
    a.plan.hdr[0] = items;
    a.plan.hdr[1] = fits ? at[2] : 0;
    a.plan.hdr[2] = a.most, a.plan.hdr[3] = a.T, a.plan.hdr[4] = a.S, a.plan.hdr[5] = a.g, a.plan.hdr[6] = a.Hkv, a.plan.hdr[7] = a.R;
  }
  if (!fits) return;
  __syncthreads();
  // Items with few rows stream, the others compute: they take turns, one of the others and kAttnPer of these, so that both have the card
  // together.
  const int both = min(at[0] / kAttnPer, at[1]), mixed = (1 + kAttnPer) * both;
  struct Place {
    AttnItem it;
    AttnSeq q;
    int kind, x;              // 1: the others; its number among its kind's
    int lo, t, j, ns, part0;  // sequence, tile, part, parts of the tile, the first of them
  };
  auto place = [&](int i) {
    const int turn = i / (1 + kAttnPer), in = i - turn * (1 + kAttnPer);
    const int kind = i < mixed ? in == 0 : i - mixed < at[1] - both;
    const int x = i < mixed ? (kind ? turn : turn * kAttnPer + in - 1) : (kind ? i - both * kAttnPer : i - at[1]);
    const int* first_l = first_s[kind];
    const int* first_g = start + kind * (a.S + 1);
    int lo = 0, hi = a.S;
    while (hi - lo > 1) {  // last s with first[s] <= x
      const int mid = (lo + hi) >> 1;
      if ((local ? first_l[mid] : first_g[mid]) <= x) lo = mid;
      else hi = mid;
    }
    const AttnSeq q = local ? seq_s[lo] : attn_seq(a, lo);
    const int first = local ? first_l[lo] : first_g[lo], end = local ? first_l[lo + 1] : first_g[lo + 1];
    const int part = local ? part_s[lo] : start[3 * (a.S + 1) + lo];
    const uint32_t ns = (uint32_t)(end - first) / (uint32_t)q.tiles, k = (uint32_t)(x - first);
    const int t = q.tiles - 1 - (int)(k / ns), j = (int)(k % ns);  // (the later tiles of a prompt see more keys: they go first)
    AttnItem it;
    it.row0 = q.row0, it.n = q.n, it.len = q.len, it.trow = q.trow, it.first = t * q.tile;
    const int last = min(it.first + q.tile, q.n * a.g) - 1;
    const int seen = max(0, min(q.len, q.len - q.n + last / a.g + 1));  // keys that the tile's last row sees
    const int64_t step = (int64_t)((seen + ns - 1) / ns + 63) / 64 * 64;
    it.kb = (int)min((int64_t)seen, j * step);
    it.ke = (int)min((int64_t)seen, (j + 1) * step);
    const int part0 = part + t * (int)ns;
    it.part = ns > 1 ? part0 + j : -1;
    return Place{it, q, kind, x, lo, t, j, (int)ns, part0};
  };
  // Where the others are most of the items, and more than the card takes at a time, the long ones go first, over all sequences (by
  // eighths of an octave): a long one that starts among the last keeps the rest of the card waiting.  Sequence by sequence and so: nine
  // prompts of 700 rows over up to 3000 tokens 242 and 227 us, 64 of 16 rows over up to 4000 151 and 123, four of 512 over up to 1500 57 and 50;
  // beside as many items with few rows it gains nothing (eight prompts of 512 rows, 128 single tokens 260 and 266).
  const bool sorted = at[1] > kAttnSlots / a.Hkv && at[1] > at[0];
  auto bin_of = [](const AttnItem& it) { return 255 - (int)((__float_as_uint((float)(it.ke - it.kb) + 1.0f) >> 20) - (127u << 3)); };
  if (sorted) {
    for (int b = tid; b < 256; b += threads) bin_s[b] = 0;
    __syncthreads();
    for (int i = tid; i < items; i += threads) {
      const Place p = place(i);
      if (p.kind) atomicAdd(&bin_s[bin_of(p.it)], 1);
    }
    __syncthreads();
    const int n = tid < 256 ? bin_s[tid] : 0;
    int before = wave_scan(n) - n;
    if (lane == 63 && wave < 4) wave_tot[wave][0] = before + n;
    __syncthreads();
    for (int w = 0; w < 4; ++w) before += w < wave ? wave_tot[w][0] : 0;
    if (tid < 256) bin_s[tid] = before;
    __syncthreads();
  }
  for (int i = tid; i < items; i += threads) {
    const Place p = place(i);
    const int x = sorted && p.kind ? atomicAdd(&bin_s[bin_of(p.it)], 1) : p.x;
    a.plan.items[!p.kind ? i : (x < both ? x * (1 + kAttnPer) : x + both * kAttnPer)] = p.it;
    if (p.ns > 1) {
      const int join = local ? join_s[p.lo] : start[2 * (a.S + 1) + p.lo];
      const int shares = attn_shares(p.q, p.ns, a.g), by = p.kind || p.ns < kAttnManyParts ? 8 : 1;
      const int rows = min(p.q.tile, p.q.n * a.g - p.it.first);
      for (int h = p.j; h < shares; h += p.ns)
        a.plan.joins[join + p.t * shares + h] = AttnJoin{p.q.row0, p.it.first, p.kind, p.part0, p.ns, h * by, shares * by, rows};
    }
  }
}

// ---- attention --------------------------------------------------------------------------------------------
struct AttnArgs {
  uint16_t* out;
  const uint16_t *q, *k, *v;
  const int* table;          // [R, M]
  AttnPlanView plan;
  float *po_small, *po_big;  // parts of the results, [part][kv head][tile row][D], not divided by their sums
  float *pm_small, *pm_big;  // [part][kv head][tile row][2]: maximum (of the scores times scale / log 2), sum
  int64_t o_row, o_head, q_row, q_head, c_page, c_head, c_slot;
  int M, n_pages, P, T, S, R, Hkv, g;
  int most;                  // M * P
  uint32_t div_mul;          // division by P: ((x * div_mul >> 32) + x) >> div_shift in 33 bits
  int div_shift;
  int whole;                 // keys from a multiple of it on, as many, that lie in one page: 16, the rows of a load, or 0
  float scale;               // times log2 e
};

typedef int i32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8 uload8(const void* p) { return *(const SMLM_CONST i32x8*)p; }
// A plan for other sizes names rows, or parts of the results, that may not be there: the call does nothing.  (h: the header's start)
__device__ __forceinline__ bool attn_fits(const AttnArgs& a, i32x8 h) {
  return ((h[2] ^ a.most) | (h[3] ^ a.T) | (h[4] ^ a.S) | (h[5] ^ a.g) | (h[6] ^ a.Hkv) | (h[7] ^ a.R)) == 0;
}

static __device__ __align__(16) const uint32_t attn_zeros[4] = {0u, 0u, 0u, 0u};

__device__ __forceinline__ int attn_div(uint32_t x, uint32_t mul, int shift) {
  return (int)(((uint64_t)__umulhi(x, mul) + x) >> shift);
}

// Element offset of a key within the pool (its kv head apart), -1 where there is none.  ke > 0.
// In two steps, the page's number a tile ahead of its use: the read is on its way meanwhile.
struct AttnKey {
  int page, slot;
};
__device__ __forceinline__ AttnKey attn_key(const AttnArgs& a, const int* trow, int key, int ke) {
  const int k = min(key, ke - 1);  // (no branch around the read)
  const int j = attn_div((uint32_t)k, a.div_mul, a.div_shift);
  return AttnKey{trow[j], key < ke ? k - j * a.P : -1};
}
__device__ __forceinline__ int64_t attn_offset(const AttnArgs& a, AttnKey k) {
  const int64_t off = (int64_t)k.page * a.c_page + (int64_t)k.slot * a.c_slot;
  return k.slot >= 0 && (uint32_t)k.page < (uint32_t)a.n_pages ? off : -1;
}
__device__ __forceinline__ int64_t attn_shfl(int64_t v, int lane) {
  const int lo = __shfl((int)(uint32_t)v, lane, kWaveSize), hi = __shfl((int)(v >> 32), lane, kWaveSize);
  return ((int64_t)hi << 32) | (uint32_t)lo;
}
__device__ __forceinline__ u32x4 attn_ld(const uint16_t* base, int64_t off, int d) {
  return ldg16(off >= 0 ? base + off + d : reinterpret_cast<const uint16_t*>(attn_zeros));
}

// A row of K or V in LDS: pieces of 16 bytes, the piece's place turned by the row.  The lanes of a matrix operand read one
// piece of sixteen rows of K: the low bits of the row turn it, and they meet all banks.  Of V, sixteen lanes of the transposing load read a
// pair of pieces of four rows, and the next sixteen the pair beside it (or the next four rows): the turn is by pairs, two apart from
// row to row.  (V turned as K is: half of LDS's cycles were conflicts.)
template <int D>
__device__ __forceinline__ int attn_place(int row, int piece) {
  return row * D + ((D == 128 ? piece ^ (row & 15) : piece ^ ((row >> 1) & 7)) << 3);
}
template <int D>
__device__ __forceinline__ int attn_place_v(int row, int piece) {
  const int pairs = D == 128 ? ((row & 3) << 1) | ((row >> 2) & 1) : (row & 2) | ((row >> 2) & 1);
  return row * D + ((piece ^ (pairs << 1)) << 3);
}

// whether an element of a pair of 16-bit values is an infinity or NaN
template <int DT>
__device__ __forceinline__ uint32_t attn_not_finite(uint32_t x) {
  return DT == SMLM_DTYPE_F16 ? ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u : ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}

// Where a lane points the transposing load for keys row .. row + 3 of its sixteen lanes and dimensions d0 .. d0 + 15: it gets
// dimension d0 + (lane & 15) of the four keys.  (Sixteen rows on, the place is the same sixteen rows on: the operands of a tile take
// few different ones, kept in registers, and constants for the rest.)
template <int D>
__device__ __forceinline__ int attn_v_place(int row, int d0) {
  const int l = threadIdx.x & 15, r = row + (l >> 2), d = d0 + (l & 3) * 4;
  return attn_place_v<D>(r, d >> 3) + (d & 7);
}
__device__ __forceinline__ u32x4 attn_v_pair(const uint16_t* a, const uint16_t* b) {
  const u32x2 x = lds_read_tr16(a), y = lds_read_tr16(b);
  return u32x4{x[0], x[1], y[0], y[1]};
}

// The weights, and so their sums and the accumulators, are held 2^bias times as large: fp16 has no normal number under 2^-14, and
// a long context's many small weights may add up to more than its few large ones.
template <int DT>
constexpr float kAttnBias = DT == SMLM_DTYPE_F16 ? 7.0f : 0.0f;

// l + the two halves of x
template <int DT>
__device__ __forceinline__ float attn_add2(uint32_t x, float l) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  if (DT == SMLM_DTYPE_F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, x), h2{(_Float16)1.0f, (_Float16)1.0f}, l, false);
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, x), b2{(__bf16)1.0f, (__bf16)1.0f}, l, false);
}

template <int DT>
__device__ __forceinline__ u32x2 attn_pack4(float a, float b, float c, float d) {
  u32x2 o;
  o[0] = pack2<DT>(a, b);
  o[1] = pack2<DT>(c, d);
  return o;
}
__device__ __forceinline__ uint16_t* attn_out_row(const AttnArgs& a, const AttnItem& it, int kvh, int p) {
  return a.out + (int64_t)(it.row0 + p / a.g) * a.o_row + (int64_t)(kvh * a.g + p % a.g) * a.o_head;
}

// the larger of a lane's and its partner's, 16 or 32 lanes on, without a trip through LDS
__device__ __forceinline__ float attn_max16(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto both = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float attn_max32(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// (the hardware's own: results under the smallest normal float are zero)
__device__ __forceinline__ float attn_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Up to 16 tile rows.  Layouts of a 16 x 16 x 32 product by lane (c = lane & 15, b = lane >> 4): operands row or column c,
// k = 8 b + 0..7; result column c, rows 4 b + 0..3.
template <int DT, int D>
__device__ __forceinline__ void attn_small(const AttnArgs& a, const AttnItem& it, int kvh, uint16_t* lds, float* ml) {
  constexpr int kSteps = D / 32, kBlk = D / 16, kVLoads = D / 16;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, b = lane >> 4;
  const int rows = it.n * a.g;
  const int* trow = a.table + (int64_t)it.trow * a.M;
  const uint16_t *kp = a.k + (int64_t)kvh * a.c_head, *vp = a.v + (int64_t)kvh * a.c_head;
  uint16_t* vl = lds + wave * 32 * D;
  const u32x4 zero4 = {0u, 0u, 0u, 0u};

  const int p = it.first + c, pc = p < rows ? p : 0;
  const int lim = min(it.ke - 1, it.len - it.n + pc / a.g);
  u32x4 q[kSteps];
  {
    const uint16_t* src = a.q + (int64_t)(it.row0 + pc / a.g) * a.q_row + (int64_t)(kvh * a.g + pc % a.g) * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const u32x4 x = ldg16(src + s * 32 + b * 8);
      q[s] = p < rows ? x : zero4;
    }
  }
  const int lim0 = it.len - it.n + it.first / a.g;  // the first row's: a tile up to it is seen whole by all

  f32x4 o[kBlk];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < kBlk; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 kr[2][kSteps], vr[kVLoads];
  constexpr int kRowLanes = D / 8, kRowsLoad = 64 / kRowLanes;  // lanes a row of V, rows a load
  int vat[kBlk];
#pragma unroll
  for (int i = 0; i < kBlk; ++i) vat[i] = attn_v_place<D>(b * 4, i * 16);
  auto load = [&](int64_t off) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t f = attn_shfl(off, u * 16 + c);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) kr[u][s] = attn_ld(kp, f, s * 32 + b * 8);
    }
#pragma unroll
    for (int i = 0; i < kVLoads; ++i)
      vr[i] = attn_ld(vp, attn_shfl(off, i * kRowsLoad + lane / kRowLanes), (lane % kRowLanes) * 8);
  };
  int64_t off = -1;
  AttnKey next{0, -1};
  if (it.kb < it.ke) {
    off = attn_offset(a, attn_key(a, trow, it.kb + wave * 32 + (lane & 31), it.ke));
    next = attn_key(a, trow, it.kb + wave * 32 + 128 + (lane & 31), it.ke);
    load(off);
  }
  for (int base = it.kb + wave * 32; base < it.ke; base += 128) {
    const uint32_t ok = (uint32_t)__ballot(off >= 0);
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kSteps; ++k) s[u] = Num<DT>::mfma(kr[u][k], q[k], s[u]);
    }
    const bool edge = base + 31 > lim0;
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < kVLoads; ++i) {
      const int r = i * kRowsLoad + lane / kRowLanes;
      *(u32x4*)(vl + attn_place_v<D>(r, lane % kRowLanes)) = vr[i];
      if (edge) odd |= attn_not_finite<DT>(vr[i][0]) | attn_not_finite<DT>(vr[i][1]) | attn_not_finite<DT>(vr[i][2]) | attn_not_finite<DT>(vr[i][3]);
    }
    off = attn_offset(a, next);
    next = attn_key(a, trow, base + 256 + (lane & 31), it.ke);
    load(off);

    const bool guard = edge && __ballot(odd != 0) != 0;
    if (edge || ok != 0xffffffffu) {
      const uint32_t there = ok >> (b * 4);
      const int seen = lim - base - b * 4;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = u * 16 + i;  // (and 4 b more)
          if (!(there >> key & 1) || key > seen) s[u][i] = -INFINITY;
        }
    }
    const float mx = attn_max32(attn_max16(fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                                 fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])))));
    const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.0f : mn * a.scale, ms = ref - kAttnBias<DT>;
    const float turn = attn_exp2(m * a.scale - ref);
    m = mn;
    float sum = 0.0f;
    u32x4 pf;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4& x = s[i >> 1];
      pf[i] = pack2<DT>(attn_exp2(x[2 * i & 3] * a.scale - ms), attn_exp2(x[(2 * i & 3) + 1] * a.scale - ms));
      sum = attn_add2<DT>(pf[i], sum);  // (the weights as V meets them: they add up to one whatever their rounding)
    }
    l = l * turn + sum;
#pragma unroll
    for (int i = 0; i < kBlk; ++i) o[i] *= turn;
    if (!guard) {
#pragma unroll
      for (int i = 0; i < kBlk; ++i) {
        const u32x4 vf = attn_v_pair(vl + vat[i], vl + vat[i] + 16 * D);
        o[i] = Num<DT>::mfma(vf, pf, o[i]);
      }
    } else {  // key by key: slot j of lane group bb
#pragma unroll 1
      for (int x = 0; x < 32; ++x) {
        const int bb = x >> 3, j = x & 7, key = (j >> 2) * 16 + bb * 4 + (j & 3);
        asm volatile("" ::: "memory");  // (V is read again for each key: kept in registers it would cost the usual path)
        u32x4 only;
#pragma unroll
        for (int e = 0; e < 4; ++e) only[e] = b == bb && (j >> 1) == e ? (j & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
#pragma unroll
        for (int i = 0; i < kBlk; ++i) {
          const u32x4 vf = attn_v_pair(vl + vat[i], vl + vat[i] + 16 * D) & only;
          const f32x4 add = Num<DT>::mfma(vf, pf & only, f32x4{0.f, 0.f, 0.f, 0.f});
          if (base + key <= lim) o[i] += add;
        }
      }
    }
    __builtin_amdgcn_wave_barrier();  // (this wave's LDS reads come before its next writes)
  }

  // the four waves' results
  float* ol = reinterpret_cast<float*>(lds);  // [4][16][D]
  l += __shfl_xor(l, 16, kWaveSize);
  l += __shfl_xor(l, 32, kWaveSize);
  __syncthreads();  // V has been read
  if (b == 0) ml[(wave * 16 + c) * 2] = m * a.scale, ml[(wave * 16 + c) * 2 + 1] = l;
#pragma unroll
  for (int i = 0; i < kBlk; ++i) *(f32x4*)(ol + (wave * 16 + c) * D + ((i * 4 + b) ^ (c & 7)) * 4) = o[i];
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * (D / 4); x += 256) {
    const int r = x / (D / 4), d4 = x % (D / 4), row = it.first + r;
    if (row >= rows) continue;
    float mw[4], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mw[w] = ml[(w * 16 + r) * 2], top = fmaxf(top, mw[w]);
    const float ref = top == -INFINITY ? 0.0f : top;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = attn_exp2(mw[w] - ref);
      sum += f * ml[(w * 16 + r) * 2 + 1];
      const f32x4 v = *(const f32x4*)(ol + (w * 16 + r) * D + (d4 ^ (r & 7)) * 4);
      acc += f * v;
    }
    if (it.part >= 0) {
      const int64_t at = ((int64_t)it.part * a.Hkv + kvh) * kAttnSmallRows + r;
      *(SMLM_GLOBAL f32x4*)(a.po_small + at * D + d4 * 4) = acc;
      if (d4 == 0) a.pm_small[at * 2] = top, a.pm_small[at * 2 + 1] = sum;
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      *(SMLM_GLOBAL u32x2*)(attn_out_row(a, it, kvh, row) + d4 * 4) =
          attn_pack4<DT>(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    }
  }
}

// 128 tile rows, 32 a wave.  Layouts of a 32 x 32 x 16 product by lane (c = lane & 31, h = lane >> 5): operands row or
// column c, k = 8 h + 0..7; result column c, rows 8 (i / 4) + 4 h + i % 4, i = 0..15.
// K and V tiles go from memory to LDS without passing through registers, the next tile's while one is worked on; the turned places are made
// by what each lane reads, as the hardware writes the lanes' pieces one after the other.
template <int DT, int D>
__device__ __forceinline__ void attn_big(const AttnArgs& a, const AttnItem& it, int kvh, uint16_t* tile0, uint16_t* tile1,
                                         uint32_t* flags) {
  constexpr int kSteps = D / 16, kBlk = D / 32, kKeys = 64;
  constexpr int kRowLanes = D / 8, kRowsLoad = 64 / kRowLanes, kLoads = 16 / kRowsLoad;  // a wave loads 16 rows of K and of V
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  const int rows = it.n * a.g;
  const int* trow = a.table + (int64_t)it.trow * a.M;
  const uint16_t *kp = a.k + (int64_t)kvh * a.c_head, *vp = a.v + (int64_t)kvh * a.c_head;
  const u32x4 zero4 = {0u, 0u, 0u, 0u};

  const bool busy = it.first + wave * 32 < rows;  // (a wave without rows loads for the others)
  const int p = it.first + wave * 32 + c, pc = p < rows ? p : 0;
  const int lim = min(it.ke - 1, it.len - it.n + pc / a.g);
  const int lim0 = it.len - it.n + it.first / a.g;  // of the workgroup's first row
  u32x4 q[kSteps];
  {
    const uint16_t* src = a.q + (int64_t)(it.row0 + pc / a.g) * a.q_row + (int64_t)(kvh * a.g + pc % a.g) * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const u32x4 x = ldg16(src + s * 16 + h * 8);
      q[s] = p < rows ? x : zero4;
    }
  }
  f32x16 o[kBlk];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < kBlk; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;

  int kat[kSteps], vat[kBlk];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) kat[k] = attn_place<D>(c, k * 2 + h);
#pragma unroll
  for (int i = 0; i < kBlk; ++i) vat[i] = attn_v_place<D>(h * 4, i * 32 + ((lane >> 4) & 1) * 16);  // (8 rows on: the same turn)

  // What a lane reads: the turn undoes itself, so the piece that is turned into the lane's place.  Rows of a load are kRowsLoad
  // apart from the next's, so their turns differ by constants.
  constexpr int kTurnsK = kLoads, kTurnsV = kLoads < 2 ? kLoads : 2;
  uint32_t kof[kTurnsK], vof[kTurnsV];  // bytes from the load's first row
  const uint32_t slot_bytes = a.whole ? (uint32_t)a.c_slot * 2u : 0u;
#pragma unroll
  for (int i = 0; i < kTurnsK; ++i) {
    const int r = i * kRowsLoad + lane / kRowLanes;
    kof[i] = (uint32_t)(lane / kRowLanes) * slot_bytes + (uint32_t)(attn_place<D>(r, lane % kRowLanes) - r * D) * 2u;
    if (i < kTurnsV) vof[i] = (uint32_t)(lane / kRowLanes) * slot_bytes + (uint32_t)(attn_place_v<D>(r, lane % kRowLanes) - r * D) * 2u;
  }
  typedef SMLM_GLOBAL const char* gptr;
  auto to_lds = [&](gptr from, uint16_t* to) {
    __builtin_amdgcn_global_load_lds((SMLM_GLOBAL void*)from, (__attribute__((address_space(3))) void*)to, 16, 0, 0);
  };
  // Rows of one page: an address for all lanes, made on the scalar side, and an offset that stays.  (Through a buffer resource: a load
  // to LDS with a lane's own address counts as an access to LDS too, and every wait for an operand then waits for all that are on their way.)
  auto page_to_lds = [&](const uint16_t* rows, uint32_t lane_bytes, uint32_t bytes, uint16_t* to) {
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(rows), 0, 0xffffffffu, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)to, 16, lane_bytes, bytes, 0, 0);
  };
  auto load_page = [&](int64_t first, uint16_t* tile) {
    uint16_t* dst = tile + wave * 16 * D;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      asm volatile("" : "+v"(kof[i]), "+v"(vof[i % kTurnsV]));  // (kept as 32 bits over the loop)
      page_to_lds(kp + first, kof[i], (uint32_t)(i * kRowsLoad) * slot_bytes, dst + i * kRowsLoad * D);
      page_to_lds(vp + first, vof[i % kTurnsV], (uint32_t)(i * kRowsLoad) * slot_bytes, dst + i * kRowsLoad * D + kKeys * D);
    }
  };
  auto load = [&](int64_t off, uint16_t* tile) {
    uint16_t* dst = tile + wave * 16 * D;
    int ln = lane;
    asm volatile("" : "+v"(ln));  // (nothing of this is kept over the loop)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = i * kRowsLoad + ln / kRowLanes;
      const int64_t f = attn_shfl(off, r);
      const int dk = attn_place<D>(r, ln % kRowLanes) - r * D, dv = attn_place_v<D>(r, ln % kRowLanes) - r * D;
      const uint16_t* zero = reinterpret_cast<const uint16_t*>(attn_zeros);
      to_lds((gptr)(f >= 0 ? kp + f + dk : zero), dst + i * kRowsLoad * D);
      to_lds((gptr)(f >= 0 ? vp + f + dv : zero), dst + i * kRowsLoad * D + kKeys * D);
    }
  };
  auto work = [&](auto may_edge, int base, const uint16_t* kl, const uint32_t* fl, auto between) {
    const uint16_t* vl = kl + kKeys * D;
    const bool edge = may_edge && base + kKeys - 1 > lim0;
    const uint64_t ok = (uint64_t)((fl[0] & 0xffffu) | (fl[1] << 16)) | ((uint64_t)((fl[2] & 0xffffu) | (fl[3] << 16)) << 32);
    f32x16 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[u][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const u32x4 kf = *(const u32x4*)(kl + kat[k] + u * 32 * D);
        s[u] = mfma32<DT>(kf, q[k], s[u]);
      }
    }
    // Six reads ahead of the products, and eight in the second: left to itself each product waits for the read before it.  (Both: 2 to 4
    // percent where the card's power is not the bound, 1 where it is.)
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
    for (int i = 0; i < 2 * kSteps - 6; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, 6, 0);
    if (edge || ok != ~0ull) {
      const uint64_t there = ok >> (4 * h);
      const int seen = lim - base - 4 * h;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = u * 32 + 8 * (e >> 2) + (e & 3);  // (and 4 h more)
          if (!(there >> key & 1) || key > seen) s[u][e] = -INFINITY;
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[u][e]);
    mx = attn_max32(mx);
    between();
    // The reference that the exponents are taken against follows the running maximum only once that is 2^8 past it: the
    // probabilities stay below 2^8 (2^15 with the bias), inside the element types, and most tiles leave the accumulators alone.
    if (__ballot((mx - m) * a.scale > 8.0f)) {
      const float mn = fmaxf(m, mx), turn = attn_exp2((mn == -INFINITY ? 0.0f : m - mn) * a.scale);
      l *= turn;
#pragma unroll
      for (int i = 0; i < kBlk; ++i) o[i] *= turn;
      m = mn;
    }
    const float ms = (m == -INFINITY ? 0.0f : m * a.scale) - kAttnBias<DT>;
    u32x4 pf[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const uint32_t two = pack2<DT>(attn_exp2(s[u][e] * a.scale - ms), attn_exp2(s[u][e + 1] * a.scale - ms));
        l = attn_add2<DT>(two, l);  // (as V meets them, as above)
        pf[u][e >> 3][(e >> 1) & 3] = two;
      }
    const bool guard = edge && ((fl[0] | fl[1] | fl[2] | fl[3]) >> 16) != 0;
    if (!guard) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int i = 0; i < kBlk; ++i) {
            const uint16_t* at = vl + (u * 32 + ks * 16) * D;
            o[i] = mfma32<DT>(attn_v_pair(at + vat[i], at + vat[i] + 8 * D), pf[u][ks], o[i]);
          }
      __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
      for (int i = 0; i < 4 * kBlk - 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
    } else {
#pragma unroll 1
      for (int x = 0; x < kKeys; ++x) {  // slot j of half hh in step st of sixteen keys
        const int st = x >> 4, hh = (x >> 3) & 1, j = x & 7, key = st * 16 + (j >> 2) * 8 + hh * 4 + (j & 3);
        asm volatile("" ::: "memory");  // (V is read again for each key: kept in registers it would cost the usual path)
        u32x4 only, pj;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          only[e] = h == hh && (j >> 1) == e ? (j & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
          pj[e] = (st == 0 ? pf[0][0][e] : st == 1 ? pf[0][1][e] : st == 2 ? pf[1][0][e] : pf[1][1][e]) & only[e];
        }
#pragma unroll
        for (int i = 0; i < kBlk; ++i) {
          const uint16_t* at = vl + st * 16 * D;
          f32x16 add;
#pragma unroll
          for (int e = 0; e < 16; ++e) add[e] = 0.0f;
          add = mfma32<DT>(attn_v_pair(at + vat[i], at + vat[i] + 8 * D) & only, pj, add);
          if (base + key <= lim) o[i] += add;
        }
      }
    }
  };
  // A tile's loads are waited for by the wave that gave them, then by all; at that point everybody is done with the tile before,
  // whose place the next loads take.
  // A tile that some rows see in part: does V, of the keys that this wave loaded, hold a value that is no number?
  auto check = [&](int base, const uint16_t* mine) -> uint32_t {
    uint32_t odd = 0;
    if (base + kKeys - 1 > lim0) {
      const uint16_t* own = mine + (kKeys + wave * 16) * D + lane * 8;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const u32x4 v = *(const u32x4*)(own + i * kRowsLoad * D);
        odd |= attn_not_finite<DT>(v[0]) | attn_not_finite<DT>(v[1]) | attn_not_finite<DT>(v[2]) | attn_not_finite<DT>(v[3]);
      }
    }
    return __ballot(odd != 0) != 0 ? 0x10000u : 0u;
  };
  int base = it.kb;
  // Where the sixteen keys of a wave lie in one page, or those of a load, what is loaded, and whether a page is there, is known on the
  // scalar side.  Of sixteen keys that reach past the end the page's other places are loaded too, and masked as later rows' keys are.
  // Pairs of tiles that every row sees, and that are not the last, go apart, so that this loop keeps its registers to itself.
  auto pages = [&](auto sixteen) {  // (two loops: the test in one of them cost up to 5 percent)
    constexpr uint32_t kAll = 0xffffu, kOne = (1u << kRowsLoad) - 1u;
    int page[kLoads], slot[kLoads];
    auto find = [&](int key) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        if (i && sixteen) break;
        const int at = key + i * kRowsLoad, k = min(at, it.ke - 1), j = attn_div((uint32_t)k, a.div_mul, a.div_shift);
        const int pg = uload(trow, j);
        slot[i] = k - j * a.P;
        page[i] = at < it.ke ? pg : -1;
      }
    };
    auto fetch = [&](uint16_t* tile) -> uint32_t {  // the keys that are there
      const uint16_t* zero = reinterpret_cast<const uint16_t*>(attn_zeros);
      uint32_t keys = 0;
      if (sixteen) {
        const bool there = (uint32_t)page[0] < (uint32_t)a.n_pages;
        uint16_t* dst = tile + wave * 16 * D;
        if (there) {
          load_page((int64_t)page[0] * a.c_page + (int64_t)slot[0] * a.c_slot, tile);
        } else {
#pragma unroll
          for (int i = 0; i < kLoads; ++i) {
            page_to_lds(zero, 0, 0, dst + i * kRowsLoad * D);
            page_to_lds(zero, 0, 0, dst + i * kRowsLoad * D + kKeys * D);
          }
        }
        return there ? kAll : 0u;
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const bool there = (uint32_t)page[i] < (uint32_t)a.n_pages;
        const int64_t first = (int64_t)page[i] * a.c_page + (int64_t)slot[i] * a.c_slot;
        uint16_t* dst = tile + (wave * 16 + i * kRowsLoad) * D;
        page_to_lds(there ? kp + first : zero, there ? kof[i] : 0u, 0, dst);
        page_to_lds(there ? vp + first : zero, there ? vof[i % kTurnsV] : 0u, 0, dst + kKeys * D);
        keys |= there ? kOne << (i * kRowsLoad) : 0u;
      }
      return keys;
    };
    find(base + wave * 16);
    uint32_t valid = fetch(tile0);
    find(base + kKeys + wave * 16);
    auto turn = [&](auto may_edge, int base, uint16_t* mine, uint16_t* other, uint32_t* fl) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      const uint32_t any_odd = may_edge ? check(base, mine) : 0u;
      if (lane == 0) fl[wave] = valid | any_odd;
      __syncthreads();
      if (!may_edge || base + kKeys < it.ke) {
        valid = fetch(other);
        if (!busy) find(base + 2 * kKeys + wave * 16);
      }
      // (the pages' numbers are asked for where nothing is waited for in LDS: the counter is one)
      if (busy) work(may_edge, base, mine, fl, [&] { find(base + 2 * kKeys + wave * 16); });
    };
    for (; base + 2 * kKeys - 1 <= lim0 && base + 2 * kKeys < it.ke; base += 2 * kKeys) {
      turn(std::false_type{}, base, tile0, tile1, flags);
      turn(std::false_type{}, base + kKeys, tile1, tile0, flags + 4);
    }
    uint16_t *mine = tile0, *other = tile1;
    uint32_t* fl = flags;
#pragma unroll 1
    for (; base < it.ke; base += kKeys) {
      turn(std::true_type{}, base, mine, other, fl);
      uint16_t* const t = mine;
      mine = other, other = t, fl = flags + (4 - (fl - flags));
    }
  };
  if (base < it.ke) {
    if (a.whole == 16) {
      pages(std::true_type{});
    } else if (a.whole) {
      pages(std::false_type{});
    } else {
      load(attn_offset(a, attn_key(a, trow, base + wave * 16 + (lane & 15), it.ke)), tile0);
      int64_t off = attn_offset(a, attn_key(a, trow, base + wave * 16 + (lane & 15), it.ke));
      AttnKey next = attn_key(a, trow, base + kKeys + wave * 16 + (lane & 15), it.ke);
      auto turn = [&](int base, uint16_t* mine, uint16_t* other, uint32_t* fl) {
        const uint32_t valid = (uint32_t)__ballot(off >= 0) & 0xffffu;
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        const uint32_t any_odd = check(base, mine);
        if (lane == 0) fl[wave] = valid | any_odd;
        __syncthreads();
        off = attn_offset(a, next);
        next = attn_key(a, trow, base + 2 * kKeys + wave * 16 + (lane & 15), it.ke);
        if (base + kKeys < it.ke) load(off, other);
        if (busy) work(std::true_type{}, base, mine, fl, [] {});
      };
      uint16_t *mine = tile0, *other = tile1;
      uint32_t* fl = flags;
#pragma unroll 1
      for (; base < it.ke; base += kKeys) {
        turn(base, mine, other, fl);
        uint16_t* const t = mine;
        mine = other, other = t, fl = flags + (4 - (fl - flags));
      }
    }
  }
  l += __shfl_xor(l, 32, kWaveSize);
  if (p >= rows) return;  // (no barrier below)
  if (it.part >= 0) {
    const int64_t at = ((int64_t)it.part * a.Hkv + kvh) * kAttnBigRows + wave * 32 + c;
#pragma unroll
    for (int i = 0; i < kBlk; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(SMLM_GLOBAL f32x4*)(a.po_big + at * D + i * 32 + 2 * e + 4 * h) = f32x4{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
    if (h == 0) a.pm_big[at * 2] = m * a.scale, a.pm_big[at * 2 + 1] = l;
  } else {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t* dst = attn_out_row(a, it, kvh, p);
#pragma unroll
    for (int i = 0; i < kBlk; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *(SMLM_GLOBAL u32x2*)(dst + i * 32 + 2 * e + 4 * h) =
            attn_pack4<DT>(o[i][e] * inv, o[i][e + 1] * inv, o[i][e + 2] * inv, o[i][e + 3] * inv);
  }
}

// Neighbouring workgroups take the kv heads of one item: with eight of them, or a multiple, a head's tiles meet in one XCD's L2.
template <int DT, int D>
__global__ __launch_bounds__(256, 2) void attn_kernel(AttnArgs a) {
  __shared__ __align__(16) uint16_t lds[2 * 64 * D], more[2 * 64 * D];
  __shared__ uint32_t side[128];
  const int i = (int)blockIdx.x / a.Hkv, kvh = (int)blockIdx.x - i * a.Hkv;
  // (there is room for an item a workgroup: it is read beside the header, not after it)
  i32x8 hdr = uload8(a.plan.hdr), item = uload8(a.plan.items + i);
  asm volatile("" : "+s"(hdr), "+s"(item));
  if (i >= hdr[0] || !attn_fits(a, hdr)) return;
  const AttnItem it = __builtin_bit_cast(AttnItem, item);
  const int rows = it.n * a.g;
  if (rows <= 0) return;
  if (rows > kAttnSmallRows) attn_big<DT, D>(a, it, kvh, lds, more, side);
  else attn_small<DT, D>(a, it, kvh, lds, reinterpret_cast<float*>(side));
}

// The parts of a tile's rows, each weighed by its maximum against the largest.  A thread takes four dimensions of a row and, where the parts
// are many, every eighth of them; the eight are then added in order.
// Workgroups of the join: the host knows a bound of the joins only, and workgroups without work cost too.  (512, 2048, 8192: a mixed batch 13,
// 8.4, 9.3 us, 256 single tokens 5.2, 4.3, 4.4.)
constexpr int kAttnJoinBlocks = 2048;
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;  // threads a row; rows, or shares of the parts, at a time
  __shared__ f32x4 acc_s[kGroups][kLanes];
  __shared__ float sum_s[kGroups], top_s[kGroups];
  const i32x8 hdr = uload8(a.plan.hdr);
  if (!attn_fits(a, hdr)) return;
  const int work = hdr[1] * a.Hkv;
  for (int w = blockIdx.x; w < work; w += gridDim.x) {
    const int i = w / a.Hkv, kvh = w - i * a.Hkv;
    const AttnJoin jn = a.plan.joins[i];
    const int tile = jn.big ? kAttnBigRows : kAttnSmallRows;
    const float *po = jn.big ? a.po_big : a.po_small, *pm = jn.big ? a.pm_big : a.pm_small;
    AttnItem it;
    it.row0 = jn.row0;
    const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
    const int64_t step = (int64_t)a.Hkv * tile;
    const bool many = jn.parts >= kAttnManyParts && !jn.big;
    const int by = many ? kGroups : 1;
    for (int r0 = jn.from; r0 < jn.rows; r0 += jn.step) {
      const int row = many ? r0 : r0 + grp, r = min(row, jn.rows - 1);
      const int64_t at0 = ((int64_t)jn.part * a.Hkv + kvh) * tile + r;
      // running maximum over this thread's parts, four on their way at a time
      float top = -INFINITY, sum = 0.0f;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      for (int j = many ? grp : 0; j < jn.parts; j += 4 * by) {
        float m[4], l[4];
        f32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int64_t at = at0 + (int64_t)min(j + u * by, jn.parts - 1) * step;
          m[u] = j + u * by < jn.parts ? pm[at * 2] : -INFINITY;
          l[u] = pm[at * 2 + 1];
          v[u] = ldg_f4(po + at * D + lane * 4);
        }
        const float now = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top), ref = now == -INFINITY ? 0.0f : now;
        const float old = attn_exp2(top - ref);
        sum *= old;
        acc *= old;
        top = now;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (j + u * by >= jn.parts) continue;
          const float f = attn_exp2(m[u] - ref);
          sum += f * l[u];
          acc += f * v[u];
        }
      }
      if (many) {
        __syncthreads();  // the last row's have been read
        acc_s[grp][lane] = acc;
        if (lane == 0) sum_s[grp] = sum, top_s[grp] = top;
        __syncthreads();
        if (grp != 0) continue;
#pragma unroll
        for (int w = 1; w < kGroups; ++w) top = fmaxf(top, top_s[w]);
        const float ref = top == -INFINITY ? 0.0f : top;
        sum = 0.0f;
        acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kGroups; ++w) {
          const float f = attn_exp2(top_s[w] - ref);
          sum += f * sum_s[w];
          acc += f * acc_s[w][lane];
        }
      } else if (grp >= 8 || row >= jn.rows) {
        continue;
      }
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      *(SMLM_GLOBAL u32x2*)(attn_out_row(a, it, kvh, jn.first + r) + lane * 4) =
          attn_pack4<DT>(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    }
  }
}

}  // namespace smlm
