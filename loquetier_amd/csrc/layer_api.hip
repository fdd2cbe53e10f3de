// C ABI of the operators between a decoder layer's projections (see include/smlm.h): rotation of queries and keys with their
// norms, the cache's pages, attention over them.  Argument checks, workspace carving, launch shapes.  No allocation, no
// host synchronisation, no state.
#include "api_common.hpp"
#include "kv_pages.hpp"
#include "paged_attn.hpp"
#include "qk_norm_rope.hpp"

using namespace smlm;

namespace {

int check_dtype(int dtype) { return dtype == SMLM_DTYPE_F16 || dtype == SMLM_DTYPE_BF16 ? SMLM_OK : SMLM_ERR_DTYPE; }

HeadsView view(const smlm_heads& h) { return {reinterpret_cast<uint16_t*>(h.data), h.row_stride, h.head_stride}; }
bool aligned(const smlm_heads& h) { return aligned16(h.data) && !(h.row_stride & 7) && !(h.head_stride & 7); }

int lanes_log2(int head_dim) {
  int l = 0;
  while ((16 << l) < head_dim) ++l;
  return l;
}

int rope_check(const smlm_qk_rope* p) {
  if (!p || p->rows < 0 || p->q_heads <= 0 || p->kv_heads <= 0 || p->head_dim <= 0 || p->rot_dim <= 0 || p->table_rows < 0 ||
      p->rot_dim > p->head_dim)
    return SMLM_ERR_ARG;
  if (int rc = check_dtype(p->dtype)) return rc;
  if ((p->head_dim & 15) || (p->rot_dim & 15)) return SMLM_ERR_ALIGN;
  if (p->head_dim > kRopeMaxDim || p->rows > (1 << 28) || p->q_heads > (1 << 16) || p->kv_heads > (1 << 16)) return SMLM_ERR_LIMIT;
  if (p->rows > 0 && (!p->table || !p->positions)) return SMLM_ERR_ARG;
  if (!aligned16(p->table) || !aligned16(p->q_weight) || !aligned16(p->k_weight)) return SMLM_ERR_ALIGN;
  return SMLM_OK;
}

// Runs of heads that a wave takes: one, where the batch has few rows and the card wants waves; two otherwise, whose loads
// are on their way together and share the row's cosines and sines.  (One, two, four: 22.0, 20.3, 21.0 us at 2112 rows of 96 heads; one, two:
// 3.4, 4.5 at 256 rows of 48.)
template <int DT, bool NORM>
int launch_rope(QkRopeArgs a, int heads, hipStream_t st) {
  const int runs = ceil_div(heads, 64 >> a.lanes_log2);
  const bool two = (int64_t)a.T * ceil_div(runs, 2) >= 4096;
  a.parts = two ? ceil_div(runs, 2) : runs;
  a.runs = ceil_div(runs, a.parts);
  const int64_t blocks = ((int64_t)a.T * a.parts + 3) / 4;
  if (blocks > 0x7fffffff) return SMLM_ERR_LIMIT;
  const dim3 grid((unsigned)blocks), bl(256);
  if (a.rot == a.D)
    return two ? launch(qk_rope_kernel<DT, NORM, true, 2>, grid, bl, st, a) : launch(qk_rope_kernel<DT, NORM, true, 1>, grid, bl, st, a);
  return two ? launch(qk_rope_kernel<DT, NORM, false, 2>, grid, bl, st, a) : launch(qk_rope_kernel<DT, NORM, false, 1>, grid, bl, st, a);
}
int launch_rope(const QkRopeArgs& a, int dtype, hipStream_t st) {
  const int heads = a.Hq + a.Hkv + (a.v_cache ? a.Hkv : 0);
  const bool norm = a.wq || a.wk;
  if (dtype == SMLM_DTYPE_F16)
    return norm ? launch_rope<SMLM_DTYPE_F16, true>(a, heads, st) : launch_rope<SMLM_DTYPE_F16, false>(a, heads, st);
  return norm ? launch_rope<SMLM_DTYPE_BF16, true>(a, heads, st) : launch_rope<SMLM_DTYPE_BF16, false>(a, heads, st);
}

// Workgroups of the backward for q or for k: each leaves a row of sums that the fold reads.  (256, 512, 1024 at most: 32.6, 26.7,
// 27.1 us at 4096 rows of 32 and 8 heads.)
int rope_bwd_blocks(int rows) {
  const int nb = ceil_div(rows, 4);
  return nb < 1 ? 1 : (nb < 512 ? nb : 512);
}

// the same numbers for extend and fork; compact uses the page arrays
size_t kv_carve(void* base, int R, int N, int S, int** owner, int** start, int** fresh, int** forked, int** src, int** dst,
                int** moved, int** head) {
  size_t off = 0;
  auto take = [&](size_t n) {
    const size_t o = off;
    off = align_up(off + n * 4, 256);
    return base ? reinterpret_cast<int*>(reinterpret_cast<char*>(base) + o) : nullptr;
  };
  int* p[8] = {take(R), take((size_t)S + 1), take(N), take(S), take(N), take(N), take(N), take(2)};
  if (owner) *owner = p[0];
  if (start) *start = p[1];
  if (fresh) *fresh = p[2];
  if (forked) *forked = p[3];
  if (src) *src = p[4];
  if (dst) *dst = p[5];
  if (moved) *moved = p[6];
  if (head) *head = p[7];
  return off;
}
int kv_check(int R, int M, int N, int S, int page_size) {
  if (R < 0 || M < 0 || N < 0 || S < 0 || page_size <= 0) return SMLM_ERR_ARG;
  if (R > (1 << 24) || M > (1 << 20) || N > (1 << 28) || S > (1 << 20) || (int64_t)N * page_size > 0x7fffffff ||
      (int64_t)M * page_size > 0x7fffffff)
    return SMLM_ERR_LIMIT;
  return SMLM_OK;
}
int kv_pool(void* pool, int N, int blocks, int page_size, int place_bytes, KvPool* out) {
  if (blocks <= 0 || place_bytes <= 0 || (N > 0 && !pool)) return SMLM_ERR_ARG;
  if (!aligned16(pool) || (place_bytes & 15)) return SMLM_ERR_ALIGN;
  if ((int64_t)page_size * place_bytes > (1 << 30) || blocks > (1 << 24)) return SMLM_ERR_LIMIT;
  const int block = page_size * place_bytes;
  out->data = reinterpret_cast<uint16_t*>(pool);
  out->page = (int64_t)blocks * block / 2;
  out->N = N;
  out->C = blocks;
  out->P = page_size;
  out->place = place_bytes / 16;
  // 32 KiB a workgroup, a block of a page to a wave at a time (16, 32, 64: 15.5, 14.4, 16.7 us for 128 part-filled pages of 512 KiB)
  int group = round_up((32 << 10) / block > 0 ? (32 << 10) / block : 1, 4);
  if (group > blocks) group = blocks;
  out->group = group;
  out->groups = ceil_div(blocks, group);
  return SMLM_OK;
}

int attn_check(int T, int S, int q_heads, int kv_heads) {
  if (T < 0 || S < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return SMLM_ERR_ARG;
  if (q_heads > 4096 || S > (1 << 20) || (int64_t)T * q_heads > 0x3fffffff) return SMLM_ERR_LIMIT;
  if ((int64_t)attn_items_max(T, S, q_heads / kv_heads, kv_heads) * kv_heads > 0x7fffffff) return SMLM_ERR_LIMIT;
  return SMLM_OK;
}
// whether a row of the table holds keys enough for a sequence to be cut
bool attn_cuts(int M, int page_size) { return (int64_t)M * page_size > kAttnMinKeys; }

size_t attn_carve(void* base, int T, int S, int most, int q_heads, int kv_heads, int head_dim, AttnArgs* a) {
  size_t off = 0;
  auto take = [&](size_t floats) {
    const size_t o = off;
    off = align_up(off + floats * 4, 256);
    return base ? reinterpret_cast<float*>(reinterpret_cast<char*>(base) + o) : nullptr;
  };
  const size_t small = (size_t)attn_parts_small(S, kv_heads, most) * kv_heads * kAttnSmallRows;
  const size_t big = (size_t)attn_parts_big(T, S, q_heads / kv_heads, kv_heads, most) * kv_heads * kAttnBigRows;
  float *p0 = take(small * head_dim), *p1 = take(big * head_dim), *p2 = take(small * 2), *p3 = take(big * 2);
  if (a) a->po_small = p0, a->po_big = p1, a->pm_small = p2, a->pm_big = p3;
  return off;
}

template <int DT, int D>
int launch_attn(const AttnArgs& a, int items, int joins, hipStream_t st) {
  const int rc = launch(attn_kernel<DT, D>, dim3((unsigned)items * a.Hkv), dim3(256), st, a);
  if (rc || joins == 0) return rc;
  const int64_t work = (int64_t)joins * a.Hkv;
  return launch(attn_join_kernel<DT, D>, dim3((unsigned)(work < kAttnJoinBlocks ? work : kAttnJoinBlocks)), dim3(256), st, a);
}

}  // namespace

extern "C" {

SMLM_API int smlm_qk_norm_rope_fwd(const smlm_qk_rope* p, void* stream) {
  if (int rc = rope_check(p)) return rc;
  if (p->rows == 0) return SMLM_OK;
  const bool cache = p->k_cache != nullptr;
  if (!p->q.data || !p->k.data || !p->q_out.data || (!cache && !p->k_out.data)) return SMLM_ERR_ARG;
  if (!aligned(p->q) || !aligned(p->k) || !aligned(p->q_out) || !aligned(p->k_out)) return SMLM_ERR_ALIGN;
  if (cache) {
    if (!p->v_cache || !p->v.data || !p->slots || p->n_pages < 0 || p->page_size <= 0) return SMLM_ERR_ARG;
    if (!aligned(p->v) || !aligned16(p->k_cache) || !aligned16(p->v_cache) || (p->page_stride & 7) || (p->head_stride & 7) ||
        (p->slot_stride & 7))
      return SMLM_ERR_ALIGN;
    if ((int64_t)p->n_pages * p->page_size > 0x7fffffff) return SMLM_ERR_LIMIT;
  }
  const QkRopeArgs a{view(p->q), view(p->k), view(p->v), view(p->q_out), view(p->k_out),
                     reinterpret_cast<const uint16_t*>(p->q_weight), reinterpret_cast<const uint16_t*>(p->k_weight), p->table,
                     p->positions, reinterpret_cast<uint16_t*>(p->k_cache), cache ? reinterpret_cast<uint16_t*>(p->v_cache) : nullptr,
                     p->slots, p->page_stride, p->head_stride, p->slot_stride, p->rows, p->q_heads, p->kv_heads, p->head_dim,
                     p->rot_dim, p->table_rows, cache ? p->page_size : 1, cache ? p->n_pages * p->page_size : 0,
                     lanes_log2(p->head_dim), 0, 0, p->eps, 1.0f};
  return launch_rope(a, p->dtype, (hipStream_t)stream);
}

SMLM_API int smlm_qk_norm_rope_bwd_workspace_size(int rows, int q_heads, int kv_heads, int head_dim, size_t* bytes) {
  if (!bytes || rows < 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0) return SMLM_ERR_ARG;
  if (head_dim > kRopeMaxDim || rows > (1 << 28)) return SMLM_ERR_LIMIT;
  *bytes = (size_t)2 * rope_bwd_blocks(rows) * head_dim * 4;
  return SMLM_OK;
}

SMLM_API int smlm_qk_norm_rope_bwd(const smlm_qk_rope* p, const smlm_heads* gq, const smlm_heads* gk, const smlm_heads* dq,
                                   const smlm_heads* dk, void* dq_weight, void* dk_weight, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (int rc = rope_check(p)) return rc;
  if (!gq || !gk || !dq || !dk) return SMLM_ERR_ARG;
  if (p->rows == 0) return p->q_weight || p->k_weight ? SMLM_ERR_ARG : SMLM_OK;  // (a weight's gradient would have nothing to sum)
  if (!gq->data || !gk->data || !dq->data || !dk->data) return SMLM_ERR_ARG;
  if (!aligned(*gq) || !aligned(*gk) || !aligned(*dq) || !aligned(*dk)) return SMLM_ERR_ALIGN;
  const smlm_heads* g[2] = {gq, gk};
  const smlm_heads* d[2] = {dq, dk};
  const smlm_heads* x[2] = {&p->q, &p->k};
  const void* w[2] = {p->q_weight, p->k_weight};
  void* dw[2] = {dq_weight, dk_weight};
  const int heads[2] = {p->q_heads, p->kv_heads}, nb = rope_bwd_blocks(p->rows);
  bool any = false;
  for (int i = 0; i < 2; ++i) {
    if (!w[i]) continue;
    any = true;
    if (!x[i]->data || !dw[i]) return SMLM_ERR_ARG;
    if (!aligned(*x[i])) return SMLM_ERR_ALIGN;
  }
  if (any && (!workspace || !aligned16(workspace))) return workspace ? SMLM_ERR_ALIGN : SMLM_ERR_ARG;
  if (any && workspace_bytes < (size_t)2 * nb * p->head_dim * 4) return SMLM_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = p->dtype == SMLM_DTYPE_F16;

  // without a weight the gradient is the rotation by the opposite angle: the forward kernel, both tensors or the one
  if (!w[0] || !w[1]) {
    QkRopeArgs a{};
    const int first = w[0] ? 1 : 0, last = w[1] ? 0 : 1;
    a.q = view(*g[first]);
    a.q_out = view(*d[first]);
    a.k = view(*g[1]);
    a.k_out = view(*d[1]);
    a.table = p->table;
    a.pos = p->positions;
    a.T = p->rows;
    a.Hq = heads[first];
    a.Hkv = first == last ? 0 : heads[1];
    a.D = p->head_dim;
    a.rot = p->rot_dim;
    a.n_pos = p->table_rows;
    a.page_size = 1;
    a.lanes_log2 = lanes_log2(p->head_dim);
    a.sign = -1.0f;
    if (int rc = launch_rope(a, p->dtype, st)) return rc;
  }
  if (!any) return SMLM_OK;
  QkRopeBwdPair both{};
  QkRopeFoldArgs fold{};
  int blocks = 0, n = 0;
  for (int i = 0; i < 2; ++i) {
    if (!w[i]) continue;
    float* partial = reinterpret_cast<float*>(workspace) + (size_t)i * nb * p->head_dim;
    both.part[n] = {view(*g[i]), view(*x[i]), view(*d[i]), reinterpret_cast<const uint16_t*>(w[i]), p->table, p->positions, partial,
                    p->rows, heads[i], p->head_dim, p->rot_dim, p->table_rows, lanes_log2(p->head_dim), nb, blocks, p->eps};
    fold.dw[n] = reinterpret_cast<uint16_t*>(dw[i]);
    fold.partial[n] = partial;
    fold.n_part[n] = nb;
    blocks += nb;
    ++n;
  }
  if (n == 1) both.part[1].first_block = 0x7fffffff;
  fold.D = p->head_dim;
  fold.blocks = p->head_dim / 16;
  int rc = f16 ? launch(qk_rope_bwd_kernel<SMLM_DTYPE_F16>, dim3((unsigned)blocks), dim3(256), st, both)
               : launch(qk_rope_bwd_kernel<SMLM_DTYPE_BF16>, dim3((unsigned)blocks), dim3(256), st, both);
  if (rc) return rc;
  return f16 ? launch(qk_rope_fold_kernel<SMLM_DTYPE_F16>, dim3((unsigned)(n * fold.blocks)), dim3(256), st, fold)
             : launch(qk_rope_fold_kernel<SMLM_DTYPE_BF16>, dim3((unsigned)(n * fold.blocks)), dim3(256), st, fold);
}

SMLM_API int smlm_kv_workspace_size(int R, int N, int S, size_t* bytes) {
  if (!bytes) return SMLM_ERR_ARG;
  if (int rc = kv_check(R, 0, N, S, 1)) return rc;
  *bytes = kv_carve(nullptr, R, N, S, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
  return SMLM_OK;
}

SMLM_API int smlm_kv_extend_upto(int32_t* table, int32_t* length, int32_t* refs, const int32_t* requests, const int32_t* counts,
                                 int32_t* q_indptr, int32_t* kv_len, int32_t* positions, int64_t* slots, void* workspace,
                                 size_t workspace_bytes, int R, int M, int N, int S, int rows, int page_size, int max_tokens,
                                 int32_t* status, void* stream) {
  if (int rc = kv_check(R, M, N, S, page_size)) return rc;
  if (rows < 0 || max_tokens < 0 || !q_indptr || !workspace || (S > 0 && (!requests || !counts || !kv_len)) ||
      (rows > 0 && (!positions || !slots)) || (R > 0 && (!length || (M > 0 && !table))) || (N > 0 && !refs))
    return SMLM_ERR_ARG;
  if (rows > (1 << 20)) return SMLM_ERR_LIMIT;
  if (!aligned16(workspace)) return SMLM_ERR_ALIGN;
  KvExtendArgs a{};
  if (workspace_bytes < kv_carve(workspace, R, N, S, &a.owner, &a.start, &a.fresh, nullptr, nullptr, nullptr, nullptr, nullptr))
    return SMLM_ERR_WORKSPACE;
  a.table = table, a.length = length, a.refs = refs, a.status = status;
  a.requests = requests, a.counts = counts;
  a.q_indptr = q_indptr, a.kv_len = kv_len, a.positions = positions, a.slots = slots;
  a.R = R, a.M = M, a.N = N, a.S = S, a.rows = rows, a.P = page_size;
  a.most = max_tokens < M * page_size ? max_tokens : M * page_size;
  if (S <= kKvThreads && rows <= kKvFewRows) return launch(kv_extend_one_kernel<true>, dim3(1), dim3(kKvThreads), (hipStream_t)stream, a);
  const int rc = launch(S <= kKvThreads ? kv_extend_one_kernel<false> : kv_extend_kernel, dim3(1), dim3(kKvThreads), (hipStream_t)stream, a);
  if (rc || rows == 0) return rc;
  return launch(kv_rows_kernel, dim3((unsigned)ceil_div(rows, 256)), dim3(256), (hipStream_t)stream, a);
}

SMLM_API int smlm_kv_extend(int32_t* table, int32_t* length, int32_t* refs, const int32_t* requests, const int32_t* counts,
                            int32_t* q_indptr, int32_t* kv_len, int32_t* positions, int64_t* slots, void* workspace,
                            size_t workspace_bytes, int R, int M, int N, int S, int rows, int page_size, int32_t* status,
                            void* stream) {
  return smlm_kv_extend_upto(table, length, refs, requests, counts, q_indptr, kv_len, positions, slots, workspace, workspace_bytes, R,
                             M, N, S, rows, page_size, 0x7fffffff, status, stream);
}

SMLM_API int smlm_kv_free(int32_t* table, int32_t* length, int32_t* refs, const int32_t* requests, int R, int M, int N, int K,
                          int page_size, int32_t* status, void* stream) {
  if (int rc = kv_check(R, M, N, K, page_size)) return rc;
  if (K == 0) return SMLM_OK;
  if (!requests || (R > 0 && (!length || (M > 0 && !table))) || (N > 0 && !refs)) return SMLM_ERR_ARG;
  const KvFreeArgs a{table, length, refs, status, requests, R, M, N, K, page_size};
  return launch(kv_free_kernel, dim3((unsigned)K), dim3(256), (hipStream_t)stream, a);
}

SMLM_API int smlm_kv_fork(void* pool, int32_t* table, int32_t* length, int32_t* refs, const int32_t* parents,
                          const int32_t* children, void* workspace, size_t workspace_bytes, int R, int M, int N, int K,
                          int blocks, int page_size, int place_bytes, int32_t* status, void* stream) {
  if (int rc = kv_check(R, M, N, K, page_size)) return rc;
  KvForkArgs a{};
  if (int rc = kv_pool(pool, N, blocks, page_size, place_bytes, &a.pool)) return rc;
  if (K == 0) return SMLM_OK;
  if (!parents || !children || !workspace || (R > 0 && (!length || (M > 0 && !table))) || (N > 0 && !refs)) return SMLM_ERR_ARG;
  if (!aligned16(workspace)) return SMLM_ERR_ALIGN;
  if (workspace_bytes < kv_carve(workspace, R, N, K, &a.owner, &a.start, &a.fresh, &a.forked, nullptr, nullptr, nullptr, nullptr))
    return SMLM_ERR_WORKSPACE;
  if ((int64_t)K * a.pool.groups > 0x7fffffff) return SMLM_ERR_LIMIT;
  a.table = table, a.length = length, a.refs = refs, a.status = status;
  a.parents = parents, a.children = children;
  a.R = R, a.M = M, a.K = K;
  const int rc = launch(kv_fork_kernel, dim3(1), dim3(kKvThreads), (hipStream_t)stream, a);
  if (rc) return rc;
  return launch(kv_fork_copy_kernel, dim3((unsigned)(K * a.pool.groups)), dim3(256), (hipStream_t)stream, a);
}

SMLM_API int smlm_kv_compact(void* pool, int32_t* table, int32_t* refs, void* workspace, size_t workspace_bytes, int R, int M,
                             int N, int blocks, int page_size, int place_bytes, void* stream) {
  if (int rc = kv_check(R, M, N, 0, page_size)) return rc;
  KvCompactArgs a{};
  if (int rc = kv_pool(pool, N, blocks, page_size, place_bytes, &a.pool)) return rc;
  if (N == 0) return SMLM_OK;
  a.entries = (int64_t)R * M;
  if (!refs || !workspace || (a.entries > 0 && !table)) return SMLM_ERR_ARG;
  if (!aligned16(workspace)) return SMLM_ERR_ALIGN;
  if (workspace_bytes < kv_carve(workspace, R, N, 0, nullptr, nullptr, nullptr, nullptr, &a.src, &a.dst, &a.moved, &a.head))
    return SMLM_ERR_WORKSPACE;
  a.table = table;
  a.refs = refs;
  const int64_t tb = (a.entries + 1023) / 1024;
  a.table_blocks = tb < 256 ? (int)tb : 256;
  int rc = launch(kv_compact_kernel, dim3(1), dim3(kKvThreads), (hipStream_t)stream, a);
  if (rc) return rc;
  const int64_t work = (int64_t)(N / 2) * a.pool.groups;  // at most half of the pages can move
  const int copies = work < 4096 ? (int)work : 4096;
  if (a.table_blocks + copies == 0) return SMLM_OK;
  return launch(kv_compact_copy_kernel, dim3((unsigned)(a.table_blocks + copies)), dim3(256), (hipStream_t)stream, a);
}

SMLM_API int smlm_kv_copy_pages(void* pool, const int32_t* src, const int32_t* dst, int K, int N, int blocks, int page_size,
                                int place_bytes, void* stream) {
  if (int rc = kv_check(0, 0, N, 0, page_size)) return rc;
  KvCopyArgs a{};
  if (K < 0) return SMLM_ERR_ARG;
  if (int rc = kv_pool(pool, N, blocks, page_size, place_bytes, &a.pool)) return rc;
  if (K == 0 || N == 0) return SMLM_OK;
  if (!src || !dst) return SMLM_ERR_ARG;
  a.src = src, a.dst = dst, a.K = K;
  const int64_t work = (int64_t)K * a.pool.groups;
  return launch(kv_copy_kernel, dim3((unsigned)(work < 8192 ? work : 8192)), dim3(256), (hipStream_t)stream, a);
}

SMLM_API int smlm_attn_plan_size(int T, int S, int q_heads, int kv_heads, size_t* bytes) {
  if (!bytes) return SMLM_ERR_ARG;
  if (int rc = attn_check(T, S, q_heads, kv_heads)) return rc;
  *bytes = attn_plan_carve(nullptr, T, S, q_heads / kv_heads, kv_heads, nullptr);
  return SMLM_OK;
}

SMLM_API int smlm_attn_plan_build(void* plan, size_t plan_bytes, const int32_t* q_indptr, const int32_t* kv_len,
                                  const int32_t* requests, int T, int S, int R, int M, int page_size, int q_heads,
                                  int kv_heads, void* stream) {
  if (int rc = attn_check(T, S, q_heads, kv_heads)) return rc;
  if (int rc = kv_check(R, M, 0, S, page_size)) return rc;
  if (!plan || !q_indptr || (S > 0 && !kv_len)) return SMLM_ERR_ARG;
  if (!aligned16(plan)) return SMLM_ERR_ALIGN;
  AttnPlanArgs a{};
  const int g = q_heads / kv_heads;
  if (plan_bytes < attn_plan_carve(plan, T, S, g, kv_heads, &a.plan)) return SMLM_ERR_WORKSPACE;
  a.q_indptr = q_indptr, a.kv_len = kv_len, a.requests = requests;
  a.T = T, a.S = S, a.g = g, a.Hkv = kv_heads, a.R = R;
  a.most = M * page_size;
  a.items_max = attn_items_max(T, S, g, kv_heads);
  a.joins_max = attn_joins_max(T, S, g, kv_heads);
  a.parts_small_max = attn_parts_small(S, kv_heads, a.most);
  a.parts_big_max = attn_parts_big(T, S, g, kv_heads, a.most);
  // (fewer waves, fewer to wait for at a barrier: two sequences 4.4 us with 512 threads, 6.1 with 1024; 256 sequences 6.2 and 8.0, with
  // 256 threads 7.2)
  return launch(attn_plan_kernel, dim3(1), dim3(S <= 256 ? 512 : kAttnPlanThreads), (hipStream_t)stream, a);
}

SMLM_API int smlm_paged_attn_workspace_size(int T, int S, int M, int page_size, int q_heads, int kv_heads, int head_dim,
                                            size_t* bytes) {
  if (!bytes || M < 0 || page_size <= 0 || head_dim <= 0) return SMLM_ERR_ARG;
  if (int rc = attn_check(T, S, q_heads, kv_heads)) return rc;
  if ((int64_t)M * page_size > 0x7fffffff) return SMLM_ERR_LIMIT;
  *bytes = attn_cuts(M, page_size) ? attn_carve(nullptr, T, S, M * page_size, q_heads, kv_heads, head_dim, nullptr) : 0;
  return SMLM_OK;
}

SMLM_API int smlm_paged_attn(const smlm_heads* out, const smlm_heads* q, const void* k_cache, const void* v_cache,
                             int64_t page_stride, int64_t head_stride, int64_t slot_stride, const int32_t* table,
                             const void* plan, size_t plan_bytes, void* workspace, size_t workspace_bytes, int T, int S, int R,
                             int M, int n_pages, int page_size, int q_heads, int kv_heads, int head_dim, int dtype, float scale,
                             void* stream) {
  if (int rc = attn_check(T, S, q_heads, kv_heads)) return rc;
  if (int rc = kv_check(R, M, n_pages < 0 ? -1 : 0, S, page_size)) return rc;
  if (int rc = check_dtype(dtype)) return rc;
  if (!(scale > 0.0f) || scale > 1.0e38f) return SMLM_ERR_ARG;
  if (head_dim != 64 && head_dim != 128) return SMLM_ERR_LIMIT;
  if (T == 0 || S == 0) return SMLM_OK;
  if (!out || !q || !out->data || !q->data || !plan || (n_pages > 0 && (!k_cache || !v_cache)) || (R > 0 && M > 0 && !table))
    return SMLM_ERR_ARG;
  if (!aligned(*out) || !aligned(*q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(plan) || !aligned16(workspace) ||
      (page_stride & 7) || (head_stride & 7) || (slot_stride & 7))
    return SMLM_ERR_ALIGN;
  const int g = q_heads / kv_heads;
  AttnArgs a{};
  if (plan_bytes < attn_plan_carve(const_cast<void*>(plan), T, S, g, kv_heads, &a.plan)) return SMLM_ERR_WORKSPACE;
  const bool cuts = attn_cuts(M, page_size);
  if (cuts) {
    if (!workspace) return SMLM_ERR_ARG;
    if (workspace_bytes < attn_carve(workspace, T, S, M * page_size, q_heads, kv_heads, head_dim, &a)) return SMLM_ERR_WORKSPACE;
  }
  a.out = reinterpret_cast<uint16_t*>(out->data);
  a.q = reinterpret_cast<const uint16_t*>(q->data);
  a.k = reinterpret_cast<const uint16_t*>(k_cache);
  a.v = reinterpret_cast<const uint16_t*>(v_cache);
  a.table = table;
  a.o_row = out->row_stride, a.o_head = out->head_stride, a.q_row = q->row_stride, a.q_head = q->head_stride;
  a.c_page = page_stride, a.c_head = head_stride, a.c_slot = slot_stride;
  a.M = M, a.most = M * page_size, a.n_pages = n_pages, a.P = page_size, a.T = T, a.S = S, a.R = R, a.Hkv = kv_heads, a.g = g;
  // x / P = (floor(x m / 2^32) + x) >> s for x < 2^32, with s = ceil(log2 P), m = floor(2^32 (2^s - P) / P) + 1
  // (Granlund and Montgomery, Division by Invariant Integers using Multiplication, 1994)
  while ((int64_t)1 << a.div_shift < page_size) ++a.div_shift;
  a.div_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << a.div_shift) - page_size)) / page_size + 1);
  const int load_rows = 512 / head_dim;
  a.whole = slot_stride < 0 || slot_stride >= (1 << 24) ? 0 : (page_size % 16 == 0 ? 16 : (page_size % load_rows == 0 ? load_rows : 0));
  a.scale = scale * 1.4426950408889634f;
  const int items = attn_items_max(T, S, g, kv_heads), joins = cuts ? attn_joins_max(T, S, g, kv_heads) : 0;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SMLM_DTYPE_F16)
    return head_dim == 64 ? launch_attn<SMLM_DTYPE_F16, 64>(a, items, joins, st) : launch_attn<SMLM_DTYPE_F16, 128>(a, items, joins, st);
  return head_dim == 64 ? launch_attn<SMLM_DTYPE_BF16, 64>(a, items, joins, st) : launch_attn<SMLM_DTYPE_BF16, 128>(a, items, joins, st);
}

}  // extern "C"
