// The life of a paged cache's pages, on the device: alloting them to growing requests, sharing them between the
// answers to one prompt, giving them back, packing the pool to its front, copying.
//
// State, all int32 on the device: table [R, M] (page ids of request r, -1 past its last page), length [R] (tokens cached),
// refs [N] (requests that hold page n; 0: free).  Free pages are taken lowest number first, so that every result is a
// function of the inputs alone; the counts are changed by integer atomics, whose order does not show.  A request's
// part-filled last page belongs to it alone (a fork copies it), so growing never has to copy.
//
// extend and fork change all they should or nothing: what they need is counted and checked first, and a call that cannot be done
// sets bits of `status`.  free takes each request by itself: there is nothing it could lack, and a number that is no request's sets a bit.
//
// The bookkeeping is a few kilobytes of integers, bound by latency: one workgroup of 1024 threads counts and takes the
// pages (scans and a pass over refs, sixteen pages a thread at a time, the next ones on their way, ended as soon as enough are found);
// what grows with tokens or page contents runs in a second launch that has the card.  us: a token for each of 256 requests, half of
// 40000 pages free, 8.1 (an empty launch takes 2.5); prompts of 128000 tokens 9.4 + 4.3; freeing 64 requests of 4000 tokens 3.4;
// forking 16 requests into 128 5.5 + 14.8 for copies of 32 MB.  Copies go at the rate of a plain copy: packing 610 MB 225 us,
// 5.4 TB/s read and written.
#pragma once
#include "smlm_common.hpp"
#include "wave_scan.hpp"

namespace smlm {

constexpr int kKvThreads = 1024;

// inclusive sum over the workgroup's 1024 threads; `total` gets the sum of all
__device__ __forceinline__ int kv_scan(int v, int* wave_tot, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();  // earlier readers of wave_tot are done
  if (lane == 63) wave_tot[wave] = v;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kKvThreads / kWaveSize; ++w) {
    const int t = wave_tot[w];
    before += w < wave ? t : 0;
    total += t;
  }
  return v + before;
}

// Atomics reach memory past the CU's own cache, so what they wrote is read the same way (a barrier orders them in a workgroup).
__device__ __forceinline__ int kv_load(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void kv_store(int* p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// This thread's sixteen pages from number `first` on, where there are as many.  (A kernel asks for its first ones as it starts, so
// that they are there when it knows how many it wants.)
struct KvRefs {
  i32x4 v[4];
};
__device__ __forceinline__ KvRefs kv_refs(const int* refs, int N, int first) {
  KvRefs x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x.v[j] = i32x4{1, 1, 1, 1};
    if (first + 16 <= N) __builtin_memcpy(&x.v[j], refs + first + 4 * j, 16);
  }
  return x;
}

// The `want` lowest pages without holders into out[0, want); returns how many there are (at most want).
__device__ __forceinline__ int kv_take_free(const int* refs, int N, int want, int* out, int* wave_tot, KvRefs x) {
  int found = 0;
  for (int base = 0; base < N && found < want; base += kKvThreads * 16) {
    const int first = base + (int)threadIdx.x * 16;
    const KvRefs next = kv_refs(refs, N, first + kKvThreads * 16);
    uint32_t mask = 0;
    if (first + 16 <= N) {
#pragma unroll
      for (int j = 0; j < 16; ++j) mask |= (x.v[j >> 2][j & 3] == 0 ? 1u : 0u) << j;
    } else {
      for (int j = 0; j < 16 && first + j < N; ++j) mask |= (refs[first + j] == 0 ? 1u : 0u) << j;
    }
    const int n = __popc(mask);
    int total;
    int at = found + kv_scan(n, wave_tot, total) - n;
    while (mask && at < want) {
      out[at++] = first + __ffs(mask) - 1;
      mask &= mask - 1;
    }
    found += total;
    x = next;
  }
  return found < want ? found : want;
}

// Marks, for each request of `list` (K entries), the first entry that names it; entry i is alone or first where kv_first gives i.
// In LDS where the requests' rows fit, else in scratch memory (two trips to L2 and back: 3 us).
constexpr int kKvOwners = 8192;
__device__ __forceinline__ void kv_mark(const int* list, int K, int R, int* owner, int* owner_s) {
  const bool local = R <= kKvOwners;
  for (int i = threadIdx.x; i < K; i += kKvThreads) {
    const int r = list[i];
    if (r < 0 || r >= R) continue;
    if (local) owner_s[r] = 0x7fffffff;
    else kv_store(owner + r, 0x7fffffff);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < K; i += kKvThreads) {
    const int r = list[i];
    if (r >= 0 && r < R) atomicMin((local ? owner_s : owner) + r, i);
  }
  __syncthreads();
}
__device__ __forceinline__ int kv_first(int r, int R, const int* owner, const int* owner_s) {
  return R <= kKvOwners ? owner_s[r] : kv_load(owner + r);
}

struct KvExtendArgs {
  int *table, *length, *refs, *status;
  const int *requests, *counts;  // [S]; a request below 0 is skipped
  int *q_indptr, *kv_len;        // [S + 1], [S]
  int* positions;                // [rows]
  int64_t* slots;                // [rows]
  int *owner, *start, *fresh;    // scratch: [R], [S + 1] running sum of new pages, [N]
  int R, M, N, S, rows, P;
  int most;                      // tokens that a request may have, at most M * P
};

// A sequence's part of a step.
struct KvNeed {
  int n, pages, err;  // new tokens, new pages
};
__device__ __forceinline__ KvNeed kv_need(const KvExtendArgs& a, int r, int count, bool first, int old) {
  KvNeed x{r < 0 ? 0 : max(count, 0), 0, 0};
  if (r >= 0) {
    if (r >= a.R || count < 0 || !first) x.err = SMLM_KV_BAD_REQUEST;
    const int64_t now = (int64_t)old + x.n, had = ((int64_t)old + a.P - 1) / a.P, has = (now + a.P - 1) / a.P;
    if (r < a.R && (now > a.most || old < 0)) x.err |= SMLM_KV_TOO_LONG;
    if (x.n > a.rows) x.err |= SMLM_KV_ROWS, x.n = 0;  // (and so the sum stays small)
    if (!x.err) x.pages = (int)(has - had);
  }
  return x;
}

// One workgroup: counts, checks, takes the pages and writes the step's tables by sequence.  q_indptr doubles as the counts' running sum.
__global__ __launch_bounds__(kKvThreads) void kv_extend_kernel(KvExtendArgs a) {
  __shared__ int wave_tot[16];
  __shared__ int owner_s[kKvOwners];
  __shared__ int bad;
  const int tid = threadIdx.x;
  const KvRefs refs0 = kv_refs(a.refs, a.N, tid * 16);
  if (tid == 0) bad = 0;
  kv_mark(a.requests, a.S, a.R, a.owner, owner_s);
  int rows = 0, pages = 0;
  for (int base = 0; base < a.S; base += kKvThreads) {
    const int i = base + tid;
    int n = 0, need = 0, err = 0;
    if (i < a.S) {
      const int r = a.requests[i];
      const bool in = r >= 0 && r < a.R;
      const KvNeed x = kv_need(a, r, r < 0 ? 0 : a.counts[i], in && kv_first(r, a.R, a.owner, owner_s) == i, in ? a.length[r] : 0);
      n = x.n, need = x.pages, err = x.err;
    }
    if (err) atomicOr(&bad, err);
    int total;
    const int upto = kv_scan(n, wave_tot, total);
    if (i < a.S) a.q_indptr[i + 1] = rows + upto;
    if (rows <= a.rows) rows += total;
    int total_pages;
    const int pages_upto = kv_scan(need, wave_tot, total_pages);
    if (i < a.S) a.start[i + 1] = pages + pages_upto;
    if (pages <= a.N) pages += total_pages;
  }
  if (tid == 0) {
    a.q_indptr[0] = a.start[0] = 0;
    if (rows > a.rows) atomicOr(&bad, SMLM_KV_ROWS);
    if (pages > a.N) atomicOr(&bad, SMLM_KV_NO_PAGES);
  }
  __syncthreads();
  if (!bad) {
    const int found = kv_take_free(a.refs, a.N, pages, a.fresh, wave_tot, refs0);
    if (tid == 0 && found < pages) bad = SMLM_KV_NO_PAGES;
  }
  __threadfence_block();
  __syncthreads();
  const int err = bad;
  if (err) {
    for (int i = tid; i <= a.S; i += kKvThreads) {
      a.q_indptr[i] = a.start[i] = 0;
      if (i < a.S) a.kv_len[i] = 0;
    }
    if (tid == 0 && a.status) atomicOr(a.status, err);
    return;
  }
  for (int i = tid; i < a.S; i += kKvThreads) {
    const int r = a.requests[i];
    const int now = r < 0 ? 0 : a.length[r] + (a.q_indptr[i + 1] - a.q_indptr[i]);
    if (r >= 0) a.length[r] = now;
    a.kv_len[i] = now;
  }
}

// last i in [0, n) with a[i] <= x, given a[0] <= x < a[n]
__device__ __forceinline__ int kv_last_le(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// The new pages' places in the table, and positions and slots of the step's rows: a thread a row (or page: there are at most as many
// as rows).  Rows past the last request's, and all of them where the step was refused, get -1.
constexpr int kKvRowsLds = 1024;  // sequences up to which the running sums are searched in LDS
__global__ __launch_bounds__(256) void kv_rows_kernel(KvExtendArgs a) {
  __shared__ int start_s[kKvRowsLds + 1], indptr_s[kKvRowsLds + 1];
  const int t = (int)blockIdx.x * 256 + (int)threadIdx.x;
  const bool local = a.S <= kKvRowsLds;
  if (local) {
    for (int i = threadIdx.x; i <= a.S; i += 256) start_s[i] = a.start[i], indptr_s[i] = a.q_indptr[i];
    __syncthreads();
  }
  if (t >= a.rows) return;
  auto start = [&](int i) { return local ? start_s[i] : a.start[i]; };
  auto indptr = [&](int i) { return local ? indptr_s[i] : a.q_indptr[i]; };
  if (t < start(a.S)) {
    const int i = local ? kv_last_le(start_s, a.S, t) : kv_last_le(a.start, a.S, t);
    const int old = a.kv_len[i] - (indptr(i + 1) - indptr(i)), id = a.fresh[t];
    a.table[(int64_t)a.requests[i] * a.M + (old + a.P - 1) / a.P + (t - start(i))] = id;
    a.refs[id] = 1;
  }
  int pos = -1;
  int64_t slot = -1;
  if (t < indptr(a.S)) {
    const int i = local ? kv_last_le(indptr_s, a.S, t) : kv_last_le(a.q_indptr, a.S, t);
    const int n = indptr(i + 1) - indptr(i), had = (a.kv_len[i] - n + a.P - 1) / a.P;
    pos = a.kv_len[i] - (indptr(i + 1) - t);
    const int j = pos / a.P;
    const int page = j < had ? a.table[(int64_t)a.requests[i] * a.M + j] : a.fresh[start(i) + j - had];
    slot = (int64_t)page * a.P + (pos - j * a.P);
  }
  a.positions[t] = pos;
  a.slots[t] = slot;
}

// The same where a thread has a sequence to itself: two trips to memory before the pages are looked for.  FEW: the rows too, which
// then find what they look up in LDS: a token for each of 256 requests 8.1 us, 6.5 + 4.1 in two launches; 4096 rows of 256
// requests 10.9 and 6.6 + 4.1, where the second launch's start is still to come; 8192 rows 14.9 and 6.7 + 4.6.
constexpr int kKvFewRows = 4096;
template <bool FEW>
__global__ __launch_bounds__(kKvThreads) void kv_extend_one_kernel(KvExtendArgs a) {
  __shared__ int wave_tot[16];
  __shared__ int owner_s[kKvOwners];
  __shared__ int indptr_s[kKvThreads + 1], start_s[kKvThreads + 1];  // running sums of new tokens and pages
  __shared__ int req_s[kKvThreads], now_s[kKvThreads], tail_s[kKvThreads];  // request; tokens; the page that was filled in part
  __shared__ int fresh_s[FEW ? kKvFewRows : 1];                                // (a new page holds a new token, so pages do not outnumber rows)
  __shared__ int bad;
  const int tid = threadIdx.x;
  const int r = tid < a.S ? a.requests[tid] : -1, count = tid < a.S ? a.counts[tid] : 0;
  const KvRefs refs0 = kv_refs(a.refs, a.N, tid * 16);
  const bool in = r >= 0 && r < a.R, local = a.R <= kKvOwners;
  if (tid == 0) bad = 0;
  if (in) {
    if (local) owner_s[r] = 0x7fffffff;
    else kv_store(a.owner + r, 0x7fffffff);
  }
  __syncthreads();
  if (in) atomicMin((local ? owner_s : a.owner) + r, tid);
  const int old = in ? a.length[r] : 0;
  __syncthreads();
  KvNeed x{0, 0, 0};
  if (tid < a.S) x = kv_need(a, r, count, in && kv_first(r, a.R, a.owner, owner_s) == tid, old);
  if (x.err) atomicOr(&bad, x.err);
  const int tail = FEW && in && old > 0 && old % a.P && old / a.P < a.M ? a.table[(int64_t)r * a.M + old / a.P] : -1;
  int rows, pages;
  const int rows_upto = kv_scan(x.n, wave_tot, rows), pages_upto = kv_scan(x.pages, wave_tot, pages);
  if (rows > a.rows || pages > a.N) {
    if (tid == 0) atomicOr(&bad, (rows > a.rows ? SMLM_KV_ROWS : 0) | (pages > a.N ? SMLM_KV_NO_PAGES : 0));
  }
  if (tid == 0) indptr_s[0] = start_s[0] = 0;
  indptr_s[tid + 1] = rows_upto, start_s[tid + 1] = pages_upto;
  req_s[tid] = r, now_s[tid] = old + x.n, tail_s[tid] = tail;
  __syncthreads();
  if (!bad) {
    const int found = FEW ? kv_take_free(a.refs, a.N, pages, fresh_s, wave_tot, refs0) : kv_take_free(a.refs, a.N, pages, a.fresh, wave_tot, refs0);
    if (tid == 0 && found < pages) bad = SMLM_KV_NO_PAGES;
  }
  __syncthreads();
  const int err = bad;
  if (tid == 0) {
    a.q_indptr[0] = 0;
    if (!FEW) a.start[0] = 0;
    if (err && a.status) atomicOr(a.status, err);
  }
  if (tid < a.S) {
    if (!FEW) a.start[tid + 1] = err ? 0 : pages_upto;
    a.q_indptr[tid + 1] = err ? 0 : rows_upto;
    a.kv_len[tid] = err || !in ? 0 : old + x.n;
    if (in && !err) a.length[r] = old + x.n;
  }
  if (!FEW) return;
  if (err) rows = pages = 0;
  for (int t = tid; t < pages; t += kKvThreads) {
    const int i = kv_last_le(start_s, a.S, t), n = indptr_s[i + 1] - indptr_s[i], id = fresh_s[t];
    a.table[(int64_t)req_s[i] * a.M + (now_s[i] - n + a.P - 1) / a.P + (t - start_s[i])] = id;
    a.refs[id] = 1;
  }
  for (int t = tid; t < a.rows; t += kKvThreads) {
    int pos = -1;
    int64_t slot = -1;
    if (t < rows) {
      const int i = kv_last_le(indptr_s, a.S, t);
      const int n = indptr_s[i + 1] - indptr_s[i], had = (now_s[i] - n + a.P - 1) / a.P;
      pos = now_s[i] - (indptr_s[i + 1] - t);
      const int j = pos / a.P, page = j < had ? tail_s[i] : fresh_s[start_s[i] + j - had];
      slot = (int64_t)page * a.P + (pos - j * a.P);
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
}

struct KvFreeArgs {
  int *table, *length, *refs, *status;
  const int* requests;  // [K]
  int R, M, N, K, P;
};

// A workgroup a request, the known ones of a list that names an unknown one too; who takes its length away gives its pages back, so a request named twice is freed once.
__global__ __launch_bounds__(256) void kv_free_kernel(KvFreeArgs a) {
  __shared__ int had;
  const int r = a.requests[blockIdx.x];
  if (r < 0) return;
  if (r >= a.R) {
    if (threadIdx.x == 0 && a.status) atomicOr(a.status, SMLM_KV_BAD_REQUEST);
    return;
  }
  if (threadIdx.x == 0) had = atomicExch(a.length + r, 0);
  __syncthreads();
  const int64_t pages = ((int64_t)had + a.P - 1) / a.P;
  int* row = a.table + (int64_t)r * a.M;
  for (int i = threadIdx.x; i < pages && i < a.M; i += 256) {
    const int id = row[i];
    if (id >= 0 && id < a.N) atomicSub(a.refs + id, 1);
    row[i] = -1;
  }
}

// ---- copies of pages --------------------------------------------------------------------------------------
// A page holds C blocks of P places of `place` 16-byte pieces (layers x keys and values x heads, tokens, dimensions);
// of each block the first `filled` places are copied.
struct KvCopy {
  int src, dst, filled;
};
struct KvPool {
  uint16_t* data;
  int64_t page;    // elements of a page
  int N, C, P, place;
  int group, groups;  // blocks a workgroup copies, workgroups a page
};

__device__ __forceinline__ void kv_copy_part(const KvPool& pool, int src, int dst, int filled, int part) {
  if (src < 0 || src >= pool.N || dst < 0 || dst >= pool.N || src == dst) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int n = filled * pool.place, block = pool.P * pool.place * 8;
  const int last = (part + 1) * pool.group < pool.C ? (part + 1) * pool.group : pool.C;
  for (int c = part * pool.group + wave; c < last; c += 4) {
    const uint16_t* from = pool.data + src * pool.page + (int64_t)c * block;
    uint16_t* to = pool.data + dst * pool.page + (int64_t)c * block;
    int i = lane;
    for (; i + 3 * kWaveSize < n; i += 4 * kWaveSize) {
      u32x4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = ldg16_nt(from + (int64_t)(i + j * kWaveSize) * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) stg16_nt(to + (int64_t)(i + j * kWaveSize) * 8, v[j]);
    }
    for (; i < n; i += kWaveSize) stg16_nt(to + (int64_t)i * 8, ldg16_nt(from + (int64_t)i * 8));
  }
}

struct KvCopyArgs {
  KvPool pool;
  const int *src, *dst;  // [K] pages
  int K;
};
__global__ __launch_bounds__(256) void kv_copy_kernel(KvCopyArgs a) {
  for (int64_t w = blockIdx.x; w < (int64_t)a.K * a.pool.groups; w += gridDim.x) {
    const int k = (int)(w / a.pool.groups);
    kv_copy_part(a.pool, a.src[k], a.dst[k], a.pool.P, (int)(w - (int64_t)k * a.pool.groups));
  }
}

struct KvForkArgs {
  KvPool pool;
  int *table, *length, *refs, *status;
  const int *parents, *children;  // [K]
  int *owner, *start, *fresh;     // scratch: [R], [K + 1] running sum of copied pages (0 everywhere: refused), [N]
  int* forked;                    // scratch: [K] tokens of the children, -1 where there is nothing to do
  int R, M, K;
};

__global__ __launch_bounds__(kKvThreads) void kv_fork_kernel(KvForkArgs a) {
  __shared__ int wave_tot[16];
  __shared__ int owner_s[kKvOwners];
  __shared__ int bad;
  const int tid = threadIdx.x, P = a.pool.P;
  const KvRefs refs0 = kv_refs(a.refs, a.pool.N, tid * 16);
  if (tid == 0) bad = 0;
  kv_mark(a.children, a.K, a.R, a.owner, owner_s);
  int pages = 0;
  for (int base = 0; base < a.K; base += kKvThreads) {
    const int i = base + tid;
    int need = 0, err = 0, n = -1;
    if (i < a.K) {
      const int p = a.parents[i], c = a.children[i];
      if (c >= 0) {
        if (p < 0 || p >= a.R || c >= a.R || kv_first(c, a.R, a.owner, owner_s) != i || a.length[c] != 0) {
          err = SMLM_KV_BAD_REQUEST;
        } else {
          n = a.length[p];
          if (n < 0 || n > (int64_t)a.M * P) err = SMLM_KV_TOO_LONG;
          else need = n % P != 0;
        }
      }
      a.forked[i] = n;
    }
    if (err) atomicOr(&bad, err);
    int total;
    const int upto = kv_scan(need, wave_tot, total);
    if (i < a.K) a.start[i + 1] = pages + upto;
    pages += total;
  }
  if (tid == 0) {
    a.start[0] = 0;
    if (pages > a.pool.N) atomicOr(&bad, SMLM_KV_NO_PAGES);
  }
  __syncthreads();
  if (!bad) {
    const int found = kv_take_free(a.refs, a.pool.N, pages, a.fresh, wave_tot, refs0);
    if (tid == 0 && found < pages) bad = SMLM_KV_NO_PAGES;
  }
  __threadfence_block();
  __syncthreads();
  const int err = bad;
  for (int i = tid; i < a.K; i += kKvThreads) {
    if (err) {
      a.forked[i] = -1;
      continue;
    }
    const int n = a.forked[i];
    if (n < 0) continue;
    const int c = a.children[i];
    a.length[c] = n;
    if (n % P != 0) {
      const int id = a.fresh[a.start[i]];
      a.table[(int64_t)c * a.M + n / P] = id;
      a.refs[id] = 1;
    }
  }
  if (tid == 0 && err && a.status) atomicOr(a.status, err);
}

// A workgroup a child and part of a page: the full pages' ids and counts (part 0), and its share of the last page's copy.
__global__ __launch_bounds__(256) void kv_fork_copy_kernel(KvForkArgs a) {
  const int k = (int)blockIdx.x / a.pool.groups, part = (int)blockIdx.x % a.pool.groups, P = a.pool.P;
  const int n = a.forked[k];
  if (n < 0) return;
  const int* from = a.table + (int64_t)a.parents[k] * a.M;
  int* to = a.table + (int64_t)a.children[k] * a.M;
  if (part == 0)
    for (int i = threadIdx.x; i < n / P; i += 256) {
      const int id = from[i];
      to[i] = id;
      if (id >= 0 && id < a.pool.N) atomicAdd(a.refs + id, 1);
    }
  if (n % P) kv_copy_part(a.pool, from[n / P], to[n / P], n % P, part);
}

struct KvCompactArgs {
  KvPool pool;
  int *table, *refs;
  int *src, *dst, *moved;  // scratch: [N] pages that move, [N] where to, [N] where a page from `live` on went
  int* head;               // scratch: [2] pages in use, pages that move
  int64_t entries;         // of the table
  int table_blocks;
};

// Pages in use from number `live` (their count) on move into the free ones below it, both in ascending order.
__global__ __launch_bounds__(kKvThreads) void kv_compact_kernel(KvCompactArgs a) {
  __shared__ int wave_tot[16];
  const int tid = threadIdx.x, N = a.pool.N;
  int mine = 0, live;
  for (int i = tid; i < N; i += kKvThreads) mine += a.refs[i] > 0;
  kv_scan(mine, wave_tot, live);
  int holes = 0, movers = 0;
  for (int base = 0; base < N; base += kKvThreads) {
    const int i = base + tid;
    const bool used = i < N && a.refs[i] > 0;
    const int hole = i < live && !used, mover = i >= live && used;
    int total;
    const int upto = kv_scan(hole | (mover << 16), wave_tot, total);
    if (hole) a.dst[holes + (upto & 0xffff) - 1] = i;
    if (mover) a.src[movers + (upto >> 16) - 1] = i;
    if (i >= live && i < N && !used) a.moved[i] = i;  // (a table may still name it)
    holes += total & 0xffff;
    movers += total >> 16;
  }
  __threadfence_block();
  __syncthreads();
  for (int k = tid; k < movers; k += kKvThreads) {
    const int from = a.src[k], to = a.dst[k];
    a.moved[from] = to;
    a.refs[to] = a.refs[from];
    a.refs[from] = 0;
  }
  if (tid == 0) a.head[0] = live, a.head[1] = movers;
}

// The first workgroups rewrite the table, the others copy.
__global__ __launch_bounds__(256) void kv_compact_copy_kernel(KvCompactArgs a) {
  if ((int)blockIdx.x < a.table_blocks) {
    const int live = a.head[0];
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.entries; i += (int64_t)a.table_blocks * 256) {
      const int id = a.table[i];
      if (id >= live && id < a.pool.N) a.table[i] = a.moved[id];
    }
    return;
  }
  const int movers = a.head[1], blocks = (int)gridDim.x - a.table_blocks;
  for (int64_t w = (int)blockIdx.x - a.table_blocks; w < (int64_t)movers * a.pool.groups; w += blocks) {
    const int k = (int)(w / a.pool.groups);
    kv_copy_part(a.pool, a.src[k], a.dst[k], a.pool.P, (int)(w - (int64_t)k * a.pool.groups));
  }
}

}  // namespace smlm
