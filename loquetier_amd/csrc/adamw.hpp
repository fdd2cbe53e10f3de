// One AdamW step of many tensors, in place, for gfx950: the adapters' weights with a step count of their own and each group's rates
// (the reference keeps a trainer and an optimizer an adapter: src/loquetier_src/trainer_utils.py).
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p - lr wd p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in float; a tensor without a gradient stays as it is and its t does not count on.  States lie in flat arrays, each tensor's from a
// multiple of 256 elements on.  In 8 bits m and sqrt(v) are e4m3 with a float scale each for 256 weights (largest / 448): half a step
// of 2^-4 of m, which the next steps average, and as much of the step's size.  The root is stored because it halves v's range of
// exponents and because a root that is not zero can be kept from becoming it (2^-9 of the scale at least): an update divided by a
// vanished v would be lr / eps of m.  The update itself takes the averages before they are rounded.  Scales follow the block's
// largest value, so what all of a block has in common, the decay above all, is kept in float.
// With float weights beside 16-bit ones the step is the float weights', and a 16-bit weight that is no longer its float weight's
// rounding (it was loaded, or set by someone) takes its place.
//
// What decides the 8-bit codes is computed as the formulas stand, operation by operation with each one's own rounding (no fused
// multiply-add, divisions and roots rounded correctly): a code's step is 2^24 times a float's, so the same step written in tensor
// expressions gives the same codes, not others here and there.
//
// Bound by HBM: 22 to 30 bytes an element with float states and 16-bit weights, 10 to 18 with 8-bit ones.  A wave takes four blocks
// of 256 in a row, all their loads on their way before the first is used; tables of a call travel in a launch's arguments, as
// put_words_kernel's do.
#pragma once
#include "add_rms_norm.hpp"

namespace smlm {

constexpr int kAdamBlock = 256;  // elements that share a scale
constexpr int kAdamRun = 4;      // blocks a wave takes
constexpr int kAdamF32 = 2;      // (element type of weights, after SMLM_DTYPE_*)

// What a step needs of a tensor; 64 bytes, read by a wave at once.
struct AdamTensor {
  uint64_t p, g;    // addresses; g 0: no gradient
  int64_t n;        // elements
  uint32_t first;   // block
  uint32_t plain;   // addresses are not aligned for pieces of four elements
  float b1, nb1, b2, nb2, size, root, eps, decay;  // size: lr / (1 - b1^t); root: 1 / sqrt(1 - b2^t); decay: lr wd
};
static_assert(sizeof(AdamTensor) == 64, "");

struct AdamEntry {
  uint64_t p, g;
  int64_t n;  // its top bit: `plain`
};
constexpr int kAdamEntries = 144;  // (a launch takes up to 4 KiB of arguments)
template <int N>
struct AdamBeginArgs {
  AdamTensor* table;
  int32_t* step;          // [n_tensors]
  const float* hyper;     // [n_groups][5] lr, b1, b2, eps, weight decay
  const int32_t* group;   // [n_tensors]
  int at, n, n_groups, pad;
  int64_t first;          // block of tensor `at`
  AdamEntry entry[N];
};

// A thread a tensor.  1 - b^t in 64 bits: near b = 1 a float's would lose it.
template <int N>
__global__ __launch_bounds__(256) void adam_begin_kernel(AdamBeginArgs<N> a) {
  __shared__ uint32_t blocks[N];
  for (int i = threadIdx.x; i < a.n; i += 256)
    blocks[i] = (uint32_t)(((a.entry[i].n & INT64_MAX) + kAdamBlock - 1) / kAdamBlock);
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += 256) {
    AdamTensor t;
    t.p = a.entry[i].p, t.g = a.entry[i].g, t.n = a.entry[i].n & INT64_MAX, t.plain = a.entry[i].n < 0;
    uint32_t first = (uint32_t)a.first;
    for (int j = 0; j < i; ++j) first += blocks[j];
    t.first = first;
    const int group = a.group[a.at + i];
    int step = a.step[a.at + i];
    if (group < 0 || group >= a.n_groups) t.g = 0;
    if (t.g) {
      a.step[a.at + i] = ++step;
      const float* h = a.hyper + 5 * group;
      const double lr = h[0], b1 = h[1], b2 = h[2];
      double p1 = 1.0, p2 = 1.0, q1 = b1, q2 = b2;
      for (int s = step > 0 ? step : 0; s; s >>= 1, q1 *= q1, q2 *= q2)
        if (s & 1) p1 *= q1, p2 *= q2;
      t.b1 = h[1], t.nb1 = (float)(1.0 - b1), t.b2 = h[2], t.nb2 = (float)(1.0 - b2);
      t.size = (float)(lr / (1.0 - p1)), t.root = (float)(1.0 / sqrt(1.0 - p2)), t.eps = h[3], t.decay = (float)(lr * (double)h[4]);
    } else {
      t.b1 = t.nb1 = t.b2 = t.nb2 = t.size = t.root = t.eps = t.decay = 0.0f;
    }
    a.table[a.at + i] = t;
  }
}

struct AdamArgs {
  const AdamTensor* table;
  void *m, *v;             // float or e4m3, [blocks * 256]
  float *m_scale, *v_scale;  // [blocks] (8 bits)
  float* master;             // [blocks * 256] or NULL
  int n_tensors;
  int64_t blocks;
};

typedef float f32x2_adam __attribute__((ext_vector_type(2)));

// Four elements of a lane as floats, and back.
template <int PT>
__device__ __forceinline__ f32x4 adam_load(uint64_t base, int64_t at, int left, bool plain) {
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (PT == kAdamF32) {
    const SMLM_GLOBAL float* p = reinterpret_cast<const SMLM_GLOBAL float*>(base) + at;
    if (left >= 4 && !plain) return *(const SMLM_GLOBAL f32x4*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) o[e] = p[e];
  } else {
    const SMLM_GLOBAL uint16_t* p = reinterpret_cast<const SMLM_GLOBAL uint16_t*>(base) + at;
    u32x2 two = {0u, 0u};
    if (left >= 4 && !plain) {
      two = *(const SMLM_GLOBAL u32x2*)p;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) two[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
    }
    constexpr int DT = PT == kAdamF32 ? 0 : PT;
    o = f32x4{Num<DT>::lo(two[0]), Num<DT>::hi(two[0]), Num<DT>::lo(two[1]), Num<DT>::hi(two[1])};
  }
  return o;
}
template <int PT>
__device__ __forceinline__ void adam_store(uint64_t base, int64_t at, int left, bool plain, f32x4 v) {
  if (PT == kAdamF32) {
    SMLM_GLOBAL float* p = reinterpret_cast<SMLM_GLOBAL float*>(base) + at;
    if (left >= 4 && !plain) {
      *(SMLM_GLOBAL f32x4*)p = v;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = v[e];
  } else {
    constexpr int DT = PT == kAdamF32 ? 0 : PT;
    SMLM_GLOBAL uint16_t* p = reinterpret_cast<SMLM_GLOBAL uint16_t*>(base) + at;
    const u32x2 two = {pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    if (left >= 4 && !plain) {
      *(SMLM_GLOBAL u32x2*)p = two;
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = (uint16_t)(two[e >> 1] >> (16 * (e & 1)));
  }
}
template <int PT>
__device__ __forceinline__ f32x4 adam_round(f32x4 v) {
  if (PT == kAdamF32) return v;
  constexpr int DT = PT == kAdamF32 ? 0 : PT;
  const uint32_t a = pack2<DT>(v[0], v[1]), b = pack2<DT>(v[2], v[3]);
  return f32x4{Num<DT>::lo(a), Num<DT>::hi(a), Num<DT>::lo(b), Num<DT>::hi(b)};
}
__device__ __forceinline__ f32x4 adam_from8(uint32_t c, float s) {
  const f32x2_adam a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  return f32x4{a[0] * s, a[1] * s, b[0] * s, b[1] * s};
}

// The last tensor that begins at block b or before it (empty ones begin where the next does): 64 guesses a round.
__device__ __forceinline__ int adam_find(const AdamTensor* table, int n, uint32_t b, int lane) {
  int lo = 0, hi = n;  // table[lo].first <= b; the answer lies in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6, i = min(lo + lane * step, n - 1);
    const uint64_t under = __ballot(lo + lane * step < hi && table[i].first <= b);
    const int k = 63 - __builtin_clzll(under | 1);
    lo += k * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

template <int PT, bool EIGHT, bool MASTER>
__global__ __launch_bounds__(256) void adam_kernel(AdamArgs a) {
#pragma clang fp contract(off)
  const int lane = threadIdx.x & 63;
  const int64_t b0 = ((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kAdamRun;
  if (b0 >= a.blocks) return;
  int ti = __builtin_amdgcn_readfirstlane(adam_find(a.table, a.n_tensors, (uint32_t)b0, lane));
  f32x4 p[kAdamRun], g[kAdamRun], w[kAdamRun], m[kAdamRun], v[kAdamRun];
  uint32_t mc[kAdamRun], vc[kAdamRun];
  float ms[kAdamRun], vs[kAdamRun];
  int tensor[kAdamRun], left[kAdamRun];
#pragma unroll
  for (int u = 0; u < kAdamRun; ++u) {
    const int64_t b = b0 + u;
    left[u] = 0;
    if (b >= a.blocks) continue;
    while (ti + 1 < a.n_tensors && a.table[ti + 1].first <= (uint32_t)b) ti = __builtin_amdgcn_readfirstlane(ti + 1);
    tensor[u] = ti;
    const AdamTensor* t = a.table + ti;
    if (!t->g) continue;
    const int64_t in = (b - t->first) * kAdamBlock + lane * 4, rest = t->n - in;
    left[u] = rest >= 4 ? 4 : rest > 0 ? (int)rest : 0;
    p[u] = adam_load<PT>(t->p, in, left[u], t->plain);
    g[u] = adam_load<PT>(t->g, in, left[u], t->plain);
    const int64_t at = b * kAdamBlock + lane * 4;
    if (MASTER) w[u] = *(const SMLM_GLOBAL f32x4*)(a.master + at);
    if (EIGHT) {
      mc[u] = *((const SMLM_GLOBAL uint32_t*)a.m + (at >> 2));
      vc[u] = *((const SMLM_GLOBAL uint32_t*)a.v + (at >> 2));
      ms[u] = *((const SMLM_GLOBAL float*)a.m_scale + b);
      vs[u] = *((const SMLM_GLOBAL float*)a.v_scale + b);
    } else {
      m[u] = *(const SMLM_GLOBAL f32x4*)((const float*)a.m + at);
      v[u] = *(const SMLM_GLOBAL f32x4*)((const float*)a.v + at);
    }
  }
#pragma unroll
  for (int u = 0; u < kAdamRun; ++u) {
    const int64_t b = b0 + u;
    if (b >= a.blocks) continue;
    const AdamTensor* t = a.table + tensor[u];
    if (!t->g) continue;
    const int64_t at = b * kAdamBlock + lane * 4, in = (b - t->first) * kAdamBlock + lane * 4;
    if (EIGHT) {
      m[u] = adam_from8(mc[u], ms[u]);
      v[u] = adam_from8(vc[u], vs[u]);
      v[u] *= v[u];
    }
    f32x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = p[u][e];
      const float gr = g[u][e];
      if (MASTER) x = adam_round<PT>(w[u])[e] == x ? w[u][e] : x;
      m[u][e] = t->b1 * m[u][e] + t->nb1 * gr;
      v[u][e] = t->b2 * v[u][e] + t->nb2 * gr * gr;
      r[e] = EIGHT ? sqrtf(v[u][e]) : __builtin_amdgcn_sqrtf(v[u][e]);
      x -= t->decay * x;
      p[u][e] = x - t->size * m[u][e] * __builtin_amdgcn_rcpf(r[e] * t->root + t->eps);
      if (e >= left[u]) m[u][e] = v[u][e] = r[e] = p[u][e] = 0.0f;  // (past the tensor's end: zeros, as the states began)
    }
    adam_store<PT>(t->p, in, left[u], t->plain, p[u]);
    if (MASTER) *(SMLM_GLOBAL f32x4*)(a.master + at) = p[u];
    if (EIGHT) {
      float most_m = 0.0f, most_r = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) most_m = max_or_nan(most_m, fabsf(m[u][e])), most_r = max_or_nan(most_r, r[e]);
      float mi, ri;
      const float sm = scale8(wave_max(most_m), mi), sr = scale8(wave_max(most_r), ri);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[u][e] = mi == 0.0f ? m[u][e] * 0.0f : m[u][e] / sm;  // (0 of 0; of a NaN, NaN)
        const float q = ri == 0.0f ? r[e] * 0.0f : r[e] / sr;
        r[e] = r[e] > 0.0f && q < 0x1p-9f && ri != 0.0f ? 0x1p-9f : q;
      }
      *((SMLM_GLOBAL uint32_t*)a.m + (at >> 2)) = pack8(m[u][0], m[u][1], m[u][2], m[u][3]);
      *((SMLM_GLOBAL uint32_t*)a.v + (at >> 2)) = pack8(r[0], r[1], r[2], r[3]);
      if (lane == 0) a.m_scale[b] = sm, a.v_scale[b] = sr;
    } else {
      *(SMLM_GLOBAL f32x4*)((float*)a.m + at) = m[u];
      *(SMLM_GLOBAL f32x4*)((float*)a.v + at) = v[u];
    }
  }
}

}  // namespace smlm
