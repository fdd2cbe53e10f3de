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
// multiply-add, quotients rounded correctly, the root a sqrtf, which is not always the nearest float): a code's step is 2^20 times a float's, so the
// same step written in tensor expressions on this card gives the same codes and scales, not others here and there.
//
// Bound by HBM: 22 to 30 bytes an element with float states and 16-bit weights, 10 to 18 with 8-bit ones.  A wave takes a block of 256:
// few registers, so many waves' loads are on their way.  (Four blocks a wave with all their loads ahead, two, one, us: 80 million
// bf16 weights with float ones, float states 455, 439, 435 (5.5 TB/s); e4m3 states 343, 286, 271 (5.3 TB/s).)  The tables of a call
// travel in launches' arguments, as put_words_kernel's do.
#pragma once
#include "add_rms_norm.hpp"
#include "wave_scan.hpp"

namespace smlm {

constexpr int kAdamBlock = 256;  // elements that share a scale
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
  static_assert(N <= 256, "a thread each");
  __shared__ uint32_t sums[4];
  const int i = threadIdx.x, wave = i >> 6;
  const bool here = i < a.n;
  const AdamEntry entry = here ? a.entry[i] : AdamEntry{0, 0, 0};
  const int group = here ? a.group[a.at + i] : -1;
  int step = here ? a.step[a.at + i] : 0;
  const bool known = group >= 0 && group < a.n_groups;
  float h[5];
#pragma unroll
  for (int e = 0; e < 5; ++e) h[e] = known ? a.hyper[5 * group + e] : 0.0f;
  const uint32_t mine = (uint32_t)(((entry.n & INT64_MAX) + kAdamBlock - 1) / kAdamBlock);
  const uint32_t upto = (uint32_t)wave_scan((int)mine);
  if ((i & 63) == 63) sums[wave] = upto;
  __syncthreads();
  if (!here) return;
  AdamTensor t;
  t.first = (uint32_t)a.first + upto - mine;
  for (int w = 0; w < wave; ++w) t.first += sums[w];
  t.p = entry.p, t.g = known ? entry.g : 0, t.n = entry.n & INT64_MAX, t.plain = entry.n < 0;
  if (t.g) {
    a.step[a.at + i] = ++step;
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

struct AdamArgs {
  const AdamTensor* table;
  void *m, *v;             // float or e4m3, [blocks * 256]
  float *m_scale, *v_scale;  // [blocks] (8 bits)
  float* master;             // [blocks * 256] or NULL
  int n_tensors;
  int64_t from, blocks;    // the launch's first block; all blocks
};
// Workgroups a launch: from 2^32 threads on HIP drops what is over, and a card's memory holds more blocks.
constexpr int64_t kAdamGroups = 1 << 22;

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
  const int64_t b = a.from + (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (b >= a.blocks) return;
  const AdamTensor* t = a.table + __builtin_amdgcn_readfirstlane(adam_find(a.table, a.n_tensors, (uint32_t)b, lane));
  if (!t->g) return;
  const int64_t in = (b - t->first) * kAdamBlock + lane * 4, at = b * kAdamBlock + lane * 4, rest = t->n - in;
  const int left = rest >= 4 ? 4 : rest > 0 ? (int)rest : 0;
  f32x4 m, v, w, r, p = adam_load<PT>(t->p, in, left, t->plain);
  const f32x4 g = adam_load<PT>(t->g, in, left, t->plain);
  if (MASTER) w = *(const SMLM_GLOBAL f32x4*)(a.master + at);
  if (EIGHT) {
    m = adam_from8(*((const SMLM_GLOBAL uint32_t*)a.m + (at >> 2)), *((const SMLM_GLOBAL float*)a.m_scale + b));
    v = adam_from8(*((const SMLM_GLOBAL uint32_t*)a.v + (at >> 2)), *((const SMLM_GLOBAL float*)a.v_scale + b));
    v *= v;
  } else {
    m = *(const SMLM_GLOBAL f32x4*)((const float*)a.m + at);
    v = *(const SMLM_GLOBAL f32x4*)((const float*)a.v + at);
  }
  if (MASTER) {
    const f32x4 rounded = adam_round<PT>(w);
#pragma unroll
    for (int e = 0; e < 4; ++e) p[e] = rounded[e] == p[e] ? w[e] : p[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = t->b1 * m[e] + t->nb1 * g[e];
    v[e] = t->b2 * v[e] + t->nb2 * g[e] * g[e];
    r[e] = EIGHT ? sqrtf(v[e]) : __builtin_amdgcn_sqrtf(v[e]);
    p[e] -= t->decay * p[e];
    p[e] -= t->size * m[e] * __builtin_amdgcn_rcpf(r[e] * t->root + t->eps);
    if (e >= left) m[e] = v[e] = r[e] = p[e] = 0.0f;  // (past the tensor's end: zeros, as the states began)
  }
  adam_store<PT>(t->p, in, left, t->plain, p);
  if (MASTER) *(SMLM_GLOBAL f32x4*)(a.master + at) = p;
  if (!EIGHT) {
    *(SMLM_GLOBAL f32x4*)((float*)a.m + at) = m;
    *(SMLM_GLOBAL f32x4*)((float*)a.v + at) = v;
    return;
  }
  float most_m = 0.0f, most_r = 0.0f, mb, mi, rb, ri;
#pragma unroll
  for (int e = 0; e < 4; ++e) most_m = max_or_nan(most_m, fabsf(m[e])), most_r = max_or_nan(most_r, r[e]);
  const float sm = scale8(wave_max(most_m), mb, mi), sr = scale8(wave_max(most_r), rb, ri);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    m[e] = divide8(m[e], mb, mi);
    const float q = divide8(r[e], rb, ri);
    r[e] = r[e] > 0.0f && q < 0x1p-9f && ri != 0.0f ? 0x1p-9f : q;
  }
  *((SMLM_GLOBAL uint32_t*)a.m + (at >> 2)) = pack8(m[0], m[1], m[2], m[3]);
  *((SMLM_GLOBAL uint32_t*)a.v + (at >> 2)) = pack8(r[0], r[1], r[2], r[3]);
  if (lane == 0) a.m_scale[b] = sm, a.v_scale[b] = sr;
}

}  // namespace smlm
