// Norms of queries and keys by head and their rotation by position, in one pass, forward and backward, and the
// serving form that also writes keys and values to a cache's pages.
//
//   y = x * r * w, r = 1 / sqrt(mean(x^2) + eps) over the head's D dimensions (no weight: y = x)
//   o[j] = y[j] c_j - y[j + h] s_j,  o[j + h] = y[j + h] c_j + y[j] s_j for j < h = rot / 2,  o[j] = y[j] for j >= rot
// and from the gradient g of o, with gy the rotation of g by the opposite angle:
//   dx = r (gy w - x r^2 mean(gy w x)),  dw = sum over rows and heads of gy x r
// Arithmetic in float, rounded once; r is made again in the backward, which reads x anyway, so nothing is saved.
//
// Streaming kernels, bound by HBM: 2 bytes read and 2 written an element (backward: 4 and 2), and by launch latency
// for decode batches.  2112 rows of 32 + 32 + 32 heads of 128 with norms into a cache 20 us (5.2 TB/s, as a plain copy of that size); 4096
// rows of 32 + 8 heads 19 us forward, 25.0 + 3.4 us backward (5.2 TB/s); 256 rows without norms into a cache 3.4 to 3.8 us.  Outputs are stored
// non-temporally (24.7 -> 21.0 us at 2112 rows): they would push out of L2 what is still to be read.  A head takes D / 16 lanes (rounded up to a power of two), each with two pieces of eight
// dimensions that are partners in the rotation, so that the pairs meet inside a lane and only the norm's sum crosses
// lanes.  A wave keeps one row: cosines and sines of its position are read once for all the heads it takes.
#pragma once
#include "smlm_common.hpp"

namespace smlm {

constexpr int kRopeMaxDim = 512;

struct HeadsView {      // [rows, heads, D] with free strides (elements), the head's dimensions next to each other
  uint16_t* data;
  int64_t row, head;
};

struct QkRopeArgs {
  HeadsView q, k, v, q_out, k_out;      // v, k_out: data may be null
  const uint16_t *wq, *wk;              // [D] or null: no norm
  const float* table;                   // [n_pos, rot]: rot / 2 cosines, then rot / 2 sines
  const int32_t* pos;                   // [T]; below 0: a row of padding, its outputs are zero; n_pos and more: NaN
  uint16_t *k_cache, *v_cache;          // or null
  const int64_t* slots;                 // [T] page * page_size + place; outside [0, n_slots): the row is not written
  int64_t c_page, c_head, c_slot;       // strides of the caches
  int T, Hq, Hkv, D, rot, n_pos, page_size, n_slots;
  int lanes_log2;                       // lanes a head
  int runs, parts;                      // runs of heads a wave, waves a row
  float eps, sign;                      // sign: -1 turns the other way
};

template <int DT>
__device__ __forceinline__ void unpack8f(u32x4 v, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[2 * e] = Num<DT>::lo(v[e]), f[2 * e + 1] = Num<DT>::hi(v[e]);
}
template <int DT>
__device__ __forceinline__ u32x4 pack8f(const float (&f)[8]) {
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = pack2<DT>(f[2 * e], f[2 * e + 1]);
  return v;
}

// the first dimensions of a lane's two pieces
__device__ __forceinline__ void rope_pieces(int lane, int rot, int& c0, int& c1) {
  const int pairs = rot >> 4;
  c0 = lane < pairs ? lane * 8 : rot + (lane - pairs) * 16;
  c1 = lane < pairs ? (rot >> 1) + lane * 8 : c0 + 8;
}

// cosines and sines of a lane's pairs at a row's position (1 and 0 where the lane's dimensions are not rotated)
__device__ __forceinline__ void rope_angles(const float* table, int pos, int n_pos, int rot, int lane, float sign, float (&c)[8],
                                            float (&s)[8]) {
  const bool in = pos >= 0 && pos < n_pos && lane < (rot >> 4);
  if (in) {
    const float* row = table + (int64_t)pos * rot + lane * 8;
    const f32x4 c0 = ldg_f4(row), c1 = ldg_f4(row + 4), s0 = ldg_f4(row + (rot >> 1)), s1 = ldg_f4(row + (rot >> 1) + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = c0[e], c[4 + e] = c1[e], s[e] = sign * s0[e], s[4 + e] = sign * s1[e];
  } else {
    const float nan = __builtin_nanf("");
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = pos >= n_pos ? nan : 1.0f, s[e] = 0.0f;
  }
}

__device__ __forceinline__ float group_sum(float x, int lanes_log2) {
  for (int d = 0; d < lanes_log2; ++d) x += __shfl_xor(x, 1 << d, kWaveSize);
  return x;
}

// A run is as many heads as a wave has groups of lanes (64 / lanes a head); heads are numbered q, then k, then v.  A wave takes
// up to HEADS runs of one row, a row's runs shared out evenly over its waves.
// FULL: every dimension is rotated.
template <int DT, bool NORM, bool FULL, int HEADS>
__global__ __launch_bounds__(256) void qk_rope_kernel(QkRopeArgs a) {
  const int lane = threadIdx.x & 63, ll = a.lanes_log2;
  const int sub = lane & ((1 << ll) - 1), grp = lane >> ll, per = kWaveSize >> ll;
  const int heads = a.Hq + a.Hkv + (a.v_cache ? a.Hkv : 0);
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int row = (int)(unit / a.parts), part = (int)(unit - (int64_t)row * a.parts);
  if (row >= a.T) return;  // (no barrier below)
  const int first = part * a.runs * per;  // of this wave's heads
  const bool lane_on = sub < (a.D >> 4), turns = FULL || sub < (a.rot >> 4);
  int c0, c1;
  rope_pieces(lane_on ? sub : 0, a.rot, c0, c1);
  const int pos = a.pos[row];
  const int64_t slot = a.k_cache ? a.slots[row] : -1;

  u32x4 x0[HEADS], x1[HEADS];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    if (i >= a.runs || first + i * per >= heads) break;  // uniform over the wave
    const int h = min(first + i * per + grp, heads - 1);  // (lanes past the last head read it too)
    const bool is_q = h < a.Hq, is_k = h < a.Hq + a.Hkv;
    const uint16_t* p = is_q ? a.q.data + row * a.q.row + h * a.q.head
                             : (is_k ? a.k.data + row * a.k.row + (h - a.Hq) * a.k.head
                                     : a.v.data + row * a.v.row + (h - a.Hq - a.Hkv) * a.v.head);
    x0[i] = ldg16(p + c0);
    x1[i] = ldg16(p + c1);
  }
  float c[8], s[8];
  rope_angles(a.table, pos, a.n_pos, a.rot, lane_on ? sub : 0, a.sign, c, s);
  u32x4 wq[2], wk[2];
  if (NORM) {
    constexpr uint32_t kOne = DT == SMLM_DTYPE_F16 ? 0x3c003c00u : 0x3f803f80u;
    const u32x4 one = {kOne, kOne, kOne, kOne};
    wq[0] = wq[1] = wk[0] = wk[1] = one;
    if (a.wq) wq[0] = ldg16(a.wq + c0), wq[1] = ldg16(a.wq + c1);
    if (a.wk) wk[0] = ldg16(a.wk + c0), wk[1] = ldg16(a.wk + c1);
  }
  const bool keep = slot >= 0 && slot < a.n_slots && pos >= 0;
  const int page = keep ? (int)slot / a.page_size : 0, at = keep ? (int)slot - page * a.page_size : 0;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    if (i >= a.runs || first + i * per >= heads) break;
    const int h = first + i * per + grp;
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    u32x4 o0 = x0[i], o1 = x1[i];
    if (first + i * per < a.Hq + a.Hkv) {  // (uniform: a run of values alone is a copy)
      float f0[8], f1[8], cr[8], sr[8];
      unpack8f<DT>(x0[i], f0);
      unpack8f<DT>(x1[i], f1);
      float r = 1.0f;
      if (NORM) {
        float ss = 0.0f, w0[8], w1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += f0[e] * f0[e] + f1[e] * f1[e];
        ss = group_sum(lane_on ? ss : 0.0f, ll);
        if (is_q ? a.wq : a.wk) r = 1.0f / sqrtf(ss / (float)a.D + a.eps);
        unpack8f<DT>(is_q ? wq[0] : wk[0], w0);
        unpack8f<DT>(is_q ? wq[1] : wk[1], w1);
#pragma unroll
        for (int e = 0; e < 8; ++e) f0[e] *= w0[e], f1[e] *= w1[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) cr[e] = NORM ? c[e] * r : c[e], sr[e] = NORM ? s[e] * r : s[e];
      float g0[8], g1[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g0[e] = f0[e] * cr[e] - (turns ? f1[e] * sr[e] : 0.0f);  // (0 times an infinity beside it would be NaN)
        g1[e] = f1[e] * cr[e] + (turns ? f0[e] * sr[e] : 0.0f);
      }
      if (!is_v) o0 = pack8f<DT>(g0), o1 = pack8f<DT>(g1);
    }
    if (pos < 0) o0 = u32x4{0u, 0u, 0u, 0u}, o1 = o0;
    if (!lane_on || h >= heads) continue;
    const int hk = is_v ? h - a.Hq - a.Hkv : h - a.Hq;
    if (is_q || (!is_v && a.k_out.data)) {
      uint16_t* p = is_q ? a.q_out.data + row * a.q_out.row + h * a.q_out.head : a.k_out.data + row * a.k_out.row + hk * a.k_out.head;
      stg16_nt(p + c0, o0);
      stg16_nt(p + c1, o1);
    }
    if (!is_q && keep) {
      uint16_t* p = (is_v ? a.v_cache : a.k_cache) + page * a.c_page + hk * a.c_head + at * a.c_slot;
      stg16_nt(p + c0, o0);
      stg16_nt(p + c1, o1);
    }
  }
}

struct QkRopeBwdArgs {
  HeadsView g, x, dx;      // of q or of k
  const uint16_t* w;       // [D]
  const float* table;
  const int32_t* pos;
  float* partial;          // [gridDim.x of this launch's part, D]
  int T, H, D, rot, n_pos, lanes_log2, blocks, first_block;
  float eps;
};
struct QkRopeBwdPair {
  QkRopeBwdArgs part[2];   // q's workgroups, then k's
};

// The backward behind a norm.  A workgroup of four waves walks the rows of q or of k; a lane keeps its sixteen
// dimensions' share of dw in registers over all rows and heads it meets.
// (Two runs of heads on their way together take a wave a SIMD its registers: 33 us where this takes 26, 4096 rows of 32 and 8 heads of 128.)
template <int DT>
__global__ __launch_bounds__(256) void qk_rope_bwd_kernel(QkRopeBwdPair both) {
  __shared__ float red[4][kRopeMaxDim];
  const QkRopeBwdArgs a = both.part[(int)blockIdx.x >= both.part[1].first_block ? 1 : 0];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ll = a.lanes_log2;
  const int sub = lane & ((1 << ll) - 1), grp = lane >> ll, per = kWaveSize >> ll;
  const int block = (int)blockIdx.x - a.first_block;
  const bool lane_on = sub < (a.D >> 4), turns = sub < (a.rot >> 4);
  int c0, c1;
  rope_pieces(lane_on ? sub : 0, a.rot, c0, c1);
  float w0[8], w1[8], dw0[8], dw1[8];
  unpack8f<DT>(ldg16(a.w + c0), w0);
  unpack8f<DT>(ldg16(a.w + c1), w1);
#pragma unroll
  for (int e = 0; e < 8; ++e) dw0[e] = dw1[e] = 0.0f;
  const float inv = 1.0f / (float)a.D;
  for (int row = block * 4 + wave; row < a.T; row += a.blocks * 4) {
    const int pos = a.pos[row];
    float c[8], s[8];
    rope_angles(a.table, pos, a.n_pos, a.rot, lane_on ? sub : 0, -1.0f, c, s);
    for (int h0 = 0; h0 < a.H; h0 += per) {
      const int h = h0 + grp, hc = min(h, a.H - 1);  // (lanes past the last head read it too)
      const uint16_t* xp = a.x.data + row * a.x.row + hc * a.x.head;
      const uint16_t* gp = a.g.data + row * a.g.row + hc * a.g.head;
      float x0[8], x1[8], g0[8], g1[8], ss = 0.0f, dot = 0.0f, y0[8], y1[8];
      unpack8f<DT>(ldg16(xp + c0), x0);
      unpack8f<DT>(ldg16(xp + c1), x1);
      unpack8f<DT>(ldg16(gp + c0), g0);
      unpack8f<DT>(ldg16(gp + c1), g1);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y0[e] = g0[e] * c[e] - (turns ? g1[e] * s[e] : 0.0f);
        y1[e] = g1[e] * c[e] + (turns ? g0[e] * s[e] : 0.0f);
        ss += x0[e] * x0[e] + x1[e] * x1[e];
        dot += y0[e] * w0[e] * x0[e] + y1[e] * w1[e] * x1[e];
      }
      ss = group_sum(lane_on ? ss : 0.0f, ll);
      dot = group_sum(lane_on ? dot : 0.0f, ll);
      if (!lane_on || h >= a.H) continue;
      const float r = 1.0f / sqrtf(ss * inv + a.eps), coef = dot * inv * r * r;
      u32x4 o0 = {0u, 0u, 0u, 0u}, o1 = o0;
      if (pos >= 0) {
        float d0[8], d1[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          d0[e] = r * (y0[e] * w0[e] - x0[e] * coef);
          d1[e] = r * (y1[e] * w1[e] - x1[e] * coef);
          dw0[e] += y0[e] * x0[e] * r;
          dw1[e] += y1[e] * x1[e] * r;
        }
        o0 = pack8f<DT>(d0);
        o1 = pack8f<DT>(d1);
      }
      uint16_t* dp = a.dx.data + row * a.dx.row + h * a.dx.head;
      stg16_nt(dp + c0, o0);
      stg16_nt(dp + c1, o1);
    }
  }
  // the heads' groups of lanes, then the four waves, always in the same order
#pragma unroll
  for (int e = 0; e < 8; ++e)
    for (int d = ll; d < 6; ++d) {
      dw0[e] += __shfl_xor(dw0[e], 1 << d, kWaveSize);
      dw1[e] += __shfl_xor(dw1[e], 1 << d, kWaveSize);
    }
  if (grp == 0 && lane_on)
#pragma unroll
    for (int e = 0; e < 8; ++e) red[wave][c0 + e] = dw0[e], red[wave][c1 + e] = dw1[e];
  __syncthreads();
  for (int j = threadIdx.x; j < a.D; j += 256)
    a.partial[(int64_t)block * a.D + j] = (red[0][j] + red[1][j]) + (red[2][j] + red[3][j]);
}

struct QkRopeFoldArgs {
  uint16_t* dw[2];
  const float* partial[2];
  int n_part[2];
  int D, blocks;           // workgroups a tensor
};

// dw from the workgroups' sums, sixteen columns a workgroup: a thread adds every 64th row of four columns, eight rows on their way
// at a time, and the 64 sums are added in order of a tree.
template <int DT>
__global__ __launch_bounds__(256) void qk_rope_fold_kernel(QkRopeFoldArgs a) {
  __shared__ f32x4 red[64][4];
  const int t = (int)blockIdx.x / a.blocks, c4 = threadIdx.x & 3, r = threadIdx.x >> 2;
  const int col = ((int)blockIdx.x - t * a.blocks) * 16;
  const float* from = a.partial[t] + col + c4 * 4;
  const int n = a.n_part[t];
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int p = r; p < n; p += 64 * 8) {
    f32x4 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ldg_f4(from + (int64_t)(p + 64 * j < n ? p + 64 * j : r) * a.D);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (p + 64 * j < n) s += v[j];
  }
  red[r][c4] = s;
  for (int d = 32; d >= 1; d >>= 1) {
    __syncthreads();
    if (r < d) red[r][c4] += red[r + d][c4];
  }
  if (r == 0) {
    const f32x4 v = red[0][c4];
    *(SMLM_GLOBAL u32x2*)(a.dw[t] + col + c4 * 4) = u32x2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
  }
}

}  // namespace smlm
