// Softmax cross entropy of a batch's rows against a vocabulary's matrix, and its gradients, without the logits in memory (the
// reference makes all of them and calls torch's loss a train partition: src/loquetier_src/models/mixed_llama.py:382-415).
//
//   z[t, v] = x[t] . w[v],  lse[t] = log sum_v exp z[t, v],  loss[t] = lse[t] - z[t, label[t]]
//   G[t, v] = c[t] (exp(z[t, v] - lse[t]) - [v == label[t]]),  dx = G w,  dw = G^T x
//
// Rows without a label cost nothing but their zeros: the labelled ones are numbered on the device, copied side by side where they
// are not already, and everything below runs over these n rows.  The forward multiplies tile by tile and keeps of each tile its
// rows' maximum and sum; the backward makes the logits again, a piece of the vocabulary at a time, turns them into G in 16 bits,
// and multiplies that with w and x.  All three are gemm_tile's products, bound by the matrix cores from some hundred rows on and by
// the reading of w below.
//
// G's rounding: half a step of 16 bits an entry, as any product of 16-bit operands has it.  In fp16 G is held 2^15 times as large,
// relative to the largest |c|: probabilities of a large vocabulary lie below fp16's normal numbers.
#pragma once
#include "gemm_tile.hpp"
#include "wave_scan.hpp"

namespace smlm {

constexpr int kLossTileV = 256;   // vocabulary entries a workgroup
constexpr int kLossRows = 256;    // rows a workgroup where there are many
constexpr int kLossFewRows = 64;  // ... and where all fit one tile of these
constexpr int kLossScanThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What the labelled rows are numbered into; n = count[0].
struct LossRows {
  int32_t* count;    // [1]
  int32_t* row;      // [T] row of the batch
  int32_t* label;    // [T]
  int32_t* number;   // [T] of a row of the batch, -1: none (backward)
  float* coef;       // [T] c, in fp16 relative to `unit` (backward)
  float* lse2;       // [T] lse in powers of two (backward)
  float* unit;       // [1] what gradients are multiplied with in the end (backward)
  uint16_t* x;       // [n, H] the rows side by side, unless n == T
};

struct LossScanArgs {
  LossRows to;
  const int64_t* labels;  // [T]
  float* loss;            // [T], zeros where there is no label (forward)
  float* lse;             // [T] (forward: written; backward: read)
  const float* grad;      // [T], or [P] (backward)
  const int32_t* partition;  // [P + 1] or NULL
  const float* weight;       // [P] (backward)
  int T, V, P, f16;
};

// Index of the partition that row t lies in, -1: none.
__device__ __forceinline__ int loss_partition(const int32_t* partition, int P, int t) {
  if (t < partition[0]) return -1;
  int lo = 0, hi = P;  // partition[lo] <= t < partition[hi]
  if (t >= partition[P]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (partition[mid] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

// One workgroup numbers the rows in order; a thread takes kLossScanEach rows in turn.
constexpr int kLossScanEach = 4;
template <bool BWD>
__global__ __launch_bounds__(kLossScanThreads) void loss_scan_kernel(LossScanArgs a) {
  __shared__ int32_t waves[kLossScanThreads / 64];
  __shared__ float most[kLossScanThreads / 64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int before = 0;
  float top = 0.0f;
  for (int base = 0; base < a.T; base += kLossScanThreads * kLossScanEach) {
    int64_t label[kLossScanEach];
    float c[kLossScanEach];
    int mine = 0;
    const int t0 = base + (int)threadIdx.x * kLossScanEach;
#pragma unroll
    for (int e = 0; e < kLossScanEach; ++e) {
      const int t = t0 + e;
      label[e] = t < a.T ? a.labels[t] : -1;
      c[e] = 0.0f;
      bool ok = label[e] >= 0 && label[e] < a.V;
      if (ok && a.partition) {
        const int p = loss_partition(a.partition, a.P, t);
        ok = p >= 0;
        if (BWD && ok) c[e] = a.grad[p] * a.weight[p];
      } else if (BWD && ok) {
        c[e] = a.grad[t];
      }
      if (BWD && c[e] == 0.0f) ok = false;  // (nothing hangs on this row)
      if (!ok) label[e] = -1;
      mine += ok;
      if (BWD && fabsf(c[e]) < INFINITY) top = fmaxf(top, fabsf(c[e]));
    }
    int upto = wave_scan(mine);
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    int at = before + upto - mine, all = 0;
    for (int w = 0; w < kLossScanThreads / 64; ++w) {
      if (w < wave) at += waves[w];
      all += waves[w];
    }
    before += all;
#pragma unroll
    for (int e = 0; e < kLossScanEach; ++e) {
      const int t = t0 + e;
      if (t >= a.T) break;
      const bool ok = label[e] >= 0;
      if (BWD) a.to.number[t] = ok ? at : -1;
      if (!BWD && !ok) a.loss[t] = 0.0f, a.lse[t] = 0.0f;
      if (!ok) continue;
      a.to.row[at] = t;
      a.to.label[at] = (int32_t)label[e];
      if (BWD) a.to.coef[at] = c[e], a.to.lse2[at] = a.lse[t] * kLog2e;
      ++at;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) a.to.count[0] = before;
  if (BWD) {
    for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d, kWaveSize));
    if (lane == 0) most[wave] = top;
    __syncthreads();
    for (int w = 0; w < kLossScanThreads / 64; ++w) top = fmaxf(top, most[w]);
    const bool turn = a.f16 && top > 0.0f;
    if (threadIdx.x == 0) a.to.unit[0] = turn ? top * 0x1p-15f : 1.0f;
    if (turn)  // (dividing first: neither quotient nor product leaves the floats)
      for (int i = threadIdx.x; i < before; i += kLossScanThreads) a.to.coef[i] = a.to.coef[i] / top * 0x1p15f;
  }
}

struct LossGatherArgs {
  LossRows rows;
  const uint16_t* x;
  int T, H;
};
// A wave a row.
__global__ __launch_bounds__(256) void loss_gather_kernel(LossGatherArgs a) {
  const int n = uload(a.rows.count, 0), lane = threadIdx.x & 63;
  if (n == a.T) return;
  for (int i = (int)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (int)gridDim.x * 4) {
    const uint16_t* from = a.x + (int64_t)a.rows.row[i] * a.H;
    uint16_t* to = a.rows.x + (int64_t)i * a.H;
    for (int c = lane * 8; c < a.H; c += 512) stg16(to + c, ldg16(from + c));
  }
}

struct LossTileArgs {
  LossRows rows;
  const uint16_t* x;  // [T, H]
  const uint16_t* w;  // [V, H]
  float* part;        // [parts][pad][2] a row's maximum and sum of a part of the vocabulary (forward)
  float* at_label;    // [pad] (forward)
  uint16_t* g;        // [n, ldg] (backward)
  float* dx;          // [splits][n, H] (backward)
  uint16_t* dw;       // [V, H] (backward)
  int T, H, V, pad;
  int v0, v1, ldg;    // the piece of the vocabulary
  int most_splits, add;
};

__device__ __forceinline__ const uint16_t* loss_x(const LossTileArgs& a, int n) { return n == a.T ? a.x : a.rows.x; }

// Which tiles a workgroup takes: workgroups go to the eight XCDs in turn, and each XCD takes a run of the tiles, eight row tiles by
// the next after another, so that its L2 holds what its 32 workgroups share (8 x 4 tiles: 12 operands' stages for 32 workgroups).
struct LossUnit {
  int rows, other;
  bool any;
};
__device__ __forceinline__ LossUnit loss_unit(int n_rows, int n_other) {
  const int units = n_rows * n_other, per = (units + 7) >> 3;
  const int local = (int)blockIdx.x >> 3, u = ((int)blockIdx.x & 7) * per + local;
  if (local >= per || u >= units) return {0, 0, false};
  const int group = u / (8 * n_other), in = u - group * 8 * n_other, wide = min(8, n_rows - group * 8);
  return {group * 8 + in % wide, in / wide, true};
}

template <int IA, int JB>
__device__ __forceinline__ void loss_zero(f32x16 (&acc)[IA][JB]) {
#pragma unroll
  for (int i = 0; i < IA; ++i)
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
}

// A wave's sums as 16-bit rows of memory: row b of out + (b of the wave's first) * ld, IA * 32 columns, through LDS so that a row's
// pieces leave together.  lds: IA * JB * 1024 elements of the wave's own, nobody reading or loading there.
template <int DT, int IA, int JB>
__device__ __forceinline__ void loss_store(const f32x16 (&acc)[IA][JB], uint16_t* lds, uint16_t* out, int64_t ld, int rows, int cols) {
  constexpr int kPieces = IA * 4, kWide = IA * 32;
  const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < JB; ++j) {
    const int row = j * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < IA; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        u32x2 two;
        two[0] = pack2<DT>(acc[i][j][e], acc[i][j][e + 1]);
        two[1] = pack2<DT>(acc[i][j][e + 2], acc[i][j][e + 3]);
        *(u32x2*)(lds + row * kWide + (((i * 4 + (e >> 2)) ^ (row & (kPieces - 1))) << 3) + h * 4) = two;
      }
  }
  // (a wave reads what itself wrote: the compiler waits for the writes)
#pragma unroll 4
  for (int r0 = 0; r0 < JB * 32; r0 += 64 / kPieces) {
    const int row = r0 + lane / kPieces, piece = lane % kPieces;
    const u32x4 v = *(const u32x4*)(lds + row * kWide + ((piece ^ (row & (kPieces - 1))) << 3));
    if (row < rows && piece * 8 < cols) stg16(out + (int64_t)row * ld + piece * 8, v);
  }
}

// Waits until nobody reads the stages and no load to them is on its way.
__device__ __forceinline__ void loss_lds_free() {
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
}

// The logits' tiles.  FEW: one tile of kLossFewRows rows holds all of them.  GRAD: they become G, otherwise their rows' statistics.
template <int DT, bool FEW, bool GRAD>
__global__ __launch_bounds__(256, 1) void loss_logits_kernel(LossTileArgs a) {
  constexpr int WA = FEW ? 4 : 2, IA = FEW ? 2 : 4, WB = FEW ? 1 : 2, JB = FEW ? 2 : 4;
  typedef GemmShape<WA, IA, false, WB, JB, false> S;
  __shared__ __align__(16) uint16_t lds[2 * S::kStage];
  const int n = uload(a.rows.count, 0);
  const LossUnit u = loss_unit((n + S::kB - 1) / S::kB, (a.v1 - a.v0 + kLossTileV - 1) / kLossTileV);
  if (!u.any) return;
  f32x16 acc[IA][JB];
  loss_zero(acc);
  const int first_v = a.v0 + u.other * kLossTileV, first_t = u.rows * S::kB;
  gemm_tile<DT, WA, IA, false, WB, JB, false>(acc, lds, GemmOperand{a.w, a.H, a.V}, first_v,
                                              GemmOperand{loss_x(a, n), a.H, n}, first_t, 0, a.H);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int v = first_v + (wave / WB) * IA * 32, t = first_t + (wave % WB) * JB * 32 + (lane & 31);
  const bool ends = v + IA * 32 > a.v1;  // the vocabulary ends inside the wave's part
  if (!GRAD) {
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      const int tj = t + j * 32;
      if (ends) {
#pragma unroll
        for (int i = 0; i < IA; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (v + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3) >= a.v1) acc[i][j][e] = -INFINITY;
      }
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
      m = fmaxf(m, __shfl_xor(m, 32, kWaveSize));
      const float m2 = m == -INFINITY ? 0.0f : m * kLog2e;
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) l += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -m2));
      l += __shfl_xor(l, 32, kWaveSize);
      const bool there = tj < n;
      const int at = there ? a.rows.label[tj] - v : -1;
      if (__ballot(at >= 0 && at < IA * 32)) {
        float z = 0.0f;
        bool here = false;
#pragma unroll
        for (int i = 0; i < IA; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at == i * 32 + 8 * (e >> 2) + 4 * h + (e & 3)) z = acc[i][j][e], here = true;
        if (here) a.at_label[tj] = z;
      }
      if (there && h == 0) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        *(SMLM_GLOBAL f32x2_t*)(a.part + ((int64_t)(u.other * WA + wave / WB) * a.pad + tj) * 2) = f32x2_t{m == -INFINITY ? m : m2, l};
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      const int tj = min(t + j * 32, n - 1);
      const float c = a.rows.coef[tj], lse2 = a.rows.lse2[tj];
      const int at = a.rows.label[tj] - v - 4 * h;
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -lse2)) * c;
      if (__ballot(at >= -4 && at < IA * 32)) {
#pragma unroll
        for (int i = 0; i < IA; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[i][j][e] -= at == i * 32 + 8 * (e >> 2) + (e & 3) ? c : 0.0f;
      }
      if (ends) {
#pragma unroll
        for (int i = 0; i < IA; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (v + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3) >= a.v1) acc[i][j][e] = 0.0f;
      }
    }
    loss_lds_free();
    const int row = first_t + (wave % WB) * JB * 32;
    loss_store<DT>(acc, lds + wave * IA * JB * 1024, a.g + (int64_t)row * a.ldg + (v - a.v0), a.ldg, n - row, IA * 32);
  }
}

// How many parts the vocabulary's axis of dx is cut into: as many as leave no compute unit without a tile.
__device__ __host__ __forceinline__ int loss_splits(int row_tiles, int h_tiles, int most) {
  const int tiles = row_tiles * h_tiles;
  if (tiles <= 0) return 1;
  const int s = 256 / tiles;
  return s < 1 ? 1 : s > most ? most : s;
}

// dx's sums over a piece of the vocabulary (added to what is there already with `add`), in float.
template <int DT, bool FEW>
__global__ __launch_bounds__(256, 1) void loss_dx_kernel(LossTileArgs a) {
  constexpr int WA = FEW ? 4 : 2, IA = FEW ? 2 : 4, WB = FEW ? 1 : 2, JB = FEW ? 2 : 4;
  typedef GemmShape<WA, IA, true, WB, JB, false> S;
  __shared__ __align__(16) uint16_t lds[2 * S::kStage];
  const int n = uload(a.rows.count, 0);
  const int row_tiles = (n + S::kB - 1) / S::kB, h_tiles = (a.H + S::kA - 1) / S::kA;
  const int splits = loss_splits(row_tiles, h_tiles, a.most_splits);
  const LossUnit u = loss_unit(row_tiles, h_tiles * splits);
  if (!u.any) return;
  const int split = u.other / h_tiles, first_h = (u.other - split * h_tiles) * S::kA, first_t = u.rows * S::kB;
  const int stages = (a.v1 - a.v0 + kGemmK - 1) / kGemmK, each = (stages + splits - 1) / splits;
  const int k0 = min(split * each, stages) * kGemmK, k1 = min((split + 1) * each, stages) * kGemmK;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  float* out = a.dx + (int64_t)split * n * a.H;
  const int hh = first_h + (wave / WB) * IA * 32 + 4 * h, t = first_t + (wave % WB) * JB * 32 + (lane & 31);
  f32x16 acc[IA][JB];
  loss_zero(acc);
  if (a.add) {
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          if (t + j * 32 < n && hh + i * 32 + 2 * e < a.H) {
            const f32x4 v = ldg_f4(out + (int64_t)(t + j * 32) * a.H + hh + i * 32 + 2 * e);
            acc[i][j][e] = v[0], acc[i][j][e + 1] = v[1], acc[i][j][e + 2] = v[2], acc[i][j][e + 3] = v[3];
          }
  }
  gemm_tile<DT, WA, IA, true, WB, JB, false>(acc, lds, GemmOperand{a.w + (int64_t)a.v0 * a.H, a.H, a.V - a.v0}, first_h,
                                             GemmOperand{a.g, a.ldg, n}, first_t, k0, k1);
#pragma unroll
  for (int j = 0; j < JB; ++j)
#pragma unroll
    for (int i = 0; i < IA; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        if (t + j * 32 < n && hh + i * 32 + 2 * e < a.H)
          *(SMLM_GLOBAL f32x4*)(out + (int64_t)(t + j * 32) * a.H + hh + i * 32 + 2 * e) =
              f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
}

// dw's rows of a piece of the vocabulary.
template <int DT>
__global__ __launch_bounds__(256, 1) void loss_dw_kernel(LossTileArgs a) {
  constexpr int WA = 2, IA = 4, WB = 2, JB = 4;
  typedef GemmShape<WA, IA, true, WB, JB, true> S;
  __shared__ __align__(16) uint16_t lds[2 * S::kStage];
  const int n = uload(a.rows.count, 0);
  const LossUnit u = loss_unit((a.H + S::kA - 1) / S::kA, (a.v1 - a.v0 + S::kB - 1) / S::kB);
  if (!u.any) return;
  f32x16 acc[IA][JB];
  loss_zero(acc);
  const int first_h = u.rows * S::kA, first_v = u.other * S::kB;
  gemm_tile<DT, WA, IA, true, WB, JB, true>(acc, lds, GemmOperand{loss_x(a, n), a.H, n}, first_h, GemmOperand{a.g, a.ldg, n},
                                            first_v, 0, n);
  const float unit = uload(a.rows.unit, 0);
#pragma unroll
  for (int i = 0; i < IA; ++i)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[i][j] *= unit;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hh = first_h + (wave / WB) * IA * 32, v = a.v0 + first_v + (wave % WB) * JB * 32;
  loss_lds_free();
  loss_store<DT>(acc, lds + wave * IA * JB * 1024, a.dw + (int64_t)v * a.H + hh, a.H, a.v1 - v, a.H - hh);
}

struct LossFoldArgs {
  LossRows rows;
  const float* part;      // [parts][pad][2]
  const float* at_label;
  float* loss;
  float* lse;
  int parts, pad;
};
// Sixteen rows a workgroup, sixteen threads a row: a line of sixteen rows' parts a load.
__global__ __launch_bounds__(256) void loss_fold_kernel(LossFoldArgs a) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  __shared__ f32x2_t sums[16][16];
  const int n = uload(a.rows.count, 0), r = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int t = (int)blockIdx.x * 16 + r;
  if ((int)blockIdx.x * 16 >= n) return;
  float m = -INFINITY, l = 0.0f;
  auto join = [&](float m1, float l1) {
    const float top = fmaxf(m, m1), at = top == -INFINITY ? 0.0f : top;
    l = l * __builtin_amdgcn_exp2f(m - at) + l1 * __builtin_amdgcn_exp2f(m1 - at);
    m = top;
  };
  if (t < n)
    for (int p0 = q; p0 < a.parts; p0 += 16 * 8) {
      f32x2_t v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int p = min(p0 + e * 16, a.parts - 1);
        v[e] = *(const SMLM_GLOBAL f32x2_t*)(a.part + ((int64_t)p * a.pad + t) * 2);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (p0 + e * 16 < a.parts) join(v[e][0], v[e][1]);
    }
  sums[q][r] = f32x2_t{m, l};
  __syncthreads();
  if (q || t >= n) return;
  for (int p = 1; p < 16; ++p) join(sums[p][r][0], sums[p][r][1]);
  // (the label's logit meets the maximum in the product that made it: what m lost in rounding is in l, and a certain label's loss is
  // 0 however large the logits are)
  const int row = a.rows.row[t];
  const float log_l = __builtin_amdgcn_logf(l);
  a.lse[row] = (m + log_l) * kLn2;
  a.loss[row] = (__builtin_fmaf(-a.at_label[t], kLog2e, m) + log_l) * kLn2;
}

struct LossMeansArgs {
  const float* loss;         // [T]
  const int64_t* labels;     // [T]
  const int32_t* partition;  // [P + 1]
  float* means;              // [P]
  float* weight;             // [P] one over the labelled rows, 0 where there are none
  int T, V;
};
// A workgroup a partition; the sum in a fixed order.
__global__ __launch_bounds__(1024) void loss_means_kernel(LossMeansArgs a) {
  __shared__ float sums[16];
  __shared__ int counts[16];
  const int from = max(a.partition[blockIdx.x], 0), to = min(a.partition[blockIdx.x + 1], a.T);
  float s = 0.0f;
  int c = 0;
  for (int t = from + (int)threadIdx.x; t < to; t += 1024) {
    const int64_t label = a.labels[t];
    if (label >= 0 && label < a.V) s += a.loss[t], ++c;
  }
  for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d, kWaveSize), c += __shfl_xor(c, d, kWaveSize);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s, counts[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < 16; ++w) s += sums[w], c += counts[w];
  const float weight = c ? 1.0f / (float)c : 0.0f;
  a.means[blockIdx.x] = c ? s / (float)c : 0.0f;
  a.weight[blockIdx.x] = weight;
}

struct LossDxFoldArgs {
  LossRows rows;
  const float* part;  // [splits][n, H]
  uint16_t* dx;       // [T, H]
  int T, H, few, most_splits;
};
// A wave a row of the batch: its parts summed in order, rounded once; zeros without a label.
template <int DT>
__global__ __launch_bounds__(256) void loss_dx_fold_kernel(LossDxFoldArgs a) {
  const int n = uload(a.rows.count, 0), lane = threadIdx.x & 63, tile = a.few ? kLossFewRows : kLossRows;
  const int splits = loss_splits((n + tile - 1) / tile, (a.H + 255) / 256, a.most_splits);
  const float unit = uload(a.rows.unit, 0);
  const int t = (int)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  const int i = a.rows.number[t];
  uint16_t* to = a.dx + (int64_t)t * a.H;
  for (int c = lane * 8; c < a.H; c += 512) {
    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    if (i >= 0)
      for (int s = 0; s < splits; ++s) {
        const float* p = a.part + ((int64_t)s * n + i) * a.H + c;
        lo += ldg_f4(p);
        hi += ldg_f4(p + 4);
      }
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      o[e] = pack2<DT>(lo[2 * e] * unit, lo[2 * e + 1] * unit);
      o[2 + e] = pack2<DT>(hi[2 * e] * unit, hi[2 * e + 1] * unit);
    }
    stg16(to + c, o);
  }
}

}  // namespace smlm
