// Softmax cross entropy of a batch's rows against a vocabulary's matrix, and its gradients, without the logits in memory (the
// reference makes all of them and calls torch's loss a train partition: src/loquetier_src/models/mixed_llama.py:382-415).
//
//   z[t, v] = x[t] . w[v],  lse[t] = log sum_v exp z[t, v],  loss[t] = lse[t] - z[t, label[t]]
//   G[t, v] = c[t] (exp(z[t, v] - lse[t]) - [v == label[t]]),  dx = G w,  dw = G^T x
//
// Rows without a label cost nothing but their zeros: the labelled ones are numbered on the device, copied side by side where they
// are not already, and everything below runs over these n rows.  All products are gemm_tile's, bound by the matrix cores from some
// hundred rows on and by the reading of w below.
//
// The loss alone: tile by tile, of each row and 128 (64) entries of the vocabulary the sum of exponentials against a whole power of two.
//
// The loss and the gradient of x (the usual fine-tuning step: the vocabulary's matrix is frozen) take two products, no third that makes the
// logits again: dx is linear in c, so what it needs is sum_v exp(z - ref) w[v] and sum_v exp(z - ref), and ref need not be the maximum.
// A piece of the vocabulary at a time the exponentials are stored in 16 bits, each row's against its reference of the pieces
// before, and multiplied with w.  Where the piece outgrows the reference (or there is none yet) a part is stored against its own,
// and turned to the row's new one before the product, as the sums so far are: references are whole powers of two, so turning rounds
// nothing but what it takes down among fp16's subnormal numbers.  The backward divides and multiplies with c.
//
// With the gradient of w the backward makes the logits again, by piece, turns them into G in 16 bits, and multiplies that with w and x.
//
// The label has no part in the sums and the 16-bit entries: with `others` = sum_{v != label} exp(z - ref) and e = exp(z[label] - ref), the
// loss is log(1 + others / e) and dx = c (sum_{v != label} exp(z - ref) w[v] - others w[label]) / (others + e), the label's share in
// float: where a label is nearly certain nothing cancels, and the gradient is as exact, relative to its size, as anywhere.
//
// Rounding to 16 bits: half a step of each entry, as any product of 16-bit operands has it (of G at the label too, where dw is
// wanted: what dx loses by it is given back in float).  fp16 entries are held 2^15 times as large: probabilities of a large vocabulary lie
// below fp16's normal numbers.  G is held relative to the largest |c|, in fp16 as 2^14 (and rows of far smaller |c| by their own: kLossLeast).
//
// Measured, us (4096 columns; PFLOP/s): 4099 rows of 128256 entries, bf16, logits with exponentials 3977 (1.08), dx 3919 (1.10), fold 65; 2458
// labelled rows of 4096, 32000 entries, 618 (1.04), 708 (0.91), 30; 2048 rows of 32000, fp16, logits 493 (1.09), again for G 494,
// dx 521 (1.03), dw 582 (0.92); 200 rows of 128256 the loss alone 274 (3.8 TB/s of w).
// What bounds the products: a wave a SIMD and a tile a workgroup, so that a tile's first loads and everything after its last product stand alone, with
// the matrix cores busy in 67 to 69 % of a compute unit's cycles (logits), 57 to 60 (dx) and 55 (dw).  The tiles of 256 rows take all 512 registers and
// keep 68 to 264 bytes a lane of the logits' epilogue, 364 of dx's `add`, in scratch memory, outside of the loops: 501 tiles of the losses alone
// write 34 MB where their parts are 2.  The card's power is the bound beyond: the tile alone does 1.23, with zeros 1.75.
#pragma once
#include "gemm_tile.hpp"
#include "rms_norm.hpp"
#include "wave_scan.hpp"

namespace smlm {

constexpr int kLossTileV = 256;   // vocabulary entries a workgroup
constexpr int kLossRows = 256;    // rows a workgroup where there are many
constexpr int kLossFewRows = 64;  // ... and where rows or tiles are few (FEW)
constexpr int kLossScanThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// What the labelled rows are numbered into; n = count[0].
struct LossRows {
  int32_t* count;    // [2] n; whether any `rest` is not 1 (backward)
  int32_t* row;      // [T] row of the batch
  int32_t* label;    // [T]
  int32_t* number;   // [T] of a row of the batch, -1: none (backward)
  float* coef;       // [T] c relative to `unit`, or a power of two (backward)
  float* rest;       // [T] what c is of coef, up to 1, or NULL: all 1 (backward)
  float* lse2;       // [T] lse in powers of two (backward)
  float* own;        // [T] exp(-loss) - 1 (backward)
  float* lost;       // [T] what rounding took from G at the label (backward)
  float* unit;       // [1] what gradients are multiplied with in the end (backward)
  float* ref;        // [T] the power of two that a row's exponentials are taken against
  float* sum;        // [T] of them without the label's; in the end one over their sum with it
  float* share;      // [T] in the end: the part of them that is not the label's
  float* turn;       // [T] what the sums so far are multiplied with
  int32_t* moved;    // [T / 16] whether anything of sixteen rows' entries is to be turned
  uint16_t* x;       // [n, H] the rows side by side, unless n == T
  uint16_t* y;       // [n, H], or [64, H] where G is held twice: the rows times `rest`, for dw (backward; NULL: x will do)
};

struct LossScanArgs {
  LossRows to;
  const int64_t* labels;  // [T]
  float* loss;            // [T] (forward: zeros where there is no label; backward: read)
  float* lse;             // [T] (the same)
  const float* grad;      // [T], or [P] (backward)
  const int32_t* partition;  // [P + 1] or NULL
  const float* weight;       // [P] (backward)
  int T, V, P, f16, number, split;  // number: rows' numbers are wanted; split: coef is a power of two (backward)
};
// fp16's entries of G are multiples of 2^-24, and a coefficient far below the largest, which is 2^14, would leave its row's none.  From 2^-11 of the
// largest down, G therefore takes 2^-11 of it and the rows the rest (rounded for dw; dx takes it in float): G's entries are off by half a step or
// 2^-28 of c, the rows' elements in dw by half a step or 2^-36 of the largest c.
constexpr float kLossLeast = 8.0f;

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
      if (a.number) a.to.number[t] = ok ? at : -1;
      if (!BWD && !ok) a.loss[t] = 0.0f, a.lse[t] = 0.0f;
      if (!ok) continue;
      a.to.row[at] = t;
      a.to.label[at] = (int32_t)label[e];
      if (BWD) a.to.coef[at] = c[e], a.to.lse2[at] = a.lse[t] * kLog2e, a.to.own[at] = expm1f(-a.loss[t]);
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
    const bool turn = top > 0.0f;
    const float up = a.f16 ? 0x1p14f : 1.0f;  // (fp16: out of the subnormal numbers)
    if (threadIdx.x == 0) a.to.unit[0] = turn ? top / up : 1.0f;
    bool any = false;
    for (int i = threadIdx.x; i < before; i += kLossScanThreads) {
      float c = a.to.coef[i];
      if (turn) c = c / top * up;  // (dividing first: neither quotient nor product leaves the floats)
      if (a.to.rest) {
        const float two = 2.0f * __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, c) & 0xff800000u);
        float held = c;
        if (a.f16 && fabsf(c) < kLossLeast) held = copysignf(kLossLeast, c);
        else if (a.split && fabsf(c) < INFINITY && two != 0.0f) held = two;
        const bool plain = !(fabsf(held) > fabsf(c));
        a.to.rest[i] = plain ? 1.0f : c / held;
        c = plain ? c : held;
        any |= !plain;
      }
      a.to.coef[i] = c;
    }
    any = __syncthreads_or(any);
    if (threadIdx.x == 0) a.to.count[1] = any;
  }
}

// Up to 32 rows, where dw is made: G is held as its rounding (rows 0 to 31 of 64) and what that took (32 to 63), both against the same rows of
// x.  In dw a row of w meets one entry of size c, its label's, and rounding is one relative error of all its columns, of all a
// partition's labels even; in a sum of many rows such errors are of random sign, here they would be the result's: 7 rows of 5304 columns
// in fp16 3.2e-4 off for the 2.1e-4 of the output's own rounding.  The second half of a tile of 64 rows, and of a stage of
// 64, is empty otherwise, so it costs nothing.
constexpr int kLossTwice = 32;

// Of a partition's rows c is one number, and its rounding at their labels, where G is nearly -c, would be one error of all of them: in dw up to
// eps / 2, where the output's own rounding is 0.41 of that in the mean square.  So coef is the power of two above c, and dw's other operand, the rows,
// is multiplied with the rest, c / coef, and rounded: errors of random sign, none for the partition of the largest c.  dx takes the rest in float.
// (Nothing is copied for it where every rest is 1.)
struct LossGatherArgs {
  LossRows rows;
  const uint16_t* x;
  int T, H, twice;
};
// Whether dw takes the rows from y.
__device__ __forceinline__ bool loss_y(const LossRows& r, int twice) { return r.y && (twice || uload(r.count, 1)); }
// A wave a row.
template <int DT>
__global__ __launch_bounds__(256) void loss_gather_kernel(LossGatherArgs a) {
  const int n = uload(a.rows.count, 0), lane = threadIdx.x & 63, all = a.twice ? 2 * kLossTwice : n;
  const bool y = loss_y(a.rows, a.twice);
  if (n == a.T && !y) return;
  for (int i = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6); i < all; i += (int)gridDim.x * 4) {
    const int at = a.twice ? i & (kLossTwice - 1) : i;
    const bool none = at >= n;
    const uint16_t* from = a.x + (none ? 0 : (int64_t)a.rows.row[at] * a.H);
    const float rest = none || !a.rows.rest ? 1.0f : a.rows.rest[at];
    for (int c = lane * 8; c < a.H; c += 512) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (!none) v = ldg16(from + c);
      if (n != a.T && i < n) stg16(a.rows.x + (int64_t)i * a.H + c, v);
      if (!y) continue;
      float f[8];
      unpack8<DT>(v, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = pack2<DT>(f[2 * e] * rest, f[2 * e + 1] * rest);
      stg16(a.rows.y + (int64_t)i * a.H + c, v);
    }
  }
}

struct LossTileArgs {
  LossRows rows;
  const uint16_t* x;  // [T, H]
  const uint16_t* w;  // [V, H]
  float* part;        // [parts][pad][2] a row's reference and sum of a part of the vocabulary (forward)
  float* at_label;    // [pad] (forward)
  uint16_t* g;        // [n, ldg] G, or the exponentials
  float* dx;          // [n, H]: sums for dx
  float* cut;         // [parts][tile]: those of tiles whose axis is cut
  uint16_t* dw;       // [V, H] (backward)
  int T, H, V, pad;
  int v0, v1, ldg;    // the piece of the vocabulary
  int stages, add;    // of a whole piece; add: to what is there of dx, turned (`turned`)
  int turned;
  int twice;          // G is held twice (backward, up to kLossTwice rows)
};

__device__ __forceinline__ const uint16_t* loss_x(const LossTileArgs& a, int n) { return n == a.T ? a.x : a.rows.x; }

// Which tiles a workgroup takes: workgroups go to the eight XCDs in turn, and each XCD takes a run of the tiles, four row tiles by
// the next after another, so that its L2 holds what its 32 workgroups share.  (Eight row tiles: 1.16 PFLOP/s for 1.23 at 32000 x 4096 x
// 4096, 1.11 for 1.26 at 8192 x 8192 x 8192; two: 1.17 and 1.10.)
constexpr int kLossGroup = 4;
struct LossUnit {
  int rows, other;
  bool any;
};
__device__ __forceinline__ LossUnit loss_tile(int u, int n_rows, int n_other) {
  const int group = u / (kLossGroup * n_other), in = u - group * kLossGroup * n_other, wide = min(kLossGroup, n_rows - group * kLossGroup);
  return {group * kLossGroup + in % wide, in / wide, true};
}
__device__ __forceinline__ int loss_tile_number(int rows, int other, int n_rows, int n_other) {
  const int group = rows / kLossGroup, wide = min(kLossGroup, n_rows - group * kLossGroup);
  return group * kLossGroup * n_other + other * wide + rows % kLossGroup;
}
__device__ __forceinline__ LossUnit loss_unit(int n_rows, int n_other) {
  const int units = n_rows * n_other, per = (units + 7) >> 3;
  const int local = (int)blockIdx.x >> 3, u = ((int)blockIdx.x & 7) * per + local;
  if (local >= per || u >= units) return {0, 0, false};
  return loss_tile(u, n_rows, n_other);
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

// The same of sums whose operands both lie across: row 4 n + j of the wave's blocks, columns 4 m + i.
template <int DT>
__device__ __forceinline__ void loss_store_across(const f32x16 (&acc)[4][4], uint16_t* lds, uint16_t* out, int64_t ld, int rows, int cols) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = gemm_row<true, 4>(j, lane & 31);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int m = gemm_sum_row(e, lane);
      u32x2 two;
      two[0] = pack2<DT>(acc[0][j][e], acc[1][j][e]);
      two[1] = pack2<DT>(acc[2][j][e], acc[3][j][e]);
      *(u32x2*)(lds + row * 128 + (((m >> 1) ^ ((row >> 2) & 15)) << 3) + (m & 1) * 4) = two;
    }
  }
#pragma unroll 4
  for (int r0 = 0; r0 < 128; r0 += 4) {
    const int row = r0 + (lane >> 4), piece = lane & 15;
    const u32x4 v = *(const u32x4*)(lds + row * 128 + ((piece ^ ((row >> 2) & 15)) << 3));
    if (row < rows && piece * 8 < cols) stg16(out + (int64_t)row * ld + piece * 8, v);
  }
}

// Waits until nobody reads the stages and no load to them is on its way.
__device__ __forceinline__ void loss_lds_free() {
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
}

constexpr int kLossSums = 0, kLossSoft = 1, kLossGrad = 2;  // what becomes of the logits: sums alone, exponentials too, G

// A reference of a part's own is above its maximum by less than one, or by the room that is left for later pieces: bf16 has exponents
// enough for any (60 above), fp16 gets 2^4 at the price of bits of entries below 2^-24 of the maximum: that one is 2^10 to 2^11 against a new
// reference, smaller entries are multiples of 2^-24 and off by 2^-35 of the maximum at most.  bf16's first piece takes 1
// as every row's reference, where the part's maximum is within 2^+-60: a model's logits are, and nothing needs to be turned.  (Of 4099 rows
// of 64128 entries, 0.5 GB: 200 us.)
template <int DT>
constexpr float kLossRoom = DT == SMLM_DTYPE_F16 ? 4.0f : 0.0f;
template <int DT>
constexpr float kLossAbove = DT == SMLM_DTYPE_F16 ? 0.0f : 60.0f;
template <int DT>
constexpr float kLossBias = DT == SMLM_DTYPE_F16 ? 15.0f : 0.0f;  // fp16 entries are 2^15 times as large, and so are their sums

// The logits' tiles.
template <int DT, bool FEW, int MODE>
__global__ __launch_bounds__(256, FEW ? 2 : 1) void loss_logits_kernel(LossTileArgs a) {
  constexpr int WA = FEW ? 4 : 2, IA = FEW ? 2 : 4, WB = FEW ? 1 : 2, JB = FEW ? 2 : 4;
  typedef GemmShape<WA, IA, false, WB, JB, false> S;
  __shared__ __align__(16) uint16_t lds[kGemmStages * S::kStage];
  const int n = uload(a.rows.count, 0);
  const LossUnit u = loss_unit((n + S::kB - 1) / S::kB, (a.v1 - a.v0 + kLossTileV - 1) / kLossTileV);
  if (!u.any) return;
  f32x16 acc[IA][JB];
  loss_zero(acc);
  const int first_v = a.v0 + u.other * kLossTileV, first_t = u.rows * S::kB;
  const GemmOperand w{a.w, a.H, a.V}, x{loss_x(a, n), a.H, n};
  // Where w comes from HBM at its rate (few rows), neighbouring workgroups begin at different columns: rows of w are often a multiple of
  // 4 KiB apart, and all workgroups at one column meet in few channels.  (200 rows against 128256 of 4096: 286 us, 254 so; with many
  // rows x is what workgroups at one column share.)
  const int row_tiles = (n + S::kB - 1) / S::kB;
  const int turn = row_tiles * S::kB <= 256 ? (u.other & 15) * (a.H >> 4) / kGemmK * kGemmK : 0;
#pragma unroll 1
  for (int s = 0; s < 2; ++s)
    GemmTile<DT, WA, IA, false, WB, JB, false>::run(acc, lds, w, first_v, x, first_t, s ? 0 : turn, s ? turn : a.H);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
  const int v = first_v + (wave / WB) * IA * 32, t = first_t + (wave % WB) * JB * 32 + (lane & 31);
  const bool ends = v + IA * 32 > a.v1;  // the vocabulary ends inside the wave's part
#pragma unroll
  for (int j = 0; j < JB; ++j) {
    const int tj = t + j * 32, tc = min(tj, n - 1);
    if (ends) {
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (v + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3) >= a.v1) acc[i][j][e] = -INFINITY;
    }
    const int at = a.rows.label[tc] - v - 4 * h;  // the label's place among the lane's logits
    const bool near = __ballot(at >= 0 && at < IA * 32) != 0;
    if (MODE != kLossGrad) {
      float m = -INFINITY, l = 0.0f;
      if (near) {
        float z = 0.0f;
        bool here = false;
#pragma unroll
        for (int i = 0; i < IA; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at == i * 32 + 8 * (e >> 2) + (e & 3)) z = acc[i][j][e], acc[i][j][e] = -INFINITY, here = true;
        if (here && tj < n) a.at_label[tj] = z;
      }
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
      m = fmaxf(m, __shfl_xor(m, 32, kWaveSize)) * kLog2e;
      float c = MODE == kLossSoft && a.add ? a.rows.ref[tc] : -INFINITY;
      if (MODE == kLossSoft && DT == SMLM_DTYPE_BF16 && !a.add && fabsf(m) <= kLossAbove<DT>) c = 0.0f;
      if (!(m <= c + kLossAbove<DT>)) c = ceilf(m) + (MODE == kLossSoft ? kLossRoom<DT> : 0.0f);
      const float to = (c == -INFINITY ? 0.0f : c) - (MODE == kLossSoft ? kLossBias<DT> : 0.0f);
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -to));
          if (MODE == kLossSoft) acc[i][j][e] = y;
          l += y;
        }
      l += __shfl_xor(l, 32, kWaveSize);
      if (tj < n && h == 0) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        *(SMLM_GLOBAL f32x2_t*)(a.part + ((int64_t)(u.other * WA + wave / WB) * a.pad + tj) * 2) = f32x2_t{c, l};
      }
    } else {
      const float c = a.rows.coef[tc], lse2 = a.rows.lse2[tc];
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -lse2)) * c;
      if (near) {
        float lost = 0.0f;
        bool here = false;
#pragma unroll
        for (int i = 0; i < IA; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at == i * 32 + 8 * (e >> 2) + (e & 3)) {
              acc[i][j][e] = c * a.rows.own[tc];
              lost = acc[i][j][e] - Num<DT>::lo(pack2<DT>(acc[i][j][e], 0.0f)), here = true;
            }
        if (here && tj < n) a.rows.lost[tj] = lost;
      }
      if (FEW && a.twice) {  // (the tile's first 32 rows are all: what lies in the others is made of them)
#pragma unroll
        for (int i = 0; i < IA; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float y = tj < n ? acc[i][0][e] : 0.0f;
            const float took = y - Num<DT>::lo(pack2<DT>(y, 0.0f));
            acc[i][0][e] = y, acc[i][JB - 1][e] = fabsf(took) < INFINITY ? took : 0.0f;  // (infinities stay what they are)
          }
        break;
      }
    }
  }
  if (MODE != kLossSums) {
    loss_lds_free();
    const int row = first_t + (wave % WB) * JB * 32;
    loss_store<DT>(acc, lds + wave * IA * JB * 1024, a.g + (int64_t)row * a.ldg + (v - a.v0), a.ldg,
                   FEW && MODE == kLossGrad && a.twice ? 2 * kLossTwice : n - row, IA * 32);
  }
}

// The tiles of dx that fill whole rounds of the compute units take the vocabulary's axis whole; of the others it is cut into as many
// parts as take the least time: rounds of a part's stages, and what a part costs to write and add up (a tile of floats, both ways at
// HBM's rate: a 17th of a stage each).  Whatever the piece, the cuts are those of a whole one.
struct LossCuts {
  int whole, parts, rest;  // tiles that are whole; parts of each other; their number
};
constexpr int kLossMostParts = 512;
__host__ __device__ __forceinline__ LossCuts loss_cuts(int tiles, int stages, bool few) {
  const int slots = few ? 512 : 256, rest = tiles % slots;
  int best = 1, least = 0x7fffffff;
  for (int s = 1; s <= 64 && s <= stages && (s == 1 || rest * s <= kLossMostParts); ++s) {
    const int cost = (rest * s + slots - 1) / slots * ((stages + s - 1) / s) * 64 + rest * s * (few ? 1 : 4);
    if (cost < least) least = cost, best = s;
  }
  return best == 1 ? LossCuts{tiles, 1, 0} : LossCuts{tiles - rest, best, rest};
}

// dx's sums over a piece of the vocabulary (added to what is there already with `add`), in float.
template <int DT, bool FEW>
__global__ __launch_bounds__(256, FEW ? 2 : 1) void loss_dx_kernel(LossTileArgs a) {
  constexpr int WA = FEW ? 4 : 2, IA = FEW ? 2 : 4, WB = FEW ? 1 : 2, JB = FEW ? 2 : 4;
  typedef GemmShape<WA, IA, true, WB, JB, false> S;
  typedef float sums __attribute__((ext_vector_type(IA)));
  __shared__ __align__(16) uint16_t lds[kGemmStages * S::kStage];
  const int n = uload(a.rows.count, 0);
  const int row_tiles = (n + S::kB - 1) / S::kB, h_tiles = (a.H + S::kA - 1) / S::kA;
  const LossCuts cuts = loss_cuts(row_tiles * h_tiles, a.stages, FEW);
  // (each XCD takes its share of the whole tiles, then of the parts)
  const int xcd = (int)blockIdx.x & 7, whole = (cuts.whole + 7) >> 3, parts = (cuts.rest * cuts.parts + 7) >> 3;
  int local = (int)blockIdx.x >> 3, tile, part = 0, at = -1;
  if (local < whole) {
    tile = xcd * whole + local;
    if (tile >= cuts.whole) return;
  } else {
    local -= whole;
    const int p = xcd * parts + local;
    if (local >= parts || p >= cuts.rest * cuts.parts) return;
    part = p / cuts.rest;
    at = p - part * cuts.rest;
    tile = cuts.whole + at;
    at = at * cuts.parts + part;
  }
  const LossUnit u = loss_tile(tile, row_tiles, h_tiles);
  const int first_h = u.other * S::kA, first_t = u.rows * S::kB, cols = a.v1 - a.v0;
  const int each = at < 0 ? a.stages : (a.stages + cuts.parts - 1) / cuts.parts;
  const int k0 = min(part * each * kGemmK, cols), k1 = min((part + 1) * each * kGemmK, cols);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  // (a cut tile's sums lie as a tile by itself)
  const int ld = at < 0 ? a.H : S::kA;
  float* out = at < 0 ? a.dx + (int64_t)first_t * a.H + first_h : a.cut + (int64_t)at * S::kA * S::kB;
  const int rows = n - first_t, wide = a.H - first_h;
  const int row0 = (wave % WB) * JB * 32 + (lane & 31), col0 = (wave / WB) * IA * 32;
  f32x16 acc[IA][JB];
  loss_zero(acc);
  if (a.add) {
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      const int row = row0 + j * 32;
      const float turn = a.turned && row < rows ? a.rows.turn[first_t + row] : 1.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int col = col0 + IA * gemm_sum_row(e, lane);
        if (row < rows && col < wide) {
          const sums v = *(const SMLM_GLOBAL sums*)(out + (int64_t)row * ld + col) * turn;
#pragma unroll
          for (int i = 0; i < IA; ++i) acc[i][j][e] = v[i];
        }
      }
    }
  }
  GemmTile<DT, WA, IA, true, WB, JB, false>::run(acc, lds, GemmOperand{a.w + (int64_t)a.v0 * a.H, a.H, a.V - a.v0}, first_h,
                                             GemmOperand{a.g, a.ldg, n}, first_t, k0, k1);
#pragma unroll
  for (int j = 0; j < JB; ++j) {
    const int row = row0 + j * 32;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int col = col0 + IA * gemm_sum_row(e, lane);
      sums v;
#pragma unroll
      for (int i = 0; i < IA; ++i) v[i] = acc[i][j][e];
      if (row < rows && col < wide) *(SMLM_GLOBAL sums*)(out + (int64_t)row * ld + col) = v;
    }
  }
}

// dw's rows of a piece of the vocabulary.
template <int DT>
__global__ __launch_bounds__(256, 1) void loss_dw_kernel(LossTileArgs a) {
  constexpr int WA = 2, IA = 4, WB = 2, JB = 4;
  typedef GemmShape<WA, IA, true, WB, JB, true> S;
  __shared__ __align__(16) uint16_t lds[kGemmStages * S::kStage];
  const int rows = uload(a.rows.count, 0), n = a.twice && rows ? 2 * kLossTwice : rows;
  const LossUnit u = loss_unit((a.H + S::kA - 1) / S::kA, (a.v1 - a.v0 + S::kB - 1) / S::kB);
  if (!u.any) return;
  f32x16 acc[IA][JB];
  loss_zero(acc);
  const int first_h = u.rows * S::kA, first_v = u.other * S::kB;
  GemmTile<DT, WA, IA, true, WB, JB, true>::run(acc, lds, GemmOperand{loss_y(a.rows, a.twice) ? a.rows.y : loss_x(a, n), a.H, n}, first_h,
                                            GemmOperand{a.g, a.ldg, n}, first_v, 0, n);
  const float unit = uload(a.rows.unit, 0);
#pragma unroll
  for (int i = 0; i < IA; ++i)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[i][j] *= unit;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hh = first_h + (wave / WB) * IA * 32, v = a.v0 + first_v + (wave % WB) * JB * 32;
  loss_lds_free();
  loss_store_across<DT>(acc, lds + wave * IA * JB * 1024, a.dw + (int64_t)v * a.H + hh, a.H, a.v1 - v, a.H - hh);
}

struct LossRefsArgs {
  LossRows rows;
  const float* part;      // [parts][pad][2]
  const float* at_label;
  float* loss;
  float* lse;
  int parts, pad, first, last;  // the piece's parts; whether it is the first, the last
  float bias;                   // the sums are 2^bias as large
};
// The rows' references and sums after a piece of the vocabulary; after the last, the losses.  Sixteen rows a workgroup, sixteen threads a
// row: a line of sixteen rows' parts a load.
__global__ __launch_bounds__(256) void loss_refs_kernel(LossRefsArgs a) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  __shared__ f32x2_t sums[16][16];
  __shared__ float lows[16][16];
  const int n = uload(a.rows.count, 0), r = threadIdx.x & 15, q = threadIdx.x >> 4;
  const int t = (int)blockIdx.x * 16 + r;
  if ((int)blockIdx.x * 16 >= n) return;
  float m = -INFINITY, l = 0.0f, least = INFINITY;
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
        if (p0 + e * 16 < a.parts) {
          join(v[e][0], v[e][1]);
          if (v[e][0] != -INFINITY) least = fminf(least, v[e][0]);
        }
    }
  sums[q][r] = f32x2_t{m, l};
  lows[q][r] = least;
  __syncthreads();
  if (q) return;  // (the first sixteen lanes are left)
  for (int p = 1; p < 16; ++p) {
    join(sums[p][r][0], sums[p][r][1]);
    least = fminf(least, lows[p][r]);
  }
  const float was = a.first || t >= n ? -INFINITY : a.rows.ref[t];
  const uint64_t any = __ballot(t < n && !(least >= fmaxf(m, was)));
  if (r == 0) a.rows.moved[blockIdx.x] = any != 0;
  if (t >= n) return;
  if (!a.first) {
    join(was, a.rows.sum[t]);
    a.rows.turn[t] = m == was ? 1.0f : __builtin_amdgcn_exp2f(was - m);
  }
  a.rows.ref[t] = m, a.rows.sum[t] = l;
  if (!a.last) return;
  // e = 2^x, in the sums' units; on the side where neither overflows
  const float z = a.at_label[t], x = (m == -INFINITY ? INFINITY : __builtin_fmaf(z, kLog2e, -m)) + a.bias;
  float loss, lse, over, share;
  if (x >= 0.0f) {
    const float e = __builtin_amdgcn_exp2f(-x), y = l * e;
    loss = y < 0x1p-10f ? y * (1.0f - y * (0.5f - y * (1.0f / 3.0f))) : __builtin_amdgcn_logf(1.0f + y) * kLn2;
    over = e / (1.0f + y), share = y / (1.0f + y), lse = z + loss;
  } else {
    const float all = l + __builtin_amdgcn_exp2f(x);
    loss = (__builtin_amdgcn_logf(all) - x) * kLn2;
    over = 1.0f / all, share = l / all, lse = (m - a.bias + __builtin_amdgcn_logf(all)) * kLn2;  // (not of z, which may be far below)
  }
  // what an infinity is divided by itself, or NaN: nothing but z may tell
  if (!(z < INFINITY) || (z == -INFINITY && m == -INFINITY)) loss = over = share = NAN;
  const int row = a.rows.row[t];
  a.loss[row] = loss, a.lse[row] = lse;
  a.rows.sum[t] = over, a.rows.share[t] = share;
}

struct LossTurnArgs {
  LossRows rows;
  const float* part;  // [parts][pad][2]
  uint16_t* g;        // [n, ldg]
  int parts, pad, ldg, wide;  // wide: entries a part, 128 or 64
};
// Exponentials that were stored against another reference than their row's: turned to it, by whole powers of two.  Sixteen lanes a row and
// a part of 128; blockIdx.y deals out the parts.
template <int DT>
__global__ __launch_bounds__(256) void loss_turn_kernel(LossTurnArgs a) {
  const int n = uload(a.rows.count, 0), i = (int)blockIdx.x * 16 + (threadIdx.x >> 4), l = threadIdx.x & 15;
  if (i >= n || !uload(a.rows.moved, (int)blockIdx.x)) return;
  const float ref = a.rows.ref[i];
  uint16_t* row = a.g + (int64_t)i * a.ldg;
  const int lanes = a.wide >> 3, each = 16 / lanes;  // (64 entries: two parts at a time)
#pragma unroll 4
  for (int p0 = (int)blockIdx.y * each; p0 < a.parts; p0 += (int)gridDim.y * each) {
    const int p = p0 + l / lanes;
    if (p >= a.parts) break;
    const float c = a.part[((int64_t)p * a.pad + i) * 2];
    if (c == ref || c == -INFINITY) continue;
    const float by = __builtin_amdgcn_exp2f(c - ref);
    uint16_t* at = row + p * a.wide + (l % lanes) * 8;
    const u32x4 v = ldg16(at);
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack2<DT>(Num<DT>::lo(v[e]) * by, Num<DT>::hi(v[e]) * by);
    stg16(at, o);
  }
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
  const float* sums;  // [n, H]
  const float* cut;   // [parts][tile]
  uint16_t* dx;       // [T, H]
  const uint16_t* w;  // [V, H]
  int from, T, H, few, stages;  // from: the launch's first row
  // of exponentials (KEPT): the rows' coefficients are found here
  const float* grad;         // [T], or [P]
  const int32_t* partition;  // [P + 1] or NULL
  const float* weight;       // [P]
  int P;
};
// A wave a row of the batch: its parts summed in order, and what the label adds; zeros without one.
template <int DT, bool KEPT>
__global__ __launch_bounds__(256) void loss_dx_fold_kernel(LossDxFoldArgs a) {
  const int n = uload(a.rows.count, 0), lane = threadIdx.x & 63, tile = a.few ? kLossFewRows : kLossRows;
  const int row_tiles = (n + tile - 1) / tile, h_tiles = (a.H + 255) / 256;
  const LossCuts cuts = loss_cuts(row_tiles * h_tiles, a.stages, a.few);
  const int t = a.from + (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6);
  if (t >= a.T) return;
  const int i = a.rows.number[t];
  uint16_t* to = a.dx + (int64_t)t * a.H;
  float by = 0.0f, label = 0.0f;  // of the sums, of w[label]
  bool none = i < 0;
  if (KEPT && i >= 0) {
    float c;
    if (a.partition) {
      const int p = loss_partition(a.partition, a.P, t);
      c = p < 0 ? 0.0f : a.grad[p] * a.weight[p];
    } else {
      c = a.grad[t];
    }
    by = c * a.rows.sum[i], label = -c * a.rows.share[i];
    none = c == 0.0f;  // (nothing hangs on this row)
  } else if (i >= 0) {
    by = a.rows.unit[0] * (a.rows.rest ? a.rows.rest[i] : 1.0f), label = a.rows.lost[i] * by;
  }
  if (none) {
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int c = lane * 8; c < a.H; c += 512) stg16(to + c, zero);
    return;
  }
  const uint16_t* w = a.w + (int64_t)a.rows.label[i] * a.H;
  for (int c = lane * 8; c < a.H; c += 512) {
    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    float f[8];
    unpack8<DT>(ldg16(w + c), f);
    const int at = loss_tile_number(i / tile, c >> 8, row_tiles, h_tiles) - cuts.whole;
    const float* p = at < 0 ? a.sums + (int64_t)i * a.H + c
                            : a.cut + ((int64_t)at * cuts.parts * tile + i % tile) * 256 + (c & 255);
    for (int s = 0; s < (at < 0 ? 1 : cuts.parts); ++s, p += tile * 256) {
      lo += ldg_f4(p);
      hi += ldg_f4(p + 4);
    }
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      o[e] = pack2<DT>(lo[2 * e] * by + f[2 * e] * label, lo[2 * e + 1] * by + f[2 * e + 1] * label);
      o[2 + e] = pack2<DT>(hi[2 * e] * by + f[4 + 2 * e] * label, hi[2 * e + 1] * by + f[5 + 2 * e] * label);
    }
    stg16(to + c, o);
  }
}

}  // namespace smlm
