// C ABI of the operators around a fine-tuning step (see include/smlm.h): the residual's addition with its norm, the loss over the
// vocabulary, the update of many tensors.  Argument checks, workspace carving, launch shapes.  No allocation, no host synchronisation, no state.
#include "adamw.hpp"
#include "api_common.hpp"
#include "rms_launch.hpp"
#include "vocab_loss.hpp"

using namespace smlm;

namespace {

int check_dtype(int dtype) { return dtype == SMLM_DTYPE_F16 || dtype == SMLM_DTYPE_BF16 ? SMLM_OK : SMLM_ERR_DTYPE; }

// ---- the loss over the vocabulary ----

constexpr int kLossMaxDim = 1 << 22;           // H: a tile's rows stay inside a resource
// Of exponentials, or of G, at a time: every piece ends the grid twice and adds to dx's sums.  Loss and dx, us, pieces of 128 / 256 / 512 / 1024
// MiB (4096 columns): 4096 rows of 128256 entries 7839 / 7347 / 7246 / 7179, 8192 rows 16225 / 15208 / 14607 / 14479, 8192 of 32000 4070 / 3806 /
// 3698 / 3698 (one piece from 512 on).
constexpr int64_t kLossPieceBytes = (int64_t)512 << 20;

// From 2^32 threads a launch on HIP drops what is over.  Workgroups a launch, and what has a workgroup for 16 rows.  (Products of matrices that
// fit a card have fewer tiles.)
constexpr int kLossGroups = 1 << 22;
constexpr int kLossMostRows = (1 << 28) - 16;

int loss_check(int T, int H, int V, int dtype) {
  if (T < 0 || H <= 0 || V <= 0) return SMLM_ERR_ARG;
  if (int rc = check_dtype(dtype)) return rc;
  if (H & 7) return SMLM_ERR_ALIGN;
  if (H > kLossMaxDim || T > kLossMostRows || V > (1 << 28)) return SMLM_ERR_LIMIT;
  if ((int64_t)ceil_div(T, kLossFewRows) * ceil_div(V, kLossTileV) > (1 << 30) ||
      (int64_t)ceil_div(H, 256) * ceil_div(V, kLossTileV) > (1 << 30))
    return SMLM_ERR_LIMIT;  // (tiles)
  return SMLM_OK;
}
// Tiles of 64 rows, two workgroups a compute unit, where rows or tiles of 256 are few: 128 tiles leave half of the card idle.  us, tiles of
// 256 rows / of 64, loss and gradient (4096 columns): 100 rows of 32000 entries (125 tiles) 235 / 193, 200 of 8000 (32) 169 / 115, 1000 of 8000
// (128) 199 / 175; 1000 of 16000 (252) 282 / 310, 500 of 64000 (500) 576 / 713.
bool loss_few(int T, int V) {
  return T <= kLossFewRows || (int64_t)ceil_div(T, kLossRows) * ceil_div(V, kLossTileV) <= 128;
}
// Vocabulary entries a piece: whole tiles, as many in each.  Of up to 64 rows as of 64, which is what G has where it is held twice, and what a
// tile has: 256 of a piece's rows then lie within 2^32 bytes, as gemm_tile's offsets have it.
int loss_piece(int T, int V) {
  const int64_t rows = T > 2 * kLossTwice ? T : 2 * kLossTwice, pieces = (2 * rows * V + kLossPieceBytes - 1) / kLossPieceBytes;
  const int64_t each = (V + pieces - 1) / pieces;
  return (int)((each + kLossTileV - 1) / kLossTileV * kLossTileV);
}
// The same where nothing is stored: all of it, or what a launch takes.
int loss_sums_piece(int T, int V) {
  const int most = kLossGroups / ceil_div(T > 0 ? T : 1, loss_few(T, V) ? kLossFewRows : kLossRows), tiles = ceil_div(V, kLossTileV);
  return kLossTileV * (tiles < most ? tiles : most);
}
int loss_stages(int T, int V) {
  const int piece = loss_piece(T, V);
  return ceil_div(piece < V ? piece : V, kGemmK);
}
// Parts of cut tiles, whatever the number of labelled rows; units of dx.
int loss_parts(int T, int H, int stages, bool few, int* most_units) {
  int parts = 0, units = 0;
  for (int r = 1; r <= ceil_div(T, few ? kLossFewRows : kLossRows); ++r) {
    const LossCuts c = loss_cuts(r * ceil_div(H, 256), stages, few);
    const int u = round_up(c.whole, 8) + round_up(c.rest * c.parts, 8);
    parts = c.rest * c.parts > parts ? c.rest * c.parts : parts;
    units = u > units ? u : units;
  }
  if (most_units) *most_units = units;
  return parts;
}

struct LossSpace {
  LossRows rows;
  float *part, *at_label, *dx, *cut;
  uint16_t* g;
  int pad, parts, piece;
};
struct LossTaker {
  char* base;
  size_t off = 0;
  template <typename P>
  void take(P*& p, size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    p = base ? reinterpret_cast<P*>(base + o) : nullptr;
  }
};
void loss_take_dx(LossTaker& k, int T, int H, int V, LossSpace* s) {
  k.take(s->dx, 4 * (size_t)T * H);
  k.take(s->cut, 4 * (size_t)loss_parts(T, H, loss_stages(T, V), loss_few(T, V), nullptr) * 256 * (loss_few(T, V) ? kLossFewRows : kLossRows));
}
bool loss_twice(int T, int what) { return T <= kLossTwice && (what == 2 || what == 3); }
// What the forward keeps for the gradient of x: its sums, and what the fold needs.
size_t loss_keep(void* base, int T, int H, int V, LossSpace* s) {
  LossTaker k{reinterpret_cast<char*>(base)};
  const size_t t = (size_t)T;
  k.take(s->rows.count, 256);
  k.take(s->rows.number, 4 * t);
  k.take(s->rows.label, 4 * t);
  k.take(s->rows.sum, 4 * t);
  k.take(s->rows.share, 4 * t);
  loss_take_dx(k, T, H, V, s);
  return k.off;
}
// what: 0 the forward, 1 the backward with dx, 2 with dw, 3 with both, 4 the forward that keeps.
size_t loss_carve(void* base, int T, int H, int V, int what, LossSpace* s) {
  LossTaker k{reinterpret_cast<char*>(base)};
  const size_t t = (size_t)T;
  if (what != 4) {
    k.take(s->rows.count, 256);
    s->rows.unit = reinterpret_cast<float*>(base ? s->rows.count + 16 : nullptr);
    k.take(s->rows.label, 4 * t);
    k.take(s->rows.sum, 4 * t);
    k.take(s->rows.share, 4 * t);
  }
  k.take(s->rows.row, 4 * t);
  const size_t twice = loss_twice(T, what) ? 2 * kLossTwice : t;  // rows of y and G
  k.take(s->rows.x, 2 * t * H);
  s->pad = round_up(T, 64);
  s->piece = what == 0 ? loss_sums_piece(T, V) : loss_piece(T, V);
  s->parts = s->piece / kLossTileV * (loss_few(T, V) ? 4 : 2);
  if (what == 0 || what == 4) {
    k.take(s->part, 8 * (size_t)s->parts * s->pad);
    k.take(s->at_label, 4 * (size_t)s->pad);
    k.take(s->rows.ref, 4 * t);
    k.take(s->rows.turn, 4 * t);
    k.take(s->rows.moved, 4 * (t / 16 + 1));
  } else {
    k.take(s->rows.number, 4 * t);
    k.take(s->rows.coef, 4 * t);
    k.take(s->rows.lse2, 4 * t);
    k.take(s->rows.own, 4 * t);
    k.take(s->rows.lost, 4 * t);
    k.take(s->rows.rest, 4 * t);
    if (what & 2) k.take(s->rows.y, 2 * twice * H);
  }
  if (what) k.take(s->g, 2 * twice * s->piece);
  if (what == 1 || what == 3) loss_take_dx(k, T, H, V, s);
  return k.off;
}

dim3 loss_grid(int64_t units) { return dim3((unsigned)((units + 7) / 8 * 8)); }

int loss_logits(int mode, bool f16, bool few, dim3 grid, hipStream_t st, const LossTileArgs& a) {
  void (*const kernels[3][2][2])(LossTileArgs) = {  // by mode, rows and type
      {{loss_logits_kernel<SMLM_DTYPE_F16, false, kLossSums>, loss_logits_kernel<SMLM_DTYPE_BF16, false, kLossSums>},
       {loss_logits_kernel<SMLM_DTYPE_F16, true, kLossSums>, loss_logits_kernel<SMLM_DTYPE_BF16, true, kLossSums>}},
      {{loss_logits_kernel<SMLM_DTYPE_F16, false, kLossSoft>, loss_logits_kernel<SMLM_DTYPE_BF16, false, kLossSoft>},
       {loss_logits_kernel<SMLM_DTYPE_F16, true, kLossSoft>, loss_logits_kernel<SMLM_DTYPE_BF16, true, kLossSoft>}},
      {{loss_logits_kernel<SMLM_DTYPE_F16, false, kLossGrad>, loss_logits_kernel<SMLM_DTYPE_BF16, false, kLossGrad>},
       {loss_logits_kernel<SMLM_DTYPE_F16, true, kLossGrad>, loss_logits_kernel<SMLM_DTYPE_BF16, true, kLossGrad>}}};
  return launch(kernels[mode][few][!f16], grid, dim3(256), st, a);
}
int loss_gather(bool f16, int rows, hipStream_t st, const LossGatherArgs& a) {
  const int groups = ceil_div(rows, 4);
  const dim3 grid((unsigned)(groups < kLossGroups ? groups : kLossGroups)), bl(256);
  return f16 ? launch(loss_gather_kernel<SMLM_DTYPE_F16>, grid, bl, st, a) : launch(loss_gather_kernel<SMLM_DTYPE_BF16>, grid, bl, st, a);
}
int loss_dx(bool f16, bool few, hipStream_t st, const LossTileArgs& a) {
  int most = 0;
  loss_parts(a.T, a.H, a.stages, few, &most);
  const dim3 grid = loss_grid(most), bl(256);
  if (few)
    return f16 ? launch(loss_dx_kernel<SMLM_DTYPE_F16, true>, grid, bl, st, a) : launch(loss_dx_kernel<SMLM_DTYPE_BF16, true>, grid, bl, st, a);
  return f16 ? launch(loss_dx_kernel<SMLM_DTYPE_F16, false>, grid, bl, st, a) : launch(loss_dx_kernel<SMLM_DTYPE_BF16, false>, grid, bl, st, a);
}
template <bool KEPT>
int loss_dx_fold(bool f16, hipStream_t st, LossDxFoldArgs a) {
  for (; a.from < a.T; a.from += kLossGroups * 4) {
    const int groups = ceil_div(a.T - a.from, 4);
    const dim3 grid((unsigned)(groups < kLossGroups ? groups : kLossGroups)), bl(256);
    const int rc = f16 ? launch(loss_dx_fold_kernel<SMLM_DTYPE_F16, KEPT>, grid, bl, st, a)
                       : launch(loss_dx_fold_kernel<SMLM_DTYPE_BF16, KEPT>, grid, bl, st, a);
    if (rc) return rc;
  }
  return SMLM_OK;
}
#define LOSS_TRY(call) \
  if (int rc = (call)) return rc

}  // namespace

SMLM_API int smlm_vocab_loss_workspace_size(int T, int H, int V, int what, size_t* bytes) {
  if (!bytes || what < 0 || what > 5) return SMLM_ERR_ARG;
  if (int rc = loss_check(T, H, V, SMLM_DTYPE_F16)) return rc;
  LossSpace s{};
  *bytes = what == 5 ? loss_keep(nullptr, T, H, V, &s) : loss_carve(nullptr, T, H, V, what, &s);
  return SMLM_OK;
}

SMLM_API int smlm_vocab_loss_fwd(float* loss, float* lse, float* means, float* weight, void* kept, size_t kept_bytes, const void* x,
                                 const void* w, const int64_t* labels, const int32_t* partition, int P, void* workspace,
                                 size_t workspace_bytes, int T, int H, int V, int dtype, void* stream) {
  if (int rc = loss_check(T, H, V, dtype)) return rc;
  if (P < 0 || (partition && P > 0 && (!means || !weight))) return SMLM_ERR_ARG;
  if (!partition) P = 0;
  if (T == 0 && P == 0) return SMLM_OK;
  if (T > 0 && (!loss || !lse || !x || !w || !labels || !workspace)) return SMLM_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(workspace) || !aligned16(kept)) return SMLM_ERR_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  if (T > 0) {
    LossSpace s{};
    if (kept && kept_bytes < loss_keep(kept, T, H, V, &s)) return SMLM_ERR_WORKSPACE;
    if (workspace_bytes < loss_carve(workspace, T, H, V, kept ? 4 : 0, &s)) return SMLM_ERR_WORKSPACE;
    const LossScanArgs sa{s.rows, labels, loss, lse, nullptr, partition, nullptr, T, V, P, 0, kept != nullptr, 0};
    LOSS_TRY(launch(loss_scan_kernel<false>, dim3(1), dim3(kLossScanThreads), st, sa));
    const LossGatherArgs ga{s.rows, reinterpret_cast<const uint16_t*>(x), T, H, 0};
    LOSS_TRY(loss_gather(dtype == SMLM_DTYPE_F16, T, st, ga));
    LossTileArgs a{};
    a.rows = s.rows, a.x = ga.x, a.w = reinterpret_cast<const uint16_t*>(w), a.part = s.part, a.at_label = s.at_label;
    a.g = s.g, a.dx = s.dx, a.T = T, a.H = H, a.V = V, a.pad = s.pad, a.ldg = s.piece, a.cut = s.cut, a.stages = loss_stages(T, V), a.turned = 1;
    const bool few = loss_few(T, V), f16 = dtype == SMLM_DTYPE_F16;
    for (int v0 = 0; v0 < V; v0 += s.piece) {
      a.v0 = v0, a.v1 = V - v0 < s.piece ? V : v0 + s.piece, a.add = v0 > 0;
      const int v_tiles = ceil_div(a.v1 - v0, kLossTileV), parts = v_tiles * (few ? 4 : 2);
      const dim3 grid = loss_grid((int64_t)ceil_div(T, few ? kLossFewRows : kLossRows) * v_tiles);
      LOSS_TRY(loss_logits(kept ? kLossSoft : kLossSums, f16, few, grid, st, a));
      const LossRefsArgs ra{s.rows, s.part, s.at_label, loss, lse, parts, s.pad, v0 == 0, a.v1 == V,
                            kept && f16 ? kLossBias<SMLM_DTYPE_F16> : 0.0f};
      const dim3 rows16((unsigned)ceil_div(T, 16));
      LOSS_TRY(launch(loss_refs_kernel, rows16, dim3(256), st, ra));
      if (!kept) continue;
      const LossTurnArgs ta{s.rows, s.part, s.g, parts, s.pad, s.piece, few ? 64 : 128};
      const dim3 gt(rows16.x, (unsigned)(ceil_div(parts, 8) < 16 ? ceil_div(parts, 8) : 16));
      LOSS_TRY(f16 ? launch(loss_turn_kernel<SMLM_DTYPE_F16>, gt, dim3(256), st, ta)
                   : launch(loss_turn_kernel<SMLM_DTYPE_BF16>, gt, dim3(256), st, ta));
      LOSS_TRY(loss_dx(f16, few, st, a));
    }
  }
  if (P == 0) return SMLM_OK;
  for (int from = 0; from < P; from += kLossGroups / 4) {  // (workgroups of 1024)
    const LossMeansArgs ma{loss, labels, partition + from, means + from, weight + from, T, V};
    LOSS_TRY(launch(loss_means_kernel, dim3((unsigned)(P - from < kLossGroups / 4 ? P - from : kLossGroups / 4)), dim3(1024), st, ma));
  }
  return SMLM_OK;
}

SMLM_API int smlm_vocab_loss_bwd_kept(void* dx, const float* grad, const void* kept, size_t kept_bytes, const void* w,
                                      const int32_t* partition, const float* weight, int P, int T, int H, int V, int dtype, void* stream) {
  if (int rc = loss_check(T, H, V, dtype)) return rc;
  if (P < 0 || (partition && P > 0 && !weight)) return SMLM_ERR_ARG;
  if (T == 0) return SMLM_OK;
  if (!dx || !grad || !kept || !w) return SMLM_ERR_ARG;
  if (!aligned16(dx) || !aligned16(kept) || !aligned16(w)) return SMLM_ERR_ALIGN;
  LossSpace s{};
  if (kept_bytes < loss_keep(const_cast<void*>(kept), T, H, V, &s)) return SMLM_ERR_WORKSPACE;
  const LossDxFoldArgs fa{s.rows, s.dx, s.cut, reinterpret_cast<uint16_t*>(dx), reinterpret_cast<const uint16_t*>(w), 0, T, H, loss_few(T, V),
                          loss_stages(T, V), grad, partition, weight, P};
  return loss_dx_fold<true>(dtype == SMLM_DTYPE_F16, (hipStream_t)stream, fa);
}

SMLM_API int smlm_vocab_loss_bwd(void* dx, void* dw, const float* grad, const float* loss, const float* lse, const void* x, const void* w,
                                 const int64_t* labels, const int32_t* partition, const float* weight, int P, void* workspace,
                                 size_t workspace_bytes, int T, int H, int V, int dtype, void* stream) {
  if (int rc = loss_check(T, H, V, dtype)) return rc;
  if (P < 0 || (partition && P > 0 && !weight) || (!dx && !dw)) return SMLM_ERR_ARG;
  if (T == 0) return dw ? SMLM_ERR_ARG : SMLM_OK;  // (dw would have nothing to sum)
  if (!grad || !loss || !lse || !x || !w || !labels || !workspace) return SMLM_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(workspace) || !aligned16(dx) || !aligned16(dw)) return SMLM_ERR_ALIGN;
  LossSpace s{};
  if (workspace_bytes < loss_carve(workspace, T, H, V, (dx ? 1 : 0) | (dw ? 2 : 0), &s)) return SMLM_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = dtype == SMLM_DTYPE_F16, few = loss_few(T, V);
  const int twice = loss_twice(T, (dx ? 1 : 0) | (dw ? 2 : 0));
  const bool split = dw && partition && !twice;  // (twice: nothing is lost that it would save)
  if (!f16 && !split) s.rows.rest = nullptr;
  if (!s.rows.rest && !twice) s.rows.y = nullptr;
  const LossScanArgs sa{s.rows, labels, const_cast<float*>(loss), const_cast<float*>(lse), grad, partition, weight, T, V, P, f16, 1, split};
  LOSS_TRY(launch(loss_scan_kernel<true>, dim3(1), dim3(kLossScanThreads), st, sa));
  const LossGatherArgs ga{s.rows, reinterpret_cast<const uint16_t*>(x), T, H, twice};
  LOSS_TRY(loss_gather(f16, twice ? 2 * kLossTwice : T, st, ga));
  LossTileArgs a{};
  a.twice = twice;
  a.rows = s.rows, a.x = ga.x, a.w = reinterpret_cast<const uint16_t*>(w), a.g = s.g, a.dx = s.dx;
  a.dw = reinterpret_cast<uint16_t*>(dw), a.T = T, a.H = H, a.V = V, a.ldg = s.piece, a.cut = s.cut, a.stages = loss_stages(T, V);
  const int tile = few ? kLossFewRows : kLossRows, h_tiles = ceil_div(H, 256);
  const dim3 bl(256);
  for (int v0 = 0; v0 < V; v0 += s.piece) {
    a.v0 = v0, a.v1 = V - v0 < s.piece ? V : v0 + s.piece, a.add = v0 > 0;
    const int v_tiles = ceil_div(a.v1 - v0, kLossTileV);
    LOSS_TRY(loss_logits(kLossGrad, f16, few, loss_grid((int64_t)ceil_div(T, tile) * v_tiles), st, a));
    if (dx) LOSS_TRY(loss_dx(f16, few, st, a));
    if (dw) {
      const dim3 gw = loss_grid((int64_t)h_tiles * v_tiles);
      LOSS_TRY(f16 ? launch(loss_dw_kernel<SMLM_DTYPE_F16>, gw, bl, st, a) : launch(loss_dw_kernel<SMLM_DTYPE_BF16>, gw, bl, st, a));
    }
  }
  if (!dx) return SMLM_OK;
  const LossDxFoldArgs fa{s.rows, s.dx, s.cut, reinterpret_cast<uint16_t*>(dx), a.w, 0, T, H, few, a.stages, nullptr, nullptr, nullptr, 0};
  return loss_dx_fold<false>(f16, st, fa);
}

// ---- the residual's addition and its norm ----

namespace {

constexpr int kAddRmsRows = 1 << 22;  // a launch, a workgroup each at most: from 2^32 threads on HIP drops what is over

template <int DT>
int launch_add_rms(hipStream_t st, const AddRmsArgs& a) {
  const dim3 bl(256);
  if (a.cols > kRmsMaxCols) return launch(add_rms_wide_kernel<DT>, dim3((unsigned)a.rows), bl, st, a);
  if (a.cols > kRmsWaveCols) {
    const dim3 grid((unsigned)a.rows);
    return a.cols <= 8192 ? launch(add_rms_kernel<DT, 4, 4>, grid, bl, st, a) : launch(add_rms_kernel<DT, 4, 8>, grid, bl, st, a);
  }
  // Four waves a row of more than 1024 columns where rows are few.  us, a wave a row / four, 2048 columns: 1 row 2.28 / 1.95, 256 3.36 / 2.89,
  // 512 3.73 / 3.36, 1024 4.23 / 4.30, 2048 6.7 / 7.3; 4096 columns: 1 row 3.03 / 2.16, 256 4.73 / 3.39, 512 4.95 / 5.15, 1024 6.7 / 7.4.  (1024
  // columns: 8 rows 2.21 / 2.20, 256 2.35 / 2.70.)
  if (a.cols > 1024 && (int64_t)a.rows * a.cols <= (1 << 20)) {
    const dim3 grid((unsigned)a.rows);
    return a.cols <= 2048 ? launch(add_rms_kernel<DT, 4, 1>, grid, bl, st, a) : launch(add_rms_kernel<DT, 4, 2>, grid, bl, st, a);
  }
  const dim3 grid((unsigned)ceil_div(a.rows, 4));
  if (a.cols <= 512) return launch(add_rms_kernel<DT, 1, 1>, grid, bl, st, a);
  if (a.cols <= 1024) return launch(add_rms_kernel<DT, 1, 2>, grid, bl, st, a);
  return a.cols <= 2048 ? launch(add_rms_kernel<DT, 1, 4>, grid, bl, st, a) : launch(add_rms_kernel<DT, 1, 8>, grid, bl, st, a);
}

}  // namespace

SMLM_API int smlm_add_rms_norm_fwd(void* out, float* rms, void* h, const void* x, const void* residual, const void* w, void* out8,
                                   float* scale, int group, int rows, int cols, float eps, int dtype, void* stream) {
  if (int rc = rms_check(rows, cols, dtype)) return rc;
  if (group != 0 && group != 128) return SMLM_ERR_ARG;
  if (group && (cols & 127)) return SMLM_ERR_ALIGN;
  if (rows == 0) return SMLM_OK;
  if ((!out && !out8 && !h) || (h && !residual) || (!out8) != (!scale)) return SMLM_ERR_ARG;
  if (!x || !w) return SMLM_ERR_ARG;
  if (!aligned16(out) || !aligned16(h) || !aligned16(x) || !aligned16(residual) || !aligned16(w) || !aligned16(out8))
    return SMLM_ERR_ALIGN;
  AddRmsArgs a{reinterpret_cast<uint16_t*>(out), rms, reinterpret_cast<uint16_t*>(h), reinterpret_cast<const uint16_t*>(x),
               reinterpret_cast<const uint16_t*>(residual), reinterpret_cast<const uint16_t*>(w),
               reinterpret_cast<uint8_t*>(out8), scale, rows, cols, group == 128, eps};
  hipStream_t st = (hipStream_t)stream;
  for (int from = 0;; from += kAddRmsRows) {
    a.rows = rows - from < kAddRmsRows ? rows - from : kAddRmsRows;
    const int rc = dtype == SMLM_DTYPE_F16 ? launch_add_rms<SMLM_DTYPE_F16>(st, a) : launch_add_rms<SMLM_DTYPE_BF16>(st, a);
    if (rc || rows - from <= kAddRmsRows) return rc;
    const int64_t n = (int64_t)kAddRmsRows * cols;
    a.x += n;
    if (out) a.out += n;
    if (rms) a.rms += kAddRmsRows;
    if (h) a.h += n;
    if (residual) a.residual += n;
    if (out8) a.out8 += n, a.scale += group ? n / 128 : kAddRmsRows;
  }
}

SMLM_API int smlm_add_rms_norm_bwd(void* dh, void* dw, const void* g, const void* gh, const void* h, const void* w, const float* rms,
                                   void* workspace, size_t workspace_bytes, int rows, int cols, int dtype, void* stream) {
  if (int rc = rms_check(rows, cols, dtype)) return rc;
  if (!dh || !dw || !g || !h || !w || !rms || !workspace) return SMLM_ERR_ARG;
  if (!aligned16(dh) || !aligned16(dw) || !aligned16(g) || !aligned16(gh) || !aligned16(h) || !aligned16(w) || !aligned16(workspace))
    return SMLM_ERR_ALIGN;
  if (rows == 0) return SMLM_ERR_ARG;  // (dw would have nothing to sum)
  const int nb = rms_bwd_blocks(rows, cols);
  if (workspace_bytes < (size_t)nb * cols * 4) return SMLM_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = dtype == SMLM_DTYPE_F16;
  const RmsBwdArgs a{reinterpret_cast<uint16_t*>(dh), reinterpret_cast<float*>(workspace), reinterpret_cast<const uint16_t*>(g),
                     reinterpret_cast<const uint16_t*>(h), reinterpret_cast<const uint16_t*>(w), rms, rows, cols,
                     reinterpret_cast<const uint16_t*>(gh)};
  const int rc = gh ? f16 ? launch_rms_bwd<SMLM_DTYPE_F16, true>(nb, st, a) : launch_rms_bwd<SMLM_DTYPE_BF16, true>(nb, st, a)
                    : f16 ? launch_rms_bwd<SMLM_DTYPE_F16, false>(nb, st, a) : launch_rms_bwd<SMLM_DTYPE_BF16, false>(nb, st, a);
  if (rc) return rc;
  const RmsFoldArgs fa{reinterpret_cast<uint16_t*>(dw), reinterpret_cast<const float*>(workspace), nb, cols};
  return f16 ? launch_rms_fold<SMLM_DTYPE_F16>(st, fa) : launch_rms_fold<SMLM_DTYPE_BF16>(st, fa);
}

// ---- the update of many tensors ----

SMLM_API int smlm_adamw_workspace_size(int n_tensors, size_t* bytes) {
  if (!bytes || n_tensors < 0) return SMLM_ERR_ARG;
  *bytes = align_up((size_t)(n_tensors > 0 ? n_tensors : 1) * sizeof(AdamTensor), 256);
  return SMLM_OK;
}

namespace {

template <int PT>
int launch_adam(bool eight, bool master, dim3 grid, hipStream_t st, const AdamArgs& a) {
  const dim3 bl(256);
  if (eight)
    return master ? launch(adam_kernel<PT, true, true>, grid, bl, st, a) : launch(adam_kernel<PT, true, false>, grid, bl, st, a);
  return master ? launch(adam_kernel<PT, false, true>, grid, bl, st, a) : launch(adam_kernel<PT, false, false>, grid, bl, st, a);
}

template <int N>
int adam_begin(const smlm_adamw* p, AdamTensor* table, int at, int n, int64_t first, int align, hipStream_t st) {
  AdamBeginArgs<N> a;
  a.table = table, a.step = p->step, a.hyper = p->hyper, a.group = p->group, a.at = at, a.n = n, a.n_groups = p->n_groups, a.pad = 0;
  a.first = first;
  for (int i = 0; i < n; ++i) {
    const uint64_t w = (uint64_t)(uintptr_t)p->params[at + i], g = (uint64_t)(uintptr_t)p->grads[at + i];
    a.entry[i] = AdamEntry{w, g, p->sizes[at + i] | (((w | g) & (uint64_t)(align - 1)) ? INT64_MIN : 0)};
  }
  return launch(adam_begin_kernel<N>, dim3(1), dim3(256), st, a);
}

}  // namespace

SMLM_API int smlm_adamw_step(const smlm_adamw* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (!p || p->n_tensors < 0 || p->n_groups < 0 || (p->state_bits != 8 && p->state_bits != 32)) return SMLM_ERR_ARG;
  const bool f32 = p->dtype == kAdamF32, eight = p->state_bits == 8;
  if (!f32)
    if (int rc = check_dtype(p->dtype)) return rc;
  if (f32 && p->master) return SMLM_ERR_ARG;
  if (p->n_tensors == 0) return SMLM_OK;
  if (!p->params || !p->grads || !p->sizes || !p->step || !p->hyper || !p->group || !workspace) return SMLM_ERR_ARG;
  int64_t blocks = 0;
  for (int i = 0; i < p->n_tensors; ++i) {
    if (p->sizes[i] < 0 || p->sizes[i] > ((int64_t)1 << 40)) return SMLM_ERR_LIMIT;
    if (p->sizes[i] > 0 && !p->params[i]) return SMLM_ERR_ARG;
    blocks += (p->sizes[i] + kAdamBlock - 1) / kAdamBlock;
  }
  if (blocks > ((int64_t)1 << 32) - 64) return SMLM_ERR_LIMIT;
  if (blocks > 0 && (!p->exp_avg || !p->exp_avg_sq || (eight && (!p->avg_scale || !p->sq_scale)))) return SMLM_ERR_ARG;
  if (!aligned16(p->exp_avg) || !aligned16(p->exp_avg_sq) || !aligned16(p->master) || !aligned16(workspace)) return SMLM_ERR_ALIGN;
  if (workspace_bytes < (size_t)p->n_tensors * sizeof(AdamTensor)) return SMLM_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  AdamTensor* table = reinterpret_cast<AdamTensor*>(workspace);
  int64_t first = 0;
  const int align = f32 ? 16 : 8;  // (bytes of a lane's four elements)
  for (int at = 0; at < p->n_tensors;) {
    const int n = p->n_tensors - at < kAdamEntries ? p->n_tensors - at : kAdamEntries;
    const int rc = n <= 16 ? adam_begin<16>(p, table, at, n, first, align, st) : adam_begin<kAdamEntries>(p, table, at, n, first, align, st);
    if (rc) return rc;
    for (int i = 0; i < n; ++i) first += (p->sizes[at + i] + kAdamBlock - 1) / kAdamBlock;
    at += n;
  }
  if (blocks == 0) return SMLM_OK;
  for (int64_t from = 0; from < blocks; from += kAdamGroups * 4) {
    const int64_t here = blocks - from < kAdamGroups * 4 ? blocks - from : kAdamGroups * 4;
    const AdamArgs a{table, p->exp_avg, p->exp_avg_sq, p->avg_scale, p->sq_scale, p->master, p->n_tensors, from, blocks};
    const dim3 grid((unsigned)((here + 3) / 4));
    const int rc = f32 ? launch_adam<kAdamF32>(eight, false, grid, st, a)
                   : p->dtype == SMLM_DTYPE_F16 ? launch_adam<SMLM_DTYPE_F16>(eight, p->master != nullptr, grid, st, a)
                                                : launch_adam<SMLM_DTYPE_BF16>(eight, p->master != nullptr, grid, st, a);
    if (rc) return rc;
  }
  return SMLM_OK;
}
