// C ABI of the operators around a fine-tuning step (see include/smlm.h): the loss over the vocabulary, the update of many
// tensors.  Argument checks, workspace carving, launch shapes.  No allocation, no host synchronisation, no state.
#include "api_common.hpp"
#include "vocab_loss.hpp"

using namespace smlm;

namespace {

int check_dtype(int dtype) { return dtype == SMLM_DTYPE_F16 || dtype == SMLM_DTYPE_BF16 ? SMLM_OK : SMLM_ERR_DTYPE; }

// ---- the loss over the vocabulary ----

constexpr int kLossMaxDim = 1 << 22;           // H: a tile's rows stay inside a resource
constexpr int64_t kLossPieceBytes = 128 << 20;  // of G at a time
constexpr int kLossMostSplits = 64;

int loss_check(int T, int H, int V, int dtype) {
  if (T < 0 || H <= 0 || V <= 0) return SMLM_ERR_ARG;
  if (int rc = check_dtype(dtype)) return rc;
  if (H & 7) return SMLM_ERR_ALIGN;
  if (H > kLossMaxDim || T > (1 << 28) || V > (1 << 28)) return SMLM_ERR_LIMIT;
  if ((int64_t)ceil_div(T, kLossFewRows) * ceil_div(V, kLossTileV) > (1 << 30) ||
      (int64_t)ceil_div(H, 256) * ceil_div(V, kLossTileV) > (1 << 30))
    return SMLM_ERR_LIMIT;  // (workgroups)
  return SMLM_OK;
}
bool loss_few(int T) { return T <= kLossFewRows; }
// Vocabulary entries a piece: whole tiles.
int loss_piece(int T, int V) {
  const int64_t most = kLossPieceBytes / (2 * (int64_t)(T > 0 ? T : 1)) / kLossTileV * kLossTileV;
  const int all = round_up(V, kLossTileV);
  return most < kLossTileV ? kLossTileV : most < all ? (int)most : all;
}
int64_t loss_dx_floats(int T, int H) {
  const int64_t one = (int64_t)T * H, tile = loss_few(T) ? kLossFewRows : kLossRows, cut = 256 * 256 * tile;
  const int64_t split = cut < kLossMostSplits * one ? cut : kLossMostSplits * one;
  return one > split ? one : split;
}

struct LossSpace {
  LossRows rows;
  float *part, *at_label, *dx;
  uint16_t* g;
  int pad, parts, piece;
};
// what: 0 the forward, 1 the backward with dx, 2 with dw, 3 with both.
size_t loss_carve(void* base, int T, int H, int V, int what, LossSpace* out) {
  size_t off = 0;
  auto take = [&](size_t bytes) {
    const size_t o = off;
    off = align_up(off + bytes, 256);
    return base ? reinterpret_cast<char*>(base) + o : nullptr;
  };
  LossSpace s{};
  const size_t t = (size_t)T;
  s.rows.count = reinterpret_cast<int32_t*>(take(256));
  s.rows.unit = reinterpret_cast<float*>(base ? s.rows.count + 16 : nullptr);
  s.rows.row = reinterpret_cast<int32_t*>(take(4 * t));
  s.rows.label = reinterpret_cast<int32_t*>(take(4 * t));
  s.rows.x = reinterpret_cast<uint16_t*>(take(2 * t * H));
  s.pad = round_up(T, 64);
  s.parts = ceil_div(V, kLossTileV) * (loss_few(T) ? 4 : 2);
  s.piece = loss_piece(T, V);
  if (what == 0) {
    s.part = reinterpret_cast<float*>(take(8 * (size_t)s.parts * s.pad));
    s.at_label = reinterpret_cast<float*>(take(4 * (size_t)s.pad));
  } else {
    s.rows.number = reinterpret_cast<int32_t*>(take(4 * t));
    s.rows.coef = reinterpret_cast<float*>(take(4 * t));
    s.rows.lse2 = reinterpret_cast<float*>(take(4 * t));
    s.g = reinterpret_cast<uint16_t*>(take(2 * t * s.piece));
    if (what & 1) s.dx = reinterpret_cast<float*>(take(4 * (size_t)loss_dx_floats(T, H)));
  }
  if (out) *out = s;
  return off;
}

dim3 loss_grid(int64_t units) { return dim3((unsigned)((units + 7) / 8 * 8)); }

template <int DT>
int loss_logits(bool few, bool grad, dim3 grid, hipStream_t st, const LossTileArgs& a) {
  const dim3 bl(256);
  if (few)
    return grad ? launch(loss_logits_kernel<DT, true, true>, grid, bl, st, a)
                : launch(loss_logits_kernel<DT, true, false>, grid, bl, st, a);
  return grad ? launch(loss_logits_kernel<DT, false, true>, grid, bl, st, a)
              : launch(loss_logits_kernel<DT, false, false>, grid, bl, st, a);
}

}  // namespace

SMLM_API int smlm_vocab_loss_workspace_size(int T, int H, int V, int what, size_t* bytes) {
  if (!bytes || what < 0 || what > 3) return SMLM_ERR_ARG;
  if (int rc = loss_check(T, H, V, SMLM_DTYPE_F16)) return rc;
  *bytes = loss_carve(nullptr, T, H, V, what, nullptr);
  return SMLM_OK;
}

SMLM_API int smlm_vocab_loss_fwd(float* loss, float* lse, float* means, float* weight, const void* x, const void* w,
                                 const int64_t* labels, const int32_t* partition, int P, void* workspace, size_t workspace_bytes,
                                 int T, int H, int V, int dtype, void* stream) {
  if (int rc = loss_check(T, H, V, dtype)) return rc;
  if (P < 0 || (partition && P > 0 && (!means || !weight))) return SMLM_ERR_ARG;
  if (!partition) P = 0;
  if (T == 0 && P == 0) return SMLM_OK;
  if (T > 0 && (!loss || !lse || !x || !w || !labels || !workspace)) return SMLM_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(workspace)) return SMLM_ERR_ALIGN;
  hipStream_t st = (hipStream_t)stream;
  if (T > 0) {
    LossSpace s;
    if (workspace_bytes < loss_carve(workspace, T, H, V, 0, &s)) return SMLM_ERR_WORKSPACE;
    const LossScanArgs sa{s.rows, labels, loss, lse, nullptr, P ? partition : nullptr, nullptr, T, V, P, 0};
    if (int rc = launch(loss_scan_kernel<false>, dim3(1), dim3(kLossScanThreads), st, sa)) return rc;
    const LossGatherArgs ga{s.rows, reinterpret_cast<const uint16_t*>(x), T, H};
    if (int rc = launch(loss_gather_kernel, dim3((unsigned)ceil_div(T, 4)), dim3(256), st, ga)) return rc;
    LossTileArgs a{};
    a.rows = s.rows, a.x = ga.x, a.w = reinterpret_cast<const uint16_t*>(w), a.part = s.part, a.at_label = s.at_label;
    a.T = T, a.H = H, a.V = V, a.pad = s.pad, a.v0 = 0, a.v1 = V;
    const bool few = loss_few(T);
    const dim3 grid = loss_grid((int64_t)ceil_div(T, few ? kLossFewRows : kLossRows) * ceil_div(V, kLossTileV));
    int rc = dtype == SMLM_DTYPE_F16 ? loss_logits<SMLM_DTYPE_F16>(few, false, grid, st, a)
                                     : loss_logits<SMLM_DTYPE_BF16>(few, false, grid, st, a);
    if (rc) return rc;
    const LossFoldArgs fa{s.rows, s.part, s.at_label, loss, lse, s.parts, s.pad};
    rc = launch(loss_fold_kernel, dim3((unsigned)ceil_div(T, 16)), dim3(256), st, fa);
    if (rc) return rc;
  }
  if (P == 0) return SMLM_OK;
  const LossMeansArgs ma{loss, labels, partition, means, weight, T, V};
  return launch(loss_means_kernel, dim3((unsigned)P), dim3(1024), st, ma);
}

SMLM_API int smlm_vocab_loss_bwd(void* dx, void* dw, const float* grad, const float* lse, const void* x, const void* w,
                                 const int64_t* labels, const int32_t* partition, const float* weight, int P, void* workspace,
                                 size_t workspace_bytes, int T, int H, int V, int dtype, void* stream) {
  if (int rc = loss_check(T, H, V, dtype)) return rc;
  if (P < 0 || (partition && P > 0 && !weight) || (!dx && !dw)) return SMLM_ERR_ARG;
  if (T == 0) return dw ? SMLM_ERR_ARG : SMLM_OK;  // (dw would have nothing to sum)
  if (!grad || !lse || !x || !w || !labels || !workspace) return SMLM_ERR_ARG;
  if (!aligned16(x) || !aligned16(w) || !aligned16(workspace) || !aligned16(dx) || !aligned16(dw)) return SMLM_ERR_ALIGN;
  LossSpace s;
  if (workspace_bytes < loss_carve(workspace, T, H, V, (dx ? 1 : 0) | (dw ? 2 : 0), &s)) return SMLM_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const bool f16 = dtype == SMLM_DTYPE_F16, few = loss_few(T);
  const LossScanArgs sa{s.rows, labels, nullptr, const_cast<float*>(lse), grad, partition, weight, T, V, P, f16};
  if (int rc = launch(loss_scan_kernel<true>, dim3(1), dim3(kLossScanThreads), st, sa)) return rc;
  const LossGatherArgs ga{s.rows, reinterpret_cast<const uint16_t*>(x), T, H};
  if (int rc = launch(loss_gather_kernel, dim3((unsigned)ceil_div(T, 4)), dim3(256), st, ga)) return rc;
  LossTileArgs a{};
  a.rows = s.rows, a.x = ga.x, a.w = reinterpret_cast<const uint16_t*>(w), a.g = s.g, a.dx = s.dx;
  a.dw = reinterpret_cast<uint16_t*>(dw), a.T = T, a.H = H, a.V = V, a.ldg = s.piece, a.most_splits = kLossMostSplits;
  const int tile = few ? kLossFewRows : kLossRows, h_tiles = ceil_div(H, 256);
  int most_units = 0;  // of dx, whatever the number of labelled rows
  for (int r = 1; r <= ceil_div(T, tile); ++r) {
    const int u = r * h_tiles * loss_splits(r, h_tiles, kLossMostSplits);
    if (u > most_units) most_units = u;
  }
  for (int v0 = 0; v0 < V; v0 += s.piece) {
    a.v0 = v0, a.v1 = V - v0 < s.piece ? V : v0 + s.piece, a.add = v0 > 0;
    const int v_tiles = ceil_div(a.v1 - v0, kLossTileV);
    const dim3 bl(256), grid = loss_grid((int64_t)ceil_div(T, tile) * v_tiles);
    int rc = f16 ? loss_logits<SMLM_DTYPE_F16>(few, true, grid, st, a) : loss_logits<SMLM_DTYPE_BF16>(few, true, grid, st, a);
    if (rc) return rc;
    if (dx) {
      const dim3 gx = loss_grid(most_units);
      if (few)
        rc = f16 ? launch(loss_dx_kernel<SMLM_DTYPE_F16, true>, gx, bl, st, a)
                 : launch(loss_dx_kernel<SMLM_DTYPE_BF16, true>, gx, bl, st, a);
      else
        rc = f16 ? launch(loss_dx_kernel<SMLM_DTYPE_F16, false>, gx, bl, st, a)
                 : launch(loss_dx_kernel<SMLM_DTYPE_BF16, false>, gx, bl, st, a);
      if (rc) return rc;
    }
    if (dw) {
      const dim3 gw = loss_grid((int64_t)h_tiles * v_tiles);
      rc = f16 ? launch(loss_dw_kernel<SMLM_DTYPE_F16>, gw, bl, st, a) : launch(loss_dw_kernel<SMLM_DTYPE_BF16>, gw, bl, st, a);
      if (rc) return rc;
    }
  }
  if (!dx) return SMLM_OK;
  const LossDxFoldArgs fa{s.rows, s.dx, reinterpret_cast<uint16_t*>(dx), T, H, few, kLossMostSplits};
  const dim3 grid((unsigned)ceil_div(T, 4));
  return f16 ? launch(loss_dx_fold_kernel<SMLM_DTYPE_F16>, grid, dim3(256), st, fa)
             : launch(loss_dx_fold_kernel<SMLM_DTYPE_BF16>, grid, dim3(256), st, fa);
}
