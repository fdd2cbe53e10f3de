// Host side of the RMSNorm kernels that the norm and the norm behind a residual's addition share: launch shapes.
#pragma once
#include "api_common.hpp"
#include "rms_norm.hpp"

namespace smlm {

inline int rms_bwd_threads(int cols) {
  const int pieces = cols / 8;  // a piece a thread, or two where a row has more than 1024
  return round_up(pieces <= 1024 ? pieces : ceil_div(pieces, 2), kWaveSize);
}
// workgroups of the RMSNorm kernels: the forward gives every row group its own workgroup; the backward's fill the
// chip once (up to 512 threads a CU, the same number on every CU) with two rows each or more, so that the partial sums
// of dw stay small next to x and g.
inline int rms_blocks(int rows, int cols, bool backward) {
  int nb, cap = 1 << 22;
  if (cols > kRmsMaxCols) {  // wide rows: a workgroup per row; the backward's partial rows are whole rows of floats
    nb = rows;
    if (backward) cap = 128;
  } else if (backward) {
    const int threads = rms_bwd_threads(cols);
    nb = ceil_div(rows, 2);
    cap = 256 * (threads >= 512 ? 1 : 512 / threads);
  } else {
    nb = ceil_div(rows, cols <= kRmsWaveCols ? 4 : 1);
  }
  if (nb > cap) nb = cap;
  return nb < 1 ? 1 : nb;
}
inline int rms_bwd_blocks(int rows, int cols) { return rms_blocks(rows, cols, true); }

inline int rms_check(int rows, int cols, int dtype) {
  if (rows < 0 || cols <= 0) return SMLM_ERR_ARG;
  if (dtype != SMLM_DTYPE_F16 && dtype != SMLM_DTYPE_BF16) return SMLM_ERR_DTYPE;
  if (cols & 7) return SMLM_ERR_ALIGN;
  if (cols > (1 << 24) || rows > (1 << 30)) return SMLM_ERR_LIMIT;
  return SMLM_OK;
}

// ADD: the gradient that reaches the norm's input by another way is added to dx.
template <int DT, bool ADD>
int launch_rms_bwd(int nb, hipStream_t st, const RmsBwdArgs& a) {
  const dim3 grid((unsigned)nb), bl((unsigned)rms_bwd_threads(a.cols));
  if (a.cols > kRmsMaxCols) return launch(rms_bwd_wide_kernel<DT, ADD>, grid, dim3(256), st, a);
  if (a.cols <= 8192) return launch(rms_bwd_kernel<DT, 1, 2, ADD>, grid, bl, st, a);
  return launch(rms_bwd_kernel<DT, 2, 1, ADD>, grid, bl, st, a);
}

// Columns a workgroup of the RMSNorm backward's fold takes: 16 where a row is short, so that its workgroups fill the
// chip; of wider rows 32 and 64, as the pieces of 64 bytes that 16 columns read of every partial row fetch the lines
// twice.  Whole backward, us, 16 / 32 / 64 columns: 4096 x 2048 16.9 / 16.9 / -, 1000 x 4096 12.4 / 11.0 / -,
// 1000 x 8192 21.8 / 18.8 / 18.6, 1000 x 11008 28.7 / 25.1 / 24.8, 64 x 20480 16.9 / - / 14.5.
template <int DT>
int launch_rms_fold(hipStream_t st, const RmsFoldArgs& a) {
  const dim3 bl(256);
  if (a.cols <= 2048) return launch(rms_fold_kernel<DT, 4>, dim3((unsigned)ceil_div(a.cols, 16)), bl, st, a);
  if (a.cols <= 4096) return launch(rms_fold_kernel<DT, 8>, dim3((unsigned)ceil_div(a.cols, 32)), bl, st, a);
  return launch(rms_fold_kernel<DT, 16>, dim3((unsigned)ceil_div(a.cols, 64)), bl, st, a);
}

}  // namespace smlm
