// Sums over the 64 lanes of a wave with DPP adds.
#pragma once
#include "smlm_common.hpp"

namespace smlm {

// Inclusive sums over a wave: shifts inside rows of 16 lanes, then the rows' totals.
#define SMLM_DPP(x, ctrl, rmask) __builtin_amdgcn_update_dpp(0, x, ctrl, rmask, 0xf, false)
__device__ __forceinline__ int wave_scan(int v) {
  v += SMLM_DPP(v, 0x111, 0xf);  // row_shr:1
  v += SMLM_DPP(v, 0x112, 0xf);
  v += SMLM_DPP(v, 0x114, 0xf);
  v += SMLM_DPP(v, 0x118, 0xf);
  v += SMLM_DPP(v, 0x142, 0xa);  // row_bcast:15 into rows 1 and 3
  v += SMLM_DPP(v, 0x143, 0xc);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ float wave_total(float v) {
  auto add = [&](int moved) { v += __builtin_bit_cast(float, moved); };
  add(SMLM_DPP(__builtin_bit_cast(int, v), 0x111, 0xf));
  add(SMLM_DPP(__builtin_bit_cast(int, v), 0x112, 0xf));
  add(SMLM_DPP(__builtin_bit_cast(int, v), 0x114, 0xf));
  add(SMLM_DPP(__builtin_bit_cast(int, v), 0x118, 0xf));
  add(SMLM_DPP(__builtin_bit_cast(int, v), 0x142, 0xa));
  add(SMLM_DPP(__builtin_bit_cast(int, v), 0x143, 0xc));
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
#undef SMLM_DPP

}  // namespace smlm
