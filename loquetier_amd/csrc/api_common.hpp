// Host helpers shared by the translation units of the C ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smlm.h"

namespace smlm {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int ceil_div(int a, int b) { return (a + b - 1) / b; }
inline int round_up(int a, int b) { return ceil_div(a, b) * b; }

// Every kernel takes one argument struct.  hipLaunchKernel hands back the
// status of this launch itself; the thread's "last error" slot is shared with
// every other HIP user in the process (torch leaves benign codes there), so it
// is neither read nor cleared here.
template <typename A>
int launch(void (*kernel)(A), dim3 grid, dim3 block, hipStream_t st, const A& a) {
  void* params[] = {const_cast<A*>(&a)};
  return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, params, 0, st) ==
                 hipSuccess
             ? SMLM_OK
             : SMLM_ERR_LAUNCH;
}

}  // namespace smlm
