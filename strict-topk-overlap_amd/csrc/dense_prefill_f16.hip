// Dense attention of many query rows, F16 (dense_prefill.hpp).
#include "dense_prefill.hpp"

namespace stk {

template <>
int launch_prefill<f16s>(int d, int mode, const DenseArgs& a, const Plan& p, const Parts& split,
                          const Parts& whole, int grid, bool direct, hipStream_t st) {
#define STK_MODE(D)                                                                              \
  switch (mode) {                                                                                \
    case 0: hipLaunchKernelGGL((k_prefill<f16s, D, 0>), dim3(grid), dim3(256), 0, st, a, p,      \
                               split, whole, direct); break;                                     \
    case 1: hipLaunchKernelGGL((k_prefill<f16s, D, 1>), dim3(grid), dim3(256), 0, st, a, p,      \
                               split, whole, direct); break;                                     \
    case 2: hipLaunchKernelGGL((k_prefill<f16s, D, 2>), dim3(grid), dim3(256), 0, st, a, p,      \
                               split, whole, direct); break;                                     \
    default: hipLaunchKernelGGL((k_prefill<f16s, D, 3>), dim3(grid), dim3(256), 0, st, a, p,     \
                                split, whole, direct);                                           \
  }
  if (d == 64) {
    STK_MODE(64)
  } else if (d == 128) {
    STK_MODE(128)
  } else {
    STK_MODE(256)
  }
#undef STK_MODE
  return stk_check_launch("k_prefill");
}

}  // namespace stk
