// Dense decode attention, F16 (dense_decode.hpp).
#include "dense_decode.hpp"

namespace stk {

template <>
int launch_decode<f16s>(int d, int mode, const DenseArgs& a, const Parts& split, const Parts& whole,
                         int32_t* place, int grid, hipStream_t st) {
#define STK_MODE(D)                                                                            \
  switch (mode) {                                                                              \
    case 0: hipLaunchKernelGGL((k_decode<f16s, D, 0>), dim3(grid), dim3(256), 0, st, a, split, \
                               whole, place); break;                                           \
    case 1: hipLaunchKernelGGL((k_decode<f16s, D, 1>), dim3(grid), dim3(256), 0, st, a, split, \
                               whole, place); break;                                           \
    case 2: hipLaunchKernelGGL((k_decode<f16s, D, 2>), dim3(grid), dim3(256), 0, st, a, split, \
                               whole, place); break;                                           \
    default: hipLaunchKernelGGL((k_decode<f16s, D, 3>), dim3(grid), dim3(256), 0, st, a,       \
                                split, whole, place);                                          \
  }
  if (d == 64) {
    STK_MODE(64)
  } else if (d == 128) {
    STK_MODE(128)
  } else {
    STK_MODE(256)
  }
#undef STK_MODE
  return stk_check_launch("k_decode");
}

}  // namespace stk
