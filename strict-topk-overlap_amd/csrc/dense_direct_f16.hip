// Dense attention of many rows, F16, no tile split (k_prefill).
#include "dense_prefill.hpp"

namespace stk {

template <>
int launch_direct<f16s>(int d, int mode, const DenseArgs& a, int grid, hipStream_t st) {
#define STK_MODE(D)                                                                           \
  switch (mode) {                                                                             \
    case 0: k_prefill<f16s, D, 0, DIRECT><<<grid, 256, 0, st>>>(a, Plan{}, Parts{}); break;   \
    case 1: k_prefill<f16s, D, 1, DIRECT><<<grid, 256, 0, st>>>(a, Plan{}, Parts{}); break;   \
    case 2: k_prefill<f16s, D, 2, DIRECT><<<grid, 256, 0, st>>>(a, Plan{}, Parts{}); break;   \
    default: k_prefill<f16s, D, 3, DIRECT><<<grid, 256, 0, st>>>(a, Plan{}, Parts{}); break;  \
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
