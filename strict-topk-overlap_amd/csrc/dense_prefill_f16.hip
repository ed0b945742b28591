// Dense attention of many rows, F16 (k_prefill).
#include "dense_prefill.hpp"

namespace stk {

template <>
int launch_prefill<f16s>(int d, int mode, const DenseArgs& a, const Plan& p, const Parts& split,
                       int grid, hipStream_t st) {
#define STK_MODE(D)                                                                    \
  switch (mode) {                                                                      \
    case 0: k_prefill<f16s, D, 0, LISTED><<<grid, 256, 0, st>>>(a, p, split); break;   \
    case 1: k_prefill<f16s, D, 1, LISTED><<<grid, 256, 0, st>>>(a, p, split); break;   \
    case 2: k_prefill<f16s, D, 2, LISTED><<<grid, 256, 0, st>>>(a, p, split); break;   \
    default: k_prefill<f16s, D, 3, LISTED><<<grid, 256, 0, st>>>(a, p, split); break;  \
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
