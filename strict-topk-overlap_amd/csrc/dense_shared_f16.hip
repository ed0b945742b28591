// Dense attention over shared blocks, F16 (k_shared).
#include "dense_shared.hpp"

namespace stk {

template <>
int launch_shared<f16s>(int d, int mode, const DenseArgs& a, const Plan& p, const Parts& psplit,
                      const Parts& pwhole, int pgrid, const Parts& split, const Parts& whole,
                      int32_t* place, int grid, hipStream_t st) {
#define STK_MODE(D)                                                                                                        \
  switch (mode) {                                                                                                          \
    case 0: k_shared<f16s, D, 0><<<pgrid + grid, 256, 0, st>>>(a, p, psplit, pwhole, pgrid, split, whole, place); break;   \
    case 1: k_shared<f16s, D, 1><<<pgrid + grid, 256, 0, st>>>(a, p, psplit, pwhole, pgrid, split, whole, place); break;   \
    case 2: k_shared<f16s, D, 2><<<pgrid + grid, 256, 0, st>>>(a, p, psplit, pwhole, pgrid, split, whole, place); break;   \
    default: k_shared<f16s, D, 3><<<pgrid + grid, 256, 0, st>>>(a, p, psplit, pwhole, pgrid, split, whole, place); break;  \
  }
  if (d == 64) {
    STK_MODE(64)
  } else if (d == 128) {
    STK_MODE(128)
  } else {
    STK_MODE(256)
  }
#undef STK_MODE
  return stk_check_launch("k_shared");
}

}  // namespace stk
