// Dense attention over shared blocks, F16 (k_shared).
#include "dense_shared.hpp"

namespace stk {

template <>
int launch_shared<f16s>(int d, int mode, const DenseArgs& a, const Plan& p, const Parts& psplit,
                      const Parts& pwhole, int pgrid, const Parts& split, const Parts& whole,
                      int32_t* place, int grid, hipStream_t st) {
#define STK_RUN(D, M)                                                                  \
  k_shared<f16s, D, M><<<pgrid + grid, 256, 0, st>>>(a, p, psplit, pwhole, pgrid,      \
                                                     split, whole, place)
#define STK_MODE(D)                 \
  switch (mode) {                   \
    case 0: STK_RUN(D, 0); break;   \
    case 1: STK_RUN(D, 1); break;   \
    case 2: STK_RUN(D, 2); break;   \
    default: STK_RUN(D, 3); break;  \
  }
  if (d == 64) {
    STK_MODE(64)
  } else if (d == 128) {
    STK_MODE(128)
  } else {
    STK_MODE(256)
  }
#undef STK_MODE
#undef STK_RUN
  return stk_check_launch("k_shared");
}

}  // namespace stk
