// Dense decode attention, F16 (k_decode).
#include "dense_decode.hpp"

namespace stk {

template <>
int launch_decode<f16s>(int d, int mode, const DenseArgs& a, const Parts& split, int32_t* place,
                      int grid, hipStream_t st) {
#define STK_MODE(D)                                                               \
  switch (mode) {                                                                 \
    case 0: k_decode<f16s, D, 0, false><<<grid, 256, 0, st>>>(a, split, place); break;   \
    case 1: k_decode<f16s, D, 1, false><<<grid, 256, 0, st>>>(a, split, place); break;   \
    case 2: k_decode<f16s, D, 2, false><<<grid, 256, 0, st>>>(a, split, place); break;   \
    default: k_decode<f16s, D, 3, false><<<grid, 256, 0, st>>>(a, split, place); break;  \
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
