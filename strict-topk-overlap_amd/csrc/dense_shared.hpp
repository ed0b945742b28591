// Dense attention of single tokens whose requests share leading blocks.
//
// One launch of two kinds of workgroup: the first pgrid work on the groups' shared
// blocks, each tile 128 query rows of a group's requests (dense_prefill.hpp), the others
// on the requests' own keys (dense_decode.hpp).  All leave parts, which
// k_join_rows joins.  96 requests, 32 query heads over 8, D = 128, of which 32768 keys
// are shared and 1 to 2000 their own: 90 us, 62 of them on the shared blocks' 51
// GFLOP, then 20 to 30 on the others' 100 MB (a CU holds two workgroups of
// either kind, so the kinds hardly overlap), and 11 for the join of 33 MB of parts.
#pragma once

#include "dense_decode.hpp"
#include "dense_prefill.hpp"

namespace stk {

template <typename T, int D, int MODE>
__global__ __launch_bounds__(256, 2) void k_shared(DenseArgs a, Plan pl, Parts psplit,
                                                                  Parts pwhole, int pgrid,
                                                                  Parts split, Parts whole,
                                                                  int32_t* place) {
  constexpr size_t N = kPrefillLds<D> > kDecodeLds<D> ? kPrefillLds<D> : kDecodeLds<D>;
  __shared__ __attribute__((aligned(1024))) char lds[N];
  const int wg = (int)blockIdx.x;
  if (wg < pgrid) {
    prefill<T, D, MODE, GROUPED>(a, pl, psplit, pwhole, lds, wg, pgrid);
  } else {
    decode<T, D, MODE, true>(a, split, whole, place, lds, wg - pgrid, (int)gridDim.x - pgrid);
  }
}

}  // namespace stk
