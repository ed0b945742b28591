// Dense attention of many query rows over the paged cache: chunks of prompts,
// whole prompts, and the shared leading blocks of a decode batch.
//
// A tile is up to 128 query rows (token, head) of one KV head, so that the
// heads of a KV group share its keys; four waves own 32 rows each, and walk
// the tile's keys in units of TK.  K and V of a unit pass through LDS, double
// buffered: the next unit's rows travel to registers while this one is
// worked on, and one barrier per unit hands them over.
//   S[key, row] = K Q^T (32x32x16), O^T[dim, row] += V^T P^T
// Column `row` of both products is one lane (and its partner 32 lanes on), so
// the softmax needs no exchange but that of the two halves' maxima, and the
// output's rescaling is one multiplier per lane.  Lane half h holds keys 8j + 4h
// .. + 3 of S; taking them in that order as the second product's keys leaves
// P in its lane, and V is read transposed from LDS to match.
// LDS rows are swizzled (16-byte chunks of K, 64-byte blocks of V) so that
// neither read has bank conflicts.
//
// Masks are one range of keys per row; units that every row of the tile sees whole
// (all but the first and last ones) skip them.  In the others a value that no
// row sees is zeroed on its way to LDS, and should a value that some rows see
// and others do not be infinite or NaN, the unit's product is done by rows,
// skipping the hidden keys.
#pragma once

#include "dense.hpp"

namespace stk {

__device__ __forceinline__ bool nonfinite16(u16x8 v, uint16_t expo) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) bad |= (v[i] & expo) == expo;
  return bad;
}

template <typename T, int D, int MODE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_prefill(DenseArgs a, Plan pl,
                                                                   Parts split, Parts whole,
                                                                   int direct) {
  constexpr int TK = kTk<D>;
  constexpr int KB = TK / 32;           // 32-key blocks of S
  constexpr int KS = D / 16;            // QK steps
  constexpr int DB = D / 32;            // output blocks
  constexpr int CPR = D / 8;            // 16-byte chunks per row
  constexpr int RP = 256 / CPR;         // rows per load instruction of the workgroup
  constexpr int KN = TK / RP;           // load instructions per unit and thread
  constexpr int GR = TK / 16;           // runs of 16 keys per unit
  constexpr int PS = D == 64 ? 4 * 32 * TK : 8;   // room for P by rows beside K's own
  constexpr uint16_t EXPO = __is_same(T, bf16s) ? 0x7f80 : 0x7c00;
  __shared__ __attribute__((aligned(16))) uint16_t s_k[2][TK * D], s_v[2][TK * D], s_p[PS];
  __shared__ int s_bad[2];
  const int tid = threadIdx.x, lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(wave_id());
  const int n32 = lane & 31, h = lane >> 5, i16 = lane & 15, gq = (lane >> 4) & 1;

  // rows of no request
  if (a.fill && a.starts) {
    const int f0 = min(max(a.starts[0], 0), a.t);
    const int f1 = max(f0, min(max(a.starts[a.requests], 0), a.t));
    const int64_t wide = (int64_t)a.hq * D / 8;
    for (int t = (int)blockIdx.x; t < f0 + (a.t - f1); t += (int)gridDim.x) {
      uint16_t* o = a.out + (int64_t)(t < f0 ? t : f1 + t - f0) * a.hq * D;
      for (int64_t x = tid; x < wide; x += 256) *reinterpret_cast<u16x8*>(o + 8 * x) = u16x8{};
    }
  }

  const int per = pl.head[0], ntiles = pl.head[1];
  int64_t u, u1;
  int kvh, it;
  if (direct) {
    const int total = ntiles * a.hkv;
    if ((int)blockIdx.x >= total) return;
    const int x = xcd_remap((int)blockIdx.x, total);
    kvh = x / ntiles;
    it = x % ntiles;
    u = 0;
    u1 = 1;
  } else {
    const int64_t total = (int64_t)per * a.hkv;
    const int grid = split_grid(total, (int)gridDim.x);
    if ((int)blockIdx.x >= grid) return;
    u = unit_at(total, (int)blockIdx.x, grid);
    u1 = unit_at(total, (int)blockIdx.x + 1, grid);
    kvh = (int)(u / per);
    const int rem = (int)(u % per);
    int lo = 0, hi = ntiles - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (pl.tiles[mid].cum <= rem) lo = mid;
      else hi = mid - 1;
    }
    it = __builtin_amdgcn_readfirstlane(lo);
  }
  if (tid < 2) s_bad[tid] = 0;
  int serial = 0;                       // units handed over so far, in this workgroup

  // LDS addresses (elements)
  auto fk = [](int row) { return D == 64 ? (row >> 1) & 7 : row & 15; };
  auto fv = [](int row) { return D == 64 ? (row >> 1) & 1 : row & 3; };
  const int lrow = tid / CPR, lch = tid % CPR;
  int kw[KN], vw[KN], ka[KS], va[DB];
#pragma unroll
  for (int i = 0; i < KN; ++i) {
    const int row = i * RP + lrow;
    kw[i] = row * D + (lch ^ fk(row)) * 8;
    vw[i] = row * D + ((((lch >> 2) ^ fv(row)) << 2) | (lch & 3)) * 8;
  }
#pragma unroll
  for (int s = 0; s < KS; ++s) ka[s] = n32 * D + ((2 * s + h) ^ fk(n32)) * 8;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const int row = 4 * h + (i16 >> 2);
    va[db] = row * D + (db ^ fv(row)) * 32 + 16 * gq + 4 * (i16 & 3);
  }

  while (u < u1) {
    const Tile tl = pl.tiles[it];
    const int seq = __builtin_amdgcn_readfirstlane(tl.seq);
    const int tile = __builtin_amdgcn_readfirstlane(tl.tile);
    const int kstart = __builtin_amdgcn_readfirstlane(tl.kstart);
    const int klo = __builtin_amdgcn_readfirstlane(tl.klo);
    const int khi = __builtin_amdgcn_readfirstlane(tl.khi);
    const int max_lo = __builtin_amdgcn_readfirstlane(tl.max_lo);
    const int min_hi = __builtin_amdgcn_readfirstlane(tl.min_hi);
    const int n = max(1, (khi - kstart + TK - 1) / TK);
    int j0 = 0, j1 = n;
    if (!direct) {
      const int64_t first = (int64_t)kvh * per + __builtin_amdgcn_readfirstlane(tl.cum);
      j0 = (int)(u - first);
      j1 = (int)min((int64_t)n, j0 + (u1 - u));
      u += j1 - j0;
    } else {
      u = u1;
    }
    int s0, s1;
    seq_rows(a, seq, s0, s1);
    const int64_t rown = (int64_t)tile * kDenseRows + 32 * w + n32;
    const bool valid = rown < (int64_t)(s1 - s0) * a.g;
    const int tok = s0 + (int)(valid ? rown / a.g : 0);
    const int head = kvh * a.g + (int)(valid ? rown % a.g : 0);
    int p = 0;
    Span sp = seq_span(a, seq, s0, s1, tok, p);
    if (!valid) sp = Span{0, 0x7fffffff};
    // keys that some row of this wave sees
    int wlo = valid && sp.hi > sp.lo ? sp.lo : 0x7fffffff;
    int whi = valid && sp.hi > sp.lo ? sp.hi : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      wlo = min(wlo, __shfl_xor(wlo, o));
      whi = max(whi, __shfl_xor(whi, o));
    }
    wlo = __builtin_amdgcn_readfirstlane(wlo);
    whi = __builtin_amdgcn_readfirstlane(whi);
    u16x8 qf[KS];
    const uint16_t* qp = a.q + (int64_t)tok * a.qs + (int64_t)head * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u16x8*>(qp + 16 * s);
    float slope = 0.f;
    if constexpr (MODE & 2) slope = a.slopes[head] * 1.44269504f;
    const int32_t* row =
        a.table + ((int64_t)(a.groups ? min(max(s0, 0), a.requests - 1) : seq) * a.hkv + kvh) * a.nb;
    const int kbase = kstart + j0 * TK, kend = min(kstart + j1 * TK, khi);
    const int cnt = j1 - j0;

    auto window = [&](int i) {                        // rows of 64 runs of 16 keys
      const int key = kbase + 16 * (64 * i + lane);
      const int x = pool_row(a, row, min(key, kend));
      return key < kend ? x : -1;
    };
    int ent = window(0), nxt = window(1);
    u16x8 kf[KN], vf[KN];
    int rows[GR];                                     // of the unit in kf, vf
    auto load = [&](int j) {
      if (j > 0 && (j * GR) % 64 == 0) {
        ent = nxt;
        nxt = window(j * GR / 64 + 1);
      }
#pragma unroll
      for (int x = 0; x < GR; ++x) rows[x] = __builtin_amdgcn_readlane(ent, (j * GR + x) & 63);
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        // this wave's rows of load i lie in one run of 16 keys
        const int run = (i * RP + w * (RP / 4)) / 16;
        const int x = D == 64 ? (w < 2 ? rows[2 * i < GR ? 2 * i : 0] : rows[2 * i + 1 < GR ? 2 * i + 1 : 0])
                              : rows[i * RP / 16];
        const int64_t at = (int64_t)max(x, 0) * D;
        const int off = (i * RP + lrow - 16 * run) * D + 8 * lch;
        kf[i] = *reinterpret_cast<const u16x8*>(a.kp + at + off);
        vf[i] = *reinterpret_cast<const u16x8*>(a.vp + at + off);
      }
    };
    // unit j sees no mask
    auto inner = [&](int key0) {
      bool ok = key0 >= max_lo && key0 + TK <= min_hi;
#pragma unroll
      for (int x = 0; x < GR; ++x) ok = ok && rows[x] >= 0;
      return ok;
    };
    int crow[GR];                                     // of the unit in LDS
    auto stage = [&](int j, int buf) {                // kf, vf to LDS
      const int key0 = kbase + j * TK;
      if (!inner(key0)) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < KN; ++i) {
          const int kr = i * RP + lrow, key = key0 + kr;
          bool ok = key >= klo && key < khi;
#pragma unroll
          for (int x = 0; x < GR; ++x) ok = ok && !(kr / 16 == x && rows[x] < 0);
          if (!ok) vf[i] = u16x8{};
          bad |= nonfinite16(vf[i], EXPO);
        }
        if (bad) s_bad[buf] = serial + 1;
      }
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        *reinterpret_cast<u16x8*>(s_k[buf] + kw[i]) = kf[i];
        *reinterpret_cast<u16x8*>(s_v[buf] + vw[i]) = vf[i];
      }
    };

    float m = -INFINITY, l = 0.f;
    f32x16 acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[i][x] = 0.f;

    load(0);
    __syncthreads();                                  // the last item's LDS reads are done
    stage(0, 0);
    bool edge = !inner(kbase);
#pragma unroll
    for (int x = 0; x < GR; ++x) crow[x] = rows[x];
    if (cnt > 1) load(1);
    for (int j = 0; j < cnt; ++j) {
      const int buf = j & 1, key0 = kbase + j * TK;
      __syncthreads();
      ++serial;
      const bool bad = edge && s_bad[buf] == serial;
      const uint16_t* lk = s_k[buf];
      const uint16_t* lv = s_v[buf];
      const bool work = key0 < whi && key0 + TK > wlo;
      u16x8 pf[TK / 16];
      if (work) {
        f32x16 s[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
#pragma unroll
          for (int x = 0; x < 16; ++x) s[b][x] = 0.f;
#pragma unroll
          for (int x = 0; x < KS; ++x)
            s[b] = mma32<T>(*reinterpret_cast<const u16x8*>(lk + ka[x] + 32 * b * D), qf[x], s[b]);
        }
        const float dist = (float)(p - key0 - 4 * h);
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int off = 32 * b + 8 * (x / 4) + x % 4;
            s[b][x] = score2<MODE>(a, s[b][x], slope, dist - (float)off);
          }
        if (edge) {
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              const int key = key0 + 4 * h + 32 * b + 8 * (x / 4) + x % 4;
              const bool ok = key >= sp.lo && key < sp.hi && crow[2 * b + x / 8] >= 0;
              s[b][x] = ok ? s[b][x] : -INFINITY;
            }
        }
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x) top = fmaxf(top, s[b][x]);
        if (__any(top > m + kLazy)) {
          float mx = fmaxf(top, m);
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float f = mx == m ? 1.f : __builtin_amdgcn_exp2f(m - mx);
          m = mx;
          l *= f;
#pragma unroll
          for (int i = 0; i < DB; ++i) acc[i] *= f;
        }
        const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const float e = __builtin_amdgcn_exp2f(s[b][x] - ms);
            l += e;
            pf[2 * b + x / 8][x % 8] = to16<T>(e);
          }
      }
      if (!bad) {
        if (work) {
#pragma unroll
          for (int x = 0; x < TK / 16; ++x)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const u16x4 lo = lds_tr(lv + va[db] + 16 * x * D);
              const u16x4 hi = lds_tr(lv + va[db] + (16 * x + 8) * D);
              acc[db] = mma32<T>(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf[x],
                                 acc[db]);
            }
        }
      } else {
        // some value is infinite or NaN: by rows, hidden keys skipped.  P goes
        // through the unit's K (all waves are past it) or, at D = 64, its own room.
        __syncthreads();
        if (work) {
          uint16_t* sp16 = (D == 64 ? s_p : s_k[buf]) + w * 32 * TK;
#pragma unroll
          for (int x = 0; x < TK / 16; ++x)
#pragma unroll
            for (int e = 0; e < 8; ++e)
              sp16[n32 * TK + 16 * x + 8 * (e / 4) + 4 * h + e % 4] = pf[x][e];
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          for (int k = 0; k < TK; ++k) {
            const float pk = cvt(T{sp16[n32 * TK + k]});
            const int key = key0 + k;
            const bool ok = key >= sp.lo && key < sp.hi;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                // dims 32 db + 8 x + 4 h .. + 3
                const u16x4 v4 = *reinterpret_cast<const u16x4*>(
                    lv + k * D + (db ^ fv(k)) * 32 + 8 * x + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float o = acc[db][4 * x + e];
                  acc[db][4 * x + e] = ok ? o + pk * cvt(T{v4[e]}) : o;
                }
              }
          }
        }
      }
      if (j + 1 < cnt) {
        stage(j + 1, buf ^ 1);
        edge = !inner(key0 + TK);
#pragma unroll
        for (int x = 0; x < GR; ++x) crow[x] = rows[x];
        if (j + 2 < cnt) load(j + 2);
      }
    }
    l += __shfl_xor(l, 32);
    const bool all = j0 == 0 && j1 == n;
    if (valid) {
      if (all && !whole.m) {
        uint16_t* o = a.out + ((int64_t)tok * a.hq + head) * D + 4 * h;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            store_out<T>(o + 32 * db + 8 * x,
                         f32x4{acc[db][4 * x], acc[db][4 * x + 1], acc[db][4 * x + 2],
                               acc[db][4 * x + 3]}, l);
      } else {
        const Parts& to = all ? whole : split;
        const int64_t slot = all ? (int64_t)kvh * ntiles + it
                                 : 2 * (int64_t)blockIdx.x + (j0 > 0 ? 0 : 1);
        const int64_t pr = slot * kDenseRows + 32 * w + n32;
        float* o = to.o + pr * D + 4 * h;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *reinterpret_cast<f32x4*>(o + 32 * db + 8 * x) =
                f32x4{acc[db][4 * x], acc[db][4 * x + 1], acc[db][4 * x + 2], acc[db][4 * x + 3]};
        if (h == 0) {
          to.m[pr] = m;
          to.l[pr] = l;
        }
      }
    }
    if (++it == ntiles) {
      it = 0;
      ++kvh;
    }
  }
}

}  // namespace stk
