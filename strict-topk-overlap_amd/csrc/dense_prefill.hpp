// Dense attention of many query rows over the paged cache: chunks of prompts,
// whole prompts, and the shared leading blocks of a decode batch.
//
// A tile is up to 128 query rows (token, head) of one KV head, so that the
// heads of a KV group share its keys; four waves own 32 rows each, and walk
// the tile's keys in units of TK.  K and V of a unit come straight into LDS
// (no registers on the way), double buffered: the next unit travels while
// this one is worked on, and one barrier per unit hands it over.
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
// (all but the first and last ones) skip them.  In the others the values that no
// row sees are zeroed in LDS; should a value that some rows see and others do
// not be infinite or NaN (0 times which is not 0), the tile is done row by row
// instead, each row reading the keys that it sees (slow_rows).
#pragma once

#include "dense.hpp"

namespace stk {

__device__ __forceinline__ bool nonfinite16(u16x8 v, uint16_t expo) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) bad |= (v[i] & expo) == expo;
  return bad;
}

// 16 bytes per lane from base + off to LDS, lane after lane from byte `lds`
// (wave-uniform) on.  Counted by vmcnt like any load; the compiler does not
// know of the write, so the caller waits (copies_done) and passes a barrier
// before it reads.  (Its own intrinsic makes the compiler wait for all of these
// before every LDS read.)
__device__ __forceinline__ void copy_to_lds(uint32_t lds, const uint16_t* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Up to 32 query rows from rown on against the keys [kbase, kend), one row after the
// other: a lane is a key for the scores and D / 64 dims for the output, and
// hidden keys and their values are not read.
template <typename T, int D, int MODE>
__device__ void slow_rows(const DenseArgs& a, int seq, int s0, int s1, int64_t rown, int kvh,
                          const int32_t* row, int kbase, int kend, const Parts* to, int64_t pr) {
  constexpr int E = D / STK_WAVE;
  const int lane = lane_id();
  for (int i = 0; i < 32; ++i, ++rown, ++pr) {
    if (rown >= (int64_t)(s1 - s0) * a.g) return;
    const int tok = s0 + (int)(rown / a.g), head = kvh * a.g + (int)(rown % a.g);
    int p;
    const Span sp = seq_span(a, seq, s0, s1, tok, p);
    const uint16_t* q = a.q + (int64_t)tok * a.qs + (int64_t)head * D;
    float slope = 0.f;
    if constexpr (MODE & 2) slope = a.slopes[head] * 1.44269504f;
    float m = -INFINITY, l = 0.f, o[E] = {};
    const int lo = max(kbase, sp.lo), hi = min(kend, sp.hi);
    for (int k0 = lo & ~15; k0 < hi; k0 += STK_WAVE) {
      const int key = k0 + lane;
      const int run = pool_row(a, row, min(key, hi - 1) & ~15);
      const bool ok = key >= lo && key < hi && run >= 0;
      const int64_t at = ((int64_t)max(run, 0) + (key & 15)) * D;
      float s = 0.f;
      if (ok)
        for (int x = 0; x < D; ++x) s += cvt(T{q[x]}) * cvt(T{a.kp[at + x]});
      s = ok ? score2<MODE>(a, s, slope, (float)(p - key)) : -INFINITY;
      const float mx = fmaxf(m, wave_max(s)), ms = mx == -INFINITY ? 0.f : mx;
      const float f = part_weight(m, mx), e = ok ? __builtin_amdgcn_exp2f(s - ms) : 0.f;
      m = mx;
      l = l * f + wave_sum(e);
#pragma unroll
      for (int x = 0; x < E; ++x) o[x] *= f;
      const uint64_t seen = __ballot(ok);
      for (int k = 0; k < STK_WAVE; ++k) {
        if (!(seen >> k & 1)) continue;
        const float ek = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, e), k));
        const int rk = __builtin_amdgcn_readlane(run, k) + ((k0 + k) & 15);
#pragma unroll
        for (int x = 0; x < E; ++x)
          o[x] += ek * cvt(T{a.vp[(int64_t)rk * D + lane + STK_WAVE * x]});
      }
    }
    if (to) {
#pragma unroll
      for (int x = 0; x < E; ++x) to->o[pr * D + lane + STK_WAVE * x] = o[x];
      if (lane == 0) {
        to->m[pr] = m;
        to->l[pr] = l;
      }
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int x = 0; x < E; ++x)
        a.out[((int64_t)tok * a.hq + head) * D + lane + STK_WAVE * x] = to16<T>(o[x] * inv);
    }
  }
}

// The tile of workgroup wg where every tile has its own: tiles of one KV head after
// the other, dealt to the XCDs in runs, and within a sequence the last rows,
// which see the most keys, first.  kvh = Hkv: none.
struct TilePlace { int seq, tile, kvh; };

__device__ __forceinline__ TilePlace tile_place(const DenseArgs& a, int wg, int nwg) {
  __shared__ int s_tmp[4], s_at[2];
  const int ns = sequences(a);
  auto tiles = [&](int q) {
    int s0 = 0, s1 = 0;
    if (q < ns) seq_rows(a, q, s0, s1);
    return (int)(((int64_t)(s1 - s0) * a.g + kDenseRows - 1) / kDenseRows);
  };
  int total = 0, c0 = 0, b0 = 0, sum0 = 0;
  for (int q0 = 0; q0 < ns; q0 += 256) {
    const int c = tiles(q0 + (int)threadIdx.x);
    int sum;
    __syncthreads();
    const int before = block_excl_scan1(c, s_tmp, &sum);   // (of the first 256: from 0)
    if (q0 == 0) {
      c0 = c;
      b0 = before;
      sum0 = sum;
    }
    total += sum;
  }
  const int64_t all = min((int64_t)total * a.hkv, (int64_t)nwg);
  if (wg >= all) return TilePlace{0, 0, a.hkv};
  const int x = xcd_remap(wg, (int)all), kvh = x / total, it = x % total;
  int base = 0;
  for (int q0 = 0; q0 < ns; q0 += 256) {
    int c = c0, before = b0, sum = sum0;
    if (q0 > 0) {
      c = tiles(q0 + (int)threadIdx.x);
      __syncthreads();
      before = base + block_excl_scan1(c, s_tmp, &sum);
    }
    if (it >= before && it < before + c) {
      s_at[0] = q0 + (int)threadIdx.x;
      s_at[1] = before + c - 1 - it;
    }
    base += sum;
  }
  __syncthreads();
  return TilePlace{__builtin_amdgcn_readfirstlane(s_at[0]),
                   __builtin_amdgcn_readfirstlane(s_at[1]), kvh};
}

// Shared blocks: every tile of a group has the same units, those of its
// shared blocks.  The units of the groups' tiles end to end, per KV head: how many
// there are, the group that holds unit u (taken modulo them), and the units before
// it.  Workgroup 0 also leaves the units before every group, and their total, in
// place [groups + 1] for k_join_rows.
__device__ __forceinline__ int group_tiles(const DenseArgs& a, int g) {
  int s0, s1;
  seq_rows(a, g, s0, s1);
  return (int)(((int64_t)(s1 - s0) * a.g + kDenseRows - 1) / kDenseRows);
}
__device__ __forceinline__ int group_units(const DenseArgs& a, int g, int tk) {
  return max(1, (shared_of(a, g) + tk - 1) / tk);
}
struct GroupPlace { int per, g, base; };

__device__ __forceinline__ GroupPlace group_place(const DenseArgs& a, int wg, int launched, int tk,
                                                  int32_t* place) {
  __shared__ int s_tmp[4], s_at[2];
  auto units = [&](int g) {
    return g < a.ngroups ? group_tiles(a, g) * group_units(a, g, tk) : 0;
  };
  int per = 0;
  for (int g0 = 0; g0 < a.ngroups; g0 += 256) {
    const int g = g0 + (int)threadIdx.x;
    int sum;
    __syncthreads();
    const int before = per + block_excl_scan1(units(g), s_tmp, &sum);
    if (wg == 0 && g < a.ngroups) place[g] = before;
    per += sum;
  }
  if (wg == 0 && threadIdx.x == 0) place[a.ngroups] = per;
  const Deal deal(per * a.hkv, launched);
  if ((uint32_t)wg >= deal.grid) return GroupPlace{per, 0, 0};
  const int u = deal.at(wg) % per;
  int base = 0;
  for (int g0 = 0; g0 < a.ngroups; g0 += 256) {
    const int g = g0 + (int)threadIdx.x, c = units(g);
    int sum;
    __syncthreads();
    const int before = base + block_excl_scan1(c, s_tmp, &sum);
    if (u >= before && u < before + c) {
      s_at[0] = g;
      s_at[1] = before;
    }
    base += sum;
  }
  __syncthreads();
  return GroupPlace{per, __builtin_amdgcn_readfirstlane(s_at[0]),
                    __builtin_amdgcn_readfirstlane(s_at[1])};
}

// Where a whole tile of a group keeps its part: distinct for all tiles of
// groups that do not overlap.
__device__ __forceinline__ int64_t group_slot(const DenseArgs& a, int kvh, int g, int s0, int tile,
                                              int limit) {
  return (int64_t)kvh * limit + (int64_t)s0 * a.g / kDenseRows + g + tile;
}

// The work of one workgroup (wg of nwg).  DIRECT: a tile each, finished here.
// LISTED: a run of the units of k_plan's tiles.  GROUPED: a run of the units of the
// groups' shared blocks, parts only.
enum PrefillKind { DIRECT, LISTED, GROUPED };
template <int D> constexpr size_t kPrefillLds = 4 * sizeof(uint16_t) * kTk<D> * D;

template <typename T, int D, int MODE, int KIND>
__device__ __forceinline__ void prefill(const DenseArgs& a, const Plan& pl, const Parts& split,
                                        const Parts& whole, char* lds, int wg, int nwg) {
  constexpr int TK = kTk<D>;
  constexpr int KB = TK / 32;           // 32-key blocks of S
  constexpr int KS = D / 16;            // QK steps
  constexpr int DB = D / 32;            // output blocks
  constexpr int CPR = D / 8;            // 16-byte chunks per row
  constexpr int RP = 256 / CPR;         // rows per load instruction of the workgroup
  constexpr int KN = TK / RP;           // load instructions per unit and thread
  constexpr int GR = TK / 16;           // runs of 16 keys per unit
  constexpr uint16_t EXPO = __is_same(T, bf16s) ? 0x7f80 : 0x7c00;
  uint16_t* const s_k = reinterpret_cast<uint16_t*>(lds);         // [2][TK * D]
  uint16_t* const s_v = s_k + 2 * TK * D;                         // [2][TK * D]
  __shared__ int s_bad, s_range[4][4];
  const int tid = threadIdx.x, lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(wave_id());
  const int n32 = lane & 31, h = lane >> 5, i16 = lane & 15, gq = (lane >> 4) & 1;

  // rows of no request
  if (a.fill && a.starts) {
    const int f0 = min(max(a.starts[0], 0), a.t);
    const int f1 = max(f0, min(max(a.starts[a.requests], 0), a.t));
    const int64_t wide = (int64_t)a.hq * D / 8;
    for (int t = wg; t < f0 + (a.t - f1); t += nwg) {
      uint16_t* o = a.out + (int64_t)(t < f0 ? t : f1 + t - f0) * a.hq * D;
      for (int64_t x = tid; x < wide; x += 256) *reinterpret_cast<u16x8*>(o + 8 * x) = u16x8{};
    }
  }

  int u = 0, u1 = 1, kvh, it = 0, per = 0, ntiles = 0, gbase = 0;
  TilePlace mine{0, 0, 0};
  if constexpr (KIND == DIRECT) {
    mine = tile_place(a, wg, nwg);
    if (mine.kvh >= a.hkv) return;
    kvh = mine.kvh;
  } else if constexpr (KIND == GROUPED) {
    const GroupPlace at = group_place(a, wg, nwg, TK, pl.base);
    per = at.per;
    it = at.g;
    gbase = at.base;
    const Deal deal(per * a.hkv, nwg);
    if ((uint32_t)wg >= deal.grid) return;
    u = deal.at(wg);
    u1 = deal.at(wg + 1);
    kvh = u / per;
  } else {
    per = pl.head[0];
    ntiles = pl.head[1];
    const Deal deal(per * a.hkv, nwg);
    if ((uint32_t)wg >= deal.grid) return;
    u = deal.at(wg);
    u1 = deal.at(wg + 1);
    kvh = u / per;
    const int rem = u - kvh * per;
    int lo = 0, hi = ntiles - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (pl.tiles[mid].cum <= rem) lo = mid;
      else hi = mid - 1;
    }
    it = __builtin_amdgcn_readfirstlane(lo);
  }
  if (tid == 0) s_bad = 0;
  int serial = 0;                       // units worked on so far, in this workgroup

  // LDS addresses (elements)
  auto fk = [](int row) { return D == 64 ? (row >> 1) & 7 : row & 15; };
  auto fv = [](int row) { return D == 64 ? (row >> 1) & 1 : row & 3; };
  const int lrow = tid / CPR, lch = tid % CPR;
  // byte offsets of this lane's K (for D = 256 of both halves of a run) and V chunk
  uint32_t ko[2], vo;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    ko[i] = ((lrow & 15) * D + (lch ^ fk(lrow + (D == 256 ? 8 * i : 0))) * 8) * 2;
  vo = ((lrow & 15) * D + ((((lch >> 2) ^ fv(lrow)) << 2) | (lch & 3)) * 8) * 2;
  int ka[KS], va[DB];
#pragma unroll
  for (int s = 0; s < KS; ++s) ka[s] = n32 * D + ((2 * s + h) ^ fk(n32)) * 8;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const int row = 4 * h + (i16 >> 2);
    va[db] = row * D + (db ^ fv(row)) * 32 + 16 * gq + 4 * (i16 & 3);
  }

  while (u < u1) {
    Tile tl{mine.seq, mine.tile, 0, 0, 0, 0, 0, 0};
    int units = 0;
    if constexpr (KIND == LISTED) tl = pl.tiles[it];
    if constexpr (KIND == GROUPED) {
      if (u == (kvh + 1) * per) {                     // the next KV head's first group
        ++kvh;
        it = 0;
        gbase = 0;
      }
      const int rem = u - kvh * per;
      for (;;) {
        units = __builtin_amdgcn_readfirstlane(group_units(a, it, TK));
        const int all = units * __builtin_amdgcn_readfirstlane(group_tiles(a, it));
        if (rem < gbase + all || it + 1 >= a.ngroups) break;
        gbase += all;
        ++it;
      }
      tl.seq = it;
      tl.tile = (rem - gbase) / units;
      tl.cum = gbase + tl.tile * units;
    }
    const int seq = __builtin_amdgcn_readfirstlane(tl.seq);
    const int tile = __builtin_amdgcn_readfirstlane(tl.tile);
    int s0, s1;
    seq_rows(a, seq, s0, s1);
    const int64_t rown = (int64_t)tile * kDenseRows + 32 * w + n32;
    const bool valid = rown < (int64_t)(s1 - s0) * a.g;
    const int tok = s0 + (int)(valid ? rown / a.g : 0);
    const int head = kvh * a.g + (int)(valid ? rown % a.g : 0);
    int p = 0;
    Span sp = seq_span(a, seq, s0, s1, tok, p);
    // keys that some row of this wave sees
    int wlo = valid && sp.hi > sp.lo ? sp.lo : 0x7fffffff;
    int whi = valid && sp.hi > sp.lo ? sp.hi : 0;
    int mlo = valid ? sp.lo : 0, mhi = valid ? (sp.hi > sp.lo ? sp.hi : 0) : 0x7fffffff;
    if (!valid) sp = Span{0, 0x7fffffff};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      wlo = min(wlo, __shfl_xor(wlo, o));
      whi = max(whi, __shfl_xor(whi, o));
    }
    wlo = __builtin_amdgcn_readfirstlane(wlo);
    whi = __builtin_amdgcn_readfirstlane(whi);
    if constexpr (KIND != LISTED) {
      // the tile's range from its rows, as k_plan lists it
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        mlo = max(mlo, __shfl_xor(mlo, o));
        mhi = min(mhi, __shfl_xor(mhi, o));
      }
      if (lane == 0) {
        s_range[w][0] = wlo;
        s_range[w][1] = whi;
        s_range[w][2] = mlo;
        s_range[w][3] = mhi;
      }
      __syncthreads();                                // (rewritten only after the units' barriers)
      tl.klo = min(min(s_range[0][0], s_range[1][0]), min(s_range[2][0], s_range[3][0]));
      tl.khi = max(max(s_range[0][1], s_range[1][1]), max(s_range[2][1], s_range[3][1]));
      tl.max_lo = max(max(s_range[0][2], s_range[1][2]), max(s_range[2][2], s_range[3][2]));
      tl.min_hi = min(min(s_range[0][3], s_range[1][3]), min(s_range[2][3], s_range[3][3]));
      if (tl.khi <= tl.klo) tl.klo = tl.khi = 0;
      if constexpr (KIND == DIRECT) tl.kstart = tl.klo & ~15;
    }
    const int kstart = __builtin_amdgcn_readfirstlane(tl.kstart);
    const int klo = __builtin_amdgcn_readfirstlane(tl.klo);
    const int khi = __builtin_amdgcn_readfirstlane(tl.khi);
    const int max_lo = __builtin_amdgcn_readfirstlane(tl.max_lo);
    const int min_hi = __builtin_amdgcn_readfirstlane(tl.min_hi);
    const int n = KIND == GROUPED ? units : max(1, (khi - kstart + TK - 1) / TK);
    int j0 = 0, j1 = n;
    if constexpr (KIND != DIRECT) {
      j0 = u - (kvh * per + __builtin_amdgcn_readfirstlane(tl.cum));
      j1 = min(n, j0 + (u1 - u));
    }
    u += KIND == DIRECT ? 1 : j1 - j0;
    // units that some row sees (of a group's shared blocks, windows may hide most)
    const int ja = KIND == GROUPED ? max(j0, klo / TK) : j0;
    const int jb = KIND == GROUPED ? min(j1, (khi + TK - 1) / TK) : j1;
    u16x8 qf[KS];
    const uint16_t* qp = a.q + (int64_t)tok * a.qs + (int64_t)head * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u16x8*>(qp + 16 * s);
    float slope = 0.f;
    if constexpr (MODE & 2) slope = a.slopes[head] * 1.44269504f;
    const int32_t* row =
        a.table + ((int64_t)(KIND == GROUPED ? s0 : seq) * a.hkv + kvh) * a.nb;
    const int kbase = kstart + ja * TK, kend = min(kstart + jb * TK, khi);
    const int cnt = jb - ja;

    auto window = [&](int i) {                        // rows of 64 runs of 16 keys
      const int key = kbase + 16 * (64 * i + lane);
      const int x = pool_row(a, row, min(key, kend));
      return key < kend ? x : -1;
    };
    int ent = window(0), nxt = window(1);
    int vmask = 0;                                    // runs with a page, of the unit last issued
    // Lane l of wave w fills the 16-byte slot 256 i + 64 w + l of the unit's LDS: row
    // i RP + lrow, and of that row the chunk that the swizzle puts there.  A
    // wave's rows lie in one run of 16 keys.
    auto issue = [&](int j, int buf) {
      if (j > 0 && (j * GR) % 64 == 0) {
        ent = nxt;
        nxt = window(j * GR / 64 + 1);
      }
      int rows[GR];
      vmask = 0;
#pragma unroll
      for (int x = 0; x < GR; ++x) {
        rows[x] = __builtin_amdgcn_readlane(ent, (j * GR + x) & 63);
        vmask |= rows[x] >= 0 ? 1 << x : 0;
      }
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        int x = rows[D == 64 ? 2 * i : i * RP / 16];
        if (D == 64 && w >= 2) x = rows[D == 64 ? 2 * i + 1 : 0];
        const int64_t at = (int64_t)max(x, 0) * D + (i * RP % 16) * D;
        const uint32_t slot = (uint32_t)(256 * i + 64 * w) * 16;
        copy_to_lds(lds_address(s_k + buf * (TK * D)) + slot, a.kp + at, ko[i * RP % 16 ? 1 : 0]);
        copy_to_lds(lds_address(s_v + buf * (TK * D)) + slot, a.vp + at, vo);
      }
    };
    // whether some row of the tile does not see all of the unit
    auto masked = [&](int key0) {
      return !(key0 >= max_lo && key0 + TK <= min_hi && vmask == (1 << GR) - 1);
    };
    // Values of the unit that no row sees become zero; s_bad = serial if any other
    // is not finite.
    auto clean = [&](int key0, int mask, uint16_t* lv) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        const int kr = i * RP + lrow, key = key0 + kr;
        u16x8* at = reinterpret_cast<u16x8*>(lv + (256 * i + tid) * 8);
        if (key >= klo && key < khi && (mask >> (kr / 16) & 1)) bad |= nonfinite16(*at, EXPO);
        else *at = u16x8{};
      }
      if (bad) s_bad = serial;
    };

    float m = -INFINITY, l = 0.f;
    f32x16 acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[i][x] = 0.f;

    // P of the unit whose K is lk, as the second product's operand; m, l and
    // the output follow its maximum
    auto weights = [&](const uint16_t* lk, int key0, bool edge, int mask,
                       u16x8 (&pf)[TK / 16]) {
      f32x16 s[KB];
#pragma unroll
      for (int b = 0; b < KB; ++b) {
#pragma unroll
        for (int x = 0; x < 16; ++x) s[b][x] = 0.f;
#pragma unroll
        for (int x = 0; x < KS; ++x)
          s[b] = mma32<T>(*reinterpret_cast<const u16x8*>(lk + ka[x] + 32 * b * D), qf[x], s[b]);
      }
      // MODE 0 keeps the products as they are: their scale goes into the exponent's FMA
      const float sc = MODE ? 1.f : a.c;
      if constexpr (MODE != 0) {
        const float dist = (float)(p - key0 - 4 * h);
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int off = 32 * b + 8 * (x / 4) + x % 4;
            s[b][x] = score2<MODE>(a, s[b][x], slope, dist - (float)off);
          }
      }
      if (edge) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int key = key0 + 4 * h + 32 * b + 8 * (x / 4) + x % 4;
            const bool ok = key >= sp.lo && key < sp.hi && (mask >> (2 * b + x / 8) & 1);
            s[b][x] = ok ? s[b][x] : -INFINITY;
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int x = 0; x < 16; ++x) top = fmaxf(top, s[b][x]);
      top *= sc;
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
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][x], sc, -ms));
          l += e;
          pf[2 * b + x / 8][x % 8] = to16<T>(e);
        }
    };

    __syncthreads();                                  // the last item's LDS reads are done
    if (KIND != GROUPED || cnt > 0) issue(0, 0);
    bool bad = false;                                 // some rows must skip a value
    for (int j = 0; j < cnt && !bad; ++j) {
      const int buf = j & 1, key0 = kbase + j * TK;
      const int mask = vmask;
      const bool edge = masked(key0);
      ++serial;
      copies_done();
      __syncthreads();
      if (j + 1 < cnt) issue(j + 1, buf ^ 1);
      if (edge) {
        clean(key0, mask, s_v + buf * (TK * D));
        __syncthreads();
        bad = s_bad == serial;
      }
      if (!bad && key0 < whi && key0 + TK > wlo) {
        u16x8 pf[TK / 16];
        weights(s_k + buf * (TK * D), key0, edge, mask, pf);
        const uint16_t* lv = s_v + buf * (TK * D);
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
    }
    const bool all = j0 == 0 && j1 == n;
    const bool keep = KIND == DIRECT || (KIND == LISTED && all);    // finished here
    const Parts& to = all ? whole : split;
    const int64_t slot = all ? group_slot(a, kvh, seq, s0, tile, pl.limit)
                             : 2 * (int64_t)wg + (j0 > 0 ? 0 : 1);
    if (bad) {
      copies_done();
      __syncthreads();
      slow_rows<T, D, MODE>(a, seq, s0, s1, (int64_t)tile * kDenseRows + 32 * w, kvh, row, kbase,
                            kend, keep ? nullptr : &to, slot * kDenseRows + 32 * w);
    }
    l += __shfl_xor(l, 32);
    if (valid && !bad) {
      if (keep) {
        uint16_t* o = a.out + ((int64_t)tok * a.hq + head) * D + 4 * h;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            store_out<T>(o + 32 * db + 8 * x,
                         f32x4{acc[db][4 * x], acc[db][4 * x + 1], acc[db][4 * x + 2],
                               acc[db][4 * x + 3]}, l);
      } else {
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
    if constexpr (KIND == LISTED)
      if (++it == ntiles) {
        it = 0;
        ++kvh;
      }
  }
}

template <typename T, int D, int MODE, int KIND>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void k_prefill(DenseArgs a, Plan pl,
                                                                   Parts split) {
  __shared__ __attribute__((aligned(16))) char lds[kPrefillLds<D>];
  prefill<T, D, MODE, KIND>(a, pl, split, split, lds, (int)blockIdx.x, (int)gridDim.x);
}

}  // namespace stk
