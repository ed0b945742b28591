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
// Bound by the SIMDs: of an 8192-token causal prompt (32 query heads over 8, D =
// 128: 530 us, 1.03 PFLOP/s, where the card's library product reaches 1.19) the
// matrix instructions take 51 % and the softmax's 47 %; at D = 256 1040 us, 1.06.
// P is rounded to 16 bits for the second product, the sum of its weights is not:
// relative error 0.0020 of the prompt's output, 0.0015 of which is the output's own
// rounding.  A second part of P, as k_decode has, would be half as many matrix
// instructions again.
//
// Masks are one range of keys per row; units that every row of the tile sees whole
// (all but the first and last ones) skip them.  In the others the values that no
// row sees are zeroed in LDS; should a value that some rows see and others do
// not be infinite or NaN (0 times which is not 0), the tile is done row by row
// instead, each row reading the keys that it sees (slow_rows).
#pragma once

#include "dense.hpp"

namespace stk {

// 16 bytes per lane from base + off to LDS, lane after lane from byte `lds`
// (wave-uniform) on.  Counted by vmcnt like any load; the compiler does not
// know of the write, so the caller waits (copies_done) and passes a barrier
// before it reads.  (Its own intrinsic makes the compiler wait for all of these
// before every LDS read.  m0 is set beside each copy, and nothing else in these
// kernels uses it.)
__device__ __forceinline__ void copy_to_lds(uint32_t lds, const uint16_t* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory");
}
// The wait is one that the compiler knows: it also settles the queries' and the
// table's loads, which it would otherwise wait for where they are used, in the
// middle of every unit, and with them for the copies of the next one.
__device__ __forceinline__ void copies_done() {
  asm volatile("" ::: "memory");
  vm_drain();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Workgroups of whole tiles come in the order of their length, and each CU takes
// two: the first 256 one each, the next 256 the second ones.  Those are taken in
// reverse, so that a CU's longest tile shares it with a short one.
__device__ __forceinline__ int paired(int it, int n, int hkv) {
  const int half = 256 / hkv, top = min(n, 2 * half);
  return it >= half && it < top ? half + top - 1 - it : it;
}

// The tile of workgroup wg where every tile has its own.  Neighbouring
// workgroups take one tile of each KV head, so that with eight heads (or a divisor of
// eight) an XCD, to which every eighth workgroup goes, reads one head's keys;
// and within a sequence the last rows, which see the most keys, come first.  Up to 64
// requests' tiles are laid end to end (four requests of 1024 tokens, one after 16000: 360
// us, 441 with gaps, which moved long tiles to one CU).  Those of more, which every
// workgroup would have to add up, come after floor(s G / 128) + r others, s their
// first row: request r has at least as many places as tiles then (4096 requests of one or
// two tokens 808 us, 542).
// kvh = Hkv: none.
struct TilePlace { int seq, tile, kvh; };

__device__ __forceinline__ TilePlace tile_place(const DenseArgs& a, int wg, int nwg) {
  const int it = paired(wg / a.hkv, nwg / a.hkv, a.hkv);
  auto tiles = [&](int rows) { return (int)(((int64_t)rows * a.g + kDenseRows - 1) / kDenseRows); };
  int r = -1, tile = -1;
  if (a.requests <= STK_WAVE) {           // (every wave for itself)
    int s0 = 0, s1 = 0;
    if (lane_id() < a.requests) rows_of(a, lane_id(), s0, s1);
    const int c = tiles(s1 - s0), end = wave_incl_scan_dpp(c);
    const uint64_t mine = __ballot(it >= end - c && it < end);
    if (mine) {
      r = __builtin_ctzll(mine);
      tile = __builtin_amdgcn_readlane(end, r) - 1 - it;
    }
  } else {
    auto before = [&](int i) {
      return (int)((int64_t)min(max(a.starts[i], 0), a.t) * a.g / kDenseRows) + i;
    };
    r = last_at_most(a.requests, it, before);
    if (r >= 0) {
      int s0, s1;
      rows_of(a, r, s0, s1);
      const int c = tiles(s1 - s0);
      tile = before(r) + c - 1 - it;
      if (tile < 0 || tile >= c) r = -1;
    }
  }
  r = __builtin_amdgcn_readfirstlane(r);
  if (r < 0) return TilePlace{0, 0, a.hkv};
  return TilePlace{r, __builtin_amdgcn_readfirstlane(tile), wg % a.hkv};
}

// Shared blocks: every tile of a group has the same units, those of its
// shared blocks.  The units of the groups' tiles end to end, per KV head: how many
// there are, the group that holds unit u (taken modulo them), and the units before
// it.  u is the first unit of workgroup wg, which becomes its place among the
// workgroups with work.  Workgroup 0 also leaves the units before every group, and
// their total, in place [groups + 1] for k_join_rows.
__device__ __forceinline__ int group_tiles(const DenseArgs& a, int g) {
  int s0, s1;
  seq_rows(a, g, s0, s1);
  return (int)(((int64_t)(s1 - s0) * a.g + kDenseRows - 1) / kDenseRows);
}
// Units of a group's shared keys that its requests' windows hide: they end at or behind
// the last shared key.
__device__ __forceinline__ int group_hidden(const DenseArgs& a, int g, int tk) {
  return a.window > 0 ? max(0, shared_of(a, g) - a.window) / tk : 0;
}
__device__ __forceinline__ int group_units(const DenseArgs& a, int g, int tk) {
  return max(1, (shared_of(a, g) + tk - 1) / tk - group_hidden(a, g, tk));
}
struct GroupPlace { int per, g, base; };      // per = 0: no work

// Workgroups that the groups' units are dealt to, of those launched, in runs of at
// least two units: each run leaves a part of up to 128 rows to write and read.
// At D = 256, where units are smaller and parts larger, four, and beyond one
// workgroup per CU sixteen.
__device__ __forceinline__ int group_grid(int units, int tk, int launched) {
  const int most = tk == 64 ? units / 2 : max(min(units / 4, 256), units / 16);
  return min(launched, max(1, most));
}

__device__ __forceinline__ GroupPlace group_place(const DenseArgs& a, int& wg, int launched, int tk,
                                                  int32_t* place) {
  if (a.ngroups <= STK_WAVE) {            // as in decode_place
    const int g = lane_id();
    const int c = g < a.ngroups ? group_tiles(a, g) * group_units(a, g, tk) : 0;
    const int end = wave_incl_scan_dpp(c);
    const int per = __builtin_amdgcn_readlane(end, STK_WAVE - 1);
    if (wg == 0 && (int)threadIdx.x < a.ngroups) place[g] = end - c;
    if (wg == 0 && threadIdx.x == 0) place[a.ngroups] = per;
    const Deal deal(per * a.hkv, group_grid(per * a.hkv, tk, launched));
    if ((uint32_t)wg >= deal.grid) return GroupPlace{0, 0, 0};
    wg = xcd_remap(wg, (int)deal.grid);
    const int u = deal.at(wg) % per;
    const uint64_t mine = __ballot(u >= end - c && u < end);
    const int at = mine ? __builtin_ctzll(mine) : 0;
    return GroupPlace{per, at, __builtin_amdgcn_readlane(end - c, at)};
  }
  __shared__ int s_tmp[4], s_at[2];
  // groups per thread and pass: their loads are in flight together
  const int e = a.ngroups > 256 ? 4 : 1, pass = 256 * e;
  int units[4];
  auto scan = [&](int g0, int& before, int& sum) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int g = g0 + e * (int)threadIdx.x + j;
      units[j] = j < e && g < a.ngroups ? group_tiles(a, g) * group_units(a, g, tk) : 0;
      c += units[j];
    }
    __syncthreads();
    before = block_excl_scan1(c, s_tmp, &sum);
  };
  int per = 0, before = 0, sum = 0;
  for (int g0 = 0; g0 < a.ngroups; g0 += pass) {
    scan(g0, before, sum);
    if (wg == 0) {
      int at = per + before;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int g = g0 + e * (int)threadIdx.x + j;
        if (j < e && g < a.ngroups) place[g] = at;
        at += units[j];
      }
    }
    per += sum;
  }
  if (wg == 0 && threadIdx.x == 0) place[a.ngroups] = per;
  const Deal deal(per * a.hkv, group_grid(per * a.hkv, tk, launched));
  if ((uint32_t)wg >= deal.grid) return GroupPlace{0, 0, 0};
  wg = xcd_remap(wg, (int)deal.grid);
  const int u = deal.at(wg) % per;
  int base = 0;
  for (int g0 = 0; g0 < a.ngroups; g0 += pass) {
    if (a.ngroups > pass) scan(g0, before, sum);
    int at = base + before;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (u >= at && u < at + units[j]) {
        s_at[0] = g0 + e * (int)threadIdx.x + j;
        s_at[1] = at;
      }
      at += units[j];
    }
    base += sum;
    if (u < base) break;
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

// The work of one workgroup (wg of nwg).  The runs of neighbouring units, which
// read the same keys, go to one XCD (one L2).  DIRECT: a tile each, finished here.
// LISTED: a tile of
// k_plan's each, or a run of their units.  GROUPED: a run of the units of the
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
  constexpr bool AHEAD = D <= 128;      // operands requested ahead of their use
  constexpr uint16_t EXPO = __is_same(T, bf16s) ? 0x7f80 : 0x7c00;
  constexpr int UNIT = 2 * TK * D;      // bytes of K or V: lds holds K, K, V, V
  const uint32_t lds_k = lds_address(lds);
  __shared__ int s_bad[2], s_range[4][4];
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
  Tile alone{};
  bool whole_tile = KIND == DIRECT;
  if constexpr (KIND == DIRECT) {
    mine = tile_place(a, wg, nwg);
    if (mine.kvh >= a.hkv) return;
    kvh = mine.kvh;
  } else if constexpr (KIND == GROUPED) {
    const GroupPlace at = group_place(a, wg, nwg, TK, pl.base);
    if (at.per == 0) return;
    per = at.per;
    it = at.g;
    gbase = at.base;
    const Deal deal(per * a.hkv, group_grid(per * a.hkv, TK, nwg));
    u = deal.at(wg);
    u1 = deal.at(wg + 1);
    kvh = u / per;
  } else {
    per = pl.head[0];
    ntiles = pl.head[1];
    const int cut = pl.head[2];
    // a whole tile's entry is requested beside the head
    kvh = wg % a.hkv;
    it = min(paired(wg / a.hkv, pl.limit, a.hkv), pl.limit - 1);
    alone = pl.tiles[it];
    whole_tile = cut == 0;
    if (whole_tile) {                     // a tile each, dealt as tile_place does
      if (it >= ntiles || wg >= pl.limit * a.hkv) return;
    } else {
      const Deal deal(per * a.hkv, cut);
      if ((uint32_t)wg >= deal.grid) return;
      wg = xcd_remap(wg, (int)deal.grid);
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
  }
  if (tid < 2) s_bad[tid] = 0;
  int serial = 0;                       // units worked on so far, in this workgroup

  // K rows are swizzled in 16-byte chunks, V rows in 64-byte blocks
  auto fk = [](int row) { return D == 64 ? (row >> 1) & 7 : row & 15; };
  auto fv = [](int row) { return D == 64 ? (row >> 1) & 1 : row & 3; };
  const int lrow = tid / CPR, lch = tid % CPR;
  // byte offsets of this lane's K (for D = 256 of both halves of a run) and V
  // chunk within a run of 16 pool rows
  uint32_t ko[2], vo;
#pragma unroll
  for (int i = 0; i < 2; ++i)
    ko[i] = ((lrow & 15) * D + (lch ^ fk(lrow + (D == 256 ? 8 * i : 0))) * 8) * 2;
  vo = ((lrow & 15) * D + ((((lch >> 2) ^ fv(lrow)) << 2) | (lch & 3)) * 8) * 2;
  // LDS byte offsets of the products' operands at step 0; the others' differ
  // by an exclusive or, since a row's start is aligned to its size
  const uint32_t ka = (n32 * D + (h ^ fk(n32)) * 8) * 2;
  const int vrow = 4 * h + (i16 >> 2);
  const uint32_t va = (vrow * D + fv(vrow) * 32 + 16 * gq + 4 * (i16 & 3)) * 2;

  while (u < u1) {
    Tile tl{mine.seq, mine.tile, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    int units = 0;
    if constexpr (KIND == LISTED) tl = whole_tile ? alone : pl.tiles[it];
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
    if constexpr (KIND != LISTED) {
      int s1;
      seq_rows(a, seq, tl.s0, s1);
      tl.rows = s1 - tl.s0;
      tl.len = KIND == DIRECT ? tokens_of(a, seq) : 0;
    }
    const int s0 = __builtin_amdgcn_readfirstlane(tl.s0);
    const int nrow = __builtin_amdgcn_readfirstlane(tl.rows);
    const uint32_t rown = (uint32_t)tile * kDenseRows + 32 * w + n32;   // (T G fits an int)
    const bool valid = rown < (uint32_t)nrow * (uint32_t)a.g;
    const uint32_t rtok = valid ? rown / (uint32_t)a.g : 0;
    const int tok = s0 + (int)rtok;
    const int head = kvh * a.g + (valid ? (int)(rown - rtok * (uint32_t)a.g) : 0);
    u16x8 qf[KS];
    const uint16_t* qp = a.q + (int64_t)tok * a.qs + (int64_t)head * D + 8 * h;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u16x8*>(qp + 16 * s);
    float slope = 0.f;
    if constexpr (MODE & 2) slope = a.slopes[head] * 1.44269504f;
    int p;
    Span sp;
    if constexpr (KIND == GROUPED) {
      sp = seq_span(a, seq, s0, s0 + nrow, tok, p);
    } else {
      const int len = __builtin_amdgcn_readfirstlane(tl.len);
      p = len - nrow + (tok - s0);
      sp = span_of(a, seq, tok, p, len);
    }
    // keys that some row of this wave sees
    const bool some = valid && sp.hi > sp.lo;
    const int wlo = (int)wave_ext_u32<false>(some ? (uint32_t)sp.lo : 0x7fffffffu);
    const int whi = (int)wave_ext_u32<true>(some ? (uint32_t)sp.hi : 0u);
    if constexpr (KIND != LISTED) {
      // the tile's range from its rows, as k_plan lists it
      const uint32_t mlo = wave_ext_u32<true>(some ? (uint32_t)sp.lo : 0u);
      const uint32_t mhi = wave_ext_u32<false>(valid ? (some ? (uint32_t)sp.hi : 0u) : 0x7fffffffu);
      if (lane == 0) {
        s_range[w][0] = wlo;
        s_range[w][1] = whi;
        s_range[w][2] = (int)mlo;
        s_range[w][3] = (int)mhi;
      }
      __syncthreads();                                // (rewritten only after the units' barriers)
      tl.klo = min(min(s_range[0][0], s_range[1][0]), min(s_range[2][0], s_range[3][0]));
      tl.khi = max(max(s_range[0][1], s_range[1][1]), max(s_range[2][1], s_range[3][1]));
      tl.max_lo = max(max(s_range[0][2], s_range[1][2]), max(s_range[2][2], s_range[3][2]));
      tl.min_hi = min(min(s_range[0][3], s_range[1][3]), min(s_range[2][3], s_range[3][3]));
      if (tl.khi <= tl.klo) tl.klo = tl.khi = 0;
      tl.kstart = KIND == DIRECT ? tl.klo & ~15 : group_hidden(a, seq, TK) * TK;
    }
    const int kstart = __builtin_amdgcn_readfirstlane(tl.kstart);
    const int klo = __builtin_amdgcn_readfirstlane(tl.klo);
    const int khi = __builtin_amdgcn_readfirstlane(tl.khi);
    const int max_lo = __builtin_amdgcn_readfirstlane(tl.max_lo);
    const int min_hi = __builtin_amdgcn_readfirstlane(tl.min_hi);
    const int n = KIND == GROUPED ? units : max(1, (khi - kstart + TK - 1) / TK);
    int j0 = 0, j1 = n;
    if (!whole_tile) {
      j0 = u - (kvh * per + __builtin_amdgcn_readfirstlane(tl.cum));
      j1 = min(n, j0 + (u1 - u));
    }
    u += whole_tile ? 1 : j1 - j0;
    // units that some row sees (of a group's shared blocks, windows may hide most)
    const int ja = KIND == GROUPED ? max(j0, (klo - kstart) / TK) : j0;
    const int jb = KIND == GROUPED ? min(j1, (khi - kstart + TK - 1) / TK) : j1;
    const int32_t* row = a.table + ((int64_t)(KIND == GROUPED ? s0 : seq) * a.hkv + kvh) * a.nb;
    const int kbase = kstart + ja * TK, kend = min(kstart + jb * TK, khi);
    const int cnt = jb - ja;

    auto window = [&](int i) {                        // rows of 64 runs of 16 keys
      const int key = kbase + 16 * (64 * i + lane);
      const int x = pool_row(a, row, min(key, kend));
      return key < kend ? x : -1;
    };
    int ent = window(0), nxt = cnt * GR > 64 ? window(1) : -1;
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
        const uint32_t slot = (uint32_t)(buf * UNIT + (256 * i + 64 * w) * 16);
        copy_to_lds(lds_k + slot, a.kp + at, ko[i * RP % 16 ? 1 : 0]);
        copy_to_lds(lds_k + 2 * UNIT + slot, a.vp + at, vo);
      }
    };
    // A value that a row does not see may be infinite or NaN, and 0 times it is
    // not 0.  Where no row of the tile sees it, it becomes zero (`cut`); any
    // other one leaves the unit's serial number in s_bad.
    auto clean = [&](int key0, int mask, int buf, bool cut) {
      bool bad = false;
#pragma unroll
      for (int i = 0; i < KN; ++i) {
        const int kr = i * RP + lrow, key = key0 + kr;
        u16x8* at = reinterpret_cast<u16x8*>(lds + (2 + buf) * UNIT + (256 * i + tid) * 16);
        const bool seen = !cut || (key >= klo && key < khi && (mask >> (kr / 16) & 1));
        if (seen) bad |= nonfinite16(*at, EXPO);
        else *at = u16x8{};
      }
      if (bad) s_bad[buf] = serial;
    };

    // V^T for one step of the second product: 16 keys, 32 dims
    auto v_part = [&](const char* at) {
      const u16x4 lo = lds_tr(reinterpret_cast<const uint16_t*>(at));
      const u16x4 hi = lds_tr(reinterpret_cast<const uint16_t*>(at + 16 * D));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    u16x8 vf[AHEAD ? TK / 16 : 1][DB];
    auto read_v = [&](int buf) {
#pragma unroll
      for (int x = 0; x < (AHEAD ? TK / 16 : 1); ++x)
#pragma unroll
        for (int db = 0; db < DB; ++db)
          vf[x][db] = v_part(lds + (2 + buf) * UNIT + (va ^ (64 * db)) + 32 * x * D);
    };

    float m = -INFINITY, l = 0.f;
    f32x16 acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[i][x] = 0.f;

    __syncthreads();                                  // the last item's LDS reads are done
    if (KIND != GROUPED || cnt > 0) issue(0, 0);
    // some row must skip a value: found one barrier after the unit's check
    bool bad = false, edge = false;
    for (int j = 0; j < cnt; ++j) {
      const int buf = j & 1, key0 = kbase + j * TK, mask = vmask;
      const bool before = edge;
      edge = !(key0 >= max_lo && key0 + TK <= min_hi && mask == (1 << GR) - 1);
      copies_done();
      __syncthreads();
      if (before) bad = s_bad[buf ^ 1] == serial;
      if (bad) break;
      ++serial;
      if (j + 1 < cnt) issue(j + 1, buf ^ 1);
      if (edge) {
        const bool cut = key0 < klo || key0 + TK > khi || mask != (1 << GR) - 1;
        clean(key0, mask, buf, cut);
        if (cut) __syncthreads();
      }
      if (key0 >= whi || key0 + TK <= wlo) continue;

      // P^T of the unit; m, l and the output follow its maximum
      f32x16 s[KB];
      u16x8 pf[TK / 16];
      {
        uint32_t kb = ka;
        if constexpr (D == 256) asm volatile("" : "+v"(kb));   // (keeps 16 offsets out of registers)
        const char* lk = lds + buf * UNIT;
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x) s[b][x] = 0.f;
        // where registers allow, the unit's K is requested at once and its V before
        // the softmax: the matrix instructions find their operands
        if constexpr (AHEAD) {
          u16x8 kf[KS][KB];
#pragma unroll
          for (int x = 0; x < KS; ++x)
#pragma unroll
            for (int b = 0; b < KB; ++b)
              kf[x][b] = *reinterpret_cast<const u16x8*>(lk + (kb ^ (32 * x)) + 64 * b * D);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int x = 0; x < KS; ++x)
#pragma unroll
            for (int b = 0; b < KB; ++b) s[b] = mma32<T>(kf[x][b], qf[x], s[b]);
          __builtin_amdgcn_sched_barrier(0);
          read_v(buf);
          __builtin_amdgcn_sched_barrier(0);
        } else {
#pragma unroll
          for (int x = 0; x < KS; ++x)
#pragma unroll
            for (int b = 0; b < KB; ++b)
              s[b] = mma32<T>(
                  *reinterpret_cast<const u16x8*>(lk + (kb ^ (32 * x)) + 64 * b * D), qf[x], s[b]);
        }
      }
      // Scores are kept as y, x = y sc + off in base 2, and sc and off go into the
      // exponent's FMA: the products themselves, or -1 / (1 + e^2y) of a capped one
      const float sc = MODE == 0 ? a.c : MODE == 1 ? 2.f * a.cap_out : 1.f;
      const float off = MODE == 1 ? a.cap_out : 0.f;
      if constexpr (MODE == 1) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            s[b][x] = __builtin_amdgcn_rcpf(-1.f - __builtin_amdgcn_exp2f(s[b][x] * a.cap_in));
      } else if constexpr (MODE != 0) {
        const float dist = (float)(p - key0 - 4 * h);
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            s[b][x] = score2<MODE>(a, s[b][x], slope,
                                   dist - (float)(32 * b + 8 * (x / 4) + x % 4));
      }
      if (edge) {
        // key0 + 4 h + off in [lo, hi), as one unsigned comparison
        const int rlo = sp.lo - key0 - 4 * h;
        const uint32_t wide = (uint32_t)max(sp.hi - sp.lo, 0);
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            s[b][x] = (uint32_t)(32 * b + 8 * (x / 4) + x % 4 - rlo) < wide ? s[b][x] : -INFINITY;
        if (mask != (1 << GR) - 1) {
#pragma unroll
          for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int x = 0; x < 16; ++x)
              s[b][x] = mask >> (2 * b + x / 8) & 1 ? s[b][x] : -INFINITY;
        }
      }
      float top = s[0][0];
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int x = 0; x < 16; ++x) top = fmaxf(top, s[b][x]);
      top = __builtin_fmaf(top, sc, off);
      if (__any(top > m + kLazy)) {
        float mx = fmaxf(top, m);
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float f = mx == m ? 1.f : __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l *= f;
#pragma unroll
        for (int i = 0; i < DB; ++i) acc[i] *= f;
      }
      const float ms = off - (m == -INFINITY ? 0.f : m);
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][x], sc, ms));
          l += e;
          pf[2 * b + x / 8][x % 8] = to16<T>(e);
        }
      if constexpr (AHEAD) {
#pragma unroll
        for (int x = 0; x < TK / 16; ++x)
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[db] = mma32<T>(vf[x][db], pf[x], acc[db]);
      } else {
        uint32_t vb = va;
        asm volatile("" : "+v"(vb));
#pragma unroll
        for (int x = 0; x < TK / 16; ++x)
#pragma unroll
          for (int db = 0; db < DB; ++db)
            acc[db] = mma32<T>(v_part(lds + (2 + buf) * UNIT + (vb ^ (64 * db)) + 32 * x * D),
                               pf[x], acc[db]);
      }
    }
    if (edge && !bad) {                               // the last unit's check
      __syncthreads();
      bad = s_bad[(cnt - 1) & 1] == serial;
    }
    const bool all = j0 == 0 && j1 == n;
    const bool keep = KIND == DIRECT || (KIND == LISTED && all);    // finished here
    const Parts& to = all ? whole : split;
    const int64_t slot = all ? group_slot(a, kvh, seq, s0, tile, pl.limit)
                             : 2 * (int64_t)wg + (j0 > 0 ? 0 : 1);
    if (bad) {
      slow_rows<T, D, MODE>(a, seq, s0, s0 + nrow, (int64_t)tile * kDenseRows + 32 * w, 32, kvh,
                            row, kbase, kend, keep ? nullptr : &to, slot * kDenseRows + 32 * w);
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
__global__ __launch_bounds__(256, 2) void k_prefill(DenseArgs a, Plan pl,
                                                                   Parts split) {
  __shared__ __attribute__((aligned(1024))) char lds[kPrefillLds<D>];
  prefill<T, D, MODE, KIND>(a, pl, split, split, lds, (int)blockIdx.x, (int)gridDim.x);
}

}  // namespace stk
