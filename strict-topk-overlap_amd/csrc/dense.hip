// Dense attention over the paged cache: the C entry points, the list of row
// tiles (k_plan), and the joins of split items (k_join_tiles, k_join_rows).
#include "dense_shared.hpp"

namespace stk {

constexpr int kPlanThreads = 1024;     // and the most requests and tiles that are listed

// Cut tiles are dealt in runs of at least kRun units; whole ones have at most
// kWhole (for which there is room to sort them).
constexpr int kRun = 4, kWhole = 1024;

// Whether `units` units in `tiles` tiles of at most `most` are better left whole; times
// in us.  A unit takes `one` on a CU of its own, and a CU finishes one per `two` with
// two workgroups.  Whole tiles last as long as the longest one, or two of them where
// CUs take two, or as all of them and the longest one's tail; cut ones are even, but
// leave parts that are written, and read one after the other for a row, and each
// workgroup begins twice.  The coefficients are fitted to 216 batches of 4 to 760 tiles of
// 10 to 438 units, measured both ways: the choice is the quicker one or within 7 % of
// it.  32 query heads over 8 KV heads, D = 128 (whole, cut): 24 tokens after 1400 41.4,
// 26.9; 500 after 2500 66.3, 52.6; 1500 of three requests after 1400 50.9, 69.1.
__device__ __forceinline__ bool leave_whole(int units, int most, int tiles, int fill, int d) {
  const float wgs = (float)min(fill, max(1, units / kRun)), wide = d / 128.f;
  const float one = d == 64 ? 0.92f : d == 128 ? 1.3f : 1.55f;
  const float two = d == 64 ? 0.6f : d == 128 ? 1.f : 1.2f;
  const float load = tiles <= 256   ? 0.f
                     : tiles <= 512 ? 1.8f * two * units / tiles
                                    : two * units / 256.f + 0.2f * most;
  const float whole = fmaxf(one * most, load);
  const float cut = (wgs <= 256.f ? one : d == 64 ? 1.3f : 2.2f) * units / wgs + 5.f +
                    wide * (0.45f * wgs / max(tiles, 1) + 0.02f * wgs + 0.03f * tiles);
  return whole <= cut && most <= kWhole;
}

// Lists the row tiles: one workgroup.  Within a request the last rows, which see
// the most keys, come first; whole tiles are listed by their length, the longest
// first.  fill: workgroups that fill the device.
__global__ __launch_bounds__(kPlanThreads) void k_plan(DenseArgs a, Plan pl, int d, int fill) {
  __shared__ int s_a[kPlanThreads / STK_WAVE], s_b[kPlanThreads / STK_WAVE], s_long;
  __shared__ int s_base[kPlanThreads + 1], s_s0[kPlanThreads], s_rows[kPlanThreads],
      s_len[kPlanThreads], s_count[kWhole + 2];
  const int tid = threadIdx.x, ns = a.requests;
  if (tid == 0) s_long = 0;
  s_count[tid] = 0;
  if (tid < 2) s_count[kPlanThreads + tid] = 0;
  int s0 = 0, s1 = 0, base;
  if (tid < ns) {
    rows_of(a, tid, s0, s1);
    s_s0[tid] = s0;
    s_rows[tid] = s1 - s0;
    s_len[tid] = tokens_of(a, tid);
  }
  const int mine = (int)(((int64_t)(s1 - s0) * a.g + kDenseRows - 1) / kDenseRows);
  s_base[tid] = block_excl_scan1(mine, s_a, &base);
  __syncthreads();
  const int rt = min(min(base, pl.limit), kPlanThreads);
  // four threads look at a tile's tokens where there are enough
  const int lanes = a.first && 4 * rt <= kPlanThreads ? 4 : 1;
  const int it = tid / lanes, sub = tid % lanes;
  const bool lists = it < rt && sub == 0;
  Tile x{};
  int n = 0, cum;
  if (it < rt) {
    int lo = 0, hi = ns - 1;             // last request that begins at or before this tile
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s_base[mid] <= it) lo = mid;
      else hi = mid - 1;
    }
    x.seq = lo;
    x.tile = (lo + 1 < ns ? s_base[lo + 1] : base) - 1 - it;
    x.s0 = s_s0[lo];
    x.rows = s_rows[lo];
    x.len = s_len[lo];
    const int64_t row0 = (int64_t)x.tile * kDenseRows;
    const int64_t row1 = min(row0 + kDenseRows, (int64_t)x.rows * a.g) - 1;
    const int t0 = x.s0 + (int)(row0 / a.g), t1 = x.s0 + (int)(row1 / a.g);
    const int p0 = x.len - x.rows - x.s0;          // position of row t: p0 + t
    x.klo = 0x7fffffff;
    x.min_hi = 0x7fffffff;
    auto see = [&](int t, int first) {
      const Span s = span_at(a, lo, first, p0 + t, x.len);
      const bool some = s.hi > s.lo;
      // without starts rows after an empty one may still see keys from its lower end on
      x.klo = some || !a.first ? min(x.klo, s.lo) : x.klo;
      x.khi = some ? max(x.khi, s.hi) : x.khi;
      x.max_lo = some ? max(x.max_lo, s.lo) : x.max_lo;
      x.min_hi = some ? min(x.min_hi, s.hi) : 0;
    };
    if (a.first) {
      for (int t = t0 + sub; t <= t1; t += 8 * lanes) {
        int f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = a.first[min(t + i * lanes, t1)];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          // (past the end: the last token again)
          const int y = min(t + i * lanes, t1);
          see(y, f[i]);
        }
      }
    } else {                             // the spans of a request's tokens only move up
      see(t0, 0);
      see(t1, 0);
    }
  }
  if (lanes > 1) {
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      x.klo = min(x.klo, __shfl_xor(x.klo, o));
      x.khi = max(x.khi, __shfl_xor(x.khi, o));
      x.max_lo = max(x.max_lo, __shfl_xor(x.max_lo, o));
      x.min_hi = min(x.min_hi, __shfl_xor(x.min_hi, o));
    }
  }
  if (lists) {
    if (x.khi <= x.klo) x.klo = x.khi = 0;
    x.kstart = x.klo & ~15;
    const int tk = d == 256 ? 32 : 64;
    n = max(1, (x.khi - x.kstart + tk - 1) / tk);
    atomicMax(&s_long, n);
  }
  x.cum = block_excl_scan1(n, s_b, &cum);          // (its barrier also publishes s_long)
  const bool whole = leave_whole(cum * a.hkv, s_long, rt * a.hkv, fill, d);
  int at = it;
  if (whole) {
    // by length, the longest first; equal ones in any order
    int rank = 0, all;
    if (lists) rank = atomicAdd(&s_count[n], 1);
    __syncthreads();
    // tiles longer than kWhole - tid, by a prefix sum over the lengths from the top
    const int here = s_count[kWhole - tid];
    const int longer = block_excl_scan1(here, s_a, &all);
    s_base[tid] = longer;
    __syncthreads();
    if (lists) at = s_base[kWhole - n] + rank;
  }
  if (lists) pl.tiles[at] = x;
  if (tid == 0) {
    pl.head[0] = cum;
    pl.head[1] = rt;
    pl.head[2] = whole ? 0 : min(fill, max(1, cum * a.hkv / kRun));
  }
}

// Rows of the tiles whose units were dealt to several workgroups, kJoinRows of
// them at a time.
constexpr int kJoinRows = 16, kJoinGrid = 8192;
template <typename T, int D>
__global__ __launch_bounds__(256) void k_join_tiles(DenseArgs a, Plan pl, Parts split) {
  constexpr int SL = kDenseRows / kJoinRows;
  const int per = pl.head[0], ntiles = pl.head[1], cut = pl.head[2];
  if (cut == 0) return;
  const Deal deal(per * a.hkv, cut);
  for (int y = (int)blockIdx.x; y < ntiles * a.hkv * SL; y += (int)gridDim.x) {
    const int r0 = (y % SL) * kJoinRows, it = y / SL % ntiles, kvh = y / SL / ntiles;
    const Tile t = pl.tiles[it];
    const int first = kvh * per + t.cum;
    const int n = (it + 1 < ntiles ? pl.tiles[it + 1].cum : per) - t.cum;
    const int w0 = deal.wg_of(first), w1 = deal.wg_of(first + n - 1);
    if (w0 == w1) continue;
    const int64_t row0 = (int64_t)t.tile * kDenseRows + r0;
    const int nrow = (int)min((int64_t)kJoinRows, (int64_t)t.rows * a.g - row0);
#pragma unroll 2
    for (int x = threadIdx.x; x < nrow * (D / 4); x += 256) {
      const int row = x / (D / 4), dc = x % (D / 4);
      float m = -INFINITY, l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int w = w0; w <= w1; ++w) {
        const int64_t pr = (2 * (int64_t)w + (w == w0 ? 1 : 0)) * kDenseRows + r0 + row;
        const float mi = split.m[pr], li = split.l[pr], mx = fmaxf(m, mi);
        const f32x4 oi = *reinterpret_cast<const f32x4*>(split.o + pr * D + 4 * dc);
        const float f = part_weight(m, mx), fi = part_weight(mi, mx);
        m = mx;
        l = l * f + li * fi;
        o = o * f + oi * fi;
      }
      const int tok = t.s0 + (int)((row0 + row) / a.g);
      const int head = kvh * a.g + (int)((row0 + row) % a.g);
      store_out<T>(a.out + ((int64_t)tok * a.hq + head) * D + 4 * dc, o, l);
    }
  }
}

// Joins `count` parts of one row into (m, l, o): rows `pr` of slot(i), four columns per
// thread.  Four parts at a time, their loads in flight together.
template <typename F>
__device__ __forceinline__ void join_parts(const Parts& p, int i0, int count, int step, int d,
                                           int col, F row, float& m, float& l, f32x4& o) {
  for (int i = i0; i < count; i += 4 * step) {
    float pm[4], plx[4];
    f32x4 po[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int64_t r = row(min(i + x * step, count - 1));
      pm[x] = p.m[r];
      plx[x] = p.l[r];
      po[x] = *reinterpret_cast<const f32x4*>(p.o + r * d + col);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (i + x * step >= count) break;
      const float mx = fmaxf(m, pm[x]), f = part_weight(m, mx), fi = part_weight(pm[x], mx);
      m = mx;
      l = l * f + plx[x] * fi;
      o = o * f + po[x] * fi;
    }
  }
}

// ALONE: single tokens.  FEW: a few rows per request; rows of no request become zero
// (a.fill).  SHARED: single tokens, with the parts of their group's shared keys.
enum JoinKind { ALONE, FEW, SHARED };

// One row, (token, query head) of a decode batch, per workgroup or, where
// there are enough of them (`WAVE`), per wave: the parts of its own keys, and with
// SHARED those of its group's shared keys.  Bound by latency (a row's loads are four
// dependent rounds, about 5 us): 96 requests of 32 heads and 23 parts took two rounds of
// workgroups, 13 us, and take 11 as waves; 2560 of 22 at D = 64 11 and 7.6.
template <typename T, int D, JoinKind KIND, bool WAVE>
__global__ __launch_bounds__(256) void k_join_rows(DenseArgs a, Parts split, Parts whole,
                                                   const int32_t* place, int launched, Plan pl,
                                                   Parts psplit, Parts pwhole, int plaunched) {
  constexpr int CH = D / 4, NP = (WAVE ? STK_WAVE : 256) / CH;   // 4-wide columns, parts in flight
  __shared__ float s_m[NP], s_l[NP];
  __shared__ f32x4 s_o[NP][CH];
  const int x = WAVE ? (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(wave_id())
                     : (int)blockIdx.x;
  if (WAVE && x >= a.t * a.hq) return;
  const int tok = x / a.hq, head = x % a.hq, kvh = head / a.g;
  const int tid = WAVE ? lane_id() : (int)threadIdx.x, dc = tid % CH, grp = tid / CH;
  int r = tok, m0 = 0, rows = 1;                 // the token's place among its request's
  if constexpr (KIND == FEW) {
    r = last_at_most(a.requests, tok, [&](int i) { return a.starts[i]; });
    int s0 = 0, s1 = 0;
    if (r >= 0) rows_of(a, r, s0, s1);
    m0 = tok - s0;
    rows = s1 - s0;
    if (r < 0 || m0 < 0 || m0 >= rows) {
      if (a.fill && grp == 0)
        store_out<T>(a.out + ((int64_t)tok * a.hq + head) * D + 4 * dc, f32x4{}, 0.f);
      return;
    }
  }
  const int gi = m0 * a.g + head % a.g, nc = row_chunks(a, rows);
  const int item = kvh * nc + gi / kDecodeRows, hrow = gi % kDecodeRows;
  // a request has the same units for each of its items
  const int base = place[r], end = place[r + 1], total = place[a.requests];
  const int n = (end - base) / (a.hkv * nc), first = base + item * n;
  const Deal deal(total, launched);
  const int w0 = deal.wg_of(first), w1 = deal.wg_of(first + n - 1);
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  if (w0 == w1) {
    if constexpr (KIND != SHARED) return;        // finished by its workgroup
    const int64_t at = ((int64_t)r * a.hkv * nc + item) * kDecodeRows + hrow;
    join_parts(whole, grp, 1, NP, D, 4 * dc, [&](int) { return at; }, m, l, o);
  } else {
    join_parts(split, grp, w1 - w0 + 1, NP, D, 4 * dc, [&](int i) {
      return (2 * (int64_t)(w0 + i) + (i == 0 ? 1 : 0)) * kDecodeRows + hrow;
    }, m, l, o);
  }
  if constexpr (KIND == SHARED) {
    const int g = group_of(a, r);
    if (g >= 0) {
      int s0, s1;
      seq_rows(a, g, s0, s1);
      const int64_t idx = (int64_t)(r - s0) * a.g + gi;
      const int tile = (int)(idx / kDenseRows), rr = (int)(idx % kDenseRows);
      const int units = group_units(a, g, kTk<D>), per = pl.base[a.ngroups];
      const int pf = kvh * per + pl.base[g] + tile * units;
      const Deal pdeal(per * a.hkv, group_grid(per * a.hkv, kTk<D>, plaunched));
      const int v0 = pdeal.wg_of(pf), v1 = pdeal.wg_of(pf + units - 1);
      if (v0 == v1) {
        const int64_t at = group_slot(a, kvh, g, s0, tile, pl.limit) * kDenseRows + rr;
        join_parts(pwhole, grp, 1, NP, D, 4 * dc, [&](int) { return at; }, m, l, o);
      } else {
        join_parts(psplit, grp, v1 - v0 + 1, NP, D, 4 * dc, [&](int i) {
          return (2 * (int64_t)(v0 + i) + (i == 0 ? 1 : 0)) * kDenseRows + rr;
        }, m, l, o);
      }
    }
  }
  if constexpr (WAVE) {
#pragma unroll
    for (int d = CH; d < STK_WAVE; d <<= 1) {
      const float mi = __shfl_xor(m, d), li = __shfl_xor(l, d), mx = fmaxf(m, mi);
      const float f = part_weight(m, mx), fi = part_weight(mi, mx);
      m = mx;
      l = l * f + li * fi;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float oi = __shfl_xor(o[i], d);
        o[i] = o[i] * f + oi * fi;
      }
    }
  } else {
    if (dc == 0) {
      s_m[grp] = m;
      s_l[grp] = l;
    }
    s_o[grp][dc] = o;
    __syncthreads();
    if (grp == 0) {
#pragma unroll
      for (int i = 1; i < NP; ++i) {
        const float mi = s_m[i], mx = fmaxf(m, mi);
        const float f = part_weight(m, mx), fi = part_weight(mi, mx);
        m = mx;
        l = l * f + s_l[i] * fi;
        o = o * f + s_o[i][dc] * fi;
      }
    }
  }
  if (grp == 0) store_out<T>(a.out + ((int64_t)tok * a.hq + head) * D + 4 * dc, o, l);
}

// ------------------------------------------------------------------ host

constexpr int kFill = 512;          // workgroups that fill the device: two per CU

struct DenseShape {
  int tokens, requests, hq, hkv, nb, b, d, ngroups;
  bool ragged;
};

static StkCheck check_dense(const DenseShape& s, int dtype, int pages) {
  if (dtype != DT_F16 && dtype != DT_BF16) return {false, "the cache must be FP16 or BF16"};
  if (s.tokens < 0 || s.requests < 1 || s.nb < 1 || pages < 1) return {false, "bad shape"};
  StkCheck c = stk_check_kv(dtype, s.hq, s.hkv, s.nb, s.b, s.d);
  if (!c.ok) return c;
  if (s.hq < 1) return {false, "expected nonempty shapes"};
  if (s.d != 64 && s.d != 128 && s.d != 256)
    return {false, "head dimension must be 64, 128 or 256"};
  if (s.b % 16) return {false, "the block size must be a multiple of 16"};
  const int64_t keys = (int64_t)s.nb * s.b;
  if (keys > (1ll << 30) || keys * s.b > (1ll << 40) || (int64_t)pages * s.b > 0x7fffffff)
    return {false, "cache too large"};
  return {true, ""};
}

// Items per KV head of attention in 16 rows, at most.
static int64_t decode_items(const DenseShape& s) {
  const int64_t g = s.hq / s.hkv;
  return s.ragged ? s.tokens * g / kDecodeRows + s.requests
                  : s.requests * ((g + kDecodeRows - 1) / kDecodeRows);
}
static int64_t decode_units(const DenseShape& s) {
  return decode_items(s) * s.hkv * (((int64_t)s.nb * s.b + kUnit - 1) / kUnit + 1);
}
// Few rows are worked on as single tokens are, 16 of them at a time: each 16 read
// the request's keys again, but these are spread over the device, and the reads
// hit the caches.  So where there are at most as many items as CUs, and their units few, or
// the rows are about 16 per request (whoever has most of them reads its keys R + 3
// times at most).  In caches of a few units tiles are as quick.
// Measured (tiles, items), 32 query heads over 8 KV heads, D = 128: 4 tokens after
// 2000 42.6, 14.0 us, after 40000 74.6, 38.6; 8 requests of 4 after 2000 44.3, 24.4;
// 100 tokens after 2000 36.1, 32.9, after 8000 52.3, 107; 32 requests of 4 after 2000
// 36.6, 41.7.
constexpr int64_t kFewItems = 256, kFewUnits = 6144;
static bool few_rows(const DenseShape& s) {
  // (the units fit an int even if starts that decrease give every request all rows)
  return s.ragged && (int64_t)s.nb * s.b > 512 && decode_items(s) * s.hkv <= kFewItems &&
         s.requests * decode_units(s) <= 0x7fffffff &&
         (decode_units(s) <= kFewUnits ||
          (int64_t)s.tokens * (s.hq / s.hkv) <= kDecodeRows * ((int64_t)s.requests + 3));
}
// A few items alone are cut into fewer parts (32 each, but one workgroup per CU at
// least), which the join is quicker with: one request of 16000 tokens, 8 KV
// heads, D = 128: 23.4 us with 512 workgroups, 21.1 with 256; 32 requests of 200
// to 2000 tokens: 26.3 and 28.2.
static int decode_grid(const DenseShape& s) {
  const int64_t items = decode_items(s) * s.hkv, u = decode_units(s);
  const int64_t want = items * 32 < kFill / 2 ? kFill / 2 : items * 32;
  const int64_t fill = want < kFill ? want : kFill;
  return (int)(u < fill ? u : fill);
}
static int64_t tile_limit(const DenseShape& s) {
  const int ns = s.ngroups ? s.ngroups : s.requests;
  const int64_t rows = (int64_t)(s.ngroups ? s.requests : s.tokens) * (s.hq / s.hkv);
  return rows / kDenseRows + ns;
}
static int64_t prefill_units(const DenseShape& s) {
  const int tk = s.d == 256 ? 32 : 64;
  return tile_limit(s) * s.hkv * (((int64_t)s.nb * s.b + tk - 1) / tk + 1);
}
// The most units that a launch counts.  Groups come from the device: even if all
// of them held all requests, their units would have to fit an int.
static int64_t most_units(const DenseShape& s) {
  if (!s.ngroups) return prefill_units(s);
  const int64_t rows = (int64_t)s.requests * (s.hq / s.hkv);
  return (prefill_units(s) / tile_limit(s)) * (rows / kDenseRows + 1) * s.ngroups;
}
// Without cutting there is nothing to list and nothing to join, which saves 7 to 12 us.
// A small cache leaves little to cut, the less the more tiles there are (`holds` times 64
// keys), and many requests of several tiles each fill the device evenly.  More than
// k_plan's tiles are not listed.
// Measured (listed, direct), 32 query heads over 8 KV heads, D = 128, in full caches:
// 60 tokens after 600 27.5, 21.5 us, after 1400 30.3, 37.0; 260 after 1400 39.6, 37.7,
// after 2500 46.3, 57.8; 1000 after 2500 68.4, 61.6; prompts of 2048 tokens 64, 55.5.
// 128 requests of 4 tokens, one of them after 60000 tokens and the others 500: 153, 1171,
// and 375, 358 after 4000 each, so short requests are listed.
constexpr int64_t kSmall = 64, kEvenTiles = 4;
static bool prefill_direct(const DenseShape& s) {
  const int64_t tiles = tile_limit(s), wgs = tiles * s.hkv;
  const int64_t holds = ((int64_t)s.nb * s.b + 63) / 64;
  if (s.ngroups) return false;
  return tiles > kPlanThreads || (holds <= kSmall && wgs >= (s.d == 256 ? 14 : 8) * (holds - 14)) ||
         (tiles >= kEvenTiles * s.requests && wgs >= 2 * kFill);
}
static int prefill_fill(const DenseShape& s) {
  const int64_t u = prefill_units(s);
  return u < kFill ? (int)u : kFill;
}
// k_plan decides whether the tiles are cut: there are workgroups for both.
static int prefill_grid(const DenseShape& s) {
  const int64_t tiles = tile_limit(s) * s.hkv;
  const int fill = prefill_fill(s);
  return s.ngroups || (tiles < fill && !prefill_direct(s)) ? fill : (int)tiles;
}

static size_t parts_bytes(int64_t slots, int rows, int d) {
  return 2 * stk_align((size_t)slots * rows * sizeof(float)) +
         stk_align((size_t)slots * rows * d * sizeof(float));
}
static Parts take_parts(Carve& c, int64_t slots, int rows, int d) {
  Parts p;
  p.m = c.take<float>((size_t)slots * rows);
  p.l = c.take<float>((size_t)slots * rows);
  p.o = c.take<float>((size_t)slots * rows * d);
  return p;
}
// With groups there is no list of tiles: only the units before each group are kept.
static size_t plan_bytes(const DenseShape& s) {
  if (s.ngroups) return stk_align((s.ngroups + 1) * sizeof(int32_t));
  return stk_align(3 * sizeof(int32_t)) + stk_align((size_t)tile_limit(s) * sizeof(Tile));
}
static Plan take_plan(Carve& c, const DenseShape& s) {
  Plan p{};
  p.limit = (int)tile_limit(s);
  if (s.ngroups) {
    p.base = c.take<int32_t>(s.ngroups + 1);
  } else {
    p.head = c.take<int32_t>(3);
    p.tiles = c.take<Tile>(p.limit);
  }
  return p;
}

static size_t dense_bytes(const DenseShape& s) {
  const bool few = few_rows(s);
  size_t x = 0;
  if (!s.ragged || few) {
    x += stk_align((s.requests + 1) * sizeof(int32_t)) +
         parts_bytes(2 * (int64_t)decode_grid(s), kDecodeRows, s.d);
    if (s.ngroups) x += parts_bytes(decode_items(s) * s.hkv, kDecodeRows, s.d);
  }
  if ((s.ragged && !few) || s.ngroups) {
    if (!prefill_direct(s))
      x += plan_bytes(s) + parts_bytes(2 * (int64_t)prefill_fill(s), kDenseRows, s.d);
    if (s.ngroups) x += parts_bytes(tile_limit(s) * s.hkv, kDenseRows, s.d);
  }
  return x ? x : 256;
}

static int launch_plan(const DenseArgs& a, const Plan& p, int d, int fill, hipStream_t st) {
  hipLaunchKernelGGL(k_plan, dim3(1), dim3(kPlanThreads), 0, st, a, p, d, fill);
  return stk_check_launch("k_plan");
}

template <typename T>
static void launch_join_tiles(const DenseArgs& a, const Plan& p, const Parts& split, int d,
                              hipStream_t st) {
  const int all = p.limit * a.hkv * (kDenseRows / kJoinRows);
  const unsigned g = (unsigned)(all < kJoinGrid ? all : kJoinGrid);
  if (d == 64) k_join_tiles<T, 64><<<g, 256, 0, st>>>(a, p, split);
  else if (d == 128) k_join_tiles<T, 128><<<g, 256, 0, st>>>(a, p, split);
  else k_join_tiles<T, 256><<<g, 256, 0, st>>>(a, p, split);
}

constexpr unsigned kJoinAlone = 2048;   // rows that have a workgroup each: one round of them
template <typename T, JoinKind KIND>
static void launch_join_rows(const DenseArgs& a, const Parts& split, const Parts& whole,
                             const int32_t* place, int grid, const Plan& p, const Parts& ps,
                             const Parts& pw, int pgrid, int d, hipStream_t st) {
  const unsigned rows = (unsigned)(a.t * a.hq);
#define STK_JOIN(D)                                                                               \
  (rows <= kJoinAlone ? k_join_rows<T, D, KIND, false><<<rows, 256, 0, st>>>(                   \
                            a, split, whole, place, grid, p, ps, pw, pgrid)                       \
                      : k_join_rows<T, D, KIND, true><<<(rows + 3) / 4, 256, 0, st>>>(          \
                            a, split, whole, place, grid, p, ps, pw, pgrid))
  if (d == 64) STK_JOIN(64);
  else if (d == 128) STK_JOIN(128);
  else STK_JOIN(256);
#undef STK_JOIN
}

template <typename T>
static int run_dense(const DenseShape& s, DenseArgs a, int mode, void* workspace, hipStream_t st) {
  Carve c(workspace);
  if (s.ragged && !few_rows(s)) {
    const int grid = prefill_grid(s);
    if (prefill_direct(s)) return launch_direct<T>(s.d, mode, a, grid, st);
    const Plan p = take_plan(c, s);
    const int fill = prefill_fill(s);
    const Parts split = take_parts(c, 2 * (int64_t)fill, kDenseRows, s.d);
    int rc = launch_plan(a, p, s.d, fill, st);
    if (rc) return rc;
    rc = launch_prefill<T>(s.d, mode, a, p, split, grid, st);
    if (rc) return rc;
    launch_join_tiles<T>(a, p, split, s.d, st);
    return stk_check_launch("k_join_tiles");
  }
  const int grid = decode_grid(s);
  int32_t* place = c.take<int32_t>(s.requests + 1);
  const Parts split = take_parts(c, 2 * (int64_t)grid, kDecodeRows, s.d);
  if (s.ngroups) {
    const Parts whole = take_parts(c, decode_items(s) * s.hkv, kDecodeRows, s.d);
    const Plan p = take_plan(c, s);
    const int pgrid = prefill_fill(s);
    const Parts ps = take_parts(c, 2 * (int64_t)pgrid, kDenseRows, s.d);
    const Parts pw = take_parts(c, tile_limit(s) * s.hkv, kDenseRows, s.d);
    const int rc = launch_shared<T>(s.d, mode, a, p, ps, pw, pgrid, split, whole, place, grid, st);
    if (rc) return rc;
    launch_join_rows<T, SHARED>(a, split, whole, place, grid, p, ps, pw, pgrid, s.d, st);
  } else {
    const int rc = s.ragged ? launch_few<T>(s.d, mode, a, split, place, grid, st)
                            : launch_decode<T>(s.d, mode, a, split, place, grid, st);
    if (rc) return rc;
    if (s.ragged)
      launch_join_rows<T, FEW>(a, split, Parts{}, place, grid, Plan{}, Parts{}, Parts{}, 0, s.d,
                               st);
    else
      launch_join_rows<T, ALONE>(a, split, Parts{}, place, grid, Plan{}, Parts{}, Parts{}, 0, s.d,
                                 st);
  }
  return stk_check_launch("k_join_rows");
}

// A cap's tanh is 1 - 2 / (1 + e^2y), within 2^-23 of the true value whatever its
// size: the capped score is within 2^-23 cap, which at 4096 is 2^-11, half a step
// of FP16.  (A cap far above the scores caps nothing; with no cap there is no such term.)
constexpr float kMaxScale = 1e30f, kMaxCap = 4096.f;

static int dense(const DenseShape& s, const void* q, int64_t q_stride, int dtype, int pages,
                 const void* k_pages, const void* v_pages, const int32_t* table,
                 const int32_t* nblocks, const int32_t* ntokens, const int32_t* starts,
                 const int32_t* groups, const int32_t* shared, float scale, float softcap,
                 const float* slopes, int window, const int32_t* prefix, const int32_t* first,
                 void* out, int fill, void* workspace, size_t workspace_bytes, void* stream) {
  STK_REQUIRE(check_dense(s, dtype, pages));
  STK_REQUIRE(s.ragged || s.tokens == s.requests, "expected one query token per request");
  STK_REQUIRE(s.tokens == 0 || (q && out), "null pointer");
  STK_REQUIRE(k_pages && v_pages && table && nblocks, "null pointer");
  STK_REQUIRE(scale > 0.f && scale <= kMaxScale, "scale must be positive and at most 1e30");
  STK_REQUIRE(softcap >= 0.f && softcap <= kMaxCap &&
                  (softcap == 0.f || scale / softcap <= kMaxScale),
              "softcap must be in (0, 4096], 0 for none, and not far below the scale");
  STK_REQUIRE(window >= 0, "window must be at least 0 (0: none)");
  STK_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) &
               15) == 0 && q_stride % 8 == 0 && q_stride >= 0,
              "rows must be 16-byte aligned");
  STK_REQUIRE(((s.ragged && !few_rows(s)) || decode_units(s) <= 0x7fffffff) &&
                  (int64_t)s.requests * s.hq <= 0x7fffffff &&
                  (int64_t)s.tokens * s.hq <= 0x7fffffff &&
                  most_units(s) <= 0x7fffffff &&
                  (int64_t)s.tokens * (s.hq / s.hkv) + kDenseRows <= 0x7fffffff,
              "batch too large");
  STK_REQUIRE(workspace && workspace_bytes >= dense_bytes(s), "workspace too small");
  STK_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "the workspace must be 16-byte aligned");
  if (s.tokens == 0) return STK_OK;
  const double log2e = 1.4426950408889634;
  DenseArgs a{};
  a.q = static_cast<const uint16_t*>(q); a.qs = q_stride;
  a.out = static_cast<uint16_t*>(out);
  a.kp = static_cast<const uint16_t*>(k_pages); a.vp = static_cast<const uint16_t*>(v_pages);
  a.table = table; a.nblocks = nblocks; a.ntokens = ntokens; a.starts = starts;
  a.t = s.tokens; a.requests = s.requests; a.hq = s.hq; a.hkv = s.hkv; a.g = s.hq / s.hkv;
  a.nb = s.nb; a.b = s.b; a.pages = pages;
  a.bdiv = (1ull << 32) / (uint64_t)(s.b / 16) + 1;
  a.c = (float)(scale * log2e);
  if (softcap > 0.f) {
    a.cap_in = (float)(2.0 * log2e * scale / softcap);
    a.cap_out = (float)(softcap * log2e);
  }
  a.slopes = slopes; a.window = window; a.prefix = prefix; a.first = first;
  a.groups = groups; a.shared = shared; a.ngroups = s.ngroups; a.fill = fill;
  const int mode = (softcap > 0.f ? 1 : 0) | (slopes ? 2 : 0);
  hipStream_t st = (hipStream_t)stream;
  return dtype == DT_BF16 ? run_dense<bf16s>(s, a, mode, workspace, st)
                          : run_dense<f16s>(s, a, mode, workspace, st);
}

}  // namespace stk

using namespace stk;

extern "C" {

STK_API size_t stk_paged_attention_workspace_bytes(int tokens, int requests, int hq, int hkv,
                                                   int nb, int b, int d, int ragged) {
  if (tokens <= 0 || requests <= 0 || hq <= 0 || hkv <= 0 || nb <= 0 || b <= 0 || d <= 0 ||
      hq % hkv)
    return 0;
  return dense_bytes({tokens, requests, hq, hkv, nb, b, d, 0, ragged != 0});
}

STK_API int stk_paged_attention(const void* q, int64_t q_stride, int dtype, int tokens,
                                int requests, int hq, int hkv, int nb, int b, int d, int pages,
                                const void* k_pages, const void* v_pages,
                                const int32_t* block_table, const int32_t* nblocks,
                                const int32_t* ntokens, const int32_t* starts, float scale,
                                float softcap, const float* slopes, int window,
                                const int32_t* prefix, const int32_t* first, void* out, int fill,
                                void* workspace, size_t workspace_bytes, void* stream) {
  return dense({tokens, requests, hq, hkv, nb, b, d, 0, starts != nullptr}, q, q_stride, dtype,
               pages, k_pages, v_pages, block_table, nblocks, ntokens, starts, nullptr, nullptr,
               scale, softcap, slopes, window, prefix, first, out, fill, workspace,
               workspace_bytes, stream);
}

STK_API size_t stk_paged_shared_workspace_bytes(int requests, int ngroups, int hq, int hkv, int nb,
                                                int b, int d) {
  if (requests <= 0 || ngroups <= 0 || hq <= 0 || hkv <= 0 || nb <= 0 || b <= 0 || d <= 0 ||
      hq % hkv)
    return 0;
  return dense_bytes({requests, requests, hq, hkv, nb, b, d, ngroups, false});
}

STK_API int stk_paged_shared_attention(const void* q, int64_t q_stride, int dtype, int requests,
                                       int hq, int hkv, int nb, int b, int d, int pages,
                                       const void* k_pages, const void* v_pages,
                                       const int32_t* block_table, const int32_t* nblocks,
                                       const int32_t* ntokens, const int32_t* groups,
                                       const int32_t* shared, int ngroups, float scale,
                                       float softcap, const float* slopes, int window,
                                       const int32_t* first, void* out, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  STK_REQUIRE(groups && shared, "null pointer");
  STK_REQUIRE(ngroups >= 1 && ngroups <= requests, "expected 1 to R groups");
  return dense({requests, requests, hq, hkv, nb, b, d, ngroups, false}, q, q_stride, dtype, pages,
               k_pages, v_pages, block_table, nblocks, ntokens, nullptr, groups, shared, scale,
               softcap, slopes, window, nullptr, first, out, 0, workspace, workspace_bytes,
               stream);
}

}  // extern "C"
