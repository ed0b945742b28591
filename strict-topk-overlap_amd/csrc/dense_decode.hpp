// Dense attention of single tokens over the paged cache, and of a few per request (FEW).
//
// An item is one request's KV head with up to 16 of its query rows (a token's heads, and
// with FEW several tokens', each with its own range of keys); its keys
// are cut into units of kUnit keys, and the units of all items, laid end to end,
// are dealt evenly over one grid that fills the device: a ragged batch, or one long
// request, keeps every CU busy to the end.  A workgroup walks its run of units
// item by item.  Items that lie whole in one workgroup are finished there; the
// parts of the others are joined by k_join_rows.  Nothing of this needs the lengths on
// the host.
//
// Within a workgroup the four waves take a quarter of the keys each (short items:
// one item each) and share nothing until the item ends.  A wave's tile is 32 keys
// (at D = 256 it is 16):
//   S[key, head] = K Q^T  (16x16x32, K straight from global memory to registers,
//                          in the operand's own layout),
//   O^T[dim, head] += V^T P^T  (V through the wave's own LDS, read transposed).
// Lane (n, g) of S holds keys 4g .. 4g + 3 of both 16-key halves for head n, and
// the order of the keys within the second product is free: taking {4g .. 4g + 3,
// 16 + 4g .. 16 + 4g + 3} as its eight, P never leaves its lane.
// The next tile's K and V are in flight while a tile is worked on.
//
// Bound by HBM: every key and value is read once (per 16 query heads of its KV
// head).  16 requests of 8192 to 131000 tokens, 8 KV heads, D = 128: 2.6 GB in 434 us, 6.0
// TB/s; one request of 16000 tokens 15 us, of which 5 pass before its first tile.
#pragma once

#include "dense.hpp"

namespace stk {

// Decode work of request r: the keys that it sees, cut into n units from lo16, and
// items per KV head.  With starts a request has any number of query tokens, and an
// item is 16 of their rows (token, head); the keys are those that any of them sees.
struct DecodeSpan { int lo, hi, lo16, n, nc; };

__device__ __forceinline__ int row_chunks(const DenseArgs& a, int tokens) {
  return (int)(((int64_t)tokens * a.g + kDecodeRows - 1) / kDecodeRows);
}

template <bool FEW>
__device__ __forceinline__ DecodeSpan decode_span(const DenseArgs& a, int r) {
  const int n = tokens_of(a, r);
  if constexpr (FEW) {
    int s0, s1;
    rows_of(a, r, s0, s1);
    DecodeSpan d{0x7fffffff, 0, 0, 1, row_chunks(a, s1 - s0)};
    auto see = [&](int t, int first, bool always) {
      const Span x = span_at(a, r, first, n - (s1 - t), n);
      if (always || x.hi > x.lo) d.lo = min(d.lo, x.lo);
      if (x.hi > x.lo) d.hi = max(d.hi, x.hi);
    };
    if (a.first && s1 - s0 <= 32) {
      for (int t = s0; t < s1; t += 8) {
        int f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = a.first[min(t + i, s1 - 1)];
#pragma unroll
        for (int i = 0; i < 8; ++i) see(min(t + i, s1 - 1), f[i], false);
      }
    } else if (s1 > s0) {
      // without documents the spans only move up; documents only raise their lower ends,
      // and those of more tokens are not looked at
      see(s0, 0, true);
      see(s1 - 1, 0, true);
    }
    if (d.hi <= d.lo) d.lo = d.hi = 0;
    d.lo16 = d.lo & ~15;
    if (s1 == s0) d.n = 0;
    else if (d.hi > d.lo) d.n = (d.hi - d.lo16 + kUnit - 1) / kUnit;
    return d;
  }
  const Span s = span_of(a, r, r, n - 1, n);
  DecodeSpan d{s.lo, s.hi, 0, 1, row_chunks(a, 1)};
  if (a.groups) {
    const int g = group_of(a, r);
    const int keys = g >= 0 ? shared_of(a, g) : 0;
    if (n >= keys) d.lo = max(d.lo, keys);
  }
  d.lo16 = d.lo & ~15;
  if (d.hi > d.lo) d.n = (d.hi - d.lo16 + kUnit - 1) / kUnit;
  return d;
}

// The requests' units laid end to end: how many there are, the request that holds
// the first unit of workgroup `wg` of `launched`, and the units before that
// request (past the last workgroup with work: any).  Workgroup 0 also leaves
// the units before every request, and their total, in place [R + 1] for k_join_rows.
struct DecodePlace { int total, base, r; DecodeSpan span; };

template <bool FEW>
__device__ __forceinline__ DecodePlace decode_place(const DenseArgs& a, int wg, int launched,
                                                    int32_t* place) {
  __shared__ int s_tmp[4], s_at[2];
  __shared__ DecodeSpan s_span;
  if (a.requests <= STK_WAVE) {
    // every wave looks for itself, without barriers (one request of 16000 tokens 21.3
    // us, 20.5)
    const int r = lane_id();
    DecodeSpan x{};
    if (r < a.requests) x = decode_span<FEW>(a, r);
    const int c = x.n * x.nc * a.hkv, end = wave_incl_scan_dpp(c);
    const int total = __builtin_amdgcn_readlane(end, STK_WAVE - 1);
    if (wg == 0 && (int)threadIdx.x < a.requests) place[r] = end - c;
    if (wg == 0 && threadIdx.x == 0) place[a.requests] = total;
    const int u = Deal(total, launched).at(wg);
    const uint64_t mine = __ballot(u >= end - c && u < end);
    const int at = mine ? __builtin_ctzll(mine) : 0;
    DecodePlace p{total, __builtin_amdgcn_readlane(end - c, at), at, {}};
    p.span.lo = __builtin_amdgcn_readlane(x.lo, at);
    p.span.hi = __builtin_amdgcn_readlane(x.hi, at);
    p.span.lo16 = __builtin_amdgcn_readlane(x.lo16, at);
    p.span.n = __builtin_amdgcn_readlane(x.n, at);
    p.span.nc = __builtin_amdgcn_readlane(x.nc, at);
    return p;
  }
  // requests per thread and pass: their loads are in flight together
  const int e = a.requests > 256 ? 4 : 1, pass = 256 * e;
  DecodeSpan span[4] = {};
  int units[4];
  // units of this pass's requests before this thread's, and of all of them
  auto scan = [&](int r0, int& before, int& sum) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + e * (int)threadIdx.x + j;
      span[j].n = 0;
      if (j < e && r < a.requests) span[j] = decode_span<FEW>(a, r);
      units[j] = span[j].n * span[j].nc * a.hkv;
      c += units[j];
    }
    __syncthreads();
    before = block_excl_scan1(c, s_tmp, &sum);
  };
  if (threadIdx.x == 0) {
    s_at[0] = s_at[1] = 0;
    s_span = DecodeSpan{};
  }
  int total = 0, before = 0, sum = 0;
  for (int r0 = 0; r0 < a.requests; r0 += pass) {
    scan(r0, before, sum);
    if (wg == 0) {
      int at = total + before;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + e * (int)threadIdx.x + j;
        if (j < e && r < a.requests) place[r] = at;
        at += units[j];
      }
    }
    total += sum;
  }
  if (wg == 0 && threadIdx.x == 0) place[a.requests] = total;
  const int u = Deal(total, launched).at(wg);
  int base = 0;
  for (int r0 = 0; r0 < a.requests; r0 += pass) {
    if (a.requests > pass) scan(r0, before, sum);
    int at = base + before;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = units[j];
      if (u >= at && u < at + c) {
        s_at[0] = at;
        s_at[1] = r0 + e * (int)threadIdx.x + j;
        s_span = span[j];
      }
      at += c;
    }
    base += sum;
    if (u < base) break;
  }
  __syncthreads();
  DecodePlace p{total, s_at[0], s_at[1], s_span};
  p.base = __builtin_amdgcn_readfirstlane(p.base);
  p.r = __builtin_amdgcn_readfirstlane(p.r);
  return p;
}

// Four neighbouring items of at most kAlone units that lie whole in one workgroup are
// worked on together, each by a wave of its own: short items are bound by their chain of
// loads.  8 KV heads, D = 128, 512 requests of 1 to 100 tokens: 46.4 us, 28.6 so; 256 of
// 100 to 300: 53.2, 43.5.  With four units the times are the same.
constexpr int kAlone = 2;

// At D = 256 a tile of 32 keys and the next one's rows would leave a wave per SIMD.
template <int D> constexpr int kDecodeTile = D == 256 ? 16 : 32;
// a wave's V tile, and after its last one its output rows in FP32
template <int D> constexpr size_t kDecodeWave = 64 * D;
template <int D> constexpr size_t kDecodeLds = 4 * kDecodeWave<D>;

// The work of workgroup wg of nwg.  With FEW a value that only some of an item's rows see
// may be infinite or NaN, and 0 times it is not 0: such an item is done again row by row.
// With PARTS items that lie whole in it leave
// their parts in `whole`, too, instead of being finished.
template <typename T, int D, int MODE, bool PARTS, bool FEW = false>
__device__ __forceinline__ void decode(const DenseArgs& a, const Parts& split, const Parts& whole,
                                       int32_t* place, char* lds, int wg, int nwg) {
  constexpr int TW = kDecodeTile<D>;    // keys per tile
  constexpr int HW = TW / 16;           // its runs of 16 keys
  constexpr int KS = D / 32;            // QK steps
  constexpr int DB = D / 16;            // output blocks
  constexpr int VN = TW * D / 512;      // 16-byte chunks of a V tile per lane
  constexpr int CPR = D / 8;            // chunks per row
  constexpr int RPI = STK_WAVE / CPR;   // rows per load instruction
  constexpr uint16_t EXPO = __is_same(T, bf16s) ? 0x7f80 : 0x7c00;
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ int s_bad[4];
  const int lane = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
  const int n16 = lane & 15, kg = lane >> 4;
  const DecodePlace at = decode_place<FEW>(a, wg, nwg, place);
  const Deal deal(at.total, nwg);
  if ((uint32_t)wg >= deal.grid) return;
  int u = deal.at(wg);
  const int u1 = deal.at(wg + 1);
  int r = at.r, base = at.base;
  // V tile in LDS: row-major, 32-byte blocks swizzled so that the 16 rows of a
  // transposed read spread over all banks
  auto fsw = [](int row) { return D == 64 ? (row >> 1) & 3 : row & 7; };
  uint16_t* vt = reinterpret_cast<uint16_t*>(lds + w * kDecodeWave<D>);
  int vw[VN], va[DB];
#pragma unroll
  for (int i = 0; i < VN; ++i) {
    const int row = i * RPI + lane / CPR, ch = lane % CPR;
    vw[i] = row * D + ((((ch >> 1) ^ fsw(row)) << 1) | (ch & 1)) * 8;
  }
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const int row = 4 * kg + (n16 >> 2);
    va[db] = row * D + (db ^ fsw(row)) * 16 + 4 * (n16 & 3);
  }
  DecodeSpan next = at.span;
  while (u < u1) {
    DecodeSpan sp = next;
    sp.lo = __builtin_amdgcn_readfirstlane(sp.lo);
    sp.hi = __builtin_amdgcn_readfirstlane(sp.hi);
    sp.lo16 = __builtin_amdgcn_readfirstlane(sp.lo16);
    sp.n = __builtin_amdgcn_readfirstlane(sp.n);
    const int nc = __builtin_amdgcn_readfirstlane(sp.nc), per = a.hkv * nc * sp.n;
    if (u >= base + per) {
      if (++r >= a.requests) return;      // (starts that decrease may count past the units)
      base += per;
      next = decode_span<FEW>(a, r);
      continue;
    }
    const int j0 = (u - base) % sp.n;
    // (FEW has too few items for it)
    const bool alone = !FEW && j0 == 0 && sp.n <= kAlone && u + 4 * sp.n <= min(u1, base + per);
    const int item = (u - base) / sp.n + (alone ? w : 0);
    const int j1 = alone ? sp.n : min(sp.n, j0 + (u1 - u));
    u += alone ? 4 * sp.n : j1 - j0;
    const int kvh = item / nc, x0 = (item % nc) * kDecodeRows;
    // rows of the item, and this lane's: token, head, and its range of keys
    int s0 = r, s1 = r + 1;
    if constexpr (FEW) rows_of(a, r, s0, s1);
    const int gn = min(kDecodeRows, (s1 - s0) * a.g - x0), xr = x0 + min(n16, gn - 1);
    const int tok = FEW ? s0 + xr / a.g : r, head = kvh * a.g + (FEW ? xr % a.g : xr);
    int p = sp.hi - 1, rlo = sp.lo, rhi = sp.hi, all_lo = sp.lo, all_hi = sp.hi;
    if constexpr (FEW) {
      const int n = tokens_of(a, r);
      p = n - (s1 - tok);
      const Span rs = span_of(a, r, tok, p, n);
      const bool some = rs.hi > rs.lo;
      rlo = some ? rs.lo : 0;
      rhi = some ? rs.hi : 0;
      all_lo = (int)wave_ext_u32<true>((uint32_t)rlo);       // keys that every row sees
      all_hi = (int)wave_ext_u32<false>((uint32_t)rhi);
    }
    bool bad = false;
    const int ka = sp.lo16 + j0 * kUnit;
    const int kb = (int)min((int64_t)sp.lo16 + (int64_t)j1 * kUnit, (int64_t)sp.hi);
    const int32_t* row = a.table + ((int64_t)r * a.hkv + kvh) * a.nb;
    // this head's query as the second operand: head n16, dims 32 s + 8 kg ..
    u16x8 qf[KS];
    const uint16_t* qp = a.q + (int64_t)tok * a.qs + (int64_t)head * D + 8 * kg;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u16x8*>(qp + 32 * s);
    float slope = 0.f;
    if constexpr (MODE & 2) slope = a.slopes[head] * 1.44269504f;
    float m = -INFINITY, l = 0.f;
    f32x4 acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    const int nt = kb > ka ? (kb - ka + TW - 1) / TW : 0, tpw = alone ? nt : (nt + 3) / 4;
    const int ta = alone ? 0 : w * tpw, tb = min(nt, ta + tpw);
    if (ta < tb) {
      const int wk = ka + TW * ta;                      // the wave's first key
      auto window = [&](int i) {                        // rows of 64 runs of 16 keys
        const int key = wk + 16 * (64 * i + lane);
        const int x = pool_row(a, row, min(key, kb));
        return key < kb ? x : -1;
      };
      int ent = window(0), nxt = window(1);
      u16x8 kf[HW][KS], vf[VN];
      int rw[HW];
      auto load = [&](int t) {
        if (t > 0 && (HW * t) % 64 == 0) {
          ent = nxt;
          nxt = window(HW * t / 64 + 1);
        }
#pragma unroll
        for (int y = 0; y < HW; ++y) rw[y] = __builtin_amdgcn_readlane(ent, (HW * t + y) & 63);
#pragma unroll
        for (int y = 0; y < HW; ++y) {
          const uint16_t* kr = a.kp + (int64_t)max(rw[y], 0) * D + n16 * D + 8 * kg;
#pragma unroll
          for (int s = 0; s < KS; ++s) kf[y][s] = *reinterpret_cast<const u16x8*>(kr + 32 * s);
        }
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const int vr = i * RPI;                       // rows vr .. vr + RPI - 1
          vf[i] = *reinterpret_cast<const u16x8*>(
              a.vp + (int64_t)max(rw[vr / 16], 0) * D + ((vr & 15) + lane / CPR) * D +
              8 * (lane % CPR));
        }
      };
      load(0);
      const int cnt = tb - ta;
      for (int t = 0; t < cnt; ++t) {
        const int key0 = wk + TW * t;
        bool full = key0 >= all_lo && key0 + TW <= min(kb, all_hi);
#pragma unroll
        for (int y = 0; y < HW; ++y) full = full && rw[y] >= 0;
        if (!full) {
          // keys that are not seen: their values are not read as numbers
#pragma unroll
          for (int i = 0; i < VN; ++i) {
            const int kr = i * RPI + lane / CPR, key = key0 + kr;
            const bool ok = key >= sp.lo && key < kb && rw[i * RPI / 16] >= 0;
            if (!ok) vf[i] = u16x8{};
            else if (FEW) bad |= nonfinite16(vf[i], EXPO);
          }
        }
        int was[HW];
#pragma unroll
        for (int y = 0; y < HW; ++y) was[y] = rw[y];
#pragma unroll
        for (int i = 0; i < VN; ++i) *reinterpret_cast<u16x8*>(vt + vw[i]) = vf[i];
        f32x4 sq[HW];
#pragma unroll
        for (int y = 0; y < HW; ++y) sq[y] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int y = 0; y < HW; ++y) sq[y] = mma16<T>(kf[y][s], qf[s], sq[y]);
        if (t + 1 < cnt) load(t + 1);
        float x[4 * HW];
        const float dist = (float)(p - key0 - 4 * kg);
#pragma unroll
        for (int i = 0; i < 4 * HW; ++i)
          x[i] = score2<MODE>(a, sq[i / 4][i % 4], slope, dist - (float)(16 * (i / 4) + i % 4));
        if (!full) {
#pragma unroll
          for (int i = 0; i < 4 * HW; ++i) {
            const int key = key0 + 4 * kg + 16 * (i / 4) + i % 4;
            x[i] = key >= rlo && key < min(kb, rhi) && was[i / 4] >= 0 ? x[i] : -INFINITY;
          }
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < 4 * HW; ++i) top = fmaxf(top, x[i]);
        if (__any(top > m + kLazy)) {
          float mx = fmaxf(top, m);
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float f = mx == m ? 1.f : __builtin_amdgcn_exp2f(m - mx);
          m = mx;
          l *= f;
#pragma unroll
          for (int i = 0; i < DB; ++i) acc[i] *= f;
        }
        const float ms = m == -INFINITY ? 0.f : m;
        // P in two 16-bit parts: the second product then keeps the weights nearly as the
        // sum has them, and the matrix instructions have time to spare here
        uint16_t p[8], pr[8];
#pragma unroll
        for (int i = 0; i < 4 * HW; ++i) {
          const float e = __builtin_amdgcn_exp2f(x[i] - ms);
          l += e;
          p[i] = to16<T>(e);
          pr[i] = to16<T>(e - cvt(T{p[i]}));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if constexpr (HW == 2) {
          const u16x8 ph = {p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7]};
          const u16x8 pl = {pr[0], pr[1], pr[2], pr[3], pr[4], pr[5], pr[6], pr[7]};
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const u16x4 lo = lds_tr(vt + va[db]), hi = lds_tr(vt + va[db] + 16 * D);
            const u16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            acc[db] = mma16<T>(v, ph, acc[db]);
            acc[db] = mma16<T>(v, pl, acc[db]);
          }
        } else {
          // sixteen keys fill one product: both parts of P against the same V
          const u16x8 pp = {p[0], p[1], p[2], p[3], pr[0], pr[1], pr[2], pr[3]};
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const u16x4 v = lds_tr(vt + va[db]);
            acc[db] = mma16<T>(__builtin_shufflevector(v, v, 0, 1, 2, 3, 4, 5, 6, 7), pp, acc[db]);
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (alone) {
      const int64_t pr = ((int64_t)r * a.hkv * nc + item) * kDecodeRows + n16;   // (PARTS)
      if (n16 < gn) {
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          if constexpr (PARTS)
            *reinterpret_cast<f32x4*>(whole.o + pr * D + 16 * db + 4 * kg) = acc[db];
          else
            store_out<T>(a.out + ((int64_t)tok * a.hq + head) * D + 16 * db + 4 * kg, acc[db], l);
        }
        if (PARTS && kg == 0) {
          whole.m[pr] = m;
          whole.l[pr] = l;
        }
      }
      continue;
    }
    // the waves' states: V's LDS holds each wave's output rows
    float* so = reinterpret_cast<float*>(vt);
#pragma unroll
    for (int db = 0; db < DB; ++db)
      *reinterpret_cast<f32x4*>(so + n16 * D + 16 * db + 4 * kg) = acc[db];
    if (lane < 16) {
      s_m[w][lane] = m;
      s_l[w][lane] = l;
    }
    if constexpr (FEW) {
      const bool any = __any(bad);
      if (lane == 0) s_bad[w] = any;
    }
    __syncthreads();
    const bool all = j0 == 0 && j1 == sp.n;
    const bool keep = all && !PARTS;                    // finished here
    const Parts& to = all ? whole : split;
    const int64_t slot = all ? (int64_t)r * a.hkv * nc + item
                             : 2 * (int64_t)wg + (j0 > 0 ? 0 : 1);
    if (FEW && (s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3])) {
      // a value that only some rows see is no number: each row reads its own
      if (4 * w < gn)
        slow_rows<T, D, MODE>(a, r, s0, s1, x0 + 4 * w, min(4, gn - 4 * w), kvh, row, ka, kb,
                              keep ? nullptr : &to, slot * kDecodeRows + 4 * w);
      __syncthreads();
      continue;
    }
    for (int x = threadIdx.x; x < gn * (D / 4); x += 256) {
      const int h = x / (D / 4), dc = x % (D / 4);
      float mx = s_m[0][h];
#pragma unroll
      for (int i = 1; i < 4; ++i) mx = fmaxf(mx, s_m[i][h]);
      float sum = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float mi = s_m[i][h];
        const float f = part_weight(mi, mx);
        sum += f * s_l[i][h];
        o += f * *reinterpret_cast<const f32x4*>(
                     reinterpret_cast<const float*>(lds + i * kDecodeWave<D>) + h * D + 4 * dc);
      }
      if (keep) {
        const int y = x0 + h;
        const int64_t to_row = FEW ? (int64_t)(s0 + y / a.g) * a.hq + kvh * a.g + y % a.g
                                   : (int64_t)r * a.hq + kvh * a.g + y;
        store_out<T>(a.out + to_row * D + 4 * dc, o, sum);
      } else {
        const int64_t pr = slot * kDecodeRows + h;
        *reinterpret_cast<f32x4*>(to.o + pr * D + 4 * dc) = o;
        if (dc == 0) {
          to.m[pr] = mx;
          to.l[pr] = sum;
        }
      }
    }
    __syncthreads();
  }
}

template <typename T, int D, int MODE, bool FEW>
__global__ __launch_bounds__(256, 2) void k_decode(DenseArgs a, Parts split, int32_t* place) {
  __shared__ __attribute__((aligned(16))) char lds[kDecodeLds<D>];
  decode<T, D, MODE, false, FEW>(a, split, split, place, lds, (int)blockIdx.x, (int)gridDim.x);
}

}  // namespace stk
