// New tokens of a ragged batch into the paged cache, rotated to their
// positions on the way.
//
// Request r's new tokens are rows [starts[r], starts[r + 1]) of k_new / v_new
// (and of q); row t of them goes to token position p = positions[r] + t: block
// p / B of the request, offset p % B.  Keys and queries are rotated to p by
// the caller's cos/sin tables: a pair (x, y) of a head's first `rot`
// dimensions becomes (x cos - y sin, y cos + x sin), evaluated in FP32 and
// rounded once to the pages' type, since that is what the cache holds.  Pairs
// are (i, i + rot / 2), or (2i, 2i + 1) interleaved.
//
// One workgroup owns one (request, KV head, touched block), or of requests with
// few tokens several heads of one: it writes the
// block's new K and V rows and folds the rotated keys, as stored, into the
// page's lo/hi, so the bounds need no atomics and do not depend on an order.
// A block whose first new token has offset 0 starts its bounds over.  The
// other workgroups rotate the queries, one wave per run of 16-byte chunks of one
// token.  The host knows neither the lengths nor the positions (they stay on
// the device, so a captured graph follows them): the grid covers the most
// blocks that T tokens of R requests can touch, in places that follow from the starts
// alone, each workgroup finds its request by a search, and those with no block leave.
//
// Bound by HBM: every new row is read once and written once.  8191 tokens of
// 32 + 16 heads, D = 128, FP16: 204 MB in 35 us, 5.8 TB/s with the inputs in the
// Infinity Cache and 43 us without; one token each of 128 requests: 5.0 us, the chain
// of the search, the table and the bounds.
#include "common.hpp"
#include "api.hpp"

namespace stk {

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

struct ExtendArgs {
  const uint16_t* k; const uint16_t* v; const uint16_t* q;
  int64_t ks, vs, qs;             // elements from one token to the next
  uint16_t* qo;                   // [T, Hq, D]
  const int32_t* starts; const int32_t* positions;
  int t, requests, hq, hkv, nb, b, pages;
  const float* cos; const float* sin;   // [rows, rot / 2], or null: no rotation
  int rows, rot;
  uint16_t* kp; uint16_t* vp;
  void* lo; void* hi; int lb;
  const int32_t* table;
  int32_t* nblocks; int32_t* ntokens;
  int page_wgs, each;             // workgroups of blocks; each: one for every token
};

template <typename T> __device__ __forceinline__ uint16_t round16(float v);
template <> __device__ __forceinline__ uint16_t round16<bf16s>(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <> __device__ __forceinline__ uint16_t round16<f16s>(float v) {
  return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// Chunk c (eight elements) of a row rotated by the angles of one position.
template <typename T, bool INTER>
__device__ __forceinline__ u16x8 rotate8(const uint16_t* row, int c, const float* cs,
                                         const float* sn, int rot) {
  const u16x8 x = *reinterpret_cast<const u16x8*>(row + 8 * c);
  if (8 * c >= rot) return x;
  u16x8 r;
  if constexpr (INTER) {
    const float4 cc = *reinterpret_cast<const float4*>(cs + 4 * c);
    const float4 ss = *reinterpret_cast<const float4*>(sn + 4 * c);
    const float co[4] = {cc.x, cc.y, cc.z, cc.w}, si[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = cvt(T{x[2 * i]}), b = cvt(T{x[2 * i + 1]});
      r[2 * i] = round16<T>(a * co[i] - b * si[i]);
      r[2 * i + 1] = round16<T>(b * co[i] + a * si[i]);
    }
  } else {
    // the partner chunk lies rot / 2 elements away; the first half subtracts
    const int hc = rot / 16;
    const bool first = c < hc;
    const u16x8 y = *reinterpret_cast<const u16x8*>(row + 8 * (first ? c + hc : c - hc));
    const int ac = first ? c : c - hc;
    const float4* cp = reinterpret_cast<const float4*>(cs + 8 * ac);
    const float4* sp = reinterpret_cast<const float4*>(sn + 8 * ac);
    const float4 c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
    const float co[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float si[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = first ? -si[i] : si[i];
      r[i] = round16<T>(cvt(T{x[i]}) * co[i] + cvt(T{y[i]}) * s);
    }
  }
  return r;
}

__device__ __forceinline__ void load_bound8(const void* p, size_t o, bool lb, bool bf,
                                            float (&f)[8]) {
  if (lb) {
    const u16x8 x = *reinterpret_cast<const u16x8*>(static_cast<const uint16_t*>(p) + o);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = bf ? cvt(bf16s{x[i]}) : cvt(f16s{x[i]});
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<const float*>(p)[o + i];
  }
}
__device__ __forceinline__ void store_bound8(void* p, size_t o, bool lb, bool bf,
                                             const float (&f)[8]) {
  if (lb) {   // exact: a bound is one of the keys
    u16x8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bf ? round16<bf16s>(f[i]) : round16<f16s>(f[i]);
    *reinterpret_cast<u16x8*>(static_cast<uint16_t*>(p) + o) = x;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) static_cast<float*>(p)[o + i] = f[i];
  }
}

// Rows [s0, s1) of request r, clamped into [0, T].
__device__ __forceinline__ void request_rows(const ExtendArgs& a, int r, int& s0, int& s1) {
  s0 = min(max(a.starts[r], 0), a.t);
  s1 = min(max(a.starts[r + 1], s0), a.t);
}

// Places of blocks before request r's: the host does not know which
// blocks it touches, so there is one for every token, or where that is fewer n / B + 2 of
// its n tokens, rounded so that they add up to T / B + 2 R.
__device__ __forceinline__ int slot_of(const ExtendArgs& a, int r) {
  const int s0 = min(max(a.starts[r], 0), a.t);
  return a.each ? s0 : s0 / a.b + 2 * r;
}

// The block of place `want`: n new tokens of request r from row src on, at offset
// off; n = 0: none.  The workgroup that `counts` for the request's first block
// sets its counts where every touched block has a page for every KV head and every
// new token fits.
struct TouchedBlock { int r, blk, off, first, n; int64_t src; };

__device__ __forceinline__ TouchedBlock touched_block(const ExtendArgs& a, int want, bool counts) {
  const int64_t room = (int64_t)a.nb * a.b;
  TouchedBlock x{};
  x.r = last_at_most(a.requests, want, [&](int i) { return slot_of(a, i); });
  if (x.r < 0) return x;
  int s0, s1;
  request_rows(a, x.r, s0, s1);
  const int p0 = a.positions[x.r], k = want - slot_of(a, x.r);
  const int64_t end = (int64_t)p0 + (s1 - s0), from = max(p0, 0), to = min(end, room);
  if (from >= to || k < 0) return x;
  x.blk = (int)from / a.b + k;
  if (x.blk > (int)(to - 1) / a.b) return x;
  x.first = max(p0, x.blk * a.b);                                   // first new position here
  x.off = x.first - x.blk * a.b;
  x.n = (int)(min(end, ((int64_t)x.blk + 1) * a.b) - x.first);
  x.src = (int64_t)s0 + (x.first - p0);
  if (counts && k == 0) {
    bool ok = p0 >= 0 && end <= room;
    if (ok) {
      const int32_t* row = a.table + (int64_t)x.r * a.hkv * a.nb;
      const int cnt = (int)(end - 1) / a.b - x.blk + 1;
      for (int64_t i = threadIdx.x; i < (int64_t)cnt * a.hkv; i += 256) {
        const int pg = row[(i / cnt) * a.nb + x.blk + i % cnt];
        ok = ok && pg >= 0 && pg < a.pages;
      }
    }
    if (__syncthreads_and(ok) && threadIdx.x == 0) {
      a.nblocks[x.r] = (int)((end + a.b - 1) / a.b);
      if (a.ntokens) a.ntokens[x.r] = (int)end;
    }
  }
  return x;
}

// A block where there is a place for every token, so that it has few: 16 bytes of a
// row per thread and a KV head per D / 8 threads, token after token.  With a workgroup per
// KV head 1024 requests of one token took 39 us, 11 so.
template <typename T, int D, bool INTER>
__device__ __forceinline__ void extend_few(const ExtendArgs& a) {
  constexpr int CPR = D / 8, HP = 256 / CPR;
  const int hgs = (a.hkv + HP - 1) / HP, hg = blockIdx.x % hgs;
  const TouchedBlock x = touched_block(a, blockIdx.x / hgs, hg == 0);
  const int c = threadIdx.x % CPR, kvh = hg * HP + (int)threadIdx.x / CPR;
  if (x.n == 0 || kvh >= a.hkv) return;
  const int page = a.table[((int64_t)x.r * a.hkv + kvh) * a.nb + x.blk];
  if (page < 0 || page >= a.pages) return;
  constexpr bool BF = __is_same(T, bf16s);
  const size_t dst = ((size_t)page * a.b + x.off) * D + 8 * c, bo = (size_t)page * D + 8 * c;
  const uint16_t* kin = a.k + x.src * a.ks + kvh * D;
  const uint16_t* vin = a.v + x.src * a.vs + kvh * D + 8 * c;
  const int half = a.rot / 2;
  float lo[8], hi[8];
  if (x.off) {
    load_bound8(a.lo, bo, a.lb, BF, lo);
    load_bound8(a.hi, bo, a.lb, BF, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = INFINITY;
      hi[i] = -INFINITY;
    }
  }
  for (int t = 0; t < x.n; ++t) {
    const u16x8 v = *reinterpret_cast<const u16x8*>(vin + t * a.vs);
    const int64_t ang = (int64_t)(x.first + t) * half;
    const u16x8 k = rotate8<T, INTER>(kin + t * a.ks, c, a.cos + ang, a.sin + ang, a.rot);
    *reinterpret_cast<u16x8*>(a.vp + dst + (size_t)t * D) = v;
    *reinterpret_cast<u16x8*>(a.kp + dst + (size_t)t * D) = k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = cvt(T{k[i]});
      lo[i] = __builtin_elementwise_minimum(lo[i], f);
      hi[i] = __builtin_elementwise_maximum(hi[i], f);
    }
  }
  store_bound8(a.lo, bo, a.lb, BF, lo);
  store_bound8(a.hi, bo, a.lb, BF, hi);
}

// One KV head of a block: its rows side by side.
template <typename T, int D, bool INTER>
__device__ __forceinline__ void extend_block(const ExtendArgs& a) {
  constexpr int CPR = D / 8;            // 16-byte chunks per row
  constexpr int RP = 256 / CPR;         // rows per pass
  constexpr bool BF = __is_same(T, bf16s);
  __shared__ float s_lo[4][D], s_hi[4][D];
  const int tid = threadIdx.x, kvh = blockIdx.x % a.hkv;
  const TouchedBlock at = touched_block(a, blockIdx.x / a.hkv, kvh == 0);
  const int n = at.n, off = at.off, first = at.first;
  if (n == 0) return;
  const int page = a.table[((int64_t)at.r * a.hkv + kvh) * a.nb + at.blk];
  if (page < 0 || page >= a.pages) return;
  const int c = tid % CPR, g = tid / CPR;
  const size_t dst = ((size_t)page * a.b + off) * D + 8 * c;
  const uint16_t* kin = a.k + at.src * a.ks + kvh * D;
  const uint16_t* vin = a.v + at.src * a.vs + kvh * D + 8 * c;
  const int half = a.rot / 2;
  float lo[8], hi[8], olo[8], ohi[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo[i] = INFINITY;
    hi[i] = -INFINITY;
  }
  const size_t bo = (size_t)page * D + 8 * c;
  if (g == 0 && off) {
    load_bound8(a.lo, bo, a.lb, BF, olo);
    load_bound8(a.hi, bo, a.lb, BF, ohi);
  }
#pragma unroll 2
  for (int t = g; t < n; t += RP) {
    const u16x8 v = *reinterpret_cast<const u16x8*>(vin + t * a.vs);
    const int64_t ang = (int64_t)(first + t) * half;
    const u16x8 k = rotate8<T, INTER>(kin + t * a.ks, c, a.cos + ang, a.sin + ang, a.rot);
    *reinterpret_cast<u16x8*>(a.vp + dst + (size_t)t * D) = v;
    *reinterpret_cast<u16x8*>(a.kp + dst + (size_t)t * D) = k;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = cvt(T{k[i]});
      lo[i] = __builtin_elementwise_minimum(lo[i], f);
      hi[i] = __builtin_elementwise_maximum(hi[i], f);
    }
  }
  if (n > 1) {
    // fold the rows of a wave, then the waves
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int o = CPR; o < STK_WAVE; o <<= 1) {
        lo[i] = __builtin_elementwise_minimum(lo[i], __shfl_xor(lo[i], o));
        hi[i] = __builtin_elementwise_maximum(hi[i], __shfl_xor(hi[i], o));
      }
    }
    if (lane_id() < CPR) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s_lo[wave_id()][8 * c + i] = lo[i];
        s_hi[wave_id()][8 * c + i] = hi[i];
      }
    }
    __syncthreads();
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int w = 1; w < 4; ++w) {
          lo[i] = __builtin_elementwise_minimum(lo[i], s_lo[w][8 * c + i]);
          hi[i] = __builtin_elementwise_maximum(hi[i], s_hi[w][8 * c + i]);
        }
      }
    }
  }
  if (g == 0) {
    if (off) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        lo[i] = __builtin_elementwise_minimum(lo[i], olo[i]);
        hi[i] = __builtin_elementwise_maximum(hi[i], ohi[i]);
      }
    }
    store_bound8(a.lo, bo, a.lb, BF, lo);
    store_bound8(a.hi, bo, a.lb, BF, hi);
  }
}

// One wave: 256 chunks of one token's queries.
constexpr int kQChunks = 256;
template <typename T, int D, bool INTER>
__device__ __forceinline__ void extend_queries(const ExtendArgs& a, int wg) {
  constexpr int CPR = D / 8;
  const int chunks = a.hq * CPR, runs = (chunks + kQChunks - 1) / kQChunks;
  const int64_t x = (int64_t)wg * 4 + wave_id();
  if (x >= (int64_t)a.t * runs) return;
  const int t = (int)(x / runs), c0 = (int)(x % runs) * kQChunks;
  const int r = last_at_most(a.requests, t, [&](int i) { return a.starts[i]; });
  int64_t p = -1;
  if (r >= 0) {
    int s0, s1;
    request_rows(a, r, s0, s1);
    if (t >= s0 && t < s1) p = (int64_t)a.positions[r] + (t - s0);
  }
  const bool ok = p >= 0 && p < a.rows;
  const uint16_t* q = a.q + t * a.qs;
  uint16_t* o = a.qo + (int64_t)t * a.hq * D;
  const int64_t ang = (ok ? p : 0) * (a.rot / 2);
#pragma unroll
  for (int u = 0; u < kQChunks; u += STK_WAVE) {
    const int i = c0 + u + lane_id();
    if (i < chunks) {
      u16x8 y = rotate8<T, INTER>(q + (i / CPR) * D, i % CPR, a.cos + ang, a.sin + ang, a.rot);
      if (!ok) y = u16x8{};
      *reinterpret_cast<u16x8*>(o + 8 * (int64_t)i) = y;
    }
  }
}

template <typename T, int D, bool INTER>
__global__ __launch_bounds__(256) void k_extend(ExtendArgs a) {
  if ((int)blockIdx.x >= a.page_wgs) extend_queries<T, D, INTER>(a, (int)blockIdx.x - a.page_wgs);
  else if (a.each) extend_few<T, D, INTER>(a);
  else extend_block<T, D, INTER>(a);
}

template <typename T, int D>
void launch_extend(const ExtendArgs& a, bool inter, unsigned grid, hipStream_t st) {
  if (inter) hipLaunchKernelGGL((k_extend<T, D, true>), dim3(grid), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_extend<T, D, false>), dim3(grid), dim3(256), 0, st, a);
}

template <typename T>
void launch_extend(const ExtendArgs& a, int d, bool inter, unsigned grid, hipStream_t st) {
  if (d == 64) launch_extend<T, 64>(a, inter, grid, st);
  else if (d == 128) launch_extend<T, 128>(a, inter, grid, st);
  else launch_extend<T, 256>(a, inter, grid, st);
}

}  // namespace stk

using namespace stk;

extern "C" {

STK_API int stk_paged_extend(const void* k_new, int64_t k_stride, const void* v_new,
                             int64_t v_stride, const void* q, int64_t q_stride, void* q_out,
                             int dtype, int tokens, int requests, int hq, int hkv, int nb, int b,
                             int d, int pages, const int32_t* starts, const int32_t* positions,
                             const float* cos, const float* sin, int rows, int rot,
                             int interleaved, void* k_pages, void* v_pages, void* lo_pages,
                             void* hi_pages, int bounds_dtype, const int32_t* block_table,
                             int32_t* nblocks, int32_t* ntokens, void* stream) {
  STK_REQUIRE(dtype == DT_F16 || dtype == DT_BF16, "the cache must be FP16 or BF16");
  STK_REQUIRE(tokens >= 0 && requests > 0 && hkv > 0 && nb > 0 && b > 0 && pages > 0,
              "bad shape");
  STK_REQUIRE(d == 64 || d == 128 || d == 256, "head dimension must be 64, 128 or 256");
  STK_REQUIRE((k_new && v_new) || tokens == 0, "null pointer");
  STK_REQUIRE(k_pages && v_pages && lo_pages && hi_pages && block_table && nblocks && starts &&
                  positions,
              "null pointer");
  STK_REQUIRE(!q || (q_out && hq > 0), "queries need q_out and at least one head");
  STK_REQUIRE(!q || cos, "queries need the rotation's tables");
  STK_REQUIRE((cos != nullptr) == (sin != nullptr), "cos and sin go together");
  STK_REQUIRE((int64_t)nb * b <= 0x7fffffff, "shape too large");
  if (cos) {
    STK_REQUIRE(rot >= 16 && rot <= d && rot % 16 == 0,
                "the rotated width must be a multiple of 16 in [16, D]");
    STK_REQUIRE(rows >= nb * b, "cos and sin need a row for every position of the table");
  } else {
    rot = 0;
  }
  STK_REQUIRE(stk_bounds_ok(dtype, bounds_dtype),
              "lo and hi pages must be FP32 or the pages' 16-bit type");
  STK_REQUIRE(((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new) |
                reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) |
                reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin) |
                reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                reinterpret_cast<uintptr_t>(lo_pages) | reinterpret_cast<uintptr_t>(hi_pages)) &
               15) == 0 && k_stride % 8 == 0 && v_stride % 8 == 0 && (!q || q_stride % 8 == 0),
              "rows must be 16-byte aligned");
  STK_REQUIRE(k_stride >= 0 && v_stride >= 0 && q_stride >= 0, "negative stride");
  STK_REQUIRE(!ntokens || ntokens != positions, "positions must not be the cache's ntokens");
  if (tokens == 0) return STK_OK;
  // a request of n >= 1 tokens touches at most n blocks, and at most (n - 1) / B + 2
  const int64_t few = tokens / b + 2 * (int64_t)requests;
  const bool each = tokens <= few;
  const int heads = 256 / (d / 8);                // KV heads per workgroup of few tokens
  const int64_t touched = each ? (int64_t)tokens * ((hkv + heads - 1) / heads) : few * hkv;
  const int64_t runs = q ? ((int64_t)hq * (d / 8) + kQChunks - 1) / kQChunks : 0;
  const int64_t grid = touched + (tokens * runs + 3) / 4;
  STK_REQUIRE(grid <= 0x7fffffff, "batch too large");
  ExtendArgs a{};
  a.k = static_cast<const uint16_t*>(k_new); a.v = static_cast<const uint16_t*>(v_new);
  a.q = static_cast<const uint16_t*>(q);
  a.ks = k_stride; a.vs = v_stride; a.qs = q_stride;
  a.qo = static_cast<uint16_t*>(q_out);
  a.starts = starts; a.positions = positions;
  a.t = tokens; a.requests = requests; a.hq = hq; a.hkv = hkv; a.nb = nb; a.b = b;
  a.pages = pages;
  a.cos = cos; a.sin = sin; a.rows = rows; a.rot = rot;
  a.kp = static_cast<uint16_t*>(k_pages); a.vp = static_cast<uint16_t*>(v_pages);
  a.lo = lo_pages; a.hi = hi_pages; a.lb = bounds_dtype != 0;
  a.table = block_table; a.nblocks = nblocks; a.ntokens = ntokens;
  a.page_wgs = (int)touched; a.each = each;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) launch_extend<bf16s>(a, d, interleaved != 0, (unsigned)grid, st);
  else launch_extend<f16s>(a, d, interleaved != 0, (unsigned)grid, st);
  return stk_check_launch("k_extend");
}

}  // extern "C"
