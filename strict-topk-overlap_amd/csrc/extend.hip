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
// One workgroup owns one (request, KV head, touched block): it writes the
// block's new K and V rows and folds the rotated keys, as stored, into the
// page's lo/hi, so the bounds need no atomics and do not depend on an order.
// A block whose first new token has offset 0 starts its bounds over.  The
// other workgroups rotate the queries, one wave per run of 16-byte chunks of one
// token.  The host knows neither the lengths nor the positions (they stay on
// the device, so a captured graph follows them): the grid covers the most
// blocks that T tokens of R requests can touch, each workgroup finds its block by
// a prefix sum over the requests, and those past the last one leave.
//
// Bound by HBM: every new row is read once and written once.  8191 tokens of
// 32 + 16 heads, D = 128, FP16: 204 MB in 35 us, 5.8 TB/s with the inputs in the
// Infinity Cache and 44 us without; one token each of 128 requests: 5.9 us, the chain
// of the counts, the table and the bounds.
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
  int page_wgs;
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

template <typename T, int D, bool INTER>
__device__ __forceinline__ void extend_block(const ExtendArgs& a) {
  constexpr int CPR = D / 8;            // 16-byte chunks per row
  constexpr int RP = 256 / CPR;         // rows per pass
  constexpr bool BF = __is_same(T, bf16s);
  __shared__ int s_tmp[4], s_hit[5];
  __shared__ float s_lo[4][D], s_hi[4][D];
  const int tid = threadIdx.x, kvh = blockIdx.x % a.hkv, want = blockIdx.x / a.hkv;
  const int64_t room = (int64_t)a.nb * a.b;
  // this workgroup's request and block
  int base = 0;
  if (tid == 0) s_hit[0] = -1;
  for (int r0 = 0; r0 < a.requests; r0 += 256) {
    const int r = r0 + tid;
    int cnt = 0, s0 = 0, s1 = 0, b0 = 0, p0 = 0;
    if (r < a.requests) {
      request_rows(a, r, s0, s1);
      p0 = a.positions[r];
      const int64_t lo = max(p0, 0), hi = min((int64_t)p0 + (s1 - s0), room);
      if (lo < hi) {
        b0 = (int)lo / a.b;
        cnt = (int)(hi - 1) / a.b - b0 + 1;
      }
    }
    int total;
    __syncthreads();
    const int before = base + block_excl_scan1(cnt, s_tmp, &total);
    if (want >= before && want < before + cnt) {
      s_hit[0] = r;
      s_hit[1] = s0;
      s_hit[2] = s1;
      s_hit[3] = b0 + (want - before);
      s_hit[4] = p0;
    }
    base += total;
    __syncthreads();
    if (want < base) break;
  }
  const int r = s_hit[0];
  if (r < 0) return;
  const int s0 = s_hit[1], s1 = s_hit[2], blk = s_hit[3], p0 = s_hit[4];
  const int first = max(p0, blk * a.b);                             // first new position here
  const int off = first - blk * a.b;
  const int n = (int)(min((int64_t)p0 + (s1 - s0), ((int64_t)blk + 1) * a.b) - first);
  const int32_t* row = a.table + ((int64_t)r * a.hkv + kvh) * a.nb;
  // the counts follow when every touched block has a page for every KV head
  // and every new token fits
  if (kvh == 0 && blk == max(p0, 0) / a.b) {
    const int64_t end = (int64_t)p0 + (s1 - s0);
    bool ok = p0 >= 0 && end <= room;
    if (ok) {
      const int cnt = (int)(end - 1) / a.b - blk + 1;
      for (int64_t x = tid; x < (int64_t)cnt * a.hkv; x += 256) {
        const int pg = row[(x / cnt) * a.nb + blk + x % cnt];
        ok = ok && pg >= 0 && pg < a.pages;
      }
    }
    if (__syncthreads_and(ok) && tid == 0) {
      a.nblocks[r] = (int)((end + a.b - 1) / a.b);
      if (a.ntokens) a.ntokens[r] = (int)end;
    }
  }
  const int page = row[blk];
  if (page < 0 || page >= a.pages) return;
  const int c = tid % CPR, g = tid / CPR;
  const int64_t src = (int64_t)s0 + (first - p0);                   // row of the first token here
  const size_t dst = ((size_t)page * a.b + off) * D + 8 * c;
  const uint16_t* kin = a.k + src * a.ks + kvh * D;
  const uint16_t* vin = a.v + src * a.vs + kvh * D + 8 * c;
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
  // the requests that end at or before row t come before its own
  int r = 0;
  for (int r0 = 0; r0 < a.requests; r0 += STK_WAVE) {
    const int i = r0 + lane_id();
    const int e = a.starts[min(i, a.requests - 1) + 1];
    r += __popcll(__ballot(i < a.requests && e <= t));
  }
  int64_t p = -1;
  if (r < a.requests) {
    const int s0 = a.starts[r];
    if (s0 <= t) p = (int64_t)a.positions[r] + (t - s0);
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
  if ((int)blockIdx.x < a.page_wgs) extend_block<T, D, INTER>(a);
  else extend_queries<T, D, INTER>(a, (int)blockIdx.x - a.page_wgs);
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
  // blocks that T tokens of R requests can touch: a request of n >= 1 tokens
  // touches at most n, and at most (n - 1) / B + 2
  const int64_t some = requests < tokens ? requests : tokens;
  const int64_t touched = tokens / b + 2 * some < tokens ? tokens / b + 2 * some : tokens;
  const int64_t runs = q ? ((int64_t)hq * (d / 8) + kQChunks - 1) / kQChunks : 0;
  const int64_t grid = touched * hkv + (tokens * runs + 3) / 4;
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
  a.page_wgs = (int)(touched * hkv);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_BF16) launch_extend<bf16s>(a, d, interleaved != 0, (unsigned)grid, st);
  else launch_extend<f16s>(a, d, interleaved != 0, (unsigned)grid, st);
  return stk_check_launch("k_extend");
}

}  // extern "C"
