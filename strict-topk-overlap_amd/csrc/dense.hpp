// Dense attention over the paged cache: what its kernels share.
//
//   s_ij = cap tanh(scale q_i . k_j / cap) - slope_h |p_i - j|   (no cap: scale q_i . k_j)
//   o_i  = sum_j e^(s_ij) v_j / sum_j e^(s_ij)   over lo_i <= j < hi_i; no such j: o_i = 0
//   lo_i = max(0, first_i, p_i - window + 1)     first, window optional
//   hi_i = max(p_i + 1, min(prefix_r, n_r))      prefix optional
//
// where query token i of request r stands at position p_i and n_r is the
// request's token count.  Causal, windowed, bidirectional-prefix and document
// masks are all one range of keys per query token.
//
// Everything is kept in base 2: scores are multiplied by log2(e) once, and p =
// 2^(s - m) is one hardware exponential.  The running maximum m is only raised
// when a score exceeds it by kLazy: until then p <= 2^kLazy, which neither the
// FP32 sums nor the 16-bit p (whose relative rounding does not depend on its
// size; FP16 reaches 2^16) can tell from p <= 1, and the accumulators need no
// rescaling.
#pragma once

#include "common.hpp"
#include "api.hpp"

namespace stk {

constexpr float kLazy = 8.f;
constexpr int kDenseRows = 128;   // query rows (token, head of the KV group) per tile
constexpr int kDecodeRows = 16;   // query heads per decode item
constexpr int kUnit = 128;        // keys per unit of decode work

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ f32x4 mma16(u16x8 a, u16x8 b, f32x4 c) {
  if constexpr (__is_same(T, bf16s))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ f32x16 mma32(u16x8 a, u16x8 b, f32x16 c) {
  if constexpr (__is_same(T, bf16s))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Four rows of a 16-bit LDS matrix, transposed: within 16 lanes, lane i's
// address names row i / 4, columns 4 (i % 4) .. + 3 of a 4 x 16 block, and it
// receives column i, rows 0 .. 3.
__device__ __forceinline__ u16x4 lds_tr(const uint16_t* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef s16x4 __attribute__((address_space(3))) * lp;
  return __builtin_bit_cast(u16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(p)));
}

template <typename T> __device__ __forceinline__ uint16_t to16(float v) {
  if constexpr (__is_same(T, bf16s)) return __builtin_bit_cast(uint16_t, (__bf16)v);
  else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// -------------------------------------------------------------- arguments

struct DenseArgs {
  const uint16_t* q; int64_t qs;          // [T, Hq, D], elements from token to token
  uint16_t* out;                          // [T, Hq, D]
  const uint16_t* kp; const uint16_t* vp; // [pages, B, D]
  const int32_t* table;                   // [R, Hkv, nb]
  const int32_t* nblocks; const int32_t* ntokens;   // ntokens may be null
  const int32_t* starts;                  // [R + 1], null: one token per request
  int t, requests, hq, hkv, g, nb, b, pages;
  uint64_t bdiv;                          // 2^32 / (B / 16), rounded up past exact
  float c;                                // scale * log2(e)
  float cap_in, cap_out;                  // 2 log2(e) scale / cap, cap * log2(e)
  const float* slopes;                    // [Hq] or null
  int window;                             // 0: none
  const int32_t* prefix;                  // [R] or null
  const int32_t* first;                   // [T] or null
  // requests [groups[i], groups[i + 1]) share their first shared[i] blocks
  const int32_t* groups; const int32_t* shared; int ngroups;
  int fill;                               // rows of no request are written as zeros
};

struct Span { int lo, hi; };              // visible keys

__device__ __forceinline__ int tokens_of(const DenseArgs& a, int r) {
  const int64_t full = (int64_t)min(max(a.nblocks[r], 0), a.nb) * a.b;
  return a.ntokens ? (int)min((int64_t)max(a.ntokens[r], 0), full) : (int)full;
}

// Rows [s0, s1) of request r, clamped into [0, T].
__device__ __forceinline__ void rows_of(const DenseArgs& a, int r, int& s0, int& s1) {
  if (!a.starts) {
    s0 = r;
    s1 = r + 1;
    return;
  }
  s0 = min(max(a.starts[r], 0), a.t);
  s1 = min(max(a.starts[r + 1], s0), a.t);
}

// Keys that a query row of request r sees, at position p of n tokens and with
// its document from `first` on.
__device__ __forceinline__ Span span_at(const DenseArgs& a, int r, int first, int p, int n) {
  Span s;
  s.lo = max(a.window > 0 ? max(0, p - a.window + 1) : 0, first);
  s.hi = min(p + 1, n);
  if (a.prefix) s.hi = max(s.hi, min(a.prefix[r], n));
  return s;
}
__device__ __forceinline__ Span span_of(const DenseArgs& a, int r, int t, int p, int n) {
  return span_at(a, r, a.first ? a.first[t] : 0, p, n);
}

// Shared leading keys of group g.  A request that has fewer reads them itself.
__device__ __forceinline__ int shared_of(const DenseArgs& a, int g) {
  return (int)min((int64_t)min(max(a.shared[g], 0), a.nb) * a.b, (int64_t)0x7ffffff0);
}
// The group that holds request r, or -1: the last one that begins at or before it, found
// in rounds that narrow the range eight times.
__device__ __forceinline__ int group_of(const DenseArgs& a, int r) {
  int lo = 0, n = a.ngroups;
  while (n > 1) {
    const int step = (n + 7) / 8;
    int at[7], c = 0;
#pragma unroll
    for (int j = 0; j < 7; ++j) at[j] = a.groups[lo + min((j + 1) * step, n - 1)];
#pragma unroll
    for (int j = 0; j < 7; ++j) c += (j + 1) * step < n && at[j] <= r;
    lo += c * step;
    n = min(step, n - c * step);
  }
  return r >= a.groups[lo] && r < a.groups[lo + 1] ? lo : -1;
}

// Pool row (page * B + offset) of the 16 keys that start at key, or -1: an
// invalid page or past the table.  key is a multiple of 16, B too.
__device__ __forceinline__ int pool_row(const DenseArgs& a, const int32_t* row, int key) {
  const uint32_t k16 = (uint32_t)key >> 4;
  const int blk = (int)(((uint64_t)k16 * a.bdiv) >> 32);
  const int pg = row[min(blk, a.nb - 1)];
  const bool ok = blk < a.nb && pg >= 0 && pg < a.pages;
  return ok ? pg * a.b + (key - blk * a.b) : -1;
}

// Scores in base 2 without their cap or distance: MODE bit 0 caps, bit 1
// subtracts slope * distance.
template <int MODE>
__device__ __forceinline__ float score2(const DenseArgs& a, float s, float slope, float dist) {
  float x;
  if constexpr (MODE & 1)   // tanh(y) = 1 - 2 / (1 + e^(2y))
    x = a.cap_out - 2.f * a.cap_out *
                        __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * a.cap_in));
  else
    x = s * a.c;
  if constexpr (MODE & 2) x -= slope * __builtin_fabsf(dist);
  return x;
}

// A split item's partial results: rows of (maximum, sum, unnormalised output).
// Workgroup w of the split grid has slot 2w for an item that began before its
// range and slot 2w + 1 for one that begins inside and goes on.
struct Parts {
  float* m; float* l; float* o;
};

// Weight of a part with maximum m among parts with maximum mx.  An empty part
// (-inf) has a zero sum and output, so its weight does not matter; 1 keeps
// the NaN of a part whose scores were all NaN.
__device__ __forceinline__ float part_weight(float m, float mx) {
  return m == mx || m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mx);
}

// Four output values; a row that saw no key (sum 0) is zero.
template <typename T>
__device__ __forceinline__ void store_out(uint16_t* p, f32x4 o, float sum) {
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  u16x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = to16<T>(o[i] * inv);
  *reinterpret_cast<u16x4*>(p) = y;
}

// Work of a split grid: `total` units dealt evenly to its first workgroups (at
// most one per unit, so that none of them is without work), workgroup w taking
// [at(w), at(w + 1)).
struct Deal {
  uint32_t grid, q, rem;
  __device__ __forceinline__ Deal(int total, int launched) {
    grid = (uint32_t)min(total, launched);
    q = (uint32_t)total / grid;
    rem = (uint32_t)total - q * grid;
  }
  __device__ __forceinline__ int at(int w) const { return (int)(w * q + min((uint32_t)w, rem)); }
  __device__ __forceinline__ int wg_of(int u) const {      // the workgroup that holds unit u
    const uint32_t big = rem * (q + 1);
    return (int)((uint32_t)u < big ? (uint32_t)u / (q + 1) : rem + ((uint32_t)u - big) / q);
  }
};

// Row tiles of the attention of many rows (dense_prefill.hpp), listed on the
// device: tile `tile` of sequence `seq` (query rows s0 .. s0 + rows - 1 of a
// request of len tokens) reads units of keys from kstart on, `cum` units come
// before it (per KV head); its rows' keys lie in [klo, khi), and every row sees
// [max_lo, min_hi).
struct Tile { int seq, tile, kstart, cum, klo, khi, max_lo, min_hi, s0, rows, len; };
struct Plan {
  int32_t* head;      // {units per KV head, tiles, workgroups of the units (0: whole tiles)}
  Tile* tiles;
  int32_t* base;      // with groups, instead of a list: [groups + 1] units before each
  int limit;          // most tiles there can be
};

template <int D> constexpr int kTk = D == 256 ? 32 : 64;   // keys per unit

__device__ __forceinline__ int sequences(const DenseArgs& a) {
  return a.groups ? a.ngroups : a.requests;
}
// Query tokens of sequence q: a request's, or (shared blocks) one per request
// of a group.
__device__ __forceinline__ void seq_rows(const DenseArgs& a, int q, int& s0, int& s1) {
  if (a.groups) {
    s0 = min(max(a.groups[q], 0), a.t);
    s1 = min(max(a.groups[q + 1], s0), a.t);
  } else {
    rows_of(a, q, s0, s1);
  }
}
// Span and position of query token t of sequence q with rows [s0, s1).
__device__ __forceinline__ Span seq_span(const DenseArgs& a, int q, int s0, int s1, int t, int& p) {
  if (a.groups) {
    const int n = tokens_of(a, t);
    p = n - 1;
    Span s = span_of(a, t, t, p, n);
    const int keys = shared_of(a, q);
    s.hi = n < keys ? s.lo : min(s.hi, keys);
    return s;
  }
  const int n = tokens_of(a, q);
  p = n - (s1 - s0) + (t - s0);
  return span_of(a, q, t, p, n);
}

__device__ __forceinline__ bool nonfinite16(u16x8 v, uint16_t expo) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) bad |= (v[i] & expo) == expo;
  return bad;
}

// Up to `count` query rows from rown on against the keys [kbase, kend), one row after the
// other: a lane is a key for the scores and D / 64 dims for the output, and
// hidden keys and their values are not read.
template <typename T, int D, int MODE>
__device__ void slow_rows(const DenseArgs& a, int seq, int s0, int s1, int64_t rown,
                          int count, int kvh, const int32_t* row, int kbase, int kend,
                          const Parts* to, int64_t pr) {
  constexpr int E = D / STK_WAVE;
  const int lane = lane_id();
  for (int i = 0; i < count; ++i, ++rown, ++pr) {
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

// dense_*_{bf16,f16}.hip: one element type each
template <typename T>
int launch_decode(int d, int mode, const DenseArgs& a, const Parts& split, int32_t* place, int grid,
                  hipStream_t st);
template <typename T>
int launch_few(int d, int mode, const DenseArgs& a, const Parts& split, int32_t* place, int grid,
               hipStream_t st);
template <typename T>
int launch_prefill(int d, int mode, const DenseArgs& a, const Plan& p, const Parts& split, int grid,
                   hipStream_t st);
template <typename T>
int launch_direct(int d, int mode, const DenseArgs& a, int grid, hipStream_t st);
template <typename T>
int launch_shared(int d, int mode, const DenseArgs& a, const Plan& p, const Parts& psplit,
                  const Parts& pwhole, int pgrid, const Parts& split, const Parts& whole,
                  int32_t* place, int grid, hipStream_t st);

}  // namespace stk
