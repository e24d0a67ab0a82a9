// Attention over the paged 8-bit cache: the kernels, compiled once for each type
// of queries and each view of theirs (k_kv_attn_*.hip, k_kv_window_*.hip, k_kv_tree_*.hip).
#pragma once
#include "gn_kv.h"

namespace gn {
namespace {

// ---------------------------------------------------------------- attention
// O = softmax(scale Q K^T) V in one pass over the keys with a running maximum and
// sum per row.  A row is a (token, query head) pair; the rows of the query heads
// that share a key head lie together, so that a key is read once for all.
//
// Both products run on bf16 MFMAs (16x16x32), transposed: S^T = K Q^T and O^T =
// V^T P^T.  E4M3 values times a power of two are bf16 numbers, exactly.  The 64
// keys of a step are dealt to the four 16-row tiles of K so that a lane's sixteen
// scores belong to sixteen keys in a row of its group of 16: the operand P^T
// of the second product then is the first one's result in place, and V^T's operand
// 16 consecutive bytes of a row of the transposed cache.  P and O pass through
// registers only, for single tokens K and V too; a row's maximum and sum live in its
// four lanes.
//
// float32 queries are cut into three bf16 numbers (8 bits each, nothing lost), and
// so are the weights: three products each, as exact as float32's.  bfloat16
// queries take one and their weights are cut into two (16 bits: off by less than 2^-15
// of themselves), so that an output's error is its own rounding's.  Weights of one
// number would take 241 us where two take 307 (the prompts below), with an error
// against 64 bits of 0.0023 where rounding alone makes 0.0017.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }
// eight E4M3 bytes times a power of two
__device__ __forceinline__ bf16x8 from_e4m3(uint32_t lo, uint32_t hi, float scale) {
  u32x4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  return as_bf16x8(r);
}
__device__ __forceinline__ uint32_t pack_high(float lo, float hi) {  // the upper halves of two float32
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
// PARTS bf16 numbers that sum to each of eight float32: rounded (1), or cut at 8
// bits, the rest cut again (2, 3)
template <int PARTS>
__device__ __forceinline__ void to_parts(const float (&v)[8], bf16x8 (&o)[PARTS]) {
  if constexpr (PARTS == 1) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (__bf16)v[i];
    o[0] = r;
  } else {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v[i];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      u32x4 r;
      r.x = pack_high(x[0], x[1]);
      r.y = pack_high(x[2], x[3]);
      r.z = pack_high(x[4], x[5]);
      r.w = pack_high(x[6], x[7]);
      o[p] = as_bf16x8(r);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] -= __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u);
    }
  }
}
// any byte of four equal to NaN (0x7f or 0xff)
__device__ __forceinline__ bool has_nan(uint32_t w) {
  const uint32_t x = ~w & 0x7f7f7f7fu;  // a zero byte where NaN
  return ((x - 0x01010101u) & ~x & 0x80808080u) != 0;
}

constexpr float LOG2E = 1.4426950408889634f;
// a row's reference maximum moves only when a score passes it by this many powers
// of two: weights stay below 2^8 and outputs are rarely rescaled
constexpr float SLACK = 8.f;
// scores to powers of two; a scale of 0 is in the queries
__device__ __forceinline__ float kv_factor(float scale) { return scale == 0.f ? 1.f : fabsf(scale) * LOG2E; }

template <int V>
struct Int {
  static constexpr int value = V;
};

// The first n of 16 bits.
__device__ __forceinline__ uint32_t first_bits(int n) { return (1u << min(max(n, 0), 16)) - 1u; }

// The keys that the rows row0 .. last of a sequence see, walked without what lies between
// a window and the first tokens: the i-th of them is key i, from `at` on (a whole step of
// 64 and so a start of the walk's steps) key i + gap.
struct Span {
  int at, gap, end;  // end: how many
  template <int VIEW>
  __device__ __forceinline__ int key(int i) const {
    return VIEW == KV_WINDOW && i >= at ? i + gap : i;
  }
};
template <int VIEW>
__device__ __forceinline__ Span kv_span(const KvAttnArgs &a, const Seq &s, int row0, int last) {
  Span p{0, 0, s.len + s.n};
  if constexpr (VIEW == KV_PREFIX) {
    if (a.causal) p.end = s.len + last / a.G + 1;
  } else if constexpr (VIEW == KV_WINDOW) {
    const int near = max(s.len + row0 / a.G - a.window + 1, 0) & ~63;
    p.at = (min(a.sinks, near) + 63) & ~63;
    p.gap = near - p.at;
    p.end = s.len + last / a.G + 1 - p.gap;
  }
  return p;
}

// The work of one workgroup: a sequence's tile of rows of one key head, over one
// split of its keys.
struct Work {
  Seq s;
  Span span;
  int b, kvh, split;
  int total, rows, row0;  // keys of the sequence, its rows, the workgroup's first
  int end, k0, k1;        // what its rows see, the split's part of it
  bool any;
};
template <int VIEW>
__device__ __forceinline__ Work kv_work(const KvAttnArgs &a, const KvPlan &pl) {
  const KvArgs &c = a.c;
  Work x;
  int id = blockIdx.x;  // heads fastest: with 8 of them a head's tiles share an XCD's L2
  x.kvh = id % c.KVH;
  id /= c.KVH;
  int tile;
  if (VIEW != KV_PREFIX && !pl.by_rows) {  // tiles of a split together: they read the same keys
    tile = id % pl.tiles;
    id /= pl.tiles;
    x.split = id % pl.splits;
    x.b = id / pl.splits;
  } else {
    x.split = id % pl.splits;
    id /= pl.splits;
    tile = pl.tiles - 1 - id % pl.tiles;  // the rows that see most first
    x.b = id / pl.tiles;
  }
  x.s = kv_seq(c, x.b, c.limit);
  if (x.s.bad && c.bad && threadIdx.x == 0) c.bad[x.b] = 1;
  x.total = x.s.len + x.s.n;
  x.rows = x.s.n * a.G;
  x.row0 = tile * pl.rows_wg;
  const int last = max(min(x.rows, x.row0 + pl.rows_wg) - 1, 0);
  x.span = kv_span<VIEW>(a, x.s, min(x.row0, last), last);
  x.end = x.span.end;
  x.k0 = x.split * pl.chunk;
  x.k1 = x.end - x.k0 < pl.chunk ? x.end : x.k0 + pl.chunk;  // the sum alone could pass 32 bits
  x.any = x.row0 < x.rows && (x.split == 0 || x.k0 < x.end);
  return x;
}

// The first key of any of the workgroup's windows; without a window, behind all keys.
template <int VIEW>
__device__ __forceinline__ int kv_reach(const KvAttnArgs &a, const Work &x) {
  if constexpr (VIEW != KV_WINDOW) return 0;
  return a.window > 0 ? x.s.len + x.row0 / a.G - a.window + 1 : 0x7fffffff;
}

// A wave's 16 RT rows.  Lane n + 16 g holds, for row n of a tile: the queries'
// columns of its k slots, sixteen keys' scores of a step, and columns 4 g + i of
// each 16 of the output.
template <typename T, int R, int RT, int VIEW>
struct Rows {
  // bf16 numbers that a query and a weight are cut into
  static constexpr int PARTS = sizeof(T) == 4 ? 3 : 1, WPARTS = sizeof(T) == 4 ? 3 : 2;
  static constexpr int NK = R / 32, ND = R / 16;
  bf16x8 q[RT][NK][PARTS];
  f32x4 O[RT][ND], L[RT];  // outputs; sums, as a product with ones (four equal rows)
  float m[RT];             // the reference maxima, in powers of two
  int lim[RT], lo_lim;     // the last key of each row (KV_TREE: its token's number), that all rows see
  int hi_low;              // KV_WINDOW: the first key of the last row's window
  bool seen[RT], every;    // whether a masked step, or any other, held a key of the row

  // col(k): the first of this lane's eight columns in the k-th product
  template <typename F>
  __device__ __forceinline__ void init(const KvAttnArgs &a, const Work &x, int row0, int n, F col) {
    // maxima are taken before the factor, which is above 0
    const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;
    lo_lim = x.total - 1;
    hi_low = 0;
    every = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = row0 + r * 16 + n;
      const bool on = row < x.rows;
      const int t = on ? row / a.G : 0;
      lim[r] = VIEW == KV_TREE ? t : on && (VIEW == KV_WINDOW || a.causal) ? x.s.len + t : x.total - 1;
      lo_lim = VIEW == KV_TREE ? x.s.len - 1 : min(lo_lim, lim[r]);
      if (VIEW == KV_WINDOW && on) hi_low = max(hi_low, lim[r] - a.window + 1);
      const T *p = (const T *)a.q + (int64_t)(x.s.start + t) * a.qs + (int64_t)(x.kvh * a.G + (on ? row % a.G : 0)) * a.c.hd;
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const int d0 = col(k);
        float v[8];
        if (a.vec) {  // whole eights of columns
          float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
          if (on && d0 < a.c.hd) {
            Elem<T>::get4(p + d0, lo);
            Elem<T>::get4(p + d0 + 4, hi);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = (i < 4 ? lo[i & 3] : hi[i & 3]) * sign;
        } else {
          for (int i = 0; i < 8; ++i) v[i] = on && d0 + i < a.c.hd ? Elem<T>::get(p + d0 + i) * sign : 0.f;
        }
        to_parts<PARTS>(v, q[r][k]);
      }
      m[r] = -INFINITY;
      L[r] = f32x4{0.f, 0.f, 0.f, 0.f};
      seen[r] = false;
#pragma unroll
      for (int d = 0; d < ND; ++d) O[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if constexpr (VIEW != KV_TREE)
      for (int o = 8; o > 0; o >>= 1) lo_lim = min(lo_lim, __shfl_xor(lo_lim, o, 64));
    lo_lim = __builtin_amdgcn_readfirstlane(lo_lim);
    if constexpr (VIEW == KV_WINDOW) {
      for (int o = 8; o > 0; o >>= 1) hi_low = max(hi_low, __shfl_xor(hi_low, o, 64));
      hi_low = __builtin_amdgcn_readfirstlane(hi_low);
    }
  }
  // whether every row sees the 64 keys from j on
  __device__ __forceinline__ bool clear(const KvAttnArgs &a, int j) const {
    return j + 63 <= lo_lim && (VIEW != KV_WINDOW || j >= hi_low || j + 63 < a.sinks);
  }
  // Which of the sixteen keys from `first` on row r sees: how many (KV_PREFIX), else a
  // bit each.
  static constexpr int ALL = VIEW == KV_PREFIX ? 16 : 0xffff;
  __device__ __forceinline__ int sees(const KvAttnArgs &a, const Work &x, int r, int first) const {
    if constexpr (VIEW == KV_PREFIX) return max(0, min(16, lim[r] - first + 1));
    if constexpr (VIEW == KV_WINDOW)
      return (int)(first_bits(lim[r] - first + 1) &
                   (~first_bits(max(lim[r] - a.window + 1, 0) - first) | first_bits(a.sinks - first)));
    const int at = first - x.s.len;  // the number of the first as a new token
    const uint32_t *bits = a.mask + (int64_t)(x.s.start + lim[r]) * a.ms;
    uint32_t w = first_bits(-at);
    if (at > -16 && at < x.s.n) {
      const int i = max(at, 0) >> 5;
      const uint32_t lo = bits[i], hi = i * 32 + 32 < x.s.n ? bits[i + 1] : 0;
      w |= at < 0 ? lo << -at : (uint32_t)((((uint64_t)hi << 32) | lo) >> (at & 31));
    }
    return (int)(w & first_bits(x.total - first));
  }
  static __device__ __forceinline__ bool in_sight(int see, int k) { return VIEW == KV_PREFIX ? k < see : see >> k & 1; }

  // the lane's sixteen keys that the row does not see leave the scores
  __device__ __forceinline__ void mask(int r, f32x4 (&S)[4], int see) {
    asm volatile("" : "+v"(see));  // keeps the comparisons out of steps without a mask
    seen[r] |= see > 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) S[k >> 2][k & 3] = in_sight(see, k) ? S[k >> 2][k & 3] : -INFINITY;
  }
  // scores S (before the factor sf > 0) of tile r to weights, as the second
  // product's operands
  __device__ __forceinline__ void weights(int r, const f32x4 (&S)[4], float sf, bf16x8 (&p)[2][WPARTS]) {
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < 16; ++k) mx = fmaxf(mx, S[k >> 2][k & 3]);
    mx *= sf;
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const bool grow = mx > m[r] + SLACK;  // also the first score, over -inf
    if (__any(grow)) {
      const float mn = grow ? mx : m[r];
      const float f = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - mn);
      L[r] *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d) O[r][d] *= f;
      m[r] = mn;
    }
    const float sub = m[r] == -INFINITY ? 0.f : -m[r];
    const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * h + (i >> 2)][i & 3], sf, sub));
      to_parts<WPARTS>(v, p[h]);
#pragma unroll
      for (int i = 0; i < WPARTS; ++i)
        L[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(ones), p[h][i], L[r], 0, 0, 0);
    }
  }

  // A masked weight is 0 but 0 * NaN is not: where V holds NaN (is: ones in their
  // place, taken out of V by the caller), the rows that see it find it by a product
  // of ones.  NaN for those, else 0.
  __device__ __forceinline__ f32x4 not_numbers(const bf16x8 (&is)[2], int see) const {
    f32x4 hit = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 on;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        on[k] = (in_sight(see, 8 * h + 2 * k) ? 0x3f80u : 0u) | (in_sight(see, 8 * h + 2 * k + 1) ? 0x3f800000u : 0u);
      hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(is[h], as_bf16x8(on), hit, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) hit[i] = hit[i] > 0.f ? __uint_as_float(0x7fc00000u) : 0.f;
    return hit;
  }

  __device__ __forceinline__ void scores(const bf16x8 &k, int step, int r, f32x4 &S) const {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[r][step][p], S, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 product(const bf16x8 &v, const bf16x8 (&p)[WPARTS], f32x4 o) {
#pragma unroll
    for (int i = 0; i < WPARTS; ++i) o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[i], o, 0, 0, 0);
    return o;
  }

  __device__ __forceinline__ void finish() {  // whether any of a row's four lanes saw a key
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int any = (int)seen[r] | __shfl_xor((int)seen[r], 16, 64);
      seen[r] = every || (any | __shfl_xor(any, 32, 64));
    }
  }

  // to the output, or to the split's place in the workspace.  No key at all: 0; keys
  // whose scores are all -inf: no number, as 0 / 0 says.
  __device__ __forceinline__ void store(const KvAttnArgs &a, const KvPlan &pl, const Work &x, int row0, int n, int g) {
    const KvArgs &c = a.c;
    const bool alone = x.end <= pl.chunk;  // no other split of these rows
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = row0 + r * 16 + n;
      if (row >= x.rows) continue;
      const int t = row / a.G, h = x.kvh * a.G + row % a.G;
      const float l = L[r][0];
      if (alone) {
        T *out = (T *)a.out + (int64_t)(x.s.start + t) * a.os + (int64_t)h * c.hd;
        const float inv = 1.f / l;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const int col = d * 16 + 4 * g;
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = seen[r] ? O[r][d][i] * inv : 0.f;
          if (a.vec) {
            if (col < c.hd) Elem<T>::put4(out + col, v);
          } else {
            for (int i = 0; i < 4; ++i)
              if (col + i < c.hd) Elem<T>::put(out + col + i, v[i]);
          }
        }
      } else {
        const int64_t slot = ((int64_t)x.b * c.max_new + t) * a.H + h, slots = (int64_t)c.B * c.max_new * a.H;
        float *ml = a.work + (x.split * slots + slot) * 2;
        if (g == 0) {
          ml[0] = m[r];
          ml[1] = seen[r] && m[r] == -INFINITY ? __uint_as_float(0x7fc00000u) : l;
        }
        float *part = a.work + kv_part_at(pl.splits, slots) + (x.split * slots + slot) * R;
#pragma unroll
        for (int d = 0; d < ND; ++d)
          *reinterpret_cast<float4 *>(part + d * 16 + 4 * g) = make_float4(O[r][d][0], O[r][d][1], O[r][d][2], O[r][d][3]);
      }
    }
  }
};

// ---- prompts ---------------------------------------------------------------
// A chunk of 16 bytes in a row of R bf16 numbers of K, moved so that 16 rows' same
// chunk lies in different banks.
template <int R>
__device__ __forceinline__ int k_place(int row, int chunk) {
  constexpr int N = R / 8;
  const int turn = R == 256 ? row & 15 : R == 128 ? row & 15 : R == 96 ? (row >> 2) & 3 : R == 32 ? (row >> 2) & 3 : (row >> 1) & 7;
  if constexpr ((N & (N - 1)) == 0) return chunk ^ turn;
  const int at = chunk + turn;
  return at >= N ? at - N : at;
}
// a row of 64 keys of V: chunk 4 h + g, which the read's lanes (n, g) take in quarters
// of 16 lanes that mix two g
__device__ __forceinline__ int v_place(int row, int chunk) { return chunk ^ ((row >> 1) & 7); }

// The four waves take 16 RT rows each and walk the keys together, 64 a step.  A
// step's K and V bytes are loaded a step ahead, turned into bf16 once for all
// waves (scales included, keys behind the sequence 0) and read as operands from
// LDS; two steps' operands lie there, so one barrier a step is enough.
// Bound by the matrix units and what feeds them: two prompts of 2048 tokens behind
// 2048, 32 heads of 128 over 8, bfloat16, in 307 us, 206 GFLOP at 672 TFLOP/s of the
// definition's products and, the weights' second part among them, 1007 of the units' (a
// product of 16384^3 reaches 1369 here); the waves wait for LDS and the barrier.
// Windows of 1024 of the same prompts: 136 us, 69 GFLOP in 19 steps a workgroup, two of them
// masked and one for four first tokens; the vector units are busy 52 % of the time, the
// matrix units 37 %.  Trees of up to 64 tokens of 16 sequences of up to 8000: 122 us and
// 19 for the join, 3.3 us a step whether one or two workgroups share a CU.
template <typename T, int R, int RT, int VIEW>
__global__ __launch_bounds__(256, R <= 128 ? 2 : 1) void kv_attn_rows_kernel(KvAttnArgs a, KvPlan pl) {
  constexpr int NK = R / 32, ND = R / 16;
  extern __shared__ __align__(16) uint8_t lds[];
  const KvArgs &c = a.c;
  const Work x = kv_work<VIEW>(a, pl);
  if (!x.any) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = lane & 15, g = lane >> 4;
  const int row0 = x.row0 + w * 16 * RT;
  // the last key that this wave's rows see
  const int my_last = min(x.rows, row0 + 16 * RT) - 1;
  const int my_end = row0 >= x.rows                                       ? 0
                     : VIEW == KV_WINDOW || (VIEW == KV_PREFIX && a.causal) ? x.s.len + my_last / a.G + 1
                                                                            : x.total;
  // where this wave's windows begin
  const int my_low = VIEW == KV_WINDOW ? x.s.len + row0 / a.G - a.window + 1 : 0;
  const float sf = kv_factor(a.scale);
  Rows<T, R, RT, VIEW> A;
  A.init(a, x, row0, n, [&](int k) { return k * 32 + g * 8; });

  const int32_t *table = c.table + (int64_t)x.b * c.max_pages;
  const int last_page = (x.total - 1) >> c.lgP;
  const int64_t page_bytes = (int64_t)c.KVH * c.P * R;
  const uint8_t *kb = c.k + (int64_t)x.kvh * c.P * R, *vb = c.v + (int64_t)x.kvh * c.P * R;
  // the page of 16 keys from j on, clamped to the sequence's last
  const auto page_at = [&](int j) { return table[min(j >> c.lgP, last_page)]; };

  // This thread's part of a step: chunks of 16 bytes of K (row t * 16 + n: key 16 (n
  // >> 2) + 4 t + (n & 3), as the scores' layout asks) and of V (row: a column,
  // chunk gv: 16 keys).
  constexpr int CH = 64 * R / 16, NL = (CH + 255) / 256, KC = R / 16;
  constexpr bool SAME = 256 % (16 * KC) == 0;  // all its K chunks are of one group of 16 keys
  uint4 kr[NL], vr[NL];
  float ksc[NL], vsc;
  int pk[NL], pv = 0, have = 0;  // pages of the next step's chunks; V keys of this one's
  uint64_t there = 0;            // lanes whose V page is there: lane g speaks for group g
  const auto in = [&](int q) { return CH % 256 == 0 || q < CH; };
  const auto chunk = [&](int i) { return in(tid + i * 256) ? tid + i * 256 : 0; };
  const int gv = tid & 3;
  // whether some row may see one of the 16 keys from j on: pages that none does need not be
  // there, nor hold a scale
  const int reach = kv_reach<VIEW>(a, x);
  const auto in_reach = [&](int j) { return VIEW != KV_WINDOW || j + 15 >= reach || j < a.sinks; };
  const auto pages = [&](int j) {
#pragma unroll
    for (int i = 0; i < NL; ++i) pk[i] = SAME && i ? pk[0] : page_at(j + ((chunk(i) / KC & 15) >> 2) * 16);
    pv = page_at(j + gv * 16);
  };
  const auto load = [&](int j, int next) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int q = chunk(i), row = q / KC, tok = ((row & 15) >> 2) * 16 + (row >> 4) * 4 + (row & 3);
      const bool on = (unsigned)pk[i] < (unsigned)c.pages;
      const int p = on ? pk[i] : 0;
      kr[i] = *reinterpret_cast<const uint4 *>(kb + p * page_bytes + ((j + tok) & (c.P - 1)) * R + q % KC * 16);
      if (!(SAME && i)) ksc[i] = c.ks[(int64_t)p * c.KVH + x.kvh];
      ksc[i] = SAME && i ? ksc[0] : on ? ksc[i] : 1.f;
    }
    const bool near = in_reach(j + gv * 16), on = near && (unsigned)pv < (unsigned)c.pages;
    const int p = on ? pv : 0;
    const uint8_t *v = vb + p * page_bytes + ((j + gv * 16) & (c.P - 1));
#pragma unroll
    for (int i = 0; i < NL; ++i) vr[i] = *reinterpret_cast<const uint4 *>(v + (chunk(i) >> 2) * c.P);
    vsc = c.vs[(int64_t)p * c.KVH + x.kvh];
    vsc = on ? vsc : 1.f;
    have = on ? x.total - (j + gv * 16) : 0;
    there = __ballot(on);
    if (!on && j + gv * 16 < x.total && near && c.bad) c.bad[x.b] = 1;
    pages(next);
  };
  // the first key that some row of the workgroup does not see
  const int wg_lim = VIEW == KV_TREE ? x.s.len : VIEW == KV_WINDOW || a.causal ? x.s.len + x.row0 / a.G + 1 : x.total;
  // the first that all windows hold
  const int wg_low = VIEW == KV_WINDOW ? x.s.len + (min(x.rows, x.row0 + pl.rows_wg) - 1) / a.G - a.window + 1 : 0;
  const auto masked = [&](int j) { return j + 64 > wg_lim || (VIEW == KV_WINDOW && j < wg_low && j + 63 >= a.sinks); };
  int *first_nan = reinterpret_cast<int *>(lds + 512 * R);  // KV_PREFIX
  // other views: a bit for each of a step's 64 keys that holds NaN in a column, for two
  // steps; the step (key + 1) whose bits hold any
  uint16_t *nan_bits = reinterpret_cast<uint16_t *>(lds + 512 * R);
  int *nan_step = reinterpret_cast<int *>(lds + 528 * R);
  const auto spread = [&](int buf, int j) {
    uint8_t *kl = lds + buf * (256 * R), *vl = kl + 128 * R;
    if (have < 16) {  // keys behind the sequence, or of a page that is not there: 0
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        uint32_t *v = reinterpret_cast<uint32_t *>(&vr[i]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int h = min(max(have - 4 * k, 0), 4);
          v[k] &= h == 4 ? ~0u : (1u << (8 * h)) - 1u;
        }
      }
    }
    if (masked(j)) {
      // masked weights are 0, but 0 * NaN is not: NaN leaves V, and the first key that
      // has it in a column is noted (a row sees it if it sees that key), or every one
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        uint32_t *v = reinterpret_cast<uint32_t *>(&vr[i]);
        const bool any = has_nan(v[0]) || has_nan(v[1]) || has_nan(v[2]) || has_nan(v[3]);
        if (VIEW != KV_PREFIX && in(tid + i * 256)) nan_bits[(buf * R + (chunk(i) >> 2)) * 4 + gv] = 0;
        if (!any) continue;
        uint32_t found = 0;
        for (int k = 15; k >= 0; --k) {
          const int at = k >> 2, sh = 8 * (k & 3);
          const uint32_t word = at == 0 ? v[0] : at == 1 ? v[1] : at == 2 ? v[2] : v[3];
          if ((word >> sh & 0x7f) == 0x7f) {
            if constexpr (VIEW == KV_PREFIX) atomicMin(&first_nan[chunk(i) >> 2], j + gv * 16 + k);
            else found |= 1u << k;
          }
        }
        if (VIEW != KV_PREFIX && in(tid + i * 256)) {
          nan_bits[(buf * R + (chunk(i) >> 2)) * 4 + gv] = (uint16_t)found;
          nan_step[buf] = j + 1;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t drop = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) drop |= (v[k] >> (8 * e) & 0x7f) == 0x7f ? 0xffu << (8 * e) : 0u;
          v[k] &= ~drop;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int q = tid + i * 256;
      if (!in(q)) continue;
      const int krow = q / KC, kc = q % KC * 2, vrow = q >> 2;
      *reinterpret_cast<bf16x8 *>(kl + krow * 2 * R + k_place<R>(krow, kc) * 16) = from_e4m3(kr[i].x, kr[i].y, ksc[i]);
      *reinterpret_cast<bf16x8 *>(kl + krow * 2 * R + k_place<R>(krow, kc + 1) * 16) = from_e4m3(kr[i].z, kr[i].w, ksc[i]);
      *reinterpret_cast<bf16x8 *>(vl + vrow * 128 + v_place(vrow, gv) * 16) = from_e4m3(vr[i].x, vr[i].y, vsc);
      *reinterpret_cast<bf16x8 *>(vl + vrow * 128 + v_place(vrow, 4 + gv) * 16) = from_e4m3(vr[i].z, vr[i].w, vsc);
    }
  };

  int buf = 0;
  uint64_t groups = 0;  // of this step: whether each group's page is there
  const auto step = [&](int j) {
    const uint8_t *kl = lds + buf * (256 * R), *vl = kl + 128 * R;
    const auto k_at = [&](int t, int k) {
      const int row = t * 16 + n;
      return *reinterpret_cast<const bf16x8 *>(kl + row * 2 * R + k_place<R>(row, k * 4 + g) * 16);
    };
    const auto v_at = [&](int d, int h) {
      const int row = d * 16 + n;
      return *reinterpret_cast<const bf16x8 *>(vl + row * 128 + v_place(row, 4 * h + g) * 16);
    };
    if constexpr (VIEW != KV_PREFIX) {
      if (nan_step[buf] == j + 1) {  // NaN that left V, for the rows that see it: rare, and few registers
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int see = groups >> g & 1 ? A.sees(a, x, r, j + 16 * g) : 0;
          uint64_t row = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) row |= (uint64_t)(uint32_t)__shfl(see, n + 16 * k, 64) << (16 * k);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (reinterpret_cast<const uint64_t *>(nan_bits)[buf * R + d * 16 + 4 * g + i] & row)
                A.O[r][d][i] = __uint_as_float(0x7fc00000u);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
    // operands are read one tile ahead of their products
    f32x4 S[RT][4];
    bf16x8 kf[2][NK];
#pragma unroll
    for (int k = 0; k < NK; ++k) kf[0][k] = k_at(0, k);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t < 3) {
#pragma unroll
        for (int k = 0; k < NK; ++k) kf[(t + 1) & 1][k] = k_at(t + 1, k);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) S[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int r = 0; r < RT; ++r) A.scores(kf[t & 1][k], k, r, S[r][t]);
      __builtin_amdgcn_sched_barrier(0);  // else all tiles' reads move up and registers run out
    }
    // The wave that weighs goes before the SIMD's other, whose products can wait for the
    // matrix unit: a window of 8192 of two prompts of 2048 tokens 843 -> 805 us, of 1024 139
    // -> 136.
    if constexpr (VIEW != KV_PREFIX) __builtin_amdgcn_s_setprio(1);
    constexpr int AHEAD = 2;
    bf16x8 vf[AHEAD + 1][2];
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
      vf[d][0] = v_at(d, 0);
      vf[d][1] = v_at(d, 1);
    }
    if (!A.clear(a, j) || groups != 15) {
#pragma unroll
      for (int r = 0; r < RT; ++r) A.mask(r, S[r], groups >> g & 1 ? A.sees(a, x, r, j + 16 * g) : 0);
    } else {
      A.every = true;
    }
    bf16x8 pf[RT][2][A.WPARTS];
#pragma unroll
    for (int r = 0; r < RT; ++r) A.weights(r, S[r], sf, pf[r]);
    if constexpr (VIEW != KV_PREFIX) __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      bf16x8(&cur)[2] = vf[d % (AHEAD + 1)];
      if (d + AHEAD < ND) {
        vf[(d + AHEAD) % (AHEAD + 1)][0] = v_at(d + AHEAD, 0);
        vf[(d + AHEAD) % (AHEAD + 1)][1] = v_at(d + AHEAD, 1);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < RT; ++r) A.O[r][d] = A.product(cur[h], pf[r][h], A.O[r][d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  const auto key = [&](int i) { return x.span.key<VIEW>(i); };
  if constexpr (VIEW == KV_PREFIX) {
    for (int d = tid; d < R; d += 256) first_nan[d] = 0x7fffffff;
  } else if (tid < 2) {
    nan_step[tid] = 0;
  }
  if (x.k0 < x.k1) {
    pages(key(x.k0));
    load(key(x.k0), key(x.k0 + 64));
    __syncthreads();
    spread(0, key(x.k0));
    __syncthreads();
  }
  for (int i = x.k0; i < x.k1; i += 64) {
    const bool more = i + 64 < x.k1;
    const int j = key(i), then = key(i + 64);
    groups = there & 15;
    if (more) load(then, key(i + 128));
    if (j < my_end && (VIEW != KV_WINDOW || j + 63 >= my_low || j < a.sinks)) step(j);
    if (more) spread(buf ^ 1, then);
    __syncthreads();
    buf ^= 1;
  }
  A.finish();
  if constexpr (VIEW == KV_PREFIX) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int nan = first_nan[d * 16 + 4 * g + i];
#pragma unroll
        for (int r = 0; r < RT; ++r)
          if (A.lim[r] >= nan) A.O[r][d][i] = __uint_as_float(0x7fc00000u);
      }
  }
  A.store(a, pl, x, row0, n, g);
}

// ---- single tokens ---------------------------------------------------------
// The four waves take the same 16 rows and every fourth step of 64 keys, whose
// operands come straight from memory into the lanes that need them: four times
// the loads in flight for one set of rows, and no barrier until the waves are
// joined through LDS.
// Windows and trees of several tokens take tiles of 16 rows so too where that is faster
// than rows of their own.
// Bound by memory: one sequence of 131072 tokens, 8 key heads of 128, in 57 us with its
// join, 4.7 TB/s of cache (43 us alone: 6.2, as fast as memory is read here; float32
// queries without shared heads 50, 5.4); 64 sequences of up to 8192 in 121 us, 4.4 TB/s;
// 64 windows of 4096 in 91, 5.3 TB/s.  A step of 5 us at the least.
template <typename T, int R, int VIEW>
__global__ __launch_bounds__(256, R <= (sizeof(T) == 4 ? 96 : 128) ? 2 : 1) void kv_attn_keys_kernel(KvAttnArgs a, KvPlan pl) {
  constexpr int NK = R / 32, ND = R / 16;
  constexpr bool LEAN = R >= 192;  // registers hold K or V, not both
  extern __shared__ __align__(16) float join[];
  const KvArgs &c = a.c;
  const Work x = kv_work<VIEW>(a, pl);
  if (!x.any) return;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = VIEW == KV_PREFIX ? tid >> 6 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const float sf = kv_factor(a.scale);
  Rows<T, R, 1, VIEW> A;
  A.init(a, x, x.row0, n, [&](int k) { return k < R / 64 * 2 ? (k >> 1) * 64 + g * 16 + (k & 1) * 8 : R / 64 * 64 + g * 8; });

  const int32_t *table = c.table + (int64_t)x.b * c.max_pages;
  constexpr int STEP = 256;
  const int last_page = (x.total - 1) >> c.lgP;
  const int64_t page_bytes = (int64_t)c.KVH * c.P * R;
  const uint8_t *kb = c.k + (int64_t)x.kvh * c.P * R, *vb = c.v + (int64_t)x.kvh * c.P * R;
  // the page of the 16 keys of this lane's group, clamped to the sequence's last
  const auto page_at = [&](int j) { return table[min((j + 16 * g) >> c.lgP, last_page)]; };

  // lane n holds key 16 (n >> 2) + 4 t + (n & 3) of tile t, 16 bytes of each 64
  // columns; of V row 16 d + n, 16 keys of group g
  uint32_t kr[4][R / 16], vr[ND][4];
  float ksc = 0.f, vsc = 0.f;  // scales of that K and that V
  const auto load_k = [&](int j, int page) {
    const int pk = __shfl(page, (n >> 2) * 16, 64);
    ksc = c.ks[(int64_t)pk * c.KVH + x.kvh];
    const uint8_t *base = kb + pk * page_bytes + (int64_t)((j + 16 * (n >> 2) + (n & 3)) & (c.P - 1)) * R;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t *p = base + t * 4 * R;
#pragma unroll
      for (int k = 0; k < R / 64; ++k) {
        const uint4 y = *reinterpret_cast<const uint4 *>(p + k * 64 + g * 16);
        kr[t][k * 4] = y.x; kr[t][k * 4 + 1] = y.y; kr[t][k * 4 + 2] = y.z; kr[t][k * 4 + 3] = y.w;
      }
      if constexpr (R % 64 != 0) {
        const uint2 y = *reinterpret_cast<const uint2 *>(p + R / 64 * 64 + g * 8);
        kr[t][R / 64 * 4] = y.x; kr[t][R / 64 * 4 + 1] = y.y;
      }
    }
  };
  const auto load_v = [&](int j, int page) {
    const uint8_t *p = vb + page * page_bytes + ((j + 16 * g) & (c.P - 1)) + (int64_t)n * c.P;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const uint4 y = *reinterpret_cast<const uint4 *>(p + (int64_t)d * 16 * c.P);
      vr[d][0] = y.x; vr[d][1] = y.y; vr[d][2] = y.z; vr[d][3] = y.w;
    }
  };

  const auto key = [&](int i) { return x.span.key<VIEW>(i); };
  // pages that no row sees need not be there, nor hold a scale
  const int reach = kv_reach<VIEW>(a, x);
  const auto in_reach = [&](int at) { return VIEW != KV_WINDOW || at + 15 >= reach || at < a.sinks; };
  int j = 0, page = 0, next = 0;
  bool ok = false;
  // a step's page (0 where there is none), K and scales, and the page after it
  const auto advance = [&](int i, int p) {
    ok = (unsigned)p < (unsigned)c.pages && in_reach(key(i) + 16 * g);
    page = ok ? p : 0;
    load_k(key(i), page);
    vsc = c.vs[(int64_t)page * c.KVH + x.kvh];
    next = page_at(key(i + STEP));
  };

  const auto step = [&](auto clean_, auto &&between) {
    constexpr bool CLEAN = decltype(clean_)::value != 0;
    const bool was_ok = ok;
    const int first = j + 16 * g;  // this lane's scores are of the keys first + 4 t + i
    const float vs = ok ? vsc : 1.f;
    f32x4 S[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NK; ++k) A.scores(from_e4m3(kr[t][2 * k], kr[t][2 * k + 1], ksc), k, 0, S[t]);
    }
    between();  // K's registers are free
    bf16x8 pf[2][A.WPARTS];
    const int see = CLEAN ? A.ALL : was_ok ? A.sees(a, x, 0, first) : 0;
    if constexpr (CLEAN) A.every = true;
    else A.mask(0, S, see);
    A.weights(0, S, sf, pf);
    // keys behind the sequence and in pages that are not there hold no numbers
    const int have = CLEAN ? 16 : was_ok ? max(0, min(16, x.total - first)) : 0;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      uint32_t v[4] = {vr[d][0], vr[d][1], vr[d][2], vr[d][3]};
      if constexpr (!CLEAN) {
        bool nan = false;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int k = min(max(have - 4 * q, 0), 4);
          v[q] &= k == 4 ? ~0u : (1u << (8 * k)) - 1u;
          nan |= has_nan(v[q]);
        }
        if (__any(nan)) {
          u32x4 is[2];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t drop = 0, one[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((v[q] >> (8 * k) & 0x7f) == 0x7f) {
                drop |= 0xffu << (8 * k);
                one[k >> 1] |= 0x3f80u << (16 * (k & 1));
              }
            v[q] &= ~drop;
            is[q >> 1][(q & 1) * 2] = one[0];
            is[q >> 1][(q & 1) * 2 + 1] = one[1];
          }
          const bf16x8 at[2] = {as_bf16x8(is[0]), as_bf16x8(is[1])};
          A.O[0][d] += A.not_numbers(at, see);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) A.O[0][d] = A.product(from_e4m3(v[2 * h], v[2 * h + 1], vs), pf[h], A.O[0][d]);
    }
  };

  int i = x.k0 + w * 64;
  if (i < x.k1) advance(i, page_at(key(i)));
  const auto clean = [&]() { return A.clear(a, j) && __all(ok); };
  const auto walk = [&](auto clean_) {
    const bool more = i + STEP < x.k1, here = ok;
    if (!here && j + 16 * g < x.total && in_reach(j + 16 * g) && c.bad) c.bad[x.b] = 1;
    if constexpr (!LEAN) load_v(j, page);  // on its way while the scores are computed
    const auto between = [&]() {
      if constexpr (LEAN) load_v(j, page);
      else if (more) advance(i + STEP, next);
    };
    step(clean_, between);
    if constexpr (LEAN)
      if (more) advance(i + STEP, next);
    i += STEP;
    j = key(i);
  };
  j = key(i);
  while (i < x.k1) {
    // steps without a mask in a loop of their own: both kinds in one loop leave a window's
    // walk, which has them in any order, without registers (heads of 128: 131 in memory)
    while (i < x.k1 && clean()) walk(Int<1>());
    if (i < x.k1) walk(Int<0>());
  }
  A.finish();

  // waves 2, 3 into 0, 1, then 1 into 0
  constexpr int SIZE = (ND * 4 + 3) * 64;
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {
    __syncthreads();
    if (w >= half && w < 2 * half) {
      float *o = join + (w - half) * SIZE + lane;
      o[0] = A.m[0];
      o[64] = A.L[0][0];
      o[128] = A.seen[0] ? 1.f : 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[(3 + d * 4 + i) * 64] = A.O[0][d][i];
    }
    __syncthreads();
    if (w < half) {
      const float *o = join + w * SIZE + lane;
      const float m2 = o[0], mn = fmaxf(A.m[0], m2);
      const float f1 = A.m[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(A.m[0] - mn);
      const float f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - mn);
      A.L[0][0] = A.L[0][0] * f1 + o[64] * f2;
      A.m[0] = mn;
      A.seen[0] |= o[128] != 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) A.O[0][d][i] = A.O[0][d][i] * f1 + o[(3 + d * 4 + i) * 64] * f2;
    }
  }
  if (w == 0) A.store(a, pl, x, x.row0, n, g);
}

// Joins a row's splits.  WAVES waves per (row, head): 1 where the rows fill the card, 4
// where few rows have few splits (2048 rows of 8: 7 us, 12 with one), 16 where they
// have many (32 rows of 64: 8 us; one wave alone waits for a load per split, 150 us
// at 128).
template <typename T, int WAVES, int VIEW>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void kv_join_kernel(KvAttnArgs a, KvPlan pl) {
  constexpr int U = KV_MAX_HEAD / 64;
  const KvArgs &c = a.c;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t slots = (int64_t)c.B * c.max_new * a.H, slot = WAVES == 1 ? (int64_t)blockIdx.x * 4 + w : blockIdx.x;
  if (slot >= slots) return;
  const int h = (int)(slot % a.H), t = (int)(slot / a.H % c.max_new), b = (int)(slot / a.H / c.max_new);
  const Seq s = kv_seq(c, b, c.limit);
  if (t >= s.n) return;
  // what the row's workgroup saw, as it counted it
  const int row = t * a.G + h % a.G, wg0 = row / pl.rows_wg * pl.rows_wg;
  const int wg_end = kv_span<VIEW>(a, s, wg0, min(s.n * a.G, wg0 + pl.rows_wg) - 1).end;
  if (wg_end <= pl.chunk) return;
  const int n = (wg_end - 1) / pl.chunk + 1;
  const float *ml = a.work + slot * 2;
  // the maximum over all splits; l of a split whose scores are all -inf is NaN
  float M = -INFINITY;
  bool none = false;
  for (int i = lane; i < n; i += 64) {
    const float2 v = *reinterpret_cast<const float2 *>(ml + i * slots * 2);
    M = fmaxf(M, v.x);
    none |= v.x == -INFINITY && v.y != v.y;
  }
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  none = __any(none);
  const float *part = a.work + kv_part_at(pl.splits, slots) + slot * c.R;
  float acc[U] = {}, l = 0.f;
#pragma unroll 4
  for (int i = WAVES == 1 ? 0 : w; i < n; i += WAVES) {
    const float2 v = *reinterpret_cast<const float2 *>(ml + i * slots * 2);
    const float f = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - M);
    l += v.x == -INFINITY ? 0.f : v.y * f;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (lane + 64 * u < c.hd) acc[u] += part[i * slots * c.R + lane + 64 * u] * f;
  }
  T *out = (T *)a.out + (int64_t)(s.start + t) * a.os + (int64_t)h * c.hd;
  const float nothing = none ? __uint_as_float(0x7fc00000u) : 0.f;
  if constexpr (WAVES == 1) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (lane + 64 * u < c.hd) Elem<T>::put(out + lane + 64 * u, M != -INFINITY ? acc[u] / l : nothing);
  } else {
    __shared__ float sl[WAVES], so[WAVES][KV_MAX_HEAD];
#pragma unroll
    for (int u = 0; u < U; ++u) so[w][lane + 64 * u] = acc[u];
    if (lane == 0) sl[w] = l;
    __syncthreads();
    for (int d = threadIdx.x; d < c.hd; d += 64 * WAVES) {
      float o = 0.f, sum = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        o += so[i][d];
        sum += sl[i];
      }
      Elem<T>::put(out + d, M != -INFINITY ? o / sum : nothing);
    }
  }
}

template <typename F>
hipError_t kv_attn_run(F fn, std::atomic<int> (&set)[kAttrDevices], int lds, const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  const int64_t blocks = (int64_t)a.c.B * p.tiles * p.splits * a.c.KVH;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  if (lds > 65536) {
    const hipError_t e = ensure_lds_attr((const void *)fn, lds, set);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), lds, s, a, p);
  return hipGetLastError();
}
template <typename T, int R, int VIEW>
hipError_t kv_attn_rows(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  static std::atomic<int> set[3][kAttrDevices];
  if (!p.by_rows)  // two waves' outputs
    return kv_attn_run(kv_attn_keys_kernel<T, R, VIEW>, set[0], 2 * (R / 16 * 4 + 3) * 64 * 4, a, p, s);
  // two steps' K and V, and where V holds NaN
  constexpr int lds = VIEW == KV_PREFIX ? 516 * R : 528 * R + 16;
  if constexpr (R <= kv_two_tiles(sizeof(T)))
    if (p.rt == 2) return kv_attn_run(kv_attn_rows_kernel<T, R, 2, VIEW>, set[1], lds, a, p, s);
  return kv_attn_run(kv_attn_rows_kernel<T, R, 1, VIEW>, set[2], lds, a, p, s);
}
template <typename T, int VIEW>
hipError_t kv_attn_typed(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  const KvArgs &c = a.c;
  hipError_t e = hipErrorInvalidValue;
  switch (c.R) {
    case 32: e = kv_attn_rows<T, 32, VIEW>(a, p, s); break;
    case 64: e = kv_attn_rows<T, 64, VIEW>(a, p, s); break;
    case 96: e = kv_attn_rows<T, 96, VIEW>(a, p, s); break;
    case 128: e = kv_attn_rows<T, 128, VIEW>(a, p, s); break;
    case 192: e = kv_attn_rows<T, 192, VIEW>(a, p, s); break;
    case 256: e = kv_attn_rows<T, 256, VIEW>(a, p, s); break;
  }
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t slots = (int64_t)c.B * c.max_new * a.H;
  // windows and trees: a wave a row from 4096 rows on (8 x 40 x 32 rows of 5 splits: 44 us
  // with the attention, 51 with four), four from 512 (2048 rows of 32 splits: 77 us, 86
  // with sixteen)
  const bool few = VIEW == KV_PREFIX || slots < 512;
  if (slots >= (VIEW == KV_PREFIX ? 16384 : 4096))
    hipLaunchKernelGGL((kv_join_kernel<T, 1, VIEW>), dim3((unsigned)((slots + 3) / 4)), dim3(256), 0, s, a, p);
  else if (!few || p.splits <= 16)
    hipLaunchKernelGGL((kv_join_kernel<T, 4, VIEW>), dim3((unsigned)slots), dim3(256), 0, s, a, p);
  else
    hipLaunchKernelGGL((kv_join_kernel<T, 16, VIEW>), dim3((unsigned)slots), dim3(1024), 0, s, a, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace gn
