// Attention over the paged 8-bit cache: the kernels, compiled once for each type
// of queries (k_kv_attn_f32.hip, k_kv_attn_bf16.hip).
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
// 16 consecutive bytes of a row of the transposed cache.  K, V, P and O pass
// through registers only; a row's maximum and sum live in its four lanes.
//
// float32 queries are cut into three bf16 numbers (8 bits each, nothing lost), and
// so are the weights: three products each, as exact as float32's.  bfloat16
// queries take one, with the weights rounded to bf16.
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
// PARTS bf16 numbers that sum to each of eight float32: rounded (1) or cut at 8
// bits, the rest cut again (3)
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

// T: float or bf16 bits; R: padded head; RT: 16-row tiles of a wave.  BY_ROWS: the
// four waves take 16 RT rows each and walk the keys together (prompts: the keys
// come out of the L1 for three of the four); else they take the same rows and every
// fourth step of 64 keys, joined through LDS (single tokens: four times the
// loads in flight for one set of rows).
template <typename T, int R, int RT, bool BY_ROWS>
__global__ __launch_bounds__(256) void kv_attn_kernel(KvAttnArgs a, KvPlan pl) {
  constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
  constexpr int NK = R / 32, ND = R / 16;
  const KvArgs &c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, n = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int kvh = id % c.KVH;
  id /= c.KVH;
  const int split = id % pl.splits;
  id /= pl.splits;
  const int tile = pl.tiles - 1 - id % pl.tiles, b = id / pl.tiles;  // the rows that see most first
  const Seq s = kv_seq(c, b, min(c.max_len, c.max_pages * c.P));
  if (s.bad && c.bad && tid == 0) c.bad[b] = 1;
  const int total = s.len + s.n, rows = s.n * a.G;
  const int wg0 = tile * pl.rows_wg;
  if (wg0 >= rows) return;
  const int row0 = wg0 + (BY_ROWS ? w * 16 * RT : 0);
  // the last key that the workgroup's last row sees
  const int wg_last = min(rows, wg0 + pl.rows_wg) - 1;
  const int wg_end = a.causal ? s.len + wg_last / a.G + 1 : total;
  const int k0 = split * pl.chunk;
  if (k0 >= wg_end && split > 0) return;
  const int my_last = min(rows, row0 + 16 * RT) - 1;
  const int k1 = min(min(k0 + pl.chunk, wg_end), row0 >= rows ? 0 : a.causal ? s.len + my_last / a.G + 1 : total);

  // queries, and the last key of each row
  bf16x8 qf[RT][NK][PARTS];
  int lim[RT], lo_lim = total - 1;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = row0 + r * 16 + n;
    const bool on = row < rows;
    const int t = on ? row / a.G : 0;
    lim[r] = on && a.causal ? s.len + t : total - 1;
    lo_lim = min(lo_lim, lim[r]);
    const T *q = (const T *)a.q + (int64_t)(s.start + t) * a.qs + (int64_t)(kvh * a.G + (on ? row % a.G : 0)) * c.hd;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int d0 = k < R / 64 * 2 ? (k >> 1) * 64 + g * 16 + (k & 1) * 8 : R / 64 * 64 + g * 8;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = on && d0 + i < c.hd ? Elem<T>::get(q + d0 + i) : 0.f;
      to_parts<PARTS>(v, qf[r][k]);
    }
  }
  for (int o = 8; o > 0; o >>= 1) lo_lim = min(lo_lim, __shfl_xor(lo_lim, o, 64));
  lo_lim = __builtin_amdgcn_readfirstlane(lo_lim);

  f32x4 O[RT][ND];
  float m[RT], l[RT];
  bool seen[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    seen[r] = false;
#pragma unroll
    for (int d = 0; d < ND; ++d) O[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t *table = c.table + (int64_t)b * c.max_pages;
  const int step = BY_ROWS ? 64 : 256;
  const int last_page = (total - 1) >> c.lgP;
  const int64_t page_bytes = (int64_t)c.KVH * c.P * R;
  const uint8_t *kb = c.k + (int64_t)kvh * c.P * R, *vb = c.v + (int64_t)kvh * c.P * R;
  // the page of this lane's 16 keys (group g), clamped to the sequence's last
  const auto page_at = [&](int j) { return table[min((j + 16 * g) >> c.lgP, last_page)]; };

  uint32_t kr[4][R / 16];
  // K rows of the step at j: lane n holds key 16 (n >> 2) + 4 t + (n & 3) of tile t
  const auto load_k = [&](int j, int page) {
    const int pk = __shfl(page, (n >> 2) * 16, 64);
    const uint8_t *base = kb + pk * page_bytes + (int64_t)((j + 16 * (n >> 2) + (n & 3)) & (c.P - 1)) * R;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint8_t *p = base + t * 4 * R;
#pragma unroll
      for (int k = 0; k < R / 64; ++k) {
        const uint4 x = *reinterpret_cast<const uint4 *>(p + k * 64 + g * 16);
        kr[t][k * 4] = x.x; kr[t][k * 4 + 1] = x.y; kr[t][k * 4 + 2] = x.z; kr[t][k * 4 + 3] = x.w;
      }
      if constexpr (R % 64 != 0) {
        const uint2 x = *reinterpret_cast<const uint2 *>(p + R / 64 * 64 + g * 8);
        kr[t][R / 64 * 4] = x.x; kr[t][R / 64 * 4 + 1] = x.y;
      }
    }
  };
  const auto valid = [&](int page) { return page >= 0 && page < c.pages; };

  int j = k0 + (BY_ROWS ? 0 : w * 64);
  int page = 0, next = 0;
  bool ok = false;
  float ksc = 0.f, vsc = 0.f;
  if (j < k1) {
    page = page_at(j);
    ok = valid(page);
    page = ok ? page : 0;
    load_k(j, page);
    ksc = c.ks[(int64_t)page * c.KVH + kvh];
    vsc = c.vs[(int64_t)page * c.KVH + kvh];
    next = page_at(j + step);
  }
  for (; j < k1; j += step) {
    // this step's V rows, on their way while the scores are computed
    uint32_t vr[ND][4];
    {
      const uint8_t *p = vb + page * page_bytes + ((j + 16 * g) & (c.P - 1)) + (int64_t)n * c.P;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const uint4 x = *reinterpret_cast<const uint4 *>(p + (int64_t)d * 16 * c.P);
        vr[d][0] = x.x; vr[d][1] = x.y; vr[d][2] = x.z; vr[d][3] = x.w;
      }
    }
    // keys of this lane's scores: j + 16 g + (4 t + i)
    const bool clean = j + 63 <= lo_lim && __all(ok);
    const float sf = ksc * (a.scale * LOG2E), vs = ok ? vsc : 1.f;
    f32x4 S[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int r = 0; r < RT; ++r) S[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const bf16x8 kf = from_e4m3(kr[t][2 * k], kr[t][2 * k + 1], 1.f);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int p = 0; p < PARTS; ++p)
            S[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[r][k][p], S[r][t], 0, 0, 0);
      }
    }
    // the next step's K and scales, the page after it
    const bool was_ok = ok;
    if (j + step < k1) {
      ok = valid(next);
      page = ok ? next : 0;
      load_k(j + step, page);
      ksc = c.ks[(int64_t)page * c.KVH + kvh];
      vsc = c.vs[(int64_t)page * c.KVH + kvh];
      next = page_at(j + 2 * step);
    }
    const int first = j + 16 * g;
    bool nan = false;
    if (!clean) {
      // keys behind the sequence and in pages that are not there are no numbers
      const int have = was_ok ? max(0, min(16, total - first)) : 0;
      if (!was_ok && first < total && c.bad) c.bad[b] = 1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = min(max(have - 4 * q, 0), 4);
        const uint32_t mask = k == 4 ? ~0u : (1u << (8 * k)) - 1u;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          vr[d][q] &= mask;
          nan |= has_nan(vr[d][q]);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      float mx = -INFINITY;
      const int see = clean ? 16 : was_ok ? max(0, min(16, lim[r] - first + 1)) : 0;
      seen[r] |= see > 0;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = S[r][t][i] * sf;
          if (!clean) x = 4 * t + i < see ? x : -INFINITY;
          S[r][t][i] = x;
          mx = fmaxf(mx, x);
        }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float mn = fmaxf(m[r], mx);
      if (__any(mn > m[r])) {
        // nothing yet, or nothing but -inf: no maximum to subtract
        const float f = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - mn);
        l[r] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) O[r][d] *= f;
        m[r] = mn;
      }
      const float sub = mn == -INFINITY ? 0.f : mn;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          S[r][t][i] = __builtin_amdgcn_exp2f(S[r][t][i] - sub);
          sum += S[r][t][i];
        }
      l[r] += sum;
    }
    // masked weights are 0 but 0 * NaN is not: NaN values are taken out of the
    // product, and rows that see one find it by a product of ones
    if (!clean && __any(nan)) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        u32x4 is[2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t v = vr[d][q];
          uint32_t drop = 0, ones[2] = {0, 0};
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if ((v >> (8 * k) & 0x7f) == 0x7f) {
              drop |= 0xffu << (8 * k);
              ones[k >> 1] |= 0x3f80u << (16 * (k & 1));
            }
          vr[d][q] = v & ~drop;
          is[q >> 1][(q & 1) * 2] = ones[0];
          is[q >> 1][(q & 1) * 2 + 1] = ones[1];
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const int see = was_ok ? lim[r] - first + 1 : 0;
          f32x4 hit = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            u32x4 on;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              on[k] = (8 * h + 2 * k < see ? 0x3f80u : 0u) | (8 * h + 2 * k + 1 < see ? 0x3f800000u : 0u);
            hit = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(is[h]), as_bf16x8(on), hit, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (hit[i] > 0.f) O[r][d][i] = __uint_as_float(0x7fc00000u);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8 pf[RT][PARTS];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float v[8] = {S[r][2 * h][0], S[r][2 * h][1], S[r][2 * h][2], S[r][2 * h][3],
                            S[r][2 * h + 1][0], S[r][2 * h + 1][1], S[r][2 * h + 1][2], S[r][2 * h + 1][3]};
        to_parts<PARTS>(v, pf[r]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const bf16x8 vf = from_e4m3(vr[d][2 * h], vr[d][2 * h + 1], vs);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int p = 0; p < PARTS; ++p)
            O[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[r][p], O[r][d], 0, 0, 0);
      }
    }
  }

  // a row's sum over its four lanes
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    l[r] += __shfl_xor(l[r], 16, 64);
    l[r] += __shfl_xor(l[r], 32, 64);
    const int any = (int)seen[r] | __shfl_xor((int)seen[r], 16, 64);
    seen[r] = any | __shfl_xor(any, 32, 64);
  }
  if constexpr (!BY_ROWS) {
    // waves 2, 3 into 0, 1, then 1 into 0
    extern __shared__ __align__(16) float join[];
    constexpr int SIZE = RT * (ND * 4 + 3) * 64;
#pragma unroll
    for (int half = 2; half > 0; half >>= 1) {
      __syncthreads();
      if (w >= half && w < 2 * half) {
        float *o = join + (w - half) * SIZE + lane;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          o[(r * 3) * 64] = m[r];
          o[(r * 3 + 1) * 64] = l[r];
          o[(r * 3 + 2) * 64] = seen[r] ? 1.f : 0.f;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[(RT * 3 + (r * ND + d) * 4 + i) * 64] = O[r][d][i];
        }
      }
      __syncthreads();
      if (w < half) {
        const float *o = join + w * SIZE + lane;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const float m2 = o[(r * 3) * 64], mn = fmaxf(m[r], m2);
          const float f1 = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - mn);
          const float f2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - mn);
          l[r] = l[r] * f1 + o[(r * 3 + 1) * 64] * f2;
          m[r] = mn;
          seen[r] |= o[(r * 3 + 2) * 64] != 0.f;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[r][d][i] = O[r][d][i] * f1 + o[(RT * 3 + (r * ND + d) * 4 + i) * 64] * f2;
        }
      }
    }
    if (w != 0) return;
  }
  const bool alone = wg_end <= pl.chunk;  // no other split of these rows
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = row0 + r * 16 + n;
    if (row >= rows) continue;
    const int t = row / a.G, h = kvh * a.G + row % a.G;
    // no key at all: 0; keys whose scores are all -inf: no number, as 0 / 0 says
    if (alone) {
      T *out = (T *)a.out + (int64_t)(s.start + t) * a.os + (int64_t)h * c.hd;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int col = d * 16 + 4 * g + i;
          if (col < c.hd) Elem<T>::put(out + col, seen[r] ? O[r][d][i] / l[r] : 0.f);
        }
    } else {
      const int64_t slot = ((int64_t)b * c.max_new + t) * a.H + h, slots = (int64_t)c.B * c.max_new * a.H;
      float *ml = a.work + (split * slots + slot) * 2;
      if (g == 0) {
        ml[0] = m[r];
        ml[1] = seen[r] && m[r] == -INFINITY ? __uint_as_float(0x7fc00000u) : l[r];
      }
      float *part = a.work + pl.splits * slots * 2 + (split * slots + slot) * R;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        *reinterpret_cast<float4 *>(part + d * 16 + 4 * g) = make_float4(O[r][d][0], O[r][d][1], O[r][d][2], O[r][d][3]);
    }
  }
}

// joins a row's splits: one wave per (row, head)
template <typename T>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttnArgs a, KvPlan pl) {
  const KvArgs &c = a.c;
  const int lane = threadIdx.x & 63;
  const int64_t slots = (int64_t)c.B * c.max_new * a.H;
  const int64_t slot = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (slot >= slots) return;
  const int h = (int)(slot % a.H), t = (int)(slot / a.H % c.max_new), b = (int)(slot / a.H / c.max_new);
  const Seq s = kv_seq(c, b, min(c.max_len, c.max_pages * c.P));
  if (t >= s.n) return;
  // what the row's workgroup saw, as it counted it
  const int row = t * a.G + h % a.G, wg0 = row / pl.rows_wg * pl.rows_wg;
  const int wg_last = min(s.n * a.G, wg0 + pl.rows_wg) - 1;
  const int wg_end = a.causal ? s.len + wg_last / a.G + 1 : s.len + s.n;
  if (wg_end <= pl.chunk) return;
  const int n = (wg_end + pl.chunk - 1) / pl.chunk;
  const float *ml = a.work + slot * 2;
  float M = -INFINITY;
  bool none = false;
  for (int i = lane; i < n; i += 64) {
    const float l = ml[i * slots * 2 + 1];
    M = fmaxf(M, ml[i * slots * 2]);
    none |= l != l && ml[i * slots * 2] == -INFINITY;
  }
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  none = __any(none);
  const float *part = a.work + pl.splits * slots * 2 + slot * c.R;
  float acc[KV_MAX_HEAD / 64] = {}, l = 0.f;
  for (int i = 0; i < n; ++i) {
    const float m = ml[i * slots * 2];
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    if (m != -INFINITY) l += ml[i * slots * 2 + 1] * f;
#pragma unroll
    for (int u = 0; u < KV_MAX_HEAD / 64; ++u)
      if (lane + 64 * u < c.hd) acc[u] += part[i * slots * c.R + lane + 64 * u] * f;
  }
  T *out = (T *)a.out + (int64_t)(s.start + t) * a.os + (int64_t)h * c.hd;
#pragma unroll
  for (int u = 0; u < KV_MAX_HEAD / 64; ++u)
    if (lane + 64 * u < c.hd)
      Elem<T>::put(out + lane + 64 * u, M != -INFINITY ? acc[u] / l : none ? __uint_as_float(0x7fc00000u) : 0.f);
}

template <typename T, int R, int RT, bool BY_ROWS>
hipError_t kv_attn_run(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  const int64_t blocks = (int64_t)a.c.B * p.tiles * p.splits * a.c.KVH;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  const int lds = BY_ROWS ? 0 : 2 * RT * (R / 16 * 4 + 3) * 64 * 4;
  const auto fn = kv_attn_kernel<T, R, RT, BY_ROWS>;
  if (lds > 65536) {
    static std::atomic<int> set[kAttrDevices];
    const hipError_t e = ensure_lds_attr((const void *)fn, lds, set);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), lds, s, a, p);
  return hipGetLastError();
}
template <typename T, int R>
hipError_t kv_attn_rows(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  if (p.by_rows) return kv_attn_run<T, R, 2, true>(a, p, s);
  return p.rt == 1 ? kv_attn_run<T, R, 1, false>(a, p, s) : kv_attn_run<T, R, 2, false>(a, p, s);
}
template <typename T>
hipError_t kv_attn_typed(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  const KvArgs &c = a.c;
  hipError_t e = hipErrorInvalidValue;
  switch (c.R) {
    case 32: e = kv_attn_rows<T, 32>(a, p, s); break;
    case 64: e = kv_attn_rows<T, 64>(a, p, s); break;
    case 96: e = kv_attn_rows<T, 96>(a, p, s); break;
    case 128: e = kv_attn_rows<T, 128>(a, p, s); break;
    case 192: e = kv_attn_rows<T, 192>(a, p, s); break;
    case 256: e = kv_attn_rows<T, 256>(a, p, s); break;
  }
  if (e != hipSuccess || p.splits == 1) return e;
  const int64_t slots = (int64_t)c.B * c.max_new * a.H;
  hipLaunchKernelGGL(kv_join_kernel<T>, dim3((unsigned)((slots + 3) / 4)), dim3(256), 0, s, a, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace gn
