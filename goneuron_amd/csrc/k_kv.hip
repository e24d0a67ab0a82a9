// The paged 8-bit cache of rotated keys and values: appending to it.
//
// Layout: K pages [page][kv head][token][R], V pages [page][kv head][R][token]
// in E4M3 with a power-of-two scale per (page, kv head) for each.  V lies
// transposed so that attention's two products read both caches as their matrix
// operands lie in registers, 16 bytes a lane (single tokens with no pass through LDS);
// the writer owns a whole block anyway (its scale covers the block).
#include "gn_kv.h"

namespace gn {
namespace {

// ---------------------------------------------------------------- append
constexpr int KV_MANY = 8;  // four-value groups of new tokens a thread holds, of single tokens
constexpr int KV_ONE = 2;
constexpr int KV_TURNS = 2;  // groups of four pairs of queries a thread turns

// One workgroup per (sequence, touched page, kv head, K or V): it owns that
// block, so its new maximum, the growth of its scale and the bytes of tokens
// already there need no other workgroup.  New values stay in registers between
// the maximum and the rounding.  Blocks behind those rotate the queries.
// Single tokens: a chain of table, row and scale reads and one reduction, 4.2 us for a
// token of 4 sequences; a bfloat16 token of 256 sequences, 32 query heads and 8 key heads
// of 128, takes 9.5 (a copy moves its 5.9 MB in 1.2), most likely for the 262144 bytes of
// V, each into a line of its own (no counter was read for it).  Prompts: memory (six of up to
// 2048: 45 us for 163 MB, 3.6 TB/s, where a copy reaches 4.9).  Prompts also wait for the
// vector unit: indexes without divisions, pairs turned once and bytes rounded two at a
// time brought them from 60.
template <typename T, int KV_SLOTS>
__global__ __launch_bounds__(1024) void kv_append_kernel(KvAppendArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  const KvArgs &c = a.c;
  const int tid = threadIdx.x, NT = blockDim.x;
  const int items = c.B * a.touch * c.KVH * 2;
  // no page behind the table, whatever the limit.  (Without the minimum prompts of
  // bfloat16 rows are given 80 registers, six waves a SIMD, not 72 and seven: 1 us of 39.)
  const int limit = min(c.limit, c.max_pages * c.P);
  const int half = c.hd >> 1;
  if ((int)blockIdx.x >= items) {  // queries: KV_TURNS groups of four pairs a thread
    const int i = blockIdx.x - items, b = i / a.qtiles, tile = i % a.qtiles;
    const Seq s = kv_seq(c, b, limit);
    const T *q = (const T *)a.q;
    T *qo = (T *)a.qo;
    const int per = (half + 3) >> 2, row_groups = a.H * per;  // of a head, of a token
    const int64_t g0 = (int64_t)tile * KV_TURNS * NT;
    const int t0 = per ? (int)(g0 / row_groups) : s.n, first = per ? (int)(g0 % row_groups) : 0;
#pragma unroll
    for (int u = 0; u < KV_TURNS; ++u) {
      int g = first + u * NT + tid, t = t0;
      if (row_groups >= KV_TURNS * NT) {  // one token's end at most lies between
        t += g >= row_groups;
        g -= g >= row_groups ? row_groups : 0;
      } else if (per) {
        t += g / row_groups;
        g %= row_groups;
      }
      if (t >= s.n) break;
      const int h = divided(g, a.per_inv, per), d = (g - h * per) * 4;
      const T *row = q + (int64_t)(s.start + t) * a.qs + h * c.hd;
      T *out = qo + (int64_t)(s.start + t) * a.qos + h * c.hd;
      const float *cs = a.cs ? a.cs + (int64_t)(s.len + t) * half : nullptr;
      const float *sn = a.cs ? a.sn + (int64_t)(s.len + t) * half : nullptr;
      float lo[4], hi[4];
      if (a.vec) {
        Elem<T>::get4(row + d, lo);
        Elem<T>::get4(row + d + half, hi);
        if (a.cs) {
          const float4 c4 = *reinterpret_cast<const float4 *>(cs + d), s4 = *reinterpret_cast<const float4 *>(sn + d);
          const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) turn(lo[j], hi[j], cc[j], ss[j]);
        }
        Elem<T>::put4(out + d, lo);
        Elem<T>::put4(out + d + half, hi);
      } else {
        for (int j = d; j < min(d + 4, half); ++j) {
          float x = Elem<T>::get(row + j), y = Elem<T>::get(row + j + half);
          if (a.cs) turn(x, y, cs[j], sn[j]);
          Elem<T>::put(out + j, x);
          Elem<T>::put(out + j + half, y);
        }
      }
    }
    if (c.hd & 1)  // the last column has no partner; every tile takes its share of the rows
      for (int64_t g = (int64_t)tile * NT + tid; g < (int64_t)s.n * a.H; g += (int64_t)a.qtiles * NT) {
        const int t = (int)(g / a.H), h = (int)(g % a.H);
        Elem<T>::put(qo + (int64_t)(s.start + t) * a.qos + h * c.hd + c.hd - 1,
                     Elem<T>::get(q + (int64_t)(s.start + t) * a.qs + h * c.hd + c.hd - 1));
      }
    return;
  }

  const int which = blockIdx.x & 1;
  int i = blockIdx.x >> 1;
  const int h = i % c.KVH;
  i /= c.KVH;
  const int j = i % a.touch, b = i / a.touch;
  const Seq s = kv_seq(c, b, limit);
  if (s.bad && c.bad && j == 0 && tid == 0) c.bad[b] = 1;
  const int pi = (s.len >> c.lgP) + j;             // page of the sequence
  const int first = pi << c.lgP;                   // its first position
  const int lo = max(s.len - first, 0), hi = min(s.len + s.n - first, c.P);
  if (s.n == 0 || hi <= lo) return;
  // the rows do not wait for the page, nor the old scale for the maximum
  const int page = c.table[(int64_t)b * c.max_pages + pi];
  const int R = c.R, P = c.P, per = R >> 2;
  const bool rot = !which && a.cs;
  const T *x = (const T *)a.x[which] + h * c.hd;
  // Of a whole page of V a thread takes four columns of eight tokens, which it can
  // store by itself; of K both halves of a pair, so that a pair is read and turned
  // once.
  const bool tall = KV_SLOTS == KV_MANY && a.vec && which && hi - lo == P, pairs = a.vec && !which;
  // the token and column of this thread's u-th group of four; false: none
  const auto place = [&](int u, int &t, int &d) {
    if (tall) {
      t = (tid & ((P >> 3) - 1)) * 8 + u;
      d = (tid >> (c.lgP - 3)) * 4;
      return d < R;
    }
    const int n = pairs ? c.hd >> 3 : per, g = tid + (pairs ? u >> 1 : u) * NT, q = divided(g, pairs ? a.pair_inv : a.group_inv, n);
    t = lo + q;
    d = (g - q * n) * 4 + (pairs && (u & 1) ? half : 0);
    return t < hi;
  };

  float v[KV_SLOTS][4];
  const T *xs = x + (int64_t)(s.start + first - s.len) * a.xs[which];
  // no branch between the loads: all of them under way at once
  if (a.vec) {
#pragma unroll
    for (int u = 0; u < KV_SLOTS; ++u) {
      int t, d;
      const bool on = place(u, t, d) && d < c.hd;
      Elem<T>::get4(xs + (on ? t : lo) * a.xs[which] + (on ? d : 0), v[u]);
    }
    if (rot) {
      float4 cs[KV_SLOTS / 2], sn[KV_SLOTS / 2];
#pragma unroll
      for (int u = 0; u < KV_SLOTS; u += 2) {
        int t, d;
        const bool on = place(u, t, d);
        const int64_t at = (int64_t)(first + (on ? t : lo)) * half + (on ? d : 0);
        cs[u / 2] = *reinterpret_cast<const float4 *>(a.cs + at);
        sn[u / 2] = *reinterpret_cast<const float4 *>(a.sn + at);
      }
#pragma unroll
      for (int u = 0; u < KV_SLOTS; u += 2) {
        const float4 c4 = cs[u / 2], s4 = sn[u / 2];
        turn(v[u][0], v[u + 1][0], c4.x, s4.x);
        turn(v[u][1], v[u + 1][1], c4.y, s4.y);
        turn(v[u][2], v[u + 1][2], c4.z, s4.z);
        turn(v[u][3], v[u + 1][3], c4.w, s4.w);
      }
    }
#pragma unroll
    for (int u = 0; u < KV_SLOTS; ++u) {
      int t, d;
      const bool on = place(u, t, d) && d < c.hd;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[u][k] = on ? v[u][k] : 0.f;
    }
  } else {
#pragma unroll
    for (int u = 0; u < KV_SLOTS; ++u) {
      int t, d;
      if (!place(u, t, d)) break;
      const int64_t pos = first + t;
      load_rotated(xs + t * a.xs[which], rot ? a.cs + pos * half : nullptr, rot ? a.sn + pos * half : nullptr, c.hd, d, rot,
                   v[u]);
    }
  }
  const auto largest = [&](auto of) {
    float m = 0.f;
#pragma unroll
    for (int u = 0; u < KV_SLOTS; ++u) {
      int t, d;
      if (!place(u, t, d)) break;
#pragma unroll
      for (int k = 0; k < 4; ++k) m = fmaxf(m, of(fabsf(v[u][k])));  // passes NaN by
    }
    return m;
  };
  float amax = largest([](float y) { return y; });
  if (amax == INFINITY) amax = largest([](float y) { return y == INFINITY ? 0.f : y; });
  if (page < 0 || page >= c.pages) {
    if (c.bad && tid == 0) c.bad[b] = 1;
    return;
  }
  const int64_t blk = (int64_t)page * c.KVH + h;
  uint8_t *dst = (which ? c.v : c.k) + blk * P * R;
  float *sp = (which ? c.vs : c.ks) + blk;
  const float old = lo > 0 ? *sp : 0.f;
  // the block's maximum
  for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
  if (NT > 64) {
    __shared__ float red[16];
    if ((tid & 63) == 0) red[tid >> 6] = amax;
    __syncthreads();
    amax = red[0];
    for (int w = 1; w < NT >> 6; ++w) amax = fmaxf(amax, red[w]);
  }
  float scale = block_scale(amax);
  if (lo > 0) {
    if (old > scale) {
      scale = old;
    } else if (old < scale) {  // the tokens already here move to the larger scale
      const float ratio = old / scale;
      if (!which) {
        uint32_t *w = reinterpret_cast<uint32_t *>(dst);
        for (int g = tid; g < lo * per; g += NT) {
          const uint32_t o = w[g];
          w[g] = rescaled(o & 0xff, ratio) | rescaled(o >> 8 & 0xff, ratio) << 8 |
                 rescaled(o >> 16 & 0xff, ratio) << 16 | rescaled(o >> 24, ratio) << 24;
        }
      } else {
        for (int g = tid; g < R * lo; g += NT) {
          uint8_t *p = dst + (int64_t)(g / lo) * P + g % lo;
          *p = (uint8_t)rescaled(*p, ratio);
        }
      }
    }
    __syncthreads();  // every thread has read the old scale
  }
  if (tid == 0) *sp = scale;
  const float inv = 1.f / scale;

  if (!which) {
#pragma unroll
    for (int u = 0; u < KV_SLOTS; ++u) {
      int t, d;
      if (!place(u, t, d)) break;
      *reinterpret_cast<uint32_t *>(dst + t * R + d) = to_e4m3(v[u][0], v[u][1], v[u][2], v[u][3], inv);
    }
    const int pad = (R - c.hd) >> 2;
    if (pairs && pad)  // the rows' ends, which no pair covers
      for (int g = tid; g < (hi - lo) * pad; g += NT)
        *reinterpret_cast<uint32_t *>(dst + (lo + g / pad) * R + c.hd + g % pad * 4) = 0;
    return;
  }
  if (tall) {
    int t, d;
    if (!place(0, t, d) || d >= c.hd) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      constexpr int L = KV_SLOTS - 1;  // no slot beyond: single tokens are not tall
      uint2 w;
      w.x = to_e4m3(v[0][k], v[1][k], v[min(2, L)][k], v[min(3, L)][k], inv);
      w.y = to_e4m3(v[min(4, L)][k], v[min(5, L)][k], v[min(6, L)][k], v[L][k], inv);
      *reinterpret_cast<uint2 *>(dst + (d + k) * P + t) = w;
    }
    return;
  }
  if (hi - lo == 1) {  // one token: a byte of every row
#pragma unroll
    for (int u = 0; u < KV_SLOTS; ++u) {
      int t, d;
      if (!place(u, t, d)) break;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (d + k < c.hd) dst[(d + k) * P + lo] = (uint8_t)to_e4m3(v[u][k], inv);
    }
    return;
  }
  const int LP = P + 16;  // rows stay 16-byte aligned
#pragma unroll
  for (int u = 0; u < KV_SLOTS; ++u) {
    int t, d;
    if (!place(u, t, d)) break;
#pragma unroll
    for (int k = 0; k < 4; ++k) lds[(d + k) * LP + t] = (uint8_t)to_e4m3(v[u][k], inv);
  }
  __syncthreads();
  const int seg = P >> 4;
  for (int g = tid; g < c.hd * seg; g += NT) {
    const int d = g >> (c.lgP - 4), t = (g & (seg - 1)) * 16;
    if (t + 16 <= lo || t >= hi) continue;
    if (t >= lo && t + 16 <= hi) {
      *reinterpret_cast<uint4 *>(dst + (int64_t)d * P + t) = *reinterpret_cast<const uint4 *>(lds + d * LP + t);
    } else {
      for (int k = max(t, lo); k < min(t + 16, hi); ++k) dst[(int64_t)d * P + k] = lds[d * LP + k];
    }
  }
}

// ---------------------------------------------------------------- keep
// Token keep[i] of a sequence's new ones becomes its i-th, i < counts[b].  keep rises, so
// a token moves to its own place or an earlier one, and from the first that moves on all
// do.  One workgroup per (sequence, kv head, K or V) takes the pages in rising order: a
// page's tokens come from it or from later ones, which are as they were then.  The page's
// scale becomes the largest of its own and those its tokens come from, and all of its
// bytes are scaled to it; its tokens wait in LDS, as they were, until that is done.
// Latency: a chain of reads (bounds, numbers, pages, then scales and bytes), a page after
// the other: 64 sequences' paths in 7.3 us, a few of a small model in 5.5.
__global__ __launch_bounds__(256) void kv_keep_kernel(KvArgs c, const int32_t *keep, const int32_t *counts) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int64_t from[128];  // of a page's tokens: where their bytes begin
  __shared__ float had[128];     // and the scale they have
  __shared__ float red[4];
  const int which = blockIdx.x & 1, h = (blockIdx.x >> 1) % c.KVH, b = (blockIdx.x >> 1) / c.KVH, tid = threadIdx.x;
  const Seq s = kv_seq(c, b, c.limit);
  const int n = counts[b], R = c.R, P = c.P;
  if (s.bad || n < 0 || n > s.n) {
    if (c.bad && tid == 0) c.bad[b] = 1;
    return;
  }
  keep += s.start;
  const int32_t *table = c.table + (int64_t)b * c.max_pages;
  const auto missing = [&](int p) { return (unsigned)table[p >> c.lgP] >= (unsigned)c.pages; };
  int stay = 0;  // tokens that are in their place
  bool wrong = false;
  for (int i0 = 0; i0 < n; i0 += 256) {
    const int i = i0 + tid;
    bool same = false;
    if (i < n) {
      const int k = keep[i], before = i ? keep[i - 1] : -1;
      same = k == i;
      wrong |= k < 0 || k <= before || k >= s.n || missing(s.len + k) || missing(s.len + i);
    }
    stay += __syncthreads_count(same);
  }
  if (__syncthreads_or(wrong)) {
    if (c.bad && tid == 0) c.bad[b] = 1;
    return;
  }
  uint8_t *cache = which ? c.v : c.k;
  float *scales = which ? c.vs : c.ks;
  const int step = which ? P : 1, token = which ? 1 : R;  // from a column to the next, from a token
  for (int at = s.len + stay; at < s.len + n;) {
    const int first = at >> c.lgP << c.lgP, end = min(s.len + n, first + P), m = end - at;
    const int64_t blk = (int64_t)table[at >> c.lgP] * c.KVH + h;
    const float own = scales[blk];
    float scale = own;
    if (tid < m) {  // a page has 128 tokens at most
      const int p = s.len + keep[at - s.len + tid];
      const int64_t src = (int64_t)table[p >> c.lgP] * c.KVH + h;
      from[tid] = src * P * R + (p & (P - 1)) * token;
      scale = had[tid] = scales[src];
      scale = fmaxf(scale, own);
    }
    for (int off = 32; off > 0; off >>= 1) scale = fmaxf(scale, __shfl_xor(scale, off, 64));
    if ((tid & 63) == 0) red[tid >> 6] = scale;
    __syncthreads();
    scale = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    // columns fastest for K, tokens for V: neighbours in memory
    const uint32_t inv = inverse(which ? m : R);
    const auto place = [&](int g, int &t, int &d) {
      const int q = divided(g, inv, which ? m : R), r = g - q * (which ? m : R);
      t = which ? r : q;
      d = which ? q : r;
    };
    for (int g = tid; g < m * R; g += 256) {
      int t, d;
      place(g, t, d);
      lds[g] = cache[from[t] + d * step];
    }
    __syncthreads();
    uint8_t *dst = cache + blk * P * R;
    if (own < scale) {
      const float ratio = own / scale;
      for (int g = tid; g < P * R / 4; g += 256) {
        uint32_t *w = reinterpret_cast<uint32_t *>(dst) + g;
        const uint32_t o = *w;
        *w = rescaled(o & 0xff, ratio) | rescaled(o >> 8 & 0xff, ratio) << 8 | rescaled(o >> 16 & 0xff, ratio) << 16 |
             rescaled(o >> 24, ratio) << 24;
      }
      if (tid == 0) scales[blk] = scale;
      __syncthreads();
    }
    for (int g = tid; g < m * R; g += 256) {
      int t, d;
      place(g, t, d);
      dst[(at - first + t) * token + d * step] = (uint8_t)(had[t] == scale ? lds[g] : rescaled(lds[g], had[t] / scale));
    }
    __syncthreads();
    at = end;
  }
}

// what the other kernels flag, where a call has no row for them
__global__ __launch_bounds__(256) void kv_check_kernel(KvArgs c) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b < c.B && kv_seq(c, b, c.limit).bad) c.bad[b] = 1;
}

}  // namespace

hipError_t launch_kv_check(const KvArgs &c, hipStream_t s) {
  hipLaunchKernelGGL(kv_check_kernel, dim3((c.B + 255) / 256), dim3(256), 0, s, c);
  return hipGetLastError();
}

hipError_t launch_kv_keep(const KvArgs &c, const int32_t *keep, const int32_t *counts, hipStream_t s) {
  const int64_t blocks = (int64_t)c.B * c.KVH * 2;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  const int most = c.max_new < c.P ? c.max_new : c.P;
  hipLaunchKernelGGL(kv_keep_kernel, dim3((unsigned)blocks), dim3(256), (size_t)most * c.R, s, c, keep, counts);
  return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppendArgs &a0, int dtype, hipStream_t s) {
  KvAppendArgs a = a0;
  const KvArgs &c = a.c;
  const int most = c.max_new < c.P ? c.max_new : c.P;
  a.touch = (c.max_new + 2 * c.P - 2) / c.P;
  // a thread holds up to 32 new values of a block
  int nt = (most * c.R / (4 * KV_MANY) + 63) / 64 * 64;
  nt = nt < 64 ? 64 : nt;
  // a thread with eight groups waits eight times for memory: 17 us for 256 tokens of
  // 32 heads of 128, where two take 9.5
  const int64_t turns = (int64_t)c.max_new * a.H * ((c.hd / 2 + 3) / 4);
  const int64_t qtiles = (turns + KV_TURNS * nt - 1) / (KV_TURNS * nt);  // below 2^31: rows are
  a.qtiles = qtiles < 1 ? 1 : (int)qtiles;
  a.per_inv = inverse((c.hd / 2 + 3) / 4);
  a.group_inv = inverse(c.R / 4);
  a.pair_inv = inverse(c.hd / 8);
  const int64_t blocks = (int64_t)c.B * a.touch * c.KVH * 2 + (a.qo ? (int64_t)c.B * a.qtiles : 0);
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  const size_t sh = most > 1 ? (size_t)c.R * (c.P + 16) : 0;
  // single tokens fill two groups of a thread at most: loads of eight took 6.1 us where
  // theirs take 4 (a token of 4 sequences, 8 heads of 32)
  const bool one = c.max_new == 1;
  auto fn = one ? kv_append_kernel<float, KV_ONE> : kv_append_kernel<float, KV_MANY>;
  if (dtype != GN_DTYPE_F32) fn = one ? kv_append_kernel<uint16_t, KV_ONE> : kv_append_kernel<uint16_t, KV_MANY>;
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(nt), sh, s, a);
  return hipGetLastError();
}

}  // namespace gn
