// Appending drafted tokens to the paged 8-bit cache: rows that turn by positions of their
// own.  What is stored is what k_kv.hip stores.
#include "gn_kv.h"

namespace gn {
namespace {

constexpr int KV_RUN = 4;  // tokens in a row, of four pairs of columns, that a thread holds

// Queries, whole groups of four pairs: rows and positions are asked for together, and the
// angles as soon as the positions are there.  Three groups a thread (64 trees of up to 64
// tokens, 32 and 8 heads of 128: 25.2 us with the keys and values, two 26.0, four 27.8).
constexpr int KV_TURNS = 3;
template <typename T>
__device__ __forceinline__ void turn_queries(const KvAppendArgs &a, const Seq &s, int tile) {
  constexpr int U = KV_TURNS;
  const int hd = a.c.hd, half = hd >> 1, per = half >> 2, row_groups = a.H * per, NT = blockDim.x, tid = threadIdx.x;
  const int64_t g0 = (int64_t)tile * U * NT;
  if (g0 >= (int64_t)s.n * row_groups) return;
  const int t0 = (int)(g0 / row_groups), first = (int)(g0 % row_groups);
  int t[U], at[U], col[U], pos[U];
  float lo[U][4], hi[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    int g = first + u * NT + tid;
    t[u] = t0;
    if (row_groups >= U * NT) {  // one token's end at most lies between
      t[u] += g >= row_groups;
      g -= g >= row_groups ? row_groups : 0;
    } else {
      t[u] += g / row_groups;
      g %= row_groups;
    }
    const int h = divided(g, a.per_inv, per);
    col[u] = (g - h * per) * 4;
    at[u] = h * hd + col[u];
    pos[u] = a.at[s.start + min(t[u], s.n - 1)];
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const T *row = (const T *)a.q + (int64_t)(s.start + min(t[u], s.n - 1)) * a.qs + at[u];
    Elem<T>::get4(row, lo[u]);
    Elem<T>::get4(row + half, hi[u]);
  }
  float4 cs[U], sn[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t from = (int64_t)((unsigned)pos[u] < (unsigned)a.rope_len ? pos[u] : 0) * half + col[u];
    cs[u] = *reinterpret_cast<const float4 *>(a.cs + from);
    sn[u] = *reinterpret_cast<const float4 *>(a.sn + from);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const float cc[4] = {cs[u].x, cs[u].y, cs[u].z, cs[u].w}, ss[4] = {sn[u].x, sn[u].y, sn[u].z, sn[u].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      turn(lo[u][j], hi[u][j], cc[j], ss[j]);
      if ((unsigned)pos[u] >= (unsigned)a.rope_len) lo[u][j] = hi[u][j] = __uint_as_float(0x7fc00000u);
    }
    if (t[u] >= s.n) continue;
    T *out = (T *)a.qo + (int64_t)(s.start + t[u]) * a.qos + at[u];
    Elem<T>::put4(out, lo[u]);
    Elem<T>::put4(out + half, hi[u]);
  }
}

// One workgroup per (sequence, touched page, kv head, K or V), which owns that block, and
// behind those the queries, as in k_kv.hip.  A thread's rows are KV_RUN tokens that follow
// each other: four bytes of a column of V are a word, and its place is found by one
// division.  Rows of V that are not whole 16-byte pieces are read, filled in and written
// as such.
// Rows or heads that do not allow 4-value accesses are taken a value at a time, twice: for
// the maximum and for the bytes.
// 64 trees of up to 64 tokens, 32 and 8 heads of 128, bfloat16: 20 us, of which 13 without
// the queries; memory would take 10 (49 MB).  The kernel of k_kv.hip, which holds any eight
// groups of four values and finds each one's place anew, took 25; 256 trees of up to 16: 46,
// here 29.  Latency: a chain of bounds, positions, angles, maximum and bytes.
template <typename T>
__global__ __launch_bounds__(1024) void kv_append_at_kernel(KvAppendArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ float red[16];
  const KvArgs &c = a.c;
  const int tid = threadIdx.x, NT = blockDim.x, half = c.hd >> 1;
  const int items = c.B * a.touch * c.KVH * 2, limit = min(c.limit, c.max_pages * c.P);
  const float nan = __uint_as_float(0x7fc00000u);
  if ((int)blockIdx.x >= items) {
    const int i = blockIdx.x - items, b = i / a.qtiles, tile = i % a.qtiles;
    const Seq s = kv_seq(c, b, limit);
    if (a.vec) {
      turn_queries<T>(a, s, tile);
      return;
    }
    // pairs, and an odd head's last column
    const int per = half + (c.hd & 1);
    for (int64_t g = (int64_t)tile * NT + tid; g < (int64_t)s.n * a.H * per; g += (int64_t)a.qtiles * NT) {
      const int t = (int)(g / (a.H * per)), r = (int)(g % (a.H * per)), h = r / per, d = r % per, pos = a.at[s.start + t];
      const bool lost = (unsigned)pos >= (unsigned)a.rope_len;
      const T *q = (const T *)a.q + (int64_t)(s.start + t) * a.qs + h * c.hd;
      T *o = (T *)a.qo + (int64_t)(s.start + t) * a.qos + h * c.hd;
      if (d == half) {
        Elem<T>::put(o + c.hd - 1, lost ? nan : Elem<T>::get(q + c.hd - 1));
        continue;
      }
      const int64_t from = (int64_t)(lost ? 0 : pos) * half + d;
      float x = Elem<T>::get(q + d), y = Elem<T>::get(q + d + half);
      turn(x, y, a.cs[from], a.sn[from]);
      Elem<T>::put(o + d, lost ? nan : x);
      Elem<T>::put(o + d + half, lost ? nan : y);
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
  const int pi = (s.len >> c.lgP) + j;  // page of the sequence
  const int first = pi << c.lgP;        // its first position
  const int lo = max(s.len - first, 0), hi = min(s.len + s.n - first, c.P);
  if (s.n == 0 || hi <= lo) return;
  const int page = c.table[(int64_t)b * c.max_pages + pi];  // the rows do not wait for it
  const int R = c.R, P = c.P;
  // token t of the page is row t of xs and of at
  const T *xs = (const T *)a.x[which] + h * c.hd + (int64_t)(s.start + first - s.len) * a.xs[which];
  const int32_t *at = a.at + (s.start + first - s.len);
  const auto lost = [&](int pos) { return (unsigned)pos >= (unsigned)a.rope_len; };
  if (!which && h == 0 && c.bad)
    for (int t = lo + tid; t < hi; t += NT)
      if (lost(at[t])) c.bad[b] = 1;
  // one value by itself, as a pair's; the last column of an odd head does not turn
  const auto value = [&](int t, int d) {
    const T *row = xs + t * a.xs[which];
    float x = Elem<T>::get(row + d);
    if (which) return x;
    const int pos = at[t];
    if (lost(pos)) return nan;
    if (d < 2 * half) {
      const bool up = d >= half;
      const int k = up ? d - half : d;
      const int64_t from = (int64_t)pos * half + k;
      float y = Elem<T>::get(row + (up ? k : d + half));
      if (up) turn(y, x, a.cs[from], a.sn[from]);
      else turn(x, y, a.cs[from], a.sn[from]);
    }
    return x;
  };

  // this thread's tokens t0 + u and columns d + k, half + d + k
  const int per = c.hd >> 3, run = a.vec ? divided(tid, a.pair_inv, per) : 0;
  const int d = (tid - run * per) * 4, t0 = (lo & ~(KV_RUN - 1)) + run * KV_RUN;
  const auto on = [&](int u) { return t0 + u >= lo && t0 + u < hi; };
  float v[KV_RUN][8];
  float amax = 0.f;
  if (a.vec) {
    const auto row = [&](int u) { return min(max(t0 + u, lo), hi - 1); };
    int pos[KV_RUN];
    if (!which)
#pragma unroll
      for (int u = 0; u < KV_RUN; ++u) pos[u] = at[row(u)];
#pragma unroll
    for (int u = 0; u < KV_RUN; ++u) {
      const T *x = xs + row(u) * a.xs[which] + d;
      float p[4], q[4];
      Elem<T>::get4(x, p);
      Elem<T>::get4(x + half, q);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[u][k] = p[k];
        v[u][4 + k] = q[k];
      }
    }
    if (!which) {
      float4 cs[KV_RUN], sn[KV_RUN];
#pragma unroll
      for (int u = 0; u < KV_RUN; ++u) {
        const int64_t from = (int64_t)(lost(pos[u]) ? 0 : pos[u]) * half + d;
        cs[u] = *reinterpret_cast<const float4 *>(a.cs + from);
        sn[u] = *reinterpret_cast<const float4 *>(a.sn + from);
      }
#pragma unroll
      for (int u = 0; u < KV_RUN; ++u) {
        const float cc[4] = {cs[u].x, cs[u].y, cs[u].z, cs[u].w}, ss[4] = {sn[u].x, sn[u].y, sn[u].z, sn[u].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          turn(v[u][k], v[u][4 + k], cc[k], ss[k]);
          if (lost(pos[u])) v[u][k] = v[u][4 + k] = nan;
        }
      }
    }
    float worst = 0.f;
#pragma unroll
    for (int u = 0; u < KV_RUN; ++u)
#pragma unroll
      for (int k = 0; k < 8; ++k) worst = fmaxf(worst, on(u) ? fabsf(v[u][k]) : 0.f);  // passes NaN by
    amax = worst;
    if (worst == INFINITY) {
      amax = 0.f;
#pragma unroll
      for (int u = 0; u < KV_RUN; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k) amax = fmaxf(amax, on(u) && fabsf(v[u][k]) != INFINITY ? fabsf(v[u][k]) : 0.f);
    }
  } else {
    for (int g = tid; g < (hi - lo) * c.hd; g += NT) {
      const int t = divided(g, a.group_inv, c.hd);
      const float y = fabsf(value(lo + t, g - t * c.hd));
      amax = fmaxf(amax, y == INFINITY ? 0.f : y);
    }
  }
  if (page < 0 || page >= c.pages) {
    if (c.bad && tid == 0) c.bad[b] = 1;
    return;
  }
  const int64_t blk = (int64_t)page * c.KVH + h;
  uint8_t *dst = (which ? c.v : c.k) + blk * P * R;
  float *sp = (which ? c.vs : c.ks) + blk;
  const float old = lo > 0 ? *sp : 0.f;
  for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
  if ((tid & 63) == 0) red[tid >> 6] = amax;
  __syncthreads();
  for (int w = 0; w < NT >> 6; ++w) amax = fmaxf(amax, red[w]);
  float scale = block_scale(amax);
  if (lo > 0) {
    if (old > scale) {
      scale = old;
    } else if (old < scale) {  // the tokens already here move to the larger scale
      const float ratio = old / scale;
      if (!which) {
        uint32_t *w = reinterpret_cast<uint32_t *>(dst);
        for (int g = tid; g < lo * R / 4; g += NT) {
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
    __syncthreads();  // every thread has read the old scale, and its bytes are there
  }
  if (tid == 0) *sp = scale;
  const float inv = 1.f / scale;

  if (!a.vec) {
    for (int g = tid; g < (hi - lo) * R; g += NT) {
      const int q = divided(g, a.pair_inv, R), t = lo + q, e = g - q * R;
      if (e < c.hd) dst[which ? e * P + t : t * R + e] = (uint8_t)to_e4m3(value(t, e), inv);
      else if (!which) dst[t * R + e] = 0;
    }
    return;
  }
  if (!which) {
#pragma unroll
    for (int u = 0; u < KV_RUN; ++u) {
      if (!on(u)) continue;
      uint8_t *p = dst + (t0 + u) * R + d;
      *reinterpret_cast<uint32_t *>(p) = to_e4m3(v[u][0], v[u][1], v[u][2], v[u][3], inv);
      *reinterpret_cast<uint32_t *>(p + half) = to_e4m3(v[u][4], v[u][5], v[u][6], v[u][7], inv);
    }
    const int pad = (R - c.hd) >> 2;
    if (pad)
      for (int g = tid; g < (hi - lo) * pad; g += NT)
        *reinterpret_cast<uint32_t *>(dst + (lo + g / pad) * R + c.hd + g % pad * 4) = 0;
    return;
  }
  const int LP = P + 16;  // rows stay 16-byte aligned
  if (t0 < hi) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      *reinterpret_cast<uint32_t *>(lds + (d + (k & 3) + (k >> 2) * half) * LP + t0) =
          to_e4m3(v[0][k], v[1][k], v[2][k], v[3][k], inv);
  }
  __syncthreads();
  const int seg0 = lo >> 4, segs = ((hi - 1) >> 4) - seg0 + 1;
  for (int g = tid; g < c.hd * segs; g += NT) {
    const int e = segs == 1 ? g : g / segs, t = (seg0 + (segs == 1 ? 0 : g % segs)) * 16;
    uint4 *to = reinterpret_cast<uint4 *>(dst + (int64_t)e * P + t);
    uint4 x = *reinterpret_cast<const uint4 *>(lds + e * LP + t);
    if (t < lo || t + 16 > hi) {
      const uint4 was = *to;
      const auto mix = [&](uint32_t was_, uint32_t x_, int t_) {
        uint32_t m = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) m |= t_ + k >= lo && t_ + k < hi ? 0xffu << (8 * k) : 0u;
        return (was_ & ~m) | (x_ & m);
      };
      x = make_uint4(mix(was.x, x.x, t), mix(was.y, x.y, t + 4), mix(was.z, x.z, t + 8), mix(was.w, x.w, t + 12));
    }
    *to = x;
  }
}

}  // namespace

hipError_t launch_kv_append_at(const KvAppendArgs &a0, int dtype, hipStream_t s) {
  KvAppendArgs a = a0;
  const KvArgs &c = a.c;
  const int most = c.max_new < c.P ? c.max_new : c.P;
  a.touch = (c.max_new + 2 * c.P - 2) / c.P;
  // runs begin at a multiple of their length: one more where the tokens do not
  int runs = (most + 2 * KV_RUN - 2) / KV_RUN;
  runs = runs < c.P / KV_RUN ? runs : c.P / KV_RUN;
  // 32 runs of 32 at most; values by themselves: 64 trees of up to 64 tokens, heads of 100,
  // float32, in 50 us, with 832 threads 77
  const int nt = a.vec ? (runs * (c.hd / 8) + 63) / 64 * 64 : 256;
  const int64_t turns = (int64_t)c.max_new * a.H * (a.vec ? c.hd / 8 : (c.hd + 1) / 2);
  const int64_t per_wg = (int64_t)(a.vec ? KV_TURNS : 4) * nt, qtiles = (turns + per_wg - 1) / per_wg;
  a.qtiles = qtiles < 1 ? 1 : (int)qtiles;
  a.per_inv = inverse(c.hd / 8);
  a.group_inv = inverse(c.hd);
  a.pair_inv = inverse(a.vec ? c.hd / 8 : c.R);
  const int64_t blocks = (int64_t)c.B * a.touch * c.KVH * 2 + (a.qo ? (int64_t)c.B * a.qtiles : 0);
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  const size_t sh = a.vec ? (size_t)c.R * (c.P + 16) : 0;
  if (dtype == GN_DTYPE_F32) hipLaunchKernelGGL(kv_append_at_kernel<float>, dim3((unsigned)blocks), dim3(nt), sh, s, a);
  else hipLaunchKernelGGL(kv_append_at_kernel<uint16_t>, dim3((unsigned)blocks), dim3(nt), sh, s, a);
  return hipGetLastError();
}

}  // namespace gn
