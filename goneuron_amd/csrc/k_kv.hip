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
// x * 2^-e rounded to E4M3 (|x| <= 448 2^e by the choice of e); what is not
// finite becomes NaN (0x7f)
__device__ __forceinline__ uint32_t to_e4m3(float x, float inv) {
  const uint32_t b = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x * inv, 0.f, 0, false) & 0xff;
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? 0x7fu : b;
}
// four of them
__device__ __forceinline__ uint32_t to_e4m3(float x, float y, float z, float w, float inv) {
  const uint32_t most = max(max(__float_as_uint(x) & 0x7fffffffu, __float_as_uint(y) & 0x7fffffffu),
                            max(__float_as_uint(z) & 0x7fffffffu, __float_as_uint(w) & 0x7fffffffu));
  if (most >= 0x7f800000u) return to_e4m3(x, inv) | to_e4m3(y, inv) << 8 | to_e4m3(z, inv) << 16 | to_e4m3(w, inv) << 24;
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x * inv, y * inv, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z * inv, w * inv, lo, true);
}
// a stored byte under a larger scale; NaN stays
__device__ __forceinline__ uint32_t rescaled(uint32_t byte, float ratio) {
  if ((byte & 0x7f) == 0x7f) return byte;
  const float x = __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x * ratio, 0.f, 0, false) & 0xff;
}
// smallest power of two s >= 2^-100 with amax / s <= 448
__device__ __forceinline__ float block_scale(float amax) {
  const uint32_t u = __float_as_uint(amax / 448.f);
  int e = (int)(u >> 23) - 127 + ((u & 0x7fffffu) ? 1 : 0);
  e = max(e, KV_MAX_SCALE_EXP);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// a pair turned by an angle, in float64 and rounded once
__device__ __forceinline__ void turn(float &x, float &y, float c, float s) {
  const double a = (double)x * (double)c - (double)y * (double)s, b = (double)x * (double)s + (double)y * (double)c;
  x = (float)a;
  y = (float)b;
}
// four values of one token's head from column d on, rotated (rot) in float64 and
// rounded once: products of two float32 are exact there, so every reader of
// the definition gets the same float32.  Columns beyond hd are 0.
template <typename T>
__device__ __forceinline__ void load_rotated(const T *row, const float *cs, const float *sn, int hd, int d, bool rot,
                                             float (&o)[4]) {
  const int half = hd >> 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = d + i;
    o[i] = j < hd ? Elem<T>::get(row + j) : 0.f;
    if (rot && j < 2 * half) {  // the last column of an odd head does not turn
      const bool up = j >= half;
      const int t = up ? j - half : j;
      const float p = Elem<T>::get(row + (up ? t : j + half));
      const double a = (double)o[i] * (double)cs[t], b = (double)p * (double)sn[t];
      o[i] = (float)(up ? b + a : a - b);
    }
  }
}

// g / n by ceil(2^32 / n), exact while g n < 2^32: a division takes twenty times as long
__device__ __forceinline__ int divided(int g, uint32_t inv, int n) { return n == 1 ? g : (int)__umulhi((uint32_t)g, inv); }
inline uint32_t inverse(int n) { return n > 1 ? (uint32_t)(((1ull << 32) + n - 1) / n) : 0; }

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
