// The paged 8-bit cache of rotated keys and values: appending to it and
// attention over it.
//
// Layout: K pages [page][kv head][token][R], V pages [page][kv head][R][token]
// in E4M3 with a power-of-two scale per (page, kv head) for each.  V lies
// transposed so that attention's two products read both caches as their matrix
// operands lie in registers, 16 bytes a lane, with no pass through LDS; the
// writer owns a whole block anyway (its scale covers the block).
#include "gn_serve.h"

namespace gn {
namespace {

__device__ __forceinline__ float bf16_f32(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
// round to nearest even; NaN stays NaN
__device__ __forceinline__ uint16_t f32_bf16(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}
template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ float get(const float *p) { return *p; }
  static __device__ __forceinline__ void put(float *p, float v) { *p = v; }
  static __device__ __forceinline__ void get4(const float *p, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4 *>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  }
  static __device__ __forceinline__ void put4(float *p, const float (&v)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct Elem<uint16_t> {
  static __device__ __forceinline__ float get(const uint16_t *p) { return bf16_f32(*p); }
  static __device__ __forceinline__ void put(uint16_t *p, float v) { *p = f32_bf16(v); }
  static __device__ __forceinline__ void get4(const uint16_t *p, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2 *>(p);
    v[0] = bf16_f32((uint16_t)x.x); v[1] = bf16_f32((uint16_t)(x.x >> 16));
    v[2] = bf16_f32((uint16_t)x.y); v[3] = bf16_f32((uint16_t)(x.y >> 16));
  }
  static __device__ __forceinline__ void put4(uint16_t *p, const float (&v)[4]) {
    uint2 x;
    x.x = f32_bf16(v[0]) | ((uint32_t)f32_bf16(v[1]) << 16);
    x.y = f32_bf16(v[2]) | ((uint32_t)f32_bf16(v[3]) << 16);
    *reinterpret_cast<uint2 *>(p) = x;
  }
};

// A sequence as the call's arrays describe it; n = 0 where there is nothing to
// do.  bad: its bounds lie outside the inputs or the table, or it is larger
// than the sizes the launch was made for.
struct Seq {
  int start, n, len;
  bool bad;
};
__device__ __forceinline__ Seq kv_seq(const KvArgs &c, int b, int limit) {
  Seq s;
  s.start = c.starts[b];
  const int end = c.starts[b + 1];
  s.len = c.lens[b];
  s.bad = s.start < 0 || end < s.start || end > c.N || end - s.start > c.max_new || s.len < 0 ||
          (int64_t)s.len + (end - s.start) > limit;
  s.n = s.bad ? 0 : end - s.start;
  return s;
}

// ---------------------------------------------------------------- append
// x * 2^-e rounded to E4M3 (|x| <= 448 2^e by the choice of e); what is not
// finite becomes NaN (0x7f)
__device__ __forceinline__ uint32_t to_e4m3(float x, float inv) {
  const uint32_t b = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x * inv, 0.f, 0, false) & 0xff;
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? 0x7fu : b;
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

// four values of one token's head from column d on, rotated (rot) in float64 and
// rounded once: products of two float32 are exact there, so every reader of
// the definition gets the same float32.  Columns beyond hd are 0.
template <typename T>
__device__ __forceinline__ void load_rotated(const T *row, const float *cs, const float *sn, int hd, int d, bool rot,
                                             int vec, float (&o)[4]) {
  const int half = hd >> 1;
  if (vec) {  // hd a multiple of 8: the four and their partners lie on one side of the middle
    if (d >= hd) {
      o[0] = o[1] = o[2] = o[3] = 0.f;
      return;
    }
    Elem<T>::get4(row + d, o);
    if (!rot) return;
    const bool up = d >= half;
    float p[4];
    Elem<T>::get4(row + (up ? d - half : d + half), p);
    const float4 c4 = *reinterpret_cast<const float4 *>(cs + (up ? d - half : d));
    const float4 s4 = *reinterpret_cast<const float4 *>(sn + (up ? d - half : d));
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double a = (double)o[i] * (double)c[i], b = (double)p[i] * (double)s[i];
      o[i] = (float)(up ? b + a : a - b);
    }
    return;
  }
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

constexpr int KV_SLOTS = 8;  // four-value groups of new tokens a thread holds

// One workgroup per (sequence, touched page, kv head, K or V): it owns that
// block, so its new maximum, the growth of its scale and the bytes of tokens
// already there need no other workgroup.  New values stay in registers between
// the maximum and the rounding.  Blocks behind those rotate the queries.
// Bound by latency for single tokens (a chain of table, row and scale reads,
// one reduction) and by memory for prompts.
template <typename T>
__global__ __launch_bounds__(1024) void kv_append_kernel(KvAppendArgs a) {
  extern __shared__ __align__(16) uint8_t lds[];
  const KvArgs &c = a.c;
  const int tid = threadIdx.x, NT = blockDim.x;
  const int items = c.B * a.touch * c.KVH * 2;
  const int limit0 = c.max_pages * c.P;
  const int limit = a.cs ? min(limit0, a.rope_len) : limit0;
  const int half = c.hd >> 1;
  if ((int)blockIdx.x >= items) {  // queries: qtok tokens of one sequence
    const int i = blockIdx.x - items, b = i / a.qtiles;
    const Seq s = kv_seq(c, b, limit);
    const int t0 = (i % a.qtiles) * a.qtok, t1 = min(t0 + a.qtok, s.n);
    const T *q = (const T *)a.q;
    T *qo = (T *)a.qo;
    const int per = (half + 3) >> 2, pairs = a.H * per;  // groups of four pairs
    for (int g = tid; g < (t1 - t0) * pairs; g += NT) {
      const int t = t0 + g / pairs, h = g % pairs / per, d = (g % per) * 4;
      const T *row = q + (int64_t)(s.start + t) * a.qs + h * c.hd;
      T *out = qo + (int64_t)(s.start + t) * a.qos + h * c.hd;
      const float *cs = a.cs ? a.cs + (int64_t)(s.len + t) * half : nullptr;
      const float *sn = a.cs ? a.sn + (int64_t)(s.len + t) * half : nullptr;
      float lo[4], hi[4];
      if (a.vec) {
        load_rotated(row, cs, sn, c.hd, d, a.cs != nullptr, 1, lo);
        load_rotated(row, cs, sn, c.hd, d + half, a.cs != nullptr, 1, hi);
        Elem<T>::put4(out + d, lo);
        Elem<T>::put4(out + d + half, hi);
      } else {
        load_rotated(row, cs, sn, c.hd, d, a.cs != nullptr, 0, lo);
        load_rotated(row, cs, sn, c.hd, d + half, a.cs != nullptr, 0, hi);
        for (int j = 0; j < 4 && d + j < half; ++j) {
          Elem<T>::put(out + d + j, lo[j]);
          Elem<T>::put(out + d + j + half, hi[j]);
        }
      }
    }
    if (c.hd & 1)  // the middle-less last column
      for (int g = tid; g < (t1 - t0) * a.H; g += NT) {
        const int t = t0 + g / a.H, h = g % a.H;
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
  const int page = c.table[(int64_t)b * c.max_pages + pi];
  if (page < 0 || page >= c.pages) {
    if (c.bad && tid == 0) c.bad[b] = 1;
    return;
  }
  const int R = c.R, P = c.P, per = R >> 2;
  const int64_t blk = (int64_t)page * c.KVH + h;
  uint8_t *dst = (which ? c.v : c.k) + blk * P * R;
  float *sp = (which ? c.vs : c.ks) + blk;
  const bool rot = !which && a.cs;
  const T *x = (const T *)a.x[which] + h * c.hd;
  const int groups = (hi - lo) * per;

  float v[KV_SLOTS][4];
  float amax = 0.f;
#pragma unroll
  for (int u = 0; u < KV_SLOTS; ++u) {
    const int g = tid + u * NT;
    if (g >= groups) break;
    const int t = lo + g / per, d = (g % per) * 4;
    const int pos = first + t;
    const T *row = x + (int64_t)(s.start + pos - s.len) * a.xs[which];
    load_rotated(row, rot ? a.cs + (int64_t)pos * half : nullptr, rot ? a.sn + (int64_t)pos * half : nullptr, c.hd, d, rot,
                 a.vec, v[u]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float m = fabsf(v[u][k]);
      if (m <= 3.402823466e38f) amax = fmaxf(amax, m);
    }
  }
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
    const float old = *sp;
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
      const int g = tid + u * NT;
      if (g >= groups) break;
      reinterpret_cast<uint32_t *>(dst + (int64_t)lo * R)[g] = to_e4m3(v[u][0], inv) | to_e4m3(v[u][1], inv) << 8 |
                                                               to_e4m3(v[u][2], inv) << 16 | to_e4m3(v[u][3], inv) << 24;
    }
    return;
  }
  if (hi - lo == 1) {  // one token: a byte of every row
#pragma unroll
    for (int u = 0; u < KV_SLOTS; ++u) {
      const int g = tid + u * NT;
      if (g >= groups) break;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (g * 4 + k < c.hd) dst[(int64_t)(g * 4 + k) * P + lo] = (uint8_t)to_e4m3(v[u][k], inv);
    }
    return;
  }
  const int LP = P + 16;  // rows stay 16-byte aligned
#pragma unroll
  for (int u = 0; u < KV_SLOTS; ++u) {
    const int g = tid + u * NT;
    if (g >= groups) break;
    const int t = lo + g / per, d = (g % per) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) lds[(d + k) * LP + t] = (uint8_t)to_e4m3(v[u][k], inv);
  }
  __syncthreads();
  const int seg = P >> 4;
  for (int g = tid; g < c.hd * seg; g += NT) {
    const int d = g / seg, t = (g % seg) * 16;
    if (t + 16 <= lo || t >= hi) continue;
    if (t >= lo && t + 16 <= hi) {
      *reinterpret_cast<uint4 *>(dst + (int64_t)d * P + t) = *reinterpret_cast<const uint4 *>(lds + d * LP + t);
    } else {
      for (int k = max(t, lo); k < min(t + 16, hi); ++k) dst[(int64_t)d * P + k] = lds[d * LP + k];
    }
  }
}

// ---------------------------------------------------------------- attention
// One wave per (row, query head): 64 keys at a time, a lane each, and the
// weights against V with a lane per column.
template <typename T>
__global__ __launch_bounds__(64) void kv_attn_kernel(KvAttnArgs a) {
  __shared__ float qs[KV_MAX_HEAD];
  __shared__ float ps[64];
  const KvArgs &c = a.c;
  const int lane = threadIdx.x, h = blockIdx.y, b = blockIdx.z, t = blockIdx.x;
  const Seq s = kv_seq(c, b, min(c.max_len, c.max_pages * c.P));
  if (s.bad && c.bad && lane == 0) c.bad[b] = 1;
  if (t >= s.n) return;
  const int kvh = h / a.G, len = a.causal ? s.len + t + 1 : s.len + s.n;
  const T *q = (const T *)a.q + (int64_t)(s.start + t) * a.qs + (int64_t)h * c.hd;
  for (int d = lane; d < c.hd; d += 64) qs[d] = Elem<T>::get(q + d);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  bool any = false;
  for (int j0 = 0; j0 < len; j0 += 64) {
    const int j = j0 + lane;
    int page = -1;
    if (j < len) page = c.table[(int64_t)b * c.max_pages + (j >> c.lgP)];
    const bool on = j < len && page >= 0 && page < c.pages;
    if (j < len && !on && c.bad) c.bad[b] = 1;
    const int64_t blk = on ? (int64_t)page * c.KVH + kvh : 0;
    float x = -INFINITY;
    if (on) {
      const uint8_t *k = c.k + (blk * c.P + (j & (c.P - 1))) * c.R;
      x = 0.f;
      for (int d = 0; d < c.hd; ++d) x += qs[d] * __builtin_amdgcn_cvt_f32_fp8((int)k[d], 0);
      x *= c.ks[blk] * a.scale;
    }
    float mm = x;
    for (int off = 32; off > 0; off >>= 1) mm = fmaxf(mm, __shfl_xor(mm, off, 64));
    any = any || __any(on);
    const float mn = fmaxf(m, mm), safe = mn == -INFINITY ? 0.f : mn;
    const float f = __expf(m - safe), p = on ? __expf(x - safe) : 0.f;
    float sum = p;
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    l = l * f + sum;
    m = mn;
    __syncthreads();
    ps[lane] = on ? p * c.vs[blk] : 0.f;
    __syncthreads();
    for (int u = 0; u < 4; ++u) o[u] *= f;
    for (int jj = 0; jj < 64; ++jj) {
      const int on2 = __shfl((int)on, jj, 64);
      if (!on2) continue;
      const int64_t blk2 = __shfl(page, jj, 64) * (int64_t)c.KVH + kvh;
      const uint8_t *v = c.v + blk2 * c.P * c.R + ((j0 + jj) & (c.P - 1));
      const float w = ps[jj];
      for (int u = 0; u < 4; ++u) {
        const int d = lane + 64 * u;
        if (d < c.hd) o[u] += w * __builtin_amdgcn_cvt_f32_fp8((int)v[(int64_t)d * c.P], 0);
      }
    }
  }
  T *out = (T *)a.out + (int64_t)(s.start + t) * a.os + (int64_t)h * c.hd;
  for (int u = 0; u < 4; ++u) {
    const int d = lane + 64 * u;
    if (d < c.hd) Elem<T>::put(out + d, any ? o[u] / l : 0.f);
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs &a0, int dtype, hipStream_t s) {
  KvAppendArgs a = a0;
  const KvArgs &c = a.c;
  const int most = c.max_new < c.P ? c.max_new : c.P;
  a.touch = (c.max_new + 2 * c.P - 2) / c.P;
  // a thread holds up to 32 new values of a block
  int nt = (most * c.R / (4 * KV_SLOTS) + 63) / 64 * 64;
  nt = nt < 64 ? 64 : nt;
  const int half = c.hd / 2 > 0 ? c.hd / 2 : 1;
  a.qtok = 8192 / (a.H * half);
  a.qtok = a.qtok < 1 ? 1 : a.qtok > c.max_new ? c.max_new : a.qtok;
  a.qtiles = (c.max_new + a.qtok - 1) / a.qtok;
  const int64_t blocks = (int64_t)c.B * a.touch * c.KVH * 2 + (a.qo ? (int64_t)c.B * a.qtiles : 0);
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  const size_t sh = most > 1 ? (size_t)c.R * (c.P + 16) : 0;
  if (dtype == GN_DTYPE_F32)
    hipLaunchKernelGGL(kv_append_kernel<float>, dim3((unsigned)blocks), dim3(nt), sh, s, a);
  else
    hipLaunchKernelGGL(kv_append_kernel<uint16_t>, dim3((unsigned)blocks), dim3(nt), sh, s, a);
  return hipGetLastError();
}

int64_t kv_attn_work_floats(int B, int max_new, int max_len, int H, int KVH, int hd) { return 0; }

hipError_t launch_kv_attn(const KvAttnArgs &a, int dtype, hipStream_t s) {
  const dim3 grid(a.c.max_new, a.H, a.c.B);
  if (dtype == GN_DTYPE_F32)
    hipLaunchKernelGGL(kv_attn_kernel<float>, grid, dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL(kv_attn_kernel<uint16_t>, grid, dim3(64), 0, s, a);
  return hipGetLastError();
}

}  // namespace gn
