// Device code shared by the cache's writer (k_kv.hip) and its readers.
#pragma once
#include "gn_serve.h"

namespace gn {

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

// ---- what is stored ----
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
__host__ __device__ inline uint32_t inverse(int n) { return n > 1 ? (uint32_t)(((1ull << 32) + n - 1) / n) : 0; }

// A sequence as the call's arrays describe it; n = 0 where there is nothing to
// do.  bad: its bounds lie outside the inputs or the call's limit, or it has more
// new tokens than the launch was made for.
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

}  // namespace gn
