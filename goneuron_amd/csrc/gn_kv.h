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
