// Rules on logits before a token is drawn: penalties for repeated tokens, biases, masks.
#include "gn_kv.h"

namespace gn {
namespace {

constexpr uint32_t IN_PROMPT = 1u << 31;  // in a token's count: it stands in the prompt

// 16 bytes of logits
template <typename T>
struct Pack {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void get(const T *p, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      float x[4];
      Elem<T>::get4(p + i, x);
      for (int k = 0; k < 4; ++k) v[i + k] = x[k];
    }
  }
};
template <>
__device__ __forceinline__ void Pack<uint16_t>::get(const uint16_t *p, float (&v)[8]) {
  const uint4 x = *reinterpret_cast<const uint4 *>(p);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = bf16_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
}
__device__ __forceinline__ void put(float *p, const float (&v)[4]) { Elem<float>::put4(p, v); }
__device__ __forceinline__ void put(uint16_t *p, const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = f32_bf16(v[2 * i]) | (uint32_t)f32_bf16(v[2 * i + 1]) << 16;
  *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// One workgroup of NT threads per (TILE vocabulary entries, row).  Its logits and their
// mask wait in registers while it counts the row's text for its own entries in LDS and finds
// their last biases (whole numbers: no order shows in them).
// Tiles begin where the row's memory is 16-byte aligned, `lead` entries before a multiple
// of their size.
// Bound by memory: 128 rows of 131072 float32, every rule, texts of up to 4096, in 34 us
// (136 MB, 4.0 TB/s; 28 with a mask alone; a copy of the logits takes 26); the rest is the
// text, which every tile of a row reads again (of 8192 entries: 35 us, of 2048: 38).
// Loops that waited for a load at a time took 67.
constexpr int NT = 512, PER = 8, TILE = NT * PER;
template <typename T>
__global__ __launch_bounds__(NT) void logits_kernel(LogitArgs a) {
  constexpr int E = Pack<T>::N, G = PER / E, AHEAD = 4;
  __shared__ __align__(16) uint32_t count[TILE], last[TILE];
  const int b = blockIdx.y, tid = threadIdx.x;
  const gn_logit_rules &r = a.r;
  const T *z = (const T *)a.z + b * a.zs;
  T *out = (T *)a.out + b * a.os;
  const int lead = (int)((uintptr_t)out / sizeof(T)) & (E - 1);
  const bool same = ((int)((uintptr_t)z / sizeof(T)) & (E - 1)) == lead;
  const int v0 = (int)blockIdx.x * TILE - lead;
  if (v0 >= a.V) return;

  const auto length = [&](const int32_t *lens, int64_t stride) {
    return (int)(stride && lens ? min((int64_t)max(lens[b], 0), stride) : stride);
  };
  const int tokens = length(r.token_lens, r.tokens_stride), biases = length(r.bias_lens, r.bias_stride);
  const int32_t *text = r.tokens + b * r.tokens_stride, *named = r.bias_ids + b * r.bias_stride;
  // Loads return in the order of their issue: the first of the lists' ids are asked for
  // first, so that LDS works on them while the logits are on their way.  Branches around
  // loads are the whole workgroup's: loads under way are counted across them.
  int id[AHEAD], named_id = -1;
  const auto load = [&](const int32_t *ids, int n, int i0) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) id[k] = ids[min(i0 + k * NT, n - 1)];
  };
  if (tokens) load(text, tokens, tid);
  if (biases) named_id = named[min(tid, biases - 1)];

  // the u-th 16 bytes of this thread: entries from at(u) on
  const auto at = [&](int u) { return v0 + (u * NT + tid) * E; };
  const bool inside = v0 >= 0 && v0 + TILE <= a.V;
  float x[G][E];
  if (inside && same) {
#pragma unroll
    for (int u = 0; u < G; ++u) Pack<T>::get(z + at(u), x[u]);
  } else {
#pragma unroll
    for (int u = 0; u < G; ++u)
#pragma unroll
      for (int k = 0; k < E; ++k) x[u][k] = Elem<T>::get(z + min(max(at(u) + k, 0), a.V - 1));
  }
  const int64_t row = r.allowed_row ? r.allowed_row[b] : b;
  const bool masked = r.allowed && row >= 0 && row < r.allowed_rows;
  uint32_t bits[G], more[G];  // the mask's word that holds at(u), the one after it
  if (masked) {
    const uint32_t *may = r.allowed + row * r.allowed_stride;
    const int words = (a.V + 31) >> 5;
#pragma unroll
    for (int u = 0; u < G; ++u) bits[u] = may[min(max(at(u), 0) >> 5, words - 1)];
    if (lead) {
#pragma unroll
      for (int u = 0; u < G; ++u) more[u] = may[min((max(at(u), 0) >> 5) + 1, words - 1)];
    }
  }
  const int prompt = tokens && r.prompt_lens ? r.prompt_lens[b] : 0;
  const float rep = r.repetition ? r.repetition[b] : 1.f, freq = r.frequency ? r.frequency[b] : 0.f,
              pres = r.presence ? r.presence[b] : 0.f;

  const auto place = [&](int i) { return i >= 0 && i < a.V ? (uint32_t)(i - v0) : ~0u; };
  const auto count_loaded = [&](int i0) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = i0 + k * NT;
      const uint32_t p = place(id[k]);
      if (i >= tokens || p >= (uint32_t)TILE) continue;
      if (i < prompt) atomicOr(&count[p], IN_PROMPT);
      else atomicAdd(&count[p], 1u);
    }
  };
  const auto counted = [&]() {
    if (!tokens) return;
    count_loaded(tid);  // not in the loop, where they would wait for the logits too
    for (int i0 = tid + AHEAD * NT; i0 < tokens; i0 += AHEAD * NT) {
      load(text, tokens, i0);
      count_loaded(i0);
    }
  };
  const auto latest = [&]() {
    for (int i = tid; i < biases; i += NT) {
      const uint32_t p = place(i == tid ? named_id : named[i]);
      if (p < (uint32_t)TILE) atomicMax(&last[p], (uint32_t)i + 1);
    }
  };
  // f(u, k, what LDS holds) of this thread's entries for which it holds something
  const auto marked = [&](const uint32_t *what, auto &&f) {
    uint32_t n[G][E];
#pragma unroll
    for (int u = 0; u < G; ++u)
#pragma unroll
      for (int k = 0; k < E; k += 4)
        *reinterpret_cast<uint4 *>(&n[u][k]) = *reinterpret_cast<const uint4 *>(what + (u * NT + tid) * E + k);
#pragma unroll
    for (int u = 0; u < G; ++u) {
      uint32_t any = 0;
#pragma unroll
      for (int k = 0; k < E; ++k) any |= n[u][k];
      if (!any) continue;
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (n[u][k]) x[u][k] = f(x[u][k], n[u][k]);
    }
  };
  const auto penalised = [&](float y, uint32_t n) {
    if (rep > 0.f) y = y > 0.f ? y / rep : y * rep;
    const uint32_t later = n & ~IN_PROMPT;
    return later ? y - freq * (float)later - pres : y;
  };
  const auto biased = [&](float y, uint32_t n) { return y + r.bias[b * r.bias_stride + n - 1]; };
  if (tokens || biases) {
#pragma unroll
    for (int i = 0; i < PER / 4; ++i)
      reinterpret_cast<uint4 *>(count)[i * NT + tid] = reinterpret_cast<uint4 *>(last)[i * NT + tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    counted();
    latest();
    __syncthreads();
    marked(count, penalised);
    marked(last, biased);
  }

  if (masked) {
#pragma unroll
    for (int u = 0; u < G; ++u) {
      const int v = at(u);
      uint32_t w = bits[u] >> (v & 31);
      if (lead) w = v < 0 ? bits[u] << (-v & 31) : (uint32_t)((((uint64_t)more[u] << 32) | bits[u]) >> (v & 31));
#pragma unroll
      for (int k = 0; k < E; ++k) x[u][k] = w >> k & 1 ? x[u][k] : -INFINITY;
    }
  }
  if (inside) {
#pragma unroll
    for (int u = 0; u < G; ++u) put(out + at(u), x[u]);
    return;
  }
#pragma unroll
  for (int u = 0; u < G; ++u) {
    const int v = at(u);
    if (v >= 0 && v + E <= a.V) {
      put(out + v, x[u]);
    } else {
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (v + k >= 0 && v + k < a.V) Elem<T>::put(out + v + k, x[u][k]);
    }
  }
}

template <typename T>
hipError_t logits_run(const LogitArgs &a, hipStream_t s) {
  const int most = a.V + Pack<T>::N - 1;  // a row's lead is known to the kernel
  hipLaunchKernelGGL(logits_kernel<T>, dim3((most + TILE - 1) / TILE, a.B), dim3(NT), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_logits_adjust(const LogitArgs &a, int dtype, hipStream_t s) {
  return dtype == GN_DTYPE_F32 ? logits_run<float>(a, s) : logits_run<uint16_t>(a, s);
}

}  // namespace gn
