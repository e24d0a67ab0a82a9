// Rules on logits before a token is drawn: penalties for repeated tokens, biases, masks.
#include "gn_kv.h"

namespace gn {
namespace {

constexpr uint32_t IN_TEXT = 1u << 31;  // in a token's count: it stands in the prompt

// One workgroup per (tile of TILE vocabulary entries, row).  It counts the row's history
// and finds its biases for its own entries in LDS (whole numbers: no order shows in
// them), then passes over the logits once.
constexpr int TILE = 2048;
template <typename T>
__global__ __launch_bounds__(256) void logits_kernel(LogitArgs a) {
  __shared__ uint32_t count[TILE], last[TILE];
  const int b = blockIdx.y, v0 = blockIdx.x * TILE, nv = min(TILE, a.V - v0), tid = threadIdx.x;
  const gn_logit_rules &r = a.r;
  const int64_t tokens = r.tokens_stride ? min((int64_t)max(r.token_lens ? r.token_lens[b] : (int)r.tokens_stride, 0), r.tokens_stride) : 0;
  const int64_t biases = r.bias_stride ? min((int64_t)max(r.bias_lens ? r.bias_lens[b] : (int)r.bias_stride, 0), r.bias_stride) : 0;
  const int64_t prompt = r.prompt_lens ? r.prompt_lens[b] : 0;
  for (int i = tid; i < TILE; i += 256) count[i] = last[i] = 0;
  __syncthreads();
  const int32_t *ids = r.tokens + b * r.tokens_stride, *bids = r.bias_ids + b * r.bias_stride;
  for (int64_t i = tid; i < tokens; i += 256) {
    const uint32_t v = (uint32_t)(ids[i] - v0);
    if (ids[i] < v0 || v >= (uint32_t)nv) continue;
    if (i < prompt) atomicOr(&count[v], IN_TEXT);
    else atomicAdd(&count[v], 1u);
  }
  for (int64_t i = tid; i < biases; i += 256) {
    const uint32_t v = (uint32_t)(bids[i] - v0);
    if (bids[i] < v0 || v >= (uint32_t)nv) continue;
    atomicMax(&last[v], (uint32_t)i + 1);
  }
  __syncthreads();
  const float rep = r.repetition ? r.repetition[b] : 1.f, freq = r.frequency ? r.frequency[b] : 0.f,
              pres = r.presence ? r.presence[b] : 0.f;
  const bool repeats = rep > 0.f;
  int64_t row = r.allowed_row ? r.allowed_row[b] : b;
  const bool masked = r.allowed && row >= 0 && row < r.allowed_rows;
  const T *z = (const T *)a.z + b * a.zs + v0;
  T *out = (T *)a.out + b * a.os + v0;
  for (int i = tid; i < nv; i += 256) {
    float x = Elem<T>::get(z + i);
    const uint32_t n = count[i];
    if (n) {
      if (repeats) x = x > 0.f ? x / rep : x * rep;
      const uint32_t later = n & ~IN_TEXT;
      if (later) x = x - freq * (float)later - pres;
    }
    if (last[i]) x += r.bias[b * r.bias_stride + last[i] - 1];
    if (masked && !(r.allowed[row * r.allowed_stride + ((v0 + i) >> 5)] >> ((v0 + i) & 31) & 1)) x = -INFINITY;
    Elem<T>::put(out + i, x);
  }
}

}  // namespace

hipError_t launch_logits_adjust(const LogitArgs &a, int dtype, hipStream_t s) {
  const dim3 grid((a.V + TILE - 1) / TILE, a.B);
  if (dtype == GN_DTYPE_F32) hipLaunchKernelGGL(logits_kernel<float>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(logits_kernel<uint16_t>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace gn
