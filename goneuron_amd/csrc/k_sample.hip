// Sampling: temperature, top-k, top-p and min-p over rows of logits and one draw
// a row.
//
// Every weight exp((z - max) / T) is a float64 exponential rounded to a whole
// multiple of 2^-43, and every sum an integer one: sums of rows cut into chunks,
// over atomics and over prefixes are then the same number whatever their order,
// and a comparison with a border (top-p's share, the draw) can be made anywhere.
//
// Rows are cut into chunks, a workgroup each.  The logits are read by four passes
// (maximum, histogram, candidates, kept weights), all but the first out of cache:
// the histogram's 1024 bins of 1/32 in the exponent fix the bins in which top-k and
// top-p cut, only their elements are then selected among exactly, by
// radix over (logit, falling index), so that equal logits go by the lowest index.
#include "gn_serve.h"

namespace gn {
namespace {

constexpr int SM_BINS = 1024;
constexpr int SM_PER = 32;        // bins per unit of the exponent
constexpr int SM_CAP = 4096;      // candidates of a row kept in a list
constexpr int SM_MASS_BITS = 43;
constexpr int SM_MAX_CHUNKS = 256;

struct RowState {
  uint64_t tau;        // kept: elements whose key is at least this
  uint64_t mass_k;     // mass of the bins before kbin
  uint64_t mass_p;     // ... before plo
  uint64_t total;
  uint32_t r;          // rank of the last kept element inside kbin
  uint32_t nlist;      // candidates found (the list holds the first SM_CAP)
  int32_t kbin, plo, phi;  // -1: top-k / top-p does not cut
  int32_t pad;
};

struct SampleWs {
  uint64_t *mass, *csum, *list;
  RowState *st;
  uint32_t *count;
  float *cmax;
  int chunk, C;
};

__host__ __device__ inline size_t up64(size_t n) { return (n + 63) / 64 * 64; }

// the cut of a row into chunks: enough workgroups to fill the card, chunks long
// enough that the histogram's flush (1024 bins) stays small beside them
inline int sample_chunk(int B, int V) {
  int chunk = 4096;
  while (chunk < 16384 && (int64_t)B * ((V + chunk - 1) / chunk) > 2048) chunk *= 2;
  return chunk;
}
size_t sample_carve(char *base, int B, int V, SampleWs *w) {
  SampleWs t{};
  t.chunk = sample_chunk(B, V);
  t.C = (V + t.chunk - 1) / t.chunk;
  size_t off = 0;
  const auto take = [&](size_t bytes) {
    char *p = base ? base + off : nullptr;
    off += up64(bytes);
    return p;
  };
  t.mass = (uint64_t *)take((size_t)B * SM_BINS * 8);
  t.csum = (uint64_t *)take((size_t)B * t.C * 8);
  t.list = (uint64_t *)take((size_t)B * SM_CAP * 8);
  t.st = (RowState *)take((size_t)B * sizeof(RowState));
  t.count = (uint32_t *)take((size_t)B * SM_BINS * 4);
  t.cmax = (float *)take((size_t)B * t.C * 4);
  if (w) *w = t;
  return off;
}

template <typename T>
__device__ __forceinline__ float logit(T x);
template <>
__device__ __forceinline__ float logit<float>(float x) { return x; }
template <>
__device__ __forceinline__ float logit<uint16_t>(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// f(i, z) over [lo, hi), the elements dealt to the workgroup's threads, 16 bytes
// at a time where rows allow it (lo is a multiple of the chunk)
template <typename T, typename F>
__device__ __forceinline__ void each(const T *row, int lo, int hi, int vec, F f) {
  constexpr int N = 16 / sizeof(T);
  if (vec) {
    const int full = lo + (hi - lo) / N * N;
    for (int i = lo + threadIdx.x * N; i < full; i += blockDim.x * N) {
      const uint4 q = *reinterpret_cast<const uint4 *>(row + i);
      const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
      for (int j = 0; j < N; ++j) f(i + j, logit<T>(e[j]));
    }
    lo = full;
  }
  for (int i = lo + threadIdx.x; i < hi; i += blockDim.x) f(i, logit<T>(row[i]));
}

__device__ __forceinline__ bool usable(float z) { return z > -INFINITY; }  // neither NaN nor -inf
// rising with the logit, then with the falling index; -0 is 0
__device__ __forceinline__ uint64_t key_of(float z, int i) {
  const uint32_t u = __float_as_uint(z + 0.f);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)k << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float z_of(uint64_t key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// (z - max) / T in float64, falling with z; 0 for the maximum itself, also where
// it is infinite
__device__ __forceinline__ double scaled(float z, float m, double invT) {
  return z == m ? 0.0 : ((double)z - (double)m) * invT;
}
__device__ __forceinline__ int bin_of(double t) {
  const double x = t * -(double)SM_PER;
  return x < (double)(SM_BINS - 1) ? (int)x : SM_BINS - 1;
}
__device__ __forceinline__ double weight_scaled(double t, int up) {  // 2^up exp(t); 0 far below
  if (!(t > -40.0)) return 0.0;
  double n;
  const double r = exp_r10(t, n);
  return __builtin_ldexp(__builtin_fma(expm1_poly(r), r, 1.0), (int)n + up);
}
// a number of [0, 2^43] to the nearest whole one
__device__ __forceinline__ uint64_t whole(double w) {
  return (uint64_t)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}
__device__ __forceinline__ uint64_t mass_of(double t) { return whole(weight_scaled(t, SM_MASS_BITS)); }

struct RowSet {
  bool greedy, k_on, p_on;
  double invT;
  int k;
  float p, minp;
};
__device__ __forceinline__ RowSet row_set(const SampleArgs &a, int b) {
  RowSet s;
  const float T = a.temperature ? a.temperature[b] : 1.f;
  s.greedy = !(T > 0.f);
  s.invT = s.greedy ? 1.0 : 1.0 / (double)T;
  s.k = a.top_k ? a.top_k[b] : 0;
  s.k_on = s.k > 0;
  s.p = a.top_p ? a.top_p[b] : 1.f;
  s.p_on = s.p < 1.f;
  s.minp = a.min_p ? a.min_p[b] : 0.f;
  return s;
}
// whether the row needs the histogram
__device__ __forceinline__ bool cuts(const RowSet &s) { return !s.greedy && (s.k_on || s.p_on); }

template <typename X, typename F>
__device__ __forceinline__ X wave_reduce(X v, F f) {
  for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o, 64));
  return v;
}
template <typename X, typename F>
__device__ __forceinline__ X block_reduce(X v, X *sh, F f) {  // sh: 16 values
  v = wave_reduce(v, f);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = f(v, sh[w]);
  return v;
}
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a + b; }
};
struct Or {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a | b; }
};
// running sum over the workgroup's threads, this one's value included
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *sh) {  // sh: 16 values
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t x = __shfl_up(v, o, 64);
    if (lane >= o) v += x;
  }
  __syncthreads();
  if (lane == 63) sh[w] = v;
  __syncthreads();
  for (int i = 0; i < w; ++i) v += sh[i];
  return v;
}
__device__ __forceinline__ float row_max(const SampleWs &w, int b, float *sh) {
  float m = -INFINITY;
  for (int i = threadIdx.x; i < w.C; i += blockDim.x) m = fmaxf(m, w.cmax[(int64_t)b * w.C + i]);
  return block_reduce(m, sh, Max());
}

// the chunk's largest logit; clears what the later passes add to
template <typename T>
__global__ __launch_bounds__(256) void sample_max_kernel(SampleArgs a, SampleWs w, int vec) {
  __shared__ float sh[16];
  const int c = blockIdx.x, b = blockIdx.y;
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  for (int i = c * 256 + threadIdx.x; i < SM_BINS; i += w.C * 256) {
    w.mass[(int64_t)b * SM_BINS + i] = 0;
    w.count[(int64_t)b * SM_BINS + i] = 0;
  }
  if (c == 0 && threadIdx.x == 0) {
    w.st[b].tau = 0;
    w.st[b].nlist = 0;
  }
  float m = -INFINITY;
  each<T>(row, c * w.chunk, min(a.V, (c + 1) * w.chunk), vec, [&](int, float z) { m = fmaxf(m, z); });  // passes NaN by
  m = block_reduce(m, sh, Max());
  if (threadIdx.x == 0) w.cmax[(int64_t)b * w.C + c] = m;
}

// counts and weights by distance from the maximum
template <typename T>
__global__ __launch_bounds__(256) void sample_hist_kernel(SampleArgs a, SampleWs w, int vec) {
  __shared__ unsigned long long hm[SM_BINS];
  __shared__ uint32_t hc[SM_BINS];
  __shared__ float sh[16];
  const int c = blockIdx.x, b = blockIdx.y;
  const RowSet s = row_set(a, b);
  if (!cuts(s)) return;
  const float m = row_max(w, b, sh);
  for (int i = threadIdx.x; i < SM_BINS; i += 256) {
    hm[i] = 0;
    hc[i] = 0;
  }
  __syncthreads();
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  each<T>(row, c * w.chunk, min(a.V, (c + 1) * w.chunk), vec, [&](int, float z) {
    if (!usable(z)) return;
    const double t = scaled(z, m, s.invT);
    const int bin = bin_of(t);
    atomicAdd(&hc[bin], 1u);
    const uint64_t q = mass_of(t);
    if (q) atomicAdd(&hm[bin], (unsigned long long)q);
  });
  __syncthreads();
  for (int i = threadIdx.x; i < SM_BINS; i += 256)
    if (hc[i]) {
      atomicAdd(&w.count[(int64_t)b * SM_BINS + i], hc[i]);
      if (hm[i]) atomicAdd((unsigned long long *)&w.mass[(int64_t)b * SM_BINS + i], hm[i]);
    }
}

// whole multiples that reach the share p of a sum (at least one)
__device__ __forceinline__ uint64_t share(float p, uint64_t sum) {
  const double t = ceil((double)p * (double)sum);
  return t < 1.0 ? 1 : (uint64_t)t;
}

// The bins in which top-k and top-p cut, and their elements into the row's list.
// Every chunk finds the same bins from the histogram.
template <typename T>
__global__ __launch_bounds__(256) void sample_gather_kernel(SampleArgs a, SampleWs w, int vec) {
  __shared__ uint64_t cm[SM_BINS];  // running mass, bin included
  __shared__ uint32_t cc[SM_BINS];  // running count
  __shared__ uint64_t sh[16];
  __shared__ float shf[16];
  __shared__ int found[3];          // kbin, plo, phi
  const int c = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const RowSet s = row_set(a, b);
  if (!cuts(s)) return;
  const float m = row_max(w, b, shf);
  constexpr int PT = SM_BINS / 256;
  uint64_t mv[PT], ms = 0, ns = 0;
  uint32_t nv[PT];
  for (int i = 0; i < PT; ++i) {
    mv[i] = w.mass[(int64_t)b * SM_BINS + tid * PT + i];
    nv[i] = w.count[(int64_t)b * SM_BINS + tid * PT + i];
    ms += mv[i];
    ns += nv[i];
  }
  uint64_t mc = block_scan(ms, sh) - ms, nc = block_scan(ns, sh) - ns;
  for (int i = 0; i < PT; ++i) {
    mc += mv[i];
    nc += nv[i];
    cm[tid * PT + i] = mc;
    cc[tid * PT + i] = (uint32_t)nc;
  }
  if (tid < 3) found[tid] = -1;
  __syncthreads();
  const uint64_t total = cm[SM_BINS - 1];
  const uint32_t n = cc[SM_BINS - 1], K = s.k_on && (uint32_t)s.k < n ? (uint32_t)s.k : n;
  if (K < n)
    for (int i = tid * PT; i < tid * PT + PT; ++i)
      if (cc[i] >= K && (i == 0 || cc[i - 1] < K)) found[0] = i;
  __syncthreads();
  const int kbin = found[0];
  const uint64_t mass_k = kbin > 0 ? cm[kbin - 1] : 0;
  if (s.p_on && n > 0) {
    // top-k's sum lies between these; the exact one decides inside the bins
    const uint64_t lo = share(s.p, kbin < 0 ? total : mass_k), hi = share(s.p, kbin < 0 ? total : cm[kbin]);
    for (int i = tid * PT; i < tid * PT + PT; ++i) {
      const uint64_t before = i ? cm[i - 1] : 0;
      if (cm[i] >= lo && before < lo) found[1] = i;
      if (cm[i] >= hi && before < hi) found[2] = i;
    }
  }
  __syncthreads();
  const int plo = found[1], phi = found[2];
  if (c == 0 && tid == 0) {
    RowState &r = w.st[b];
    r.kbin = kbin;
    r.plo = plo;
    r.phi = phi;
    r.total = total;
    r.mass_k = mass_k;
    r.mass_p = plo > 0 ? cm[plo - 1] : 0;
    r.r = kbin < 0 ? 0 : K - (kbin > 0 ? cc[kbin - 1] : 0);
  }
  if (kbin < 0 && plo < 0) return;
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  each<T>(row, c * w.chunk, min(a.V, (c + 1) * w.chunk), vec, [&](int i, float z) {
    if (!usable(z)) return;
    const int bin = bin_of(scaled(z, m, s.invT));
    if (bin != kbin && !(bin >= plo && bin <= phi && plo >= 0)) return;
    const uint32_t at = atomicAdd(&w.st[b].nlist, 1u);
    if (at < (uint32_t)SM_CAP) w.list[(int64_t)b * SM_CAP + at] = key_of(z, i);
  });
}

// candidates of bins [b0, b1]: from the list where it holds them all, else from
// the row again
template <typename T>
struct Source {
  const uint64_t *list;
  const T *row;
  int n, V;  // n < 0: the row
  float m;
  double invT;
  template <typename F>
  __device__ __forceinline__ void each_key(int b0, int b1, F f) const {
    const int N = n >= 0 ? n : V;
    for (int i = threadIdx.x; i < N; i += blockDim.x) {
      uint64_t key;
      float z;
      if (n >= 0) {
        key = list[i];
        z = z_of(key);
      } else {
        z = logit<T>(row[i]);
        if (!usable(z)) continue;
        key = key_of(z, i);
      }
      const double t = scaled(z, m, invT);
      const int bin = bin_of(t);
      if (bin >= b0 && bin <= b1) f(key, t);
    }
  }
};

struct CutShared {
  unsigned long long amount[256], mass[256];
  uint32_t count[256];
  uint64_t sh[16];
  uint64_t need, prefix, above, key;
  int bucket, single;
};
// The key at which the running amount (elements, or their mass) over falling keys
// of bins [b0, b1] reaches `need`; above: the mass of the elements over that key, it
// included.
template <bool MASS, typename T>
__device__ uint64_t cut_key(const Source<T> &src, int b0, int b1, uint64_t need, CutShared &S, uint64_t &above) {
  const int tid = threadIdx.x;
  // bits in which the candidates differ at all
  uint64_t any = 0, all = ~0ull;
  src.each_key(b0, b1, [&](uint64_t key, double) {
    any |= key;
    all &= key;
  });
  any = block_reduce(any, S.sh, Or());
  all = ~block_reduce(~all, S.sh, Or());
  const uint64_t diff = any ^ all;
  int shift = diff ? (63 - __builtin_clzll(diff)) / 8 * 8 : 0;
  __syncthreads();
  if (tid == 0) {
    S.need = need;
    S.above = 0;
    S.prefix = shift == 56 ? 0 : any >> (shift + 8);
    S.single = 0;
  }
  for (;; shift -= 8) {
    if (tid < 256) {
      S.amount[tid] = 0;
      S.mass[tid] = 0;
      S.count[tid] = 0;
    }
    __syncthreads();
    const uint64_t prefix = S.prefix, want = S.need;
    src.each_key(b0, b1, [&](uint64_t key, double t) {
      if (shift < 56 && key >> (shift + 8) != prefix) return;
      const int d = 255 - (int)(key >> shift & 255);  // falling order
      const uint64_t q = mass_of(t);
      atomicAdd(&S.count[d], 1u);
      atomicAdd(&S.mass[d], (unsigned long long)q);
      atomicAdd(&S.amount[d], (unsigned long long)(MASS ? q : 1));
    });
    __syncthreads();
    const uint64_t mine = tid < 256 ? S.amount[tid] : 0, mm = tid < 256 ? S.mass[tid] : 0;
    const uint64_t sum = block_scan(mine, S.sh), summ = block_scan(mm, S.sh);
    if (tid < 256 && sum >= want && sum - mine < want) {
      S.bucket = tid;
      S.need = want - (sum - mine);
      S.above += summ - mm;
      S.prefix = (shift == 56 ? 0 : prefix << 8) | (uint64_t)(255 - tid);
      S.single = S.count[tid] == 1;
      if (S.single || shift == 0) S.above += mm;
    }
    __syncthreads();
    if (shift == 0) {
      above = S.above;
      const uint64_t key = S.prefix;
      __syncthreads();
      return key;
    }
    if (S.single) {
      const uint64_t pre = S.prefix;
      src.each_key(b0, b1, [&](uint64_t key, double) {
        if (key >> shift == pre) S.key = key;
      });
      __syncthreads();
      above = S.above;
      const uint64_t key = S.key;
      __syncthreads();
      return key;
    }
  }
}

// the exact cut among the candidates
template <typename T>
__global__ __launch_bounds__(1024) void sample_cut_kernel(SampleArgs a, SampleWs w) {
  __shared__ CutShared S;
  __shared__ float shf[16];
  const int b = blockIdx.x;
  const RowSet s = row_set(a, b);
  if (!cuts(s)) return;
  const RowState r = w.st[b];
  if (r.kbin < 0 && r.plo < 0) return;
  Source<T> src;
  src.list = w.list + (int64_t)b * SM_CAP;
  src.row = (const T *)a.z + (int64_t)b * a.stride;
  src.n = r.nlist <= (uint32_t)SM_CAP ? (int)r.nlist : -1;
  src.V = a.V;
  src.m = row_max(w, b, shf);
  src.invT = s.invT;
  uint64_t tau = 0, sum = r.total, above;
  if (r.kbin >= 0) {
    tau = cut_key<false>(src, r.kbin, r.kbin, r.r, S, above);
    sum = r.mass_k + above;
  }
  if (r.plo >= 0) {
    const uint64_t key = cut_key<true>(src, r.plo, r.phi, share(s.p, sum) - r.mass_p, S, above);
    tau = key > tau ? key : tau;
  }
  if (threadIdx.x == 0) w.st[b].tau = tau;
}

// the weight an element keeps, as a whole number
__device__ __forceinline__ uint64_t kept(float z, int i, float m, const RowSet &s, uint64_t tau) {
  if (!usable(z)) return 0;
  if (z == m) return s.greedy || key_of(z, i) >= tau ? 1ull << SM_MASS_BITS : 0;
  if (s.greedy || key_of(z, i) < tau) return 0;
  const double e = weight_scaled(scaled(z, m, s.invT), SM_MASS_BITS);
  return e >= __builtin_ldexp((double)s.minp, SM_MASS_BITS) ? whole(e) : 0;
}

template <typename T>
__global__ __launch_bounds__(256) void sample_sum_kernel(SampleArgs a, SampleWs w, int vec) {
  __shared__ float shf[16];
  __shared__ uint64_t sh[16];
  const int c = blockIdx.x, b = blockIdx.y;
  const RowSet s = row_set(a, b);
  const float m = row_max(w, b, shf);
  const uint64_t tau = w.st[b].tau;
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  uint64_t q = 0;
  each<T>(row, c * w.chunk, min(a.V, (c + 1) * w.chunk), vec, [&](int i, float z) { q += kept(z, i, m, s, tau); });
  q = block_reduce(q, sh, Add());
  if (threadIdx.x == 0) w.csum[(int64_t)b * w.C + c] = q;
}

// the chunk, the thread's run in it and the element at which the running sum
// passes u times the whole
template <typename T>
__global__ __launch_bounds__(SM_MAX_CHUNKS) void sample_pick_kernel(SampleArgs a, SampleWs w) {
  __shared__ float shf[16];
  __shared__ uint64_t sh[16];
  __shared__ uint64_t need;
  __shared__ int at;
  const int b = blockIdx.x, tid = threadIdx.x;
  const RowSet s = row_set(a, b);
  const float m = row_max(w, b, shf);
  const uint64_t tau = w.st[b].tau;
  const uint64_t mine = tid < w.C ? w.csum[(int64_t)b * w.C + tid] : 0;
  const uint64_t sum = block_scan(mine, sh);
  const uint64_t W = block_reduce(mine, sh, Add());
  if (W == 0) {
    if (tid == 0) a.ids[b] = -1;
    return;
  }
  const float u = a.u[b];
  uint64_t t = !s.greedy && u > 0.f ? (uint64_t)((double)fminf(u, 1.f) * (double)W) : 0;
  if (t >= W) t = W - 1;
  if (sum > t && sum - mine <= t) {
    at = tid;
    need = t - (sum - mine);
  }
  __syncthreads();
  const int c = at;
  t = need;
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  const int run = w.chunk / SM_MAX_CHUNKS, lo = c * w.chunk + tid * run, hi = min(a.V, lo + run);
  uint64_t q = 0;
  for (int i = lo; i < hi; ++i) q += kept(logit<T>(row[i]), i, m, s, tau);
  const uint64_t run_sum = block_scan(q, sh);
  if (run_sum > t && run_sum - q <= t) {
    t -= run_sum - q;
    for (int i = lo; i < hi; ++i) {
      const uint64_t k = kept(logit<T>(row[i]), i, m, s, tau);
      if (k > t) {
        a.ids[b] = i;
        break;
      }
      t -= k;
    }
  }
}

template <typename T>
hipError_t sample_run(const SampleArgs &a, const SampleWs &w, hipStream_t s) {
  const dim3 grid(w.C, a.B);
  const int vec = ((uintptr_t)a.z & 15) == 0 && (a.stride * sizeof(T)) % 16 == 0;
  hipLaunchKernelGGL(sample_max_kernel<T>, grid, dim3(256), 0, s, a, w, vec);
  if (a.top_k || a.top_p) {
    hipLaunchKernelGGL(sample_hist_kernel<T>, grid, dim3(256), 0, s, a, w, vec);
    hipLaunchKernelGGL(sample_gather_kernel<T>, grid, dim3(256), 0, s, a, w, vec);
    hipLaunchKernelGGL(sample_cut_kernel<T>, dim3(a.B), dim3(1024), 0, s, a, w);
  }
  hipLaunchKernelGGL(sample_sum_kernel<T>, grid, dim3(256), 0, s, a, w, vec);
  hipLaunchKernelGGL(sample_pick_kernel<T>, dim3(a.B), dim3(SM_MAX_CHUNKS), 0, s, a, w);
  return hipGetLastError();
}

}  // namespace

int64_t sample_work_floats(int B, int V) { return (int64_t)(sample_carve(nullptr, B, V, nullptr) / 4); }

hipError_t launch_sample(const SampleArgs &a, int dtype, hipStream_t s) {
  SampleWs w{};
  sample_carve((char *)a.work, a.B, a.V, &w);
  return dtype == GN_DTYPE_F32 ? sample_run<float>(a, w, s) : sample_run<uint16_t>(a, w, s);
}

}  // namespace gn
