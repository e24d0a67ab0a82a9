// Sampling: temperature, top-k, top-p and min-p over rows of logits and one draw
// a row.
//
// Every weight exp((z - max) / T) is a float64 exponential rounded to a whole
// multiple of 2^-43, and every sum an integer one: sums of rows cut into chunks,
// over atomics and over prefixes are then the same number whatever their order,
// and a comparison with a border (top-p's share, the draw) can be made anywhere.
//
// A histogram of 1024 bins of 1/32 in the exponent fixes the bins in which top-k
// and top-p cut; only their elements are then ranked exactly, by (logit, falling
// index), so that equal logits go by the lowest index.  A row of up to 16384 logits
// is one workgroup's, its logits in LDS from the first pass to the draw.  Longer rows
// are cut into chunks, a workgroup each, and read whole once: that pass leaves maxima
// and counts, and a workgroup a row then fetches the few logits in question and
// draws.  Rows of which much is kept are read once more for the sum of what is kept,
// and before it for the histogram's masses where top-p asks for them without a small
// top-k.
//
// Rows of up to 16384 are bound by the float64 operations of one CU and by latency: 4
// rows of 8000, every filter, 13.3 us.  Longer ones: the pass over the logits is
// memory's (128 rows of 131072 float32, 67 MB: 15.5 us, 4.3 TB/s), the cut a chain of
// waits (22 us there, 16.6 for one row of 50257); 42 us and 20 to 24 us in all.  With
// top-p alone 105 to 114 us, without a cut 45 to 49: a pass that weighs all 16.8 million
// logits in float64 takes 27 to 32 us, of which the operations themselves are about 9 at
// the card's rate; how the rest divides between table reads and LDS atomics was not
// measured.
#include "gn_serve.h"

namespace gn {
namespace {

constexpr int SM_BINS = 1024;
constexpr int SM_PER = 32;        // bins per unit of the exponent
constexpr int SM_CAP = 4096;      // candidates of a row kept in a list
constexpr int SM_RANK = 256;      // candidates ranked against each other; more: radix
constexpr int SM_LISTED = 2048;   // top-k up to this: kept logits from the list alone
constexpr int SM_MASS_BITS = 43;
constexpr int SM_WAVE = 1024;     // logits of a wave, 16 a lane
constexpr int SM_RUN = 256;       // logits whose kept weights are summed, 4 a lane
constexpr int SM_ONE = 16384;     // rows up to this size: one workgroup

// 2^43 exp(-b / 32), from exp(-1/32) and its powers by their series
struct ExpTable {
  double v[SM_BINS];
  static constexpr double series(double x) {  // exp(x), |x| <= 1
    double term = 1.0, sum = 1.0;
    for (int i = 1; i < 30; ++i) {
      term *= x / i;
      sum += term;
    }
    return sum;
  }
  constexpr ExpTable() : v() {
    double whole = 8796093022208.0;  // 2^43 exp(-(b / 32))
    for (int b = 0; b < SM_BINS; ++b) {
      if (b && b % SM_PER == 0) whole *= series(-1.0);
      v[b] = whole * series(-(double)(b % SM_PER) / SM_PER);
    }
  }
};
__device__ const ExpTable exp_table = ExpTable();

// where a row's cuts fall in its histogram
struct Cuts {
  uint64_t mass_k;     // mass of the bins before kbin
  uint64_t mass_p;     // ... before plo
  uint64_t total;
  uint32_t r;          // rank of the last kept element inside kbin
  int32_t kbin, plo, phi;  // -1: top-k / top-p does not cut
  int32_t last;            // bins 0 .. last hold all that is kept, SM_CAP or fewer (-1: more)
};
struct RowState {
  uint64_t tau;        // kept: elements whose key is at least this
  int32_t done, pad;   // the draw is made
};

struct SampleWs {
  uint64_t *mass, *wsum;
  RowState *st;
  uint16_t *count;  // a chunk's histogram below its own maximum
  float *cmax, *gmax;  // maxima of a chunk, of every 16 logits
  int C, waves;  // chunks of a row, waves of a chunk
};

inline size_t up64(size_t n) { return (n + 63) / 64 * 64; }

size_t sample_carve(char *base, int B, int V, SampleWs *w) {
  SampleWs t{};
  // chunks of 4096, or of 16384 where those fill the card or a row has so many that
  // joining their histograms takes longer (a row of 2^20: 52 us)
  const int few = (V + 4 * SM_WAVE - 1) / (4 * SM_WAVE);
  t.waves = (int64_t)B * few > 2048 || few > 64 ? 16 : 4;
  t.C = (V + t.waves * SM_WAVE - 1) / (t.waves * SM_WAVE);
  size_t off = 0;
  const auto take = [&](size_t bytes) {
    char *p = base ? base + off : nullptr;
    off += up64(bytes);
    return p;
  };
  if (V > SM_ONE) {
    t.mass = (uint64_t *)take((size_t)B * SM_BINS * 8);
    t.wsum = (uint64_t *)take((size_t)B * ((V + SM_RUN - 1) / SM_RUN) * 8);
    t.st = (RowState *)take((size_t)B * sizeof(RowState));
    t.count = (uint16_t *)take((size_t)B * t.C * SM_BINS * 2);
    t.cmax = (float *)take((size_t)B * t.C * 4);
    t.gmax = (float *)take((size_t)B * t.C * t.waves * 64 * 4);
  }
  if (w) *w = t;
  return off ? off : 64;  // callers hand over some workspace whatever the size
}

template <typename T>
__device__ __forceinline__ float logit(T x);
template <>
__device__ __forceinline__ float logit<float>(float x) { return x; }
template <>
__device__ __forceinline__ float logit<uint16_t>(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

template <int CTRL>
__device__ __forceinline__ float near(float v) {  // of another lane of the quad
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, false));
}
// A lane's 16 of a wave's 1024 logits from `base` on: 16 bytes at a time, group q's
// element k being base + at<T>(q, lane) + k, so that (q, lane, k) rises with the
// index.  Behind the row: NaN, which nothing counts.
template <typename T>
struct Lane {
  static constexpr int N = 16 / sizeof(T), Q = 16 / N;
  static __device__ __forceinline__ int at(int q, int lane) { return q * 64 * N + lane * N; }
  float z[16];
  int base, lane;
  __device__ __forceinline__ int index(int e) const { return base + at(e / N, lane) + e % N; }
  __device__ __forceinline__ void load(const T *row, int base_, int V, int vec) {
    base = base_;
    lane = threadIdx.x & 63;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = base + at(q, lane);
      if (vec && i + N <= V) {
        const uint4 v = *reinterpret_cast<const uint4 *>(row + i);
        const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
        for (int k = 0; k < N; ++k) z[q * N + k] = logit<T>(e[k]);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) z[q * N + k] = i + k < V ? logit<T>(row[i + k]) : __uint_as_float(0x7fc00000u);
      }
    }
  }
  // the largest of 16 that follow each other: group at<T>(q, lane) / 16 of the wave
  // for q = lane % Q, a group being Q lanes'
  __device__ __forceinline__ float group_max() const {
    float of = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < N; ++k) m = fmaxf(m, z[q * N + k]);
      m = fmaxf(m, near<0xb1>(m));          // lane ^ 1
      if (Q == 4) m = fmaxf(m, near<0x4e>(m));  // lane ^ 2
      of = lane % Q == q ? m : of;
    }
    return of;
  }
  __device__ __forceinline__ int group() const { return lane % Q * (64 / Q) + lane / Q; }
  __device__ __forceinline__ float max() const {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, z[e]);  // passes NaN by
    return m;
  }
};

// four that follow each other; NaN behind the row
template <typename T>
__device__ __forceinline__ void load4(float (&z)[4], const T *row, int i, int V, int vec) {
  if (vec && i + 4 <= V) {
    struct alignas(4 * sizeof(T)) Four {
      T e[4];
    };
    const Four v = *reinterpret_cast<const Four *>(row + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = logit<T>(v.e[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] = i + k < V ? logit<T>(row[i + k]) : __uint_as_float(0x7fc00000u);
  }
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
// 32 (max - z) / T in float64 (per: 32 / T), rising as z falls; 0 for the maximum
// itself, also where it is infinite
__device__ __forceinline__ double scaled(float z, float m, double per) {
  return z == m ? 0.0 : ((double)m - (double)z) * per;
}
__device__ __forceinline__ int bin_of(double x) { return x < (double)(SM_BINS - 1) ? (int)x : SM_BINS - 1; }
// 2^43 exp(-x / 32) for x of bin `bin`: the table's value times the series of the
// rest, 1/32 at most (its first omitted term is below 6e-15 of the value); 0 in the
// last bin, where a weight is below 2^-46
__device__ __forceinline__ double weight_of(double x, int bin, const double *tab) {
  constexpr double c = -1.0 / SM_PER;
  const double f = x - (double)bin;
  double p = c * c * c * c * c * c / 720.0;
  p = __builtin_fma(p, f, c * c * c * c * c / 120.0);
  p = __builtin_fma(p, f, c * c * c * c / 24.0);
  p = __builtin_fma(p, f, c * c * c / 6.0);
  p = __builtin_fma(p, f, c * c / 2.0);
  p = __builtin_fma(p, f, c);
  p = __builtin_fma(p, f, 1.0);
  return bin < SM_BINS - 1 ? p * tab[bin] : 0.0;
}
// a number of [0, 2^43] to the nearest whole one
__device__ __forceinline__ uint64_t whole(double w) {
  return (uint64_t)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}
__device__ __forceinline__ uint64_t mass_of(double x, const double *tab) { return whole(weight_of(x, bin_of(x), tab)); }

struct RowSet {
  bool greedy, k_on, p_on;
  double per;  // bins a unit of the logit: 32 / T
  float per4;  // the same in float32, finite
  int k;
  float p, minp;
  double least;  // min_p as a weight
};
__device__ __forceinline__ RowSet row_set(const SampleArgs &a, int b) {
  RowSet s;
  const float T = a.temperature ? a.temperature[b] : 1.f;
  s.greedy = !(T > 0.f);
  s.per = s.greedy ? 1.0 : (double)SM_PER / (double)T;
  s.per4 = fminf((float)s.per, 3.4028234e38f);
  s.k = a.top_k ? a.top_k[b] : 0;
  s.k_on = s.k > 0;
  s.p = a.top_p ? a.top_p[b] : 1.f;
  s.p_on = s.p < 1.f;
  s.minp = a.min_p ? a.min_p[b] : 0.f;
  s.least = __builtin_ldexp((double)s.minp, SM_MASS_BITS);
  return s;
}
// whether the row needs the histogram
__device__ __forceinline__ bool cuts(const RowSet &s) { return !s.greedy && (s.k_on || s.p_on); }
// whether it needs its masses too: not where top-k leaves few, which bring their own
__device__ __forceinline__ bool weighs(const RowSet &s) { return s.p_on && !(s.k_on && s.k <= SM_LISTED); }
// The histogram's bins are a grid of 1/32 in z / T, in float32: all they have to do
// is fall with z and be the same wherever they are asked for.  Grid lines are whole
// numbers, so that bins below a chunk's maximum, moved by that maximum's bin, are
// those below the row's.
__device__ __forceinline__ float line_of(float z, const RowSet &s) {
  return fminf(fmaxf(floorf(z * s.per4), -3.4028234e38f), 3.4028234e38f);
}
__device__ __forceinline__ int hbin(float z, float top, const RowSet &s) {  // top: line_of(maximum)
  return (int)fminf(fmaxf(top - line_of(z, s), 0.f), (float)(SM_BINS - 1));
}

template <typename X, typename F>
__device__ __forceinline__ X wave_reduce(X v, F f) {
  for (int o = 32; o > 0; o >>= 1) v = f(v, __shfl_xor(v, o, 64));
  return v;
}
// over a workgroup of NT threads; the waves' values are read back all at once
template <int NT, typename X, typename F>
__device__ __forceinline__ X block_reduce(X v, X *sh, F f) {  // sh: 16 values
  v = wave_reduce(v, f);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = f(v, sh[w]);
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
// running sums over a wave: within rows of 16 lanes, then the rows before (DPP moves
// on the vector unit; a shuffle through LDS per step takes four times as long)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp(uint64_t v) {
  return (uint64_t)dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | dpp<CTRL, ROWS>((uint32_t)v);
}
template <typename X>
__device__ __forceinline__ X wave_scan(X v) {
  v += dpp<0x111, 0xf>(v);
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // lane 15 of rows 0 and 2 to rows 1 and 3
  v += dpp<0x143, 0xc>(v);  // lane 31 to rows 2 and 3
  return v;
}
// places for this lane's n behind a counter, those of a wave together
__device__ __forceinline__ uint32_t places(uint32_t n, uint32_t *counter) {
  const uint32_t run = wave_scan(n), all = (uint32_t)__builtin_amdgcn_readlane((int)run, 63);
  if (all == 0) return 0;
  uint32_t first = 0;
  if ((threadIdx.x & 63) == 0) first = atomicAdd(counter, all);
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)first) + run - n;
}
// A workgroup's waves' sums, one in each of sh[0 .. NT / 64), to the sums of the waves
// before; all of them in sh[16].  One wave's work: done by each of sixteen it took
// longer than the scan itself.
template <int NT, typename X>
__device__ __forceinline__ void waves_scan(X *sh) {
  const int lane = threadIdx.x;
  const X x = lane < NT / 64 ? sh[lane] : 0;
  X v = x;
  v += dpp<0x111, 0xf>(v);
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  if (lane < NT / 64) sh[lane] = v - x;
  if (lane == NT / 64 - 1) sh[16] = v;
}
// running sum over the workgroup's threads, this one's value included; all: the sum
template <int NT>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *sh, uint64_t &all) {  // sh: 17 values
  const int w = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh[w] = v;
  __syncthreads();
  if (w == 0) waves_scan<NT>(sh);
  __syncthreads();
  all = sh[16];
  return v + sh[w];
}
// each wave for itself, without a barrier
__device__ __forceinline__ float row_max(const SampleWs &w, int b) {
  float m = -INFINITY;
  for (int i = threadIdx.x & 63; i < w.C; i += 64) m = fmaxf(m, w.cmax[(int64_t)b * w.C + i]);
  return wave_reduce(m, Max());
}

// whole multiples that reach the share p of a sum (at least one)
__device__ __forceinline__ uint64_t share(float p, uint64_t sum) {
  const double t = ceil((double)p * (double)sum);
  return t < 1.0 ? 1 : (uint64_t)t;
}

struct Bins {
  uint64_t cm[SM_BINS];  // running mass, bin included
  uint32_t cc[SM_BINS];  // running count
  uint64_t sm[17];
  uint32_t sn[17];
  int found[3];          // kbin, plo, phi
  uint64_t lo, hi;
  Cuts cuts;
};
// The bins in which top-k and, with `masses`, top-p cut, from a row's histogram in
// S.cm and S.cc (NT threads).
template <int NT>
__device__ Cuts cut_bins(const RowSet &s, float m, bool masses, Bins &S) {
  constexpr int PT = SM_BINS / NT;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  uint64_t mv[PT], ms = 0;
  uint32_t nv[PT], ns = 0;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    mv[i] = S.cm[tid * PT + i];
    nv[i] = S.cc[tid * PT + i];
    ms += mv[i];
    ns += nv[i];
  }
  uint64_t mc = wave_scan(ms);
  uint32_t nc = wave_scan(ns);
  if (lane == 63) {
    S.sm[w] = mc;
    S.sn[w] = nc;
  }
  if (tid < 3) S.found[tid] = -1;
  __syncthreads();
  if (w == 0) {
    waves_scan<NT>(S.sm);
    waves_scan<NT>(S.sn);
  }
  __syncthreads();
  mc += S.sm[w];
  nc += S.sn[w];
  const uint32_t n = S.sn[16];
  mc -= ms;
  nc -= ns;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    mc += mv[i];
    nc += nv[i];
    S.cm[tid * PT + i] = mc;
    S.cc[tid * PT + i] = nc;
  }
  __syncthreads();
  const uint32_t K = s.k_on && (uint32_t)s.k < n ? (uint32_t)s.k : n;
  if (K < n)
    for (int i = tid * PT; i < tid * PT + PT; ++i)
      if (S.cc[i] >= K && (i == 0 || S.cc[i - 1] < K)) S.found[0] = i;
  __syncthreads();
  const bool p = s.p_on && masses && n > 0;
  if (w == 0) {  // scalar work, in float64: one wave's
    Cuts r;
    r.kbin = S.found[0];
    r.total = S.cm[SM_BINS - 1];
    r.mass_k = r.kbin > 0 ? S.cm[r.kbin - 1] : 0;
    r.r = r.kbin < 0 ? 0 : K - (r.kbin > 0 ? S.cc[r.kbin - 1] : 0);
    r.plo = r.phi = r.last = -1;
    r.mass_p = 0;
    // top-k's sum lies between these; the exact one decides inside the bins
    const uint64_t lo = p ? share(s.p, r.kbin < 0 ? r.total : r.mass_k) : 0;
    const uint64_t hi = p ? share(s.p, r.kbin < 0 ? r.total : S.cm[r.kbin]) : 0;
    if (tid == 0) {
      S.lo = lo;
      S.hi = hi;
      S.cuts = r;
    }
  }
  __syncthreads();
  Cuts r = S.cuts;
  if (p) {
    const uint64_t lo = S.lo, hi = S.hi;
    for (int i = tid * PT; i < tid * PT + PT; ++i) {
      const uint64_t before = i ? S.cm[i - 1] : 0;
      if (S.cm[i] >= lo && before < lo) S.found[1] = i;
      if (S.cm[i] >= hi && before < hi) S.found[2] = i;
    }
    __syncthreads();
    r.plo = S.found[1];
    r.phi = S.found[2];
    r.mass_p = r.plo > 0 ? S.cm[r.plo - 1] : 0;
  }
  // all that can be kept lies in bins 0 .. last; top-p without masses wants all of
  // top-k's.  min_p's bin with what the logarithm and the grid's lines may be off.
  int last = r.plo >= 0 ? r.phi : r.kbin >= 0 ? r.kbin : SM_BINS - 1;
  if (s.minp > 1e-30f && (masses || !s.p_on)) {
    const float x = -(float)SM_PER * __logf(fminf(s.minp, 1.f));
    last = min(last, (int)fminf(x + 3.f + (x + fabsf(m) * s.per4) * 0x1p-20f, (float)(SM_BINS - 1)));
  }
  r.last = S.cc[last] <= (uint32_t)SM_CAP ? last : -1;
  return r;
}
// Up to SM_RANK candidates (in any order), one a thread: how many of their bins lie
// above one, and their mass, say where the cuts fall.
struct Rank {
  uint64_t key, mass;  // mass: bit 62 of kbin, bit 63 of plo .. phi
};
struct Ranks {
  Rank at[SM_RANK];
  unsigned long long mk[SM_RANK], mp[SM_RANK];
  uint32_t ck[SM_RANK];
  uint32_t n;
  uint64_t tau_k, above_k, tau_p;
};
constexpr uint64_t RANK_K = 1ull << 62, RANK_P = 1ull << 63, RANK_MASS = RANK_K - 1;
// 1: of kbin, 2: of plo .. phi
__device__ __forceinline__ uint32_t cut_of(const Cuts &r, int bin) {
  return (bin == r.kbin ? 1u : 0u) | (r.plo >= 0 && bin >= r.plo && bin <= r.phi ? 2u : 0u);
}
// S.at[..].key holds the n candidates.  Where there are threads enough a candidate's
// comparisons are shared by several.
template <int NT>
__device__ uint64_t cut_by_rank(const RowSet &s, const Cuts &r, float m, float top, const double *tab, Ranks &S) {
  constexpr int PARTS = NT / SM_RANK;
  const int tid = threadIdx.x, n = (int)S.n, own = tid % SM_RANK, part = tid / SM_RANK;
  uint64_t key = 0, q = 0;
  uint32_t in = 0;
  if (own < n) key = S.at[own].key;
  if (tid < n) {
    q = mass_of(scaled(z_of(key), m, s.per), tab);
    in = cut_of(r, hbin(z_of(key), top, s));
    S.at[tid].mass = q | (in & 1 ? RANK_K : 0) | (in & 2 ? RANK_P : 0);
    S.mk[tid] = S.mp[tid] = S.ck[tid] = 0;
  }
  if (tid == 0) S.tau_k = S.tau_p = S.above_k = 0;
  __syncthreads();
  uint64_t mk = 0, mp = 0;
  uint32_t ck = 0;
  if (own < n) {
#pragma unroll 4
    for (int j = part; j < n; j += PARTS) {
      const Rank o = S.at[j];
      const bool over = o.key > key, k = over && (o.mass & RANK_K), p = over && (o.mass & RANK_P);
      const uint64_t qj = o.mass & RANK_MASS;
      ck += k;
      mk += k ? qj : 0;
      mp += p ? qj : 0;
    }
    if (PARTS > 1) {
      atomicAdd(&S.ck[own], ck);
      atomicAdd(&S.mk[own], (unsigned long long)mk);
      atomicAdd(&S.mp[own], (unsigned long long)mp);
    }
  }
  if (PARTS > 1) {
    __syncthreads();
    if (tid < n) {
      ck = S.ck[tid];
      mk = S.mk[tid];
      mp = S.mp[tid];
    }
  }
  if (tid < n && (in & 1) && ck == r.r - 1) {
    S.tau_k = key;
    S.above_k = mk + q;
  }
  __syncthreads();
  if (tid < n && (in & 2)) {
    const uint64_t need = share(s.p, r.kbin >= 0 ? r.mass_k + S.above_k : r.total) - r.mass_p;
    if (mp < need && mp + q >= need) S.tau_p = key;
  }
  __syncthreads();
  return S.tau_k > S.tau_p ? S.tau_k : S.tau_p;
}

struct Radix {
  unsigned long long amount[256], mass[256];
  uint32_t count[256];
  uint64_t sh[17];
  uint64_t need, prefix, above, key;
  int single;
};
// The key at which the running amount over falling keys reaches `need`; above: the
// mass of the elements over that key, it included.  each(f): f(key, amount, mass)
// for this thread's elements, the keys all different.
template <int NT, typename Each>
__device__ uint64_t find_by_radix(const Each &each, uint64_t need, Radix &S, uint64_t &above) {
  const int tid = threadIdx.x;
  // bits in which the keys differ at all
  uint64_t any = 0, none = 0;
  each([&](uint64_t key, uint64_t, uint64_t) {
    any |= key;
    none |= ~key;
  });
  any = block_reduce<NT>(any, S.sh, Or());
  none = block_reduce<NT>(none, S.sh, Or());
  const uint64_t diff = any & none;
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
    each([&](uint64_t key, uint64_t amount, uint64_t mass) {
      if (shift < 56 && key >> (shift + 8) != prefix) return;
      const int d = 255 - (int)(key >> shift & 255);  // falling order
      atomicAdd(&S.count[d], 1u);
      atomicAdd(&S.mass[d], (unsigned long long)mass);
      atomicAdd(&S.amount[d], (unsigned long long)amount);
    });
    __syncthreads();
    const uint64_t mine = tid < 256 ? S.amount[tid] : 0, mm = tid < 256 ? S.mass[tid] : 0;
    uint64_t all;
    const uint64_t sum = block_scan<NT>(mine, S.sh, all), summ = block_scan<NT>(mm, S.sh, all);
    if (tid < 256 && sum >= want && sum - mine < want) {
      S.need = want - (sum - mine);
      S.above += summ - mm;
      S.prefix = (shift == 56 ? 0 : prefix << 8) | (uint64_t)(255 - tid);
      S.single = S.count[tid] == 1;
      if (S.single || shift == 0) S.above += mm;
    }
    __syncthreads();
    if (shift == 0 || S.single) {
      const uint64_t pre = S.prefix;
      if (shift == 0) {
        if (tid == 0) S.key = pre;
      } else {
        each([&](uint64_t key, uint64_t, uint64_t) {
          if (key >> shift == pre) S.key = key;
        });
      }
      __syncthreads();
      above = S.above;
      const uint64_t key = S.key;
      __syncthreads();
      return key;
    }
  }
}
// all(f): f(key) for this thread's candidates, or for all elements of the row
template <int NT, typename All>
__device__ uint64_t cut_by_radix(const All &all, const RowSet &s, const Cuts &r, float m, float top, const double *tab,
                                 Radix &S) {
  uint64_t tau = 0, sum = r.total, above;
  const auto of = [&](uint32_t cut, bool mass, auto f) {
    all([&](uint64_t key) {
      if (!(cut_of(r, hbin(z_of(key), top, s)) & cut)) return;
      const uint64_t q = mass_of(scaled(z_of(key), m, s.per), tab);
      f(key, mass ? q : 1, q);
    });
  };
  if (r.kbin >= 0) {
    tau = find_by_radix<NT>([&](auto f) { of(1, false, f); }, r.r, S, above);
    sum = r.mass_k + above;
  }
  if (r.plo >= 0) {
    const uint64_t key = find_by_radix<NT>([&](auto f) { of(2, true, f); }, share(s.p, sum) - r.mass_p, S, above);
    tau = key > tau ? key : tau;
  }
  return tau;
}

// the weight an element keeps, as a whole number; no branch, so that a lane's
// elements run beside each other
__device__ __forceinline__ uint64_t kept(float z, int i, float m, const RowSet &s, uint64_t tau, const double *tab) {
  const double x = scaled(z, m, s.per), e = weight_of(x, bin_of(x), tab);
  const bool top = z == m, in = usable(z) && key_of(z, i) >= tau && (top || (!s.greedy && e >= s.least));
  return in ? (top ? 1ull << SM_MASS_BITS : whole(e)) : 0;
}
// the place of the draw in kept weights of sum W > 0
__device__ __forceinline__ uint64_t draw_at(const RowSet &s, float u, uint64_t W) {
  const uint64_t t = !s.greedy && u > 0.f ? (uint64_t)((double)fminf(u, 1.f) * (double)W) : 0;
  return t < W ? t : W - 1;
}

// ---- rows of up to 16384 logits: every step in one workgroup --------------------
// A thread's E logits follow each other (runs of E + 1 words, for the banks), so that
// a scan over the threads is one over the indexes.
template <typename T, int NT, int E>
__global__ __launch_bounds__(NT) void sample_row_kernel(SampleArgs a) {
  extern __shared__ float z[];
  __shared__ union {
    Bins bins;
    Ranks ranks;
    Radix radix;
  } S;
  __shared__ double tab[SM_BINS];
  __shared__ uint64_t sh[17];
  __shared__ float shf[16];
  const int b = blockIdx.x, tid = threadIdx.x;
  const RowSet s = row_set(a, b);
  const float u = a.u[b];
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  float m = -INFINITY;
  T raw[E];  // all loads in flight, behind the row's end of its last logit
#pragma unroll
  for (int e = 0; e < E; ++e) raw[e] = row[min(e * NT + tid, a.V - 1)];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * NT + tid;
    const float v = i < a.V ? logit<T>(raw[e]) : __uint_as_float(0x7fc00000u);
    z[i + (i / E)] = v;
    m = fmaxf(m, v);  // passes NaN by
  }
  const bool cut = cuts(s);
  for (int i = tid; i < SM_BINS; i += NT) {
    tab[i] = exp_table.v[i];
    S.bins.cm[i] = 0;
    S.bins.cc[i] = 0;
  }
  m = block_reduce<NT>(m, shf, Max());  // and a barrier for the rest
  const float top = line_of(m, s);
  float zr[E];
#pragma unroll
  for (int e = 0; e < E; ++e) zr[e] = z[tid * (E + 1) + e];
  uint64_t tau = 0;
  if (cut) {
    unsigned long long *hm = (unsigned long long *)S.bins.cm;
    int bin[E];  // -2: no logit to choose
#pragma unroll
    for (int e = 0; e < E; ++e) {  // no branch on the way: all chains at once
      bin[e] = hbin(zr[e], top, s);
      const bool ok = usable(zr[e]);
      if (ok) atomicAdd(&S.bins.cc[bin[e]], 1u);
      if (s.p_on) {  // top-k alone goes by the counts
        const uint64_t q = mass_of(scaled(zr[e], m, s.per), tab);
        if (ok && q) atomicAdd(&hm[bin[e]], (unsigned long long)q);
      }
      bin[e] = ok ? bin[e] : -2;
    }
    __syncthreads();
    const Cuts r = cut_bins<NT>(s, m, true, S.bins);
    if (r.kbin >= 0 || r.plo >= 0) {
      __syncthreads();  // the bins are read, the ranks lie in their place
      if (tid == 0) S.ranks.n = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (cut_of(r, bin[e])) {
          const uint32_t at = atomicAdd(&S.ranks.n, 1u);
          if (at < SM_RANK) S.ranks.at[at].key = key_of(zr[e], tid * E + e);
        }
      __syncthreads();
      if (S.ranks.n <= SM_RANK) {
        tau = cut_by_rank<NT>(s, r, m, top, tab, S.ranks);
      } else {
        __syncthreads();
        const auto all = [&](auto f) {
#pragma unroll 1
          for (int e = 0; e < E; ++e)
            if (usable(z[tid * (E + 1) + e])) f(key_of(z[tid * (E + 1) + e], tid * E + e));
        };
        tau = cut_by_radix<NT>(all, s, r, m, top, tab, S.radix);
      }
    }
  }
  uint64_t k[E], q = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    k[e] = kept(zr[e], tid * E + e, m, s, tau, tab);
    q += k[e];
  }
  uint64_t W;
  const uint64_t run = block_scan<NT>(q, sh, W);
  if (W == 0) {
    if (tid == 0) a.ids[b] = -1;
    return;
  }
  uint64_t t = draw_at(s, u, W);
  if (run > t && run - q <= t) {
    t -= run - q;
    int e = 0;
    bool more = true;
#pragma unroll
    for (int i = 0; i < E - 1; ++i) {
      more = more && t >= k[i];
      e += more;
      t -= more ? k[i] : 0;
    }
    a.ids[b] = tid * E + e;
  }
}

// ---- longer rows -------------------------------------------------------------
// The chunk's largest logit, its histogram below that, and the largest of every 16
// logits; clears what the later passes add to.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_count_kernel(SampleArgs a, SampleWs w, int vec) {
  __shared__ float sh[16];
  __shared__ uint32_t hc[SM_BINS];
  const int c = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  Lane<T> x;
  x.load((const T *)a.z + (int64_t)b * a.stride, c * NT * 16 + (tid >> 6) * SM_WAVE, a.V, vec);
  const RowSet s = row_set(a, b);
  const bool cut = cuts(s);
  if (cut) {
    for (int i = tid; i < SM_BINS; i += NT) hc[i] = 0;
    if (weighs(s))
      for (int i = c * NT + tid; i < SM_BINS; i += w.C * NT) w.mass[(int64_t)b * SM_BINS + i] = 0;
  }
  if (c == 0 && tid == 0) {
    w.st[b].tau = 0;
    w.st[b].done = 0;
  }
  const float m = block_reduce<NT>(x.max(), sh, Max());  // and a barrier for hc
  if (tid == 0) w.cmax[(int64_t)b * w.C + c] = m;
  if (!cut) return;
  w.gmax[((int64_t)b * w.C + c) * NT + (tid & ~63) + x.group()] = x.group_max();
  const float top = line_of(m, s);
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (usable(x.z[e])) atomicAdd(&hc[hbin(x.z[e], top, s)], 1u);
  __syncthreads();
  uint32_t *out = (uint32_t *)(w.count + ((int64_t)b * w.C + c) * SM_BINS);
  for (int i = tid; i < SM_BINS / 2; i += NT) out[i] = hc[2 * i] | hc[2 * i + 1] << 16;
}

// The histogram's masses, where a row needs them.
template <typename T>
__global__ __launch_bounds__(256) void sample_mass_kernel(SampleArgs a, SampleWs w, int vec) {
  constexpr int NT = 256;
  __shared__ unsigned long long hm[SM_BINS];
  __shared__ double tab[SM_BINS];
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const RowSet s = row_set(a, b);
  if (!cuts(s) || !weighs(s)) return;
  for (int i = threadIdx.x; i < SM_BINS; i += NT) {
    hm[i] = 0;
    tab[i] = exp_table.v[i];
  }
  const float m = row_max(w, b), top = line_of(m, s);
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  __syncthreads();
  for (int i = blockIdx.x * 4 + (threadIdx.x >> 6); i * SM_RUN < a.V; i += gridDim.x * 4) {
    float z[4];
    load4<T>(z, row, i * SM_RUN + lane * 4, a.V, vec);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t q = mass_of(scaled(z[e], m, s.per), tab);
      if (usable(z[e]) && q) atomicAdd(&hm[hbin(z[e], top, s)], (unsigned long long)q);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < SM_BINS; i += NT)
    if (hm[i]) atomicAdd((unsigned long long *)&w.mass[(int64_t)b * SM_BINS + i], hm[i]);
}

// A row's cuts and, mostly, its draw.  The row's histogram is joined from its chunks'
// and gives the bins of interest; the maxima of 16 say where their logits are.  These
// go into a list: all that can be kept where that is few, else (or where ties make
// them too many) what lies in the bins in which top-k and top-p cut.  Few candidates
// for a cut are ranked, more take the radix, from the list or, where it does not hold
// them all, from the row.  Where the list holds all that is kept the draw is made here
// too: the kept weights by the upper bits of their indexes, then those of one of these
// 1024 runs of indexes against each other.
//
// A workgroup a row, each step of which waits for the one before: what counts is how
// much code there is to fetch once and how many loads are under way at a time.  Hence
// loops that are not unrolled, and candidates read again rather than held.
template <typename T>
__global__ __launch_bounds__(1024) void sample_cut_kernel(SampleArgs a, SampleWs w, int vec) {
  constexpr int NT = 1024, AHEAD = 8;
  __shared__ union {
    Bins bins;
    Ranks ranks;
    Radix radix;
    unsigned long long run[1024];
  } S;
  __shared__ double tab[SM_BINS];
  __shared__ uint64_t list[SM_CAP];
  __shared__ uint16_t groups[SM_CAP];
  __shared__ uint64_t sh[17], need;
  __shared__ int which;
  __shared__ uint32_t found, nlist, ngroups;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const RowSet s = row_set(a, b);
  if (!cuts(s)) return;
  const bool masses = weighs(s);
  S.bins.cm[tid] = masses ? w.mass[(int64_t)b * SM_BINS + tid] : 0;
  S.bins.cc[tid] = 0;
  tab[tid] = exp_table.v[tid];
  if (tid == 0) nlist = ngroups = 0;
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  const int ngroup = w.C * w.waves * 64;
  const float *gmax = w.gmax + (int64_t)b * ngroup;
  // what is read first is under way before it is wanted: maxima of groups and a
  // chunk's histogram
  float gv[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) gv[i] = i * NT + tid < ngroup ? gmax[i * NT + tid] : -INFINITY;
  uint32_t v[SM_BINS / 128];
  const auto chunk = [&](int c) {
    const uint32_t *h = (const uint32_t *)(w.count + ((int64_t)b * w.C + c) * SM_BINS);
#pragma unroll
    for (int i = 0; i < SM_BINS / 128; ++i) v[i] = h[i * 64 + lane];
  };
  int c = tid >> 6;
  if (c < w.C) chunk(c);
  const float m = row_max(w, b), u = a.u[b], top = line_of(m, s);
  __syncthreads();
  while (c < w.C) {
    const int move = hbin(w.cmax[(int64_t)b * w.C + c], top, s);
#pragma unroll
    for (int i = 0; i < SM_BINS / 128; ++i) {
      const int bin = (i * 64 + lane) * 2 + move;
      if (v[i] & 0xffff) atomicAdd(&S.bins.cc[min(bin, SM_BINS - 1)], v[i] & 0xffff);
      if (v[i] >> 16) atomicAdd(&S.bins.cc[min(bin + 1, SM_BINS - 1)], v[i] >> 16);
    }
    c += NT / 64;
    if (c < w.C) chunk(c);
  }
  __syncthreads();
  Cuts r = cut_bins<NT>(s, m, masses, S.bins);
  // top-p's share is of all that top-k keeps: its last bin is wanted too
  if (r.plo >= 0 && r.kbin > r.last) r.last = -1;
  if (r.last >= 0) {  // at most SM_CAP logits, so no more groups of 16
    for (int i0 = 0; i0 < ngroup; i0 += AHEAD * NT) {
      uint32_t take = 0;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (usable(gv[i]) && hbin(gv[i], top, s) <= r.last) take |= 1u << i;
      uint32_t at = places(__popc(take), &ngroups);
      for (; take; take &= take - 1, ++at)
        if (at < SM_CAP) groups[at] = (uint16_t)(i0 + (__ffs(take) - 1) * NT + tid);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int g = i0 + (AHEAD + i) * NT + tid;
        gv[i] = g < ngroup ? gmax[g] : -INFINITY;
      }
    }
    __syncthreads();
    const int ng = min((int)ngroups, SM_CAP) * 16;
    for (int i0 = 0; i0 < ng; i0 += AHEAD * NT) {
      const auto at = [&](int i) {
        const int e = i0 + i * NT + tid;
        return e < ng ? groups[e / 16] * 16 + e % 16 : a.V;
      };
      float z[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) z[i] = at(i) < a.V ? logit<T>(row[at(i)]) : -INFINITY;
      uint32_t take = 0;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (usable(z[i]) && hbin(z[i], top, s) <= r.last) take |= 1u << i;
      uint32_t to = places(__popc(take), &nlist);
      for (; take; take &= take - 1, ++to) {
        const int i = at(__ffs(take) - 1);
        if (to < SM_CAP) list[to] = key_of(logit<T>(row[i]), i);
      }
    }
  } else {
    // the grid's lines around the bins of interest, and some more: three operations
    // pass most logits by, the bins decide on the rest (NaN goes there too)
    const int from = min(r.kbin < 0 ? SM_BINS : r.kbin, r.plo < 0 ? SM_BINS : r.plo), upto = max(r.kbin, r.phi);
    const float slack = 1.f + fabsf(top) * 0x1p-22f, hi = top - (float)from + slack;
    const float lo = upto < SM_BINS - 1 ? top - (float)upto - slack : -INFINITY;
    for (int i0 = tid >> 6; i0 * SM_WAVE < a.V; i0 += NT / 64) {
      Lane<T> x;
      x.load(row, i0 * SM_WAVE, a.V, vec);
      uint32_t take = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float y = x.z[e] * s.per4;
        take |= (!(y < lo) && !(y > hi)) ? 1u << e : 0;
      }
      for (; take; take &= take - 1) {
        const int i = x.index(__ffs(take) - 1);
        const float z = i < a.V ? logit<T>(row[i]) : -INFINITY;
        if (usable(z) && cut_of(r, hbin(z, top, s))) {
          const uint32_t to = atomicAdd(&nlist, 1u);
          if (to < SM_CAP) list[to] = key_of(z, i);
        }
      }
    }
  }
  __syncthreads();
  bool listed = nlist <= (uint32_t)SM_CAP;
  const int n = listed ? (int)nlist : 0;
  if (s.p_on && !masses) {
    // top-p's bins, from the candidates, or where ties make them too many from the row
    S.bins.cm[tid] = S.bins.cc[tid] = 0;
    __syncthreads();
    const auto add = [&](float z) {
      const int bin = hbin(z, top, s);
      atomicAdd(&S.bins.cc[bin], 1u);
      atomicAdd((unsigned long long *)&S.bins.cm[bin], (unsigned long long)mass_of(scaled(z, m, s.per), tab));
    };
    listed = listed && r.last >= 0;
    if (listed) {
#pragma unroll 1
      for (int i = tid; i < n; i += NT) add(z_of(list[i]));
    } else {
#pragma unroll 1
      for (int i = tid; i < a.V; i += NT) {
        const float z = logit<T>(row[i]);
        if (usable(z)) add(z);
      }
    }
    __syncthreads();
    r = cut_bins<NT>(s, m, true, S.bins);
    if (!listed) r.last = -1;
    __syncthreads();
  }
  if (tid == 0) S.ranks.n = 0;
  __syncthreads();
  uint64_t tau = 0;
  if (r.kbin >= 0 || r.plo >= 0) {
#pragma unroll 1
    for (int i = tid; i < n; i += NT)
      if (cut_of(r, hbin(z_of(list[i]), top, s))) {
        const uint32_t at = atomicAdd(&S.ranks.n, 1u);
        if (at < SM_RANK) S.ranks.at[at].key = list[i];
      }
    __syncthreads();
    if (listed && S.ranks.n <= SM_RANK) {
      tau = cut_by_rank<NT>(s, r, m, top, tab, S.ranks);
    } else {
      __syncthreads();
      const auto all = [&](auto f) {
        if (listed) {
#pragma unroll 1
          for (int i = tid; i < n; i += NT) f(list[i]);
        } else {
#pragma unroll 1
          for (int i = tid; i < a.V; i += NT) {
            const float z = logit<T>(row[i]);
            if (usable(z)) f(key_of(z, i));
          }
        }
      };
      tau = cut_by_radix<NT>(all, s, r, m, top, tab, S.radix);
    }
    if (tid == 0) w.st[b].tau = tau;
  }
  if (r.last < 0 || !listed) return;
  const auto index = [](uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); };
  const int shift = max(0, 32 - __clz(a.V - 1) - 10);  // indexes to 1024 runs
  __syncthreads();
  S.run[tid] = 0;
  __syncthreads();
  const auto mass = [&](uint64_t key) { return kept(z_of(key), index(key), m, s, tau, tab); };
#pragma unroll 1
  for (int i = tid; i < n; i += NT) {
    const uint64_t q = mass(list[i]);
    if (q) atomicAdd(&S.run[index(list[i]) >> shift], (unsigned long long)q);
  }
  __syncthreads();
  uint64_t W;
  const uint64_t mine = S.run[tid], upto = block_scan<NT>(mine, sh, W);
  if (W > 0) {
    const uint64_t t = draw_at(s, u, W), before = upto - mine;
    if (t >= before && t < upto) {
      which = tid;
      need = t - before;
      found = 0xffffffffu;
    }
    __syncthreads();
    // of that run: its kept elements, in a list of their own
    if (tid == 0) S.ranks.n = 0;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < n; i += NT)
      if (index(list[i]) >> shift == which) {
        const uint64_t q = mass(list[i]);
        const uint32_t at = q ? atomicAdd(&S.ranks.n, 1u) : SM_RANK;
        if (at < SM_RANK) S.ranks.at[at] = Rank{(uint64_t)index(list[i]), q};
      }
    __syncthreads();
    const int k = (int)S.ranks.n;
    if (k <= SM_RANK) {
      if (tid < k) {
        const Rank at = S.ranks.at[tid];
        uint64_t under = 0;
#pragma unroll 8
        for (int j = 0; j < k; ++j) under += S.ranks.at[j].key < at.key ? S.ranks.at[j].mass : 0;
        if (need >= under && need < under + at.mass) found = (uint32_t)at.key;
      }
    } else {
      __syncthreads();
      // falling lower halves of the keys are rising indexes
      const auto all = [&](auto f) {
#pragma unroll 1
        for (int i = tid; i < n; i += NT)
          if (index(list[i]) >> shift == which) {
            const uint64_t q = mass(list[i]);
            if (q) f(list[i] & 0xffffffffu, q, q);
          }
      };
      uint64_t above;
      const uint64_t low = find_by_radix<NT>(all, need + 1, S.radix, above);
      if (tid == 0) found = (uint32_t)index(low);
    }
    __syncthreads();
  }
  if (tid == 0) {
    a.ids[b] = W > 0 ? (int32_t)found : -1;
    w.st[b].done = 1;
  }
}

// kept weights of every 256 logits, where the list does not hold them
template <typename T>
__global__ __launch_bounds__(256) void sample_sum_kernel(SampleArgs a, SampleWs w, int vec) {
  const int b = blockIdx.y, lane = threadIdx.x & 63, n = (a.V + SM_RUN - 1) / SM_RUN;
  if (w.st[b].done) return;
  const RowSet s = row_set(a, b);
  const float m = row_max(w, b);
  const uint64_t tau = w.st[b].tau;
  const T *row = (const T *)a.z + (int64_t)b * a.stride;
  for (int run = blockIdx.x * 4 + (threadIdx.x >> 6); run < n; run += gridDim.x * 4) {
    const int i = run * SM_RUN + lane * 4;
    float z[4];
    load4<T>(z, row, i, a.V, vec);
    uint64_t q = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) q += kept(z[e], i + e, m, s, tau, exp_table.v);
    q = wave_scan(q);
    if (lane == 63) w.wsum[(int64_t)b * n + run] = q;
  }
}

// the 256 logits and the one of them at which the running sum passes the draw
template <typename T>
__global__ __launch_bounds__(1024) void sample_pick_kernel(SampleArgs a, SampleWs w) {
  constexpr int NT = 1024, PT = SAMPLE_MAX_V / SM_RUN / NT;
  __shared__ uint64_t sh[17], need;
  __shared__ int at;
  const int b = blockIdx.x, tid = threadIdx.x, n = (a.V + SM_RUN - 1) / SM_RUN;
  if (w.st[b].done) return;
  const RowSet s = row_set(a, b);
  const float m = row_max(w, b);
  const uint64_t tau = w.st[b].tau;
  uint64_t v[PT], mine = 0;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    v[i] = tid * PT + i < n ? w.wsum[(int64_t)b * n + tid * PT + i] : 0;
    mine += v[i];
  }
  uint64_t W, sum = block_scan<NT>(mine, sh, W);
  if (W == 0) {
    if (tid == 0) a.ids[b] = -1;
    return;
  }
  const uint64_t t0 = draw_at(s, a.u[b], W);
  sum -= mine;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    if (t0 >= sum && t0 < sum + v[i]) {
      at = tid * PT + i;
      need = t0 - sum;
    }
    sum += v[i];
  }
  __syncthreads();
  const int i = at * SM_RUN + tid;
  uint64_t q = 0;
  if (tid < SM_RUN && i < a.V)
    q = kept(logit<T>(((const T *)a.z + (int64_t)b * a.stride)[i]), i, m, s, tau, exp_table.v);
  const uint64_t t = need, run = block_scan<NT>(q, sh, W);
  if (run > t && run - q <= t) a.ids[b] = i;
}

template <typename T, int NT, int E>
hipError_t sample_row(const SampleArgs &a, hipStream_t s) {
  const int lds = NT * (E + 1) * 4;
  const auto fn = sample_row_kernel<T, NT, E>;
  if (E == 16) {  // with its other arrays beyond 64 KiB
    static std::atomic<int> set[kAttrDevices];
    const hipError_t e = ensure_lds_attr((const void *)fn, lds, set);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3(a.B), dim3(NT), lds, s, a);
  return hipGetLastError();
}
template <typename T, int NT>
hipError_t sample_chunks(const SampleArgs &a, const SampleWs &w, hipStream_t s) {
  const int vec = ((uintptr_t)a.z & 15) == 0 && (a.stride * sizeof(T)) % 16 == 0;
  const dim3 grid(w.C, a.B);
  // the passes that most rows do not need: workgroups enough for the card, each
  // through several runs where the rows are many
  const int all = (a.V + 4 * SM_RUN - 1) / (4 * SM_RUN);
  const auto some = [&](int workgroups) { return dim3(std::min(all, std::max(1, workgroups / a.B)), a.B); };
  hipLaunchKernelGGL((sample_count_kernel<T, NT>), grid, dim3(NT), 0, s, a, w, vec);
  if (a.top_k || a.top_p) {
    if (a.top_p) hipLaunchKernelGGL(sample_mass_kernel<T>, some(1024), dim3(256), 0, s, a, w, vec);
    hipLaunchKernelGGL(sample_cut_kernel<T>, dim3(a.B), dim3(1024), 0, s, a, w, vec);
  }
  hipLaunchKernelGGL(sample_sum_kernel<T>, some(2048), dim3(256), 0, s, a, w, vec);
  hipLaunchKernelGGL(sample_pick_kernel<T>, dim3(a.B), dim3(1024), 0, s, a, w);
  return hipGetLastError();
}
template <typename T>
hipError_t sample_run(const SampleArgs &a, const SampleWs &w, hipStream_t s) {
  // as many waves as hide the chains of float64 operations behind each other
  if (a.V <= SM_ONE / 8) return sample_row<T, 256, 8>(a, s);
  if (a.V <= SM_ONE / 2) return sample_row<T, 1024, 8>(a, s);
  if (a.V <= SM_ONE) return sample_row<T, 1024, 16>(a, s);
  return w.waves == 4 ? sample_chunks<T, 256>(a, w, s) : sample_chunks<T, 1024>(a, w, s);
}

}  // namespace

// enough for fewer rows too, which may be cut into smaller and more chunks
int64_t sample_work_floats(int B, int V) {
  const int fewer = std::min(B, 2048 / std::max(1, (V + 4 * SM_WAVE - 1) / (4 * SM_WAVE)));
  return (int64_t)(std::max(sample_carve(nullptr, B, V, nullptr), sample_carve(nullptr, fewer, V, nullptr)) / 4);
}

hipError_t launch_sample(const SampleArgs &a, int dtype, hipStream_t s) {
  SampleWs w{};
  sample_carve((char *)a.work, a.B, a.V, &w);
  return dtype == GN_DTYPE_F32 ? sample_run<float>(a, w, s) : sample_run<uint16_t>(a, w, s);
}

}  // namespace gn
