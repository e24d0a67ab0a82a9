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
// is one workgroup's, its logits in LDS from the first pass to the draw.  Longer
// rows are cut into chunks, a workgroup each, and read by three passes (maximum,
// histogram, candidates) and, where too many logits are kept to go into the list of
// candidates, a fourth, all but the first out of cache.
#include "gn_serve.h"

namespace gn {
namespace {

constexpr int SM_BINS = 1024;
constexpr int SM_PER = 32;        // bins per unit of the exponent
constexpr int SM_CAP = 4096;      // candidates of a row kept in a list
constexpr int SM_RANK = 256;      // candidates ranked against each other; more: radix
constexpr int SM_MASS_BITS = 43;
constexpr int SM_WAVE = 1024;     // logits of a wave, 16 a lane
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

struct RowState {
  uint64_t tau;        // kept: elements whose key is at least this
  uint64_t mass_k;     // mass of the bins before kbin
  uint64_t mass_p;     // ... before plo
  uint64_t total;
  uint32_t r;          // rank of the last kept element inside kbin
  uint32_t nlist;      // candidates found (the list holds the first SM_CAP)
  int32_t kbin, plo, phi;  // -1: top-k / top-p does not cut
  int32_t last;            // the list holds all of bins 0 .. last (-1: the cuts' bins)
  int32_t done;            // the draw is made
  int32_t pad;
};

struct SampleWs {
  uint64_t *mass, *wsum, *list;
  RowState *st;
  uint32_t *count;
  float *cmax;
  int C, waves;  // chunks of a row, waves of a chunk
};

inline size_t up64(size_t n) { return (n + 63) / 64 * 64; }

size_t sample_carve(char *base, int B, int V, SampleWs *w) {
  SampleWs t{};
  // chunks of 4096, or of 16384 where those fill the card: a quarter of the
  // histograms to join and to search
  t.waves = (int64_t)B * ((V + 4 * SM_WAVE - 1) / (4 * SM_WAVE)) > 2048 ? 16 : 4;
  t.C = (V + t.waves * SM_WAVE - 1) / (t.waves * SM_WAVE);
  size_t off = 0;
  const auto take = [&](size_t bytes) {
    char *p = base ? base + off : nullptr;
    off += up64(bytes);
    return p;
  };
  if (V > SM_ONE) {
    t.mass = (uint64_t *)take((size_t)B * SM_BINS * 8);
    t.wsum = (uint64_t *)take((size_t)B * t.C * t.waves * 8);
    t.list = (uint64_t *)take((size_t)B * SM_CAP * 8);
    t.st = (RowState *)take((size_t)B * sizeof(RowState));
    t.count = (uint32_t *)take((size_t)B * SM_BINS * 4);
    t.cmax = (float *)take((size_t)B * t.C * 4);
  }
  if (w) *w = t;
  return off;
}

template <typename T>
__device__ __forceinline__ float logit(T x);
template <>
__device__ __forceinline__ float logit<float>(float x) { return x; }
template <>
__device__ __forceinline__ float logit<uint16_t>(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

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
  __device__ __forceinline__ float max() const {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) m = fmaxf(m, z[e]);  // passes NaN by
    return m;
  }
};

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
__device__ __forceinline__ uint64_t mass_of(double t, int bin, const double *tab) { return whole(weight_of(t, bin, tab)); }

struct RowSet {
  bool greedy, k_on, p_on;
  double per;  // bins a unit of the logit: 32 / T
  int k;
  float p, minp;
  double least;  // min_p as a weight
};
__device__ __forceinline__ RowSet row_set(const SampleArgs &a, int b) {
  RowSet s;
  const float T = a.temperature ? a.temperature[b] : 1.f;
  s.greedy = !(T > 0.f);
  s.per = s.greedy ? 1.0 : (double)SM_PER / (double)T;
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
// running sum over the workgroup's threads, this one's value included
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *sh) {  // sh: 16 values
  const int w = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh[w] = v;
  __syncthreads();
  for (int i = 0; i < w; ++i) v += sh[i];
  return v;
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
  uint64_t sm[16];
  uint32_t sn[16];
  int found[3];          // kbin, plo, phi
};
// The bins in which top-k and top-p cut, from a row's histogram (NT threads; mass and
// count may be cm and cc).
template <int NT>
__device__ RowState cut_bins(const RowSet &s, const uint64_t *mass, const uint32_t *count, Bins &S) {
  constexpr int PT = SM_BINS / NT;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  uint64_t mv[PT], ms = 0;
  uint32_t nv[PT], ns = 0;
#pragma unroll
  for (int i = 0; i < PT; ++i) {
    mv[i] = mass[tid * PT + i];
    nv[i] = count[tid * PT + i];
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
  for (int i = 0; i < w; ++i) {
    mc += S.sm[i];
    nc += S.sn[i];
  }
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
  const uint64_t total = S.cm[SM_BINS - 1];
  const uint32_t n = S.cc[SM_BINS - 1], K = s.k_on && (uint32_t)s.k < n ? (uint32_t)s.k : n;
  if (K < n)
    for (int i = tid * PT; i < tid * PT + PT; ++i)
      if (S.cc[i] >= K && (i == 0 || S.cc[i - 1] < K)) S.found[0] = i;
  __syncthreads();
  RowState r;
  r.kbin = S.found[0];
  r.total = total;
  r.mass_k = r.kbin > 0 ? S.cm[r.kbin - 1] : 0;
  r.r = r.kbin < 0 ? 0 : K - (r.kbin > 0 ? S.cc[r.kbin - 1] : 0);
  if (s.p_on && n > 0) {
    // top-k's sum lies between these; the exact one decides inside the bins
    const uint64_t lo = share(s.p, r.kbin < 0 ? total : r.mass_k), hi = share(s.p, r.kbin < 0 ? total : S.cm[r.kbin]);
    for (int i = tid * PT; i < tid * PT + PT; ++i) {
      const uint64_t before = i ? S.cm[i - 1] : 0;
      if (S.cm[i] >= lo && before < lo) S.found[1] = i;
      if (S.cm[i] >= hi && before < hi) S.found[2] = i;
    }
  }
  __syncthreads();
  r.plo = S.found[1];
  r.phi = S.found[2];
  r.mass_p = r.plo > 0 ? S.cm[r.plo - 1] : 0;
  // all that can be kept lies in bins 0 .. last
  int last = r.plo >= 0 ? r.phi : r.kbin >= 0 ? r.kbin : SM_BINS - 1;
  if (s.minp > 0.f) last = min(last, bin_of(-(double)SM_PER * log((double)fminf(s.minp, 1.f))) + 1);
  r.last = S.cc[last] <= (uint32_t)SM_CAP ? last : -1;
  r.tau = 0;
  r.nlist = 0;
  r.done = r.pad = 0;
  return r;
}
// Up to SM_RANK candidates (in any order), one a thread: how many of their bins lie
// above one, and their mass, say where the cuts fall.
struct Rank {
  uint64_t key, mass;  // mass: bit 62 of kbin, bit 63 of plo .. phi
};
struct Ranks {
  Rank at[SM_RANK];
  uint32_t n;
  uint64_t tau_k, above_k, tau_p;
};
constexpr uint64_t RANK_K = 1ull << 62, RANK_P = 1ull << 63, RANK_MASS = RANK_K - 1;
// 1: of kbin, 2: of plo .. phi
__device__ __forceinline__ uint32_t cut_of(const RowState &r, int bin) {
  return (bin == r.kbin ? 1u : 0u) | (r.plo >= 0 && bin >= r.plo && bin <= r.phi ? 2u : 0u);
}
// S.at[..].key holds the n candidates
__device__ uint64_t cut_by_rank(const RowSet &s, const RowState &r, float m, const double *tab, Ranks &S) {
  const int tid = threadIdx.x, n = (int)S.n;
  uint64_t key = 0, q = 0;
  uint32_t in = 0;
  if (tid < n) {
    key = S.at[tid].key;
    const double x = scaled(z_of(key), m, s.per);
    const int bin = bin_of(x);
    q = mass_of(x, bin, tab);
    in = cut_of(r, bin);
    S.at[tid].mass = q | (in & 1 ? RANK_K : 0) | (in & 2 ? RANK_P : 0);
  }
  if (tid == 0) S.tau_k = S.tau_p = S.above_k = 0;
  __syncthreads();
  uint64_t mk = 0, mp = 0;
  uint32_t ck = 0;
  if (tid < n) {
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const Rank o = S.at[j];
      const bool over = o.key > key, k = over && (o.mass & RANK_K), p = over && (o.mass & RANK_P);
      const uint64_t qj = o.mass & RANK_MASS;
      ck += k;
      mk += k ? qj : 0;
      mp += p ? qj : 0;
    }
    if ((in & 1) && ck == r.r - 1) {
      S.tau_k = key;
      S.above_k = mk + q;
    }
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
  uint64_t sh[16];
  uint64_t need, prefix, above, key;
  int single;
};
// The key at which the running amount over falling keys reaches `need`; above: the
// mass of the elements over that key, it included.  each(f): f(key, amount, mass)
// for this thread's elements, the keys all different.
template <typename Each>
__device__ uint64_t find_by_radix(const Each &each, uint64_t need, Radix &S, uint64_t &above) {
  const int tid = threadIdx.x;
  // bits in which the keys differ at all
  uint64_t any = 0, none = 0;
  each([&](uint64_t key, uint64_t, uint64_t) {
    any |= key;
    none |= ~key;
  });
  any = block_reduce(any, S.sh, Or());
  none = block_reduce(none, S.sh, Or());
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
    const uint64_t sum = block_scan(mine, S.sh), summ = block_scan(mm, S.sh);
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
template <typename All>
__device__ uint64_t cut_by_radix(const All &all, const RowSet &s, const RowState &r, float m, const double *tab, Radix &S) {
  uint64_t tau = 0, sum = r.total, above;
  const auto of = [&](uint32_t cut, bool mass, auto f) {
    all([&](uint64_t key) {
      const double t = scaled(z_of(key), m, s.per);
      const int bin = bin_of(t);
      if (!(cut_of(r, bin) & cut)) return;
      const uint64_t q = mass_of(t, bin, tab);
      f(key, mass ? q : 1, q);
    });
  };
  if (r.kbin >= 0) {
    tau = find_by_radix([&](auto f) { of(1, false, f); }, r.r, S, above);
    sum = r.mass_k + above;
  }
  if (r.plo >= 0) {
    const uint64_t key = find_by_radix([&](auto f) { of(2, true, f); }, share(s.p, sum) - r.mass_p, S, above);
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
  __shared__ uint64_t sh[16];
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
  m = block_reduce(m, shf, Max());  // and a barrier for the rest
  float zr[E];
#pragma unroll
  for (int e = 0; e < E; ++e) zr[e] = z[tid * (E + 1) + e];
  uint64_t tau = 0;
  if (cut) {
    unsigned long long *hm = (unsigned long long *)S.bins.cm;
    int bin[E];  // -2: no logit to choose
#pragma unroll
    for (int e = 0; e < E; ++e) {  // no branch on the way: all chains at once
      const double x = scaled(zr[e], m, s.per);
      bin[e] = bin_of(x);
      const bool ok = usable(zr[e]);
      if (ok) atomicAdd(&S.bins.cc[bin[e]], 1u);
      if (s.p_on) {  // top-k alone goes by the counts
        const uint64_t q = mass_of(x, bin[e], tab);
        if (ok && q) atomicAdd(&hm[bin[e]], (unsigned long long)q);
      }
      bin[e] = ok ? bin[e] : -2;
    }
    __syncthreads();
    const RowState r = cut_bins<NT>(s, S.bins.cm, S.bins.cc, S.bins);
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
        tau = cut_by_rank(s, r, m, tab, S.ranks);
      } else {
        __syncthreads();
        const auto all = [&](auto f) {
#pragma unroll 1
          for (int e = 0; e < E; ++e)
            if (usable(z[tid * (E + 1) + e])) f(key_of(z[tid * (E + 1) + e], tid * E + e));
        };
        tau = cut_by_radix(all, s, r, m, tab, S.radix);
      }
    }
  }
  uint64_t k[E], q = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    k[e] = kept(zr[e], tid * E + e, m, s, tau, tab);
    q += k[e];
  }
  const uint64_t run = block_scan(q, sh);
  uint64_t W = 0;
  for (int i = 0; i < NT / 64; ++i) W += sh[i];
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
// the chunk's largest logit; clears what the later passes add to
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_max_kernel(SampleArgs a, SampleWs w, int vec) {
  __shared__ float sh[16];
  const int c = blockIdx.x, b = blockIdx.y;
  Lane<T> x;
  x.load((const T *)a.z + (int64_t)b * a.stride, c * NT * 16 + (threadIdx.x >> 6) * SM_WAVE, a.V, vec);
  for (int i = c * NT + threadIdx.x; i < SM_BINS; i += w.C * NT) {
    w.mass[(int64_t)b * SM_BINS + i] = 0;
    w.count[(int64_t)b * SM_BINS + i] = 0;
  }
  if (c == 0 && threadIdx.x == 0) {
    w.st[b].tau = 0;
    w.st[b].nlist = 0;
    w.st[b].done = 0;
  }
  const float m = block_reduce(x.max(), sh, Max());
  if (threadIdx.x == 0) w.cmax[(int64_t)b * w.C + c] = m;
}

// counts and weights by distance from the maximum
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_hist_kernel(SampleArgs a, SampleWs w, int vec) {
  __shared__ unsigned long long hm[SM_BINS];
  __shared__ uint32_t hc[SM_BINS];
  __shared__ double tab[SM_BINS];
  const int c = blockIdx.x, b = blockIdx.y;
  Lane<T> x;
  x.load((const T *)a.z + (int64_t)b * a.stride, c * NT * 16 + (threadIdx.x >> 6) * SM_WAVE, a.V, vec);
  const RowSet s = row_set(a, b);
  if (!cuts(s)) return;
  const float m = row_max(w, b);
  for (int i = threadIdx.x; i < SM_BINS; i += NT) {
    hm[i] = 0;
    hc[i] = 0;
    tab[i] = exp_table.v[i];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const double d = scaled(x.z[e], m, s.per);
    const int bin = bin_of(d);
    const bool ok = usable(x.z[e]);
    if (ok) atomicAdd(&hc[bin], 1u);
    if (s.p_on) {  // top-k alone goes by the counts
      const uint64_t q = mass_of(d, bin, tab);
      if (ok && q) atomicAdd(&hm[bin], (unsigned long long)q);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < SM_BINS; i += NT)
    if (hc[i]) {
      atomicAdd(&w.count[(int64_t)b * SM_BINS + i], hc[i]);
      if (hm[i]) atomicAdd((unsigned long long *)&w.mass[(int64_t)b * SM_BINS + i], hm[i]);
    }
}

// the bins in which a row's cuts fall
__global__ __launch_bounds__(256) void sample_bins_kernel(SampleArgs a, SampleWs w) {
  __shared__ Bins S;
  const int b = blockIdx.x;
  const RowSet s = row_set(a, b);
  if (!cuts(s)) return;
  const RowState r = cut_bins<256>(s, w.mass + (int64_t)b * SM_BINS, w.count + (int64_t)b * SM_BINS, S);
  if (threadIdx.x == 0) w.st[b] = r;
}

// the candidates into the row's list: all that can be kept where that is few, else
// the elements of the bins in which top-k and top-p cut
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_gather_kernel(SampleArgs a, SampleWs w, int vec) {
  const int c = blockIdx.x, b = blockIdx.y;
  Lane<T> x;
  x.load((const T *)a.z + (int64_t)b * a.stride, c * NT * 16 + (threadIdx.x >> 6) * SM_WAVE, a.V, vec);
  const RowSet s = row_set(a, b);
  if (!cuts(s)) return;
  const RowState r = w.st[b];
  const float m = row_max(w, b);
  // logits below this lie behind every bin of interest, with half a bin and more of
  // slack for the comparison in float32; most waves pass most of theirs by.  The last
  // bin has no end.
  const int deepest = max(max(r.last, r.kbin), r.phi);
  const double edge = (double)m - ((double)deepest + 1.5) / s.per - fabs((double)m) * 0x1p-22;
  const float least = deepest < SM_BINS - 1 && edge > -3.4e38 && edge < 3.4e38 ? (float)edge : -INFINITY;
  uint32_t take = 0;  // this lane's candidates, a bit each
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (x.z[e] >= least) {
      const int bin = bin_of(scaled(x.z[e], m, s.per));
      if (usable(x.z[e]) && (bin <= r.last || cut_of(r, bin))) take |= 1u << e;
    }
  // a wave takes its places in the list at once
  const int mine = __popc(take), lane = threadIdx.x & 63;
  const int run = (int)wave_scan((uint32_t)mine);
  const int all = __shfl(run, 63, 64);
  if (all == 0) return;
  uint32_t at = 0;
  if (lane == 0) at = atomicAdd(&w.st[b].nlist, (uint32_t)all);
  at = __shfl(at, 0, 64) + run - mine;
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (take >> e & 1) {
      if (at < (uint32_t)SM_CAP) w.list[(int64_t)b * SM_CAP + at] = key_of(x.z[e], x.index(e));
      ++at;
    }
}

// The exact cut among the candidates: few are ranked, more take the radix, from the
// list or, where it does not hold them all, from the row.  Where the list holds all
// that is kept the draw is made here too: the kept weights by the upper bits of
// their indexes, then those of one of these 1024 runs of indexes against each other.
template <typename T>
__global__ __launch_bounds__(512) void sample_cut_kernel(SampleArgs a, SampleWs w) {
  constexpr int NT = 512, PER = SM_CAP / NT;
  __shared__ union {
    Ranks ranks;
    Radix radix;
    unsigned long long run[1024];
  } S;
  __shared__ double tab[SM_BINS];
  __shared__ uint64_t sh[16], need;
  __shared__ int which;
  __shared__ uint32_t found;
  const int b = blockIdx.x, tid = threadIdx.x;
  const RowSet s = row_set(a, b);
  const RowState r = w.st[b];
  if (!cuts(s)) return;
  const uint64_t *list = w.list + (int64_t)b * SM_CAP;
  const bool listed = r.nlist <= (uint32_t)SM_CAP;
  const int n = listed ? (int)r.nlist : 0;
  uint64_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = i * NT + tid < n ? list[i * NT + tid] : 0;  // no key is 0
  for (int i = tid; i < SM_BINS; i += NT) tab[i] = exp_table.v[i];
  if (tid == 0) S.ranks.n = 0;
  const float m = row_max(w, b), u = a.u[b];
  __syncthreads();
  uint64_t tau = 0;
  if (r.kbin >= 0 || r.plo >= 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] && cut_of(r, bin_of(scaled(z_of(key[i]), m, s.per)))) {
        const uint32_t at = atomicAdd(&S.ranks.n, 1u);
        if (at < SM_RANK) S.ranks.at[at].key = key[i];
      }
    __syncthreads();
    if (listed && S.ranks.n <= SM_RANK) {
      tau = cut_by_rank(s, r, m, tab, S.ranks);
    } else {
      __syncthreads();
      const T *row = (const T *)a.z + (int64_t)b * a.stride;
      const auto all = [&](auto f) {
        if (listed) {
          for (int i = tid; i < n; i += NT) f(list[i]);
        } else {
          for (int i = tid; i < a.V; i += NT) {
            const float z = logit<T>(row[i]);
            if (usable(z)) f(key_of(z, i));
          }
        }
      };
      tau = cut_by_radix(all, s, r, m, tab, S.radix);
    }
    if (tid == 0) w.st[b].tau = tau;
  }
  if (r.last < 0 || !listed) return;
  const auto index = [](uint64_t k) { return (int)(0xffffffffu - (uint32_t)k); };
  const int shift = a.V > 1 ? max(0, 32 - __clz(a.V - 1) - 10) : 0;  // indexes to 1024 runs
  __syncthreads();
  for (int i = tid; i < 1024; i += NT) S.run[i] = 0;
  __syncthreads();
  uint64_t q[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    q[i] = key[i] ? kept(z_of(key[i]), index(key[i]), m, s, tau, tab) : 0;
    if (q[i]) atomicAdd(&S.run[index(key[i]) >> shift], (unsigned long long)q[i]);
  }
  __syncthreads();
  const uint64_t r0 = S.run[tid * 2], r1 = S.run[tid * 2 + 1];
  const uint64_t upto = block_scan(r0 + r1, sh);
  uint64_t W = 0;
  for (int i = 0; i < NT / 64; ++i) W += sh[i];
  if (W > 0) {
    const uint64_t t = draw_at(s, u, W), before = upto - r0 - r1;
    if (t >= before && t < upto) {
      which = tid * 2 + (t >= before + r0);
      need = t - before - (t >= before + r0 ? r0 : 0);
      found = 0xffffffffu;
    }
    __syncthreads();
    // of that run: its kept elements, in a list of their own
    if (tid == 0) S.ranks.n = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (q[i] && index(key[i]) >> shift == which) {
        const uint32_t at = atomicAdd(&S.ranks.n, 1u);
        if (at < SM_RANK) S.ranks.at[at] = Rank{(uint64_t)index(key[i]), q[i]};
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
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (q[i] && index(key[i]) >> shift == which) f(key[i] & 0xffffffffu, q[i], q[i]);
      };
      uint64_t above;
      const uint64_t low = find_by_radix(all, need + 1, S.radix, above);
      if (tid == 0) found = (uint32_t)index(low);
    }
    __syncthreads();
  }
  if (tid == 0) {
    a.ids[b] = W > 0 ? (int32_t)found : -1;
    w.st[b].done = 1;
  }
}

// kept weights of every 1024 logits, where the list does not hold them
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_sum_kernel(SampleArgs a, SampleWs w, int vec) {
  const int c = blockIdx.x, b = blockIdx.y, wave = c * (NT / 64) + (threadIdx.x >> 6);
  if (w.st[b].done) return;
  Lane<T> x;
  x.load((const T *)a.z + (int64_t)b * a.stride, wave * SM_WAVE, a.V, vec);
  const RowSet s = row_set(a, b);
  const float m = row_max(w, b);
  const uint64_t tau = w.st[b].tau;
  uint64_t q = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) q += kept(x.z[e], x.index(e), m, s, tau, exp_table.v);
  q = wave_reduce(q, Add());
  if ((threadIdx.x & 63) == 0) w.wsum[(int64_t)b * w.C * w.waves + wave] = q;
}

// the 1024 logits and the one of them at which the running sum passes the draw
template <typename T>
__global__ __launch_bounds__(256) void sample_pick_kernel(SampleArgs a, SampleWs w, int vec) {
  constexpr int PT = SAMPLE_MAX_V / SM_WAVE / 256, N = Lane<T>::N;
  __shared__ uint64_t sh[16], need;
  __shared__ int at;
  const int b = blockIdx.x, tid = threadIdx.x, n = w.C * w.waves;
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
  uint64_t sum = block_scan(mine, sh), W = 0;
  for (int i = 0; i < 4; ++i) W += sh[i];
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
  if (tid >= 64) return;
  Lane<T> x;
  x.load((const T *)a.z + (int64_t)b * a.stride, at * SM_WAVE, a.V, vec);
  uint64_t t = need;
#pragma unroll
  for (int g = 0; g < Lane<T>::Q; ++g) {
    uint64_t k[N], q = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      k[e] = kept(x.z[g * N + e], x.index(g * N + e), m, s, tau, exp_table.v);
      q += k[e];
    }
    const uint64_t run = wave_scan(q), all = __shfl(run, 63, 64);
    if (t < all) {
      if (run > t && run - q <= t) {
        t -= run - q;
        int e = 0;
        bool more = true;
#pragma unroll
        for (int i = 0; i < N - 1; ++i) {
          more = more && t >= k[i];
          e += more;
          t -= more ? k[i] : 0;
        }
        a.ids[b] = x.index(g * N) + e;
      }
      return;
    }
    t -= all;
  }
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
  hipLaunchKernelGGL((sample_max_kernel<T, NT>), grid, dim3(NT), 0, s, a, w, vec);
  if (a.top_k || a.top_p) {
    hipLaunchKernelGGL((sample_hist_kernel<T, NT>), grid, dim3(NT), 0, s, a, w, vec);
    hipLaunchKernelGGL(sample_bins_kernel, dim3(a.B), dim3(256), 0, s, a, w);
    hipLaunchKernelGGL((sample_gather_kernel<T, NT>), grid, dim3(NT), 0, s, a, w, vec);
    hipLaunchKernelGGL(sample_cut_kernel<T>, dim3(a.B), dim3(512), 0, s, a, w);
  }
  hipLaunchKernelGGL((sample_sum_kernel<T, NT>), grid, dim3(NT), 0, s, a, w, vec);
  hipLaunchKernelGGL(sample_pick_kernel<T>, dim3(a.B), dim3(256), 0, s, a, w, vec);
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

int64_t sample_work_floats(int B, int V) { return (int64_t)(sample_carve(nullptr, B, V, nullptr) / 4); }

hipError_t launch_sample(const SampleArgs &a, int dtype, hipStream_t s) {
  SampleWs w{};
  sample_carve((char *)a.work, a.B, a.V, &w);
  return dtype == GN_DTYPE_F32 ? sample_run<float>(a, w, s) : sample_run<uint16_t>(a, w, s);
}

}  // namespace gn
