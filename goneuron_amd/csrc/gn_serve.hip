// Entry points of the operators that answer token by token: the paged 8-bit
// cache, attention over it, the MultiHeadAttention layer on such a cache, and
// sampling.  Arguments are checked here; what lies in device memory (starts,
// lens, page tables, settings) is checked by the kernels.
#include <math.h>

#include <algorithm>
#include <new>
#include <vector>

#include "gn_ctx.h"
#include "gn_serve.h"

namespace {

constexpr int64_t kMaxRows = (int64_t)1 << 26;
// (token, query head) rows that the kernels count in 32 bits
bool too_many_rows(int B, int max_new, int heads) {
  return B > 0 && max_new > 0 && heads > KV_MAX_TOKENS / B / max_new;
}

int cache_check(gn_ctx *c, const gn_kv_cache *kv, KvArgs &a) {
  if (!kv || !kv->k || !kv->v || !kv->k_scale || !kv->v_scale || !kv->table)
    return set_err(c, GN_ERR_INVALID, "kv cache: null pointer");
  if (kv->page_size != 16 && kv->page_size != 32 && kv->page_size != 64 && kv->page_size != 128)
    return set_err(c, GN_ERR_INVALID, "kv cache: page size %d is not 16, 32, 64 or 128", kv->page_size);
  if (kv->head_dim < 1 || kv->head_dim > KV_MAX_HEAD)
    return set_err(c, GN_ERR_UNSUPPORTED, "kv cache: head size %d is not 1 to %d", kv->head_dim, KV_MAX_HEAD);
  if (kv->pages < 1 || kv->kv_heads < 1 || kv->max_pages < 1 ||
      (int64_t)kv->max_pages * kv->page_size > KV_MAX_TOKENS)
    return set_err(c, GN_ERR_INVALID, "kv cache: %d pages, %d heads, %d pages a sequence", kv->pages, kv->kv_heads,
                   kv->max_pages);
  if (((uintptr_t)kv->k | (uintptr_t)kv->v) & 15)
    return set_err(c, GN_ERR_INVALID, "kv cache: k and v must be 16-byte aligned");
  a.k = (uint8_t *)kv->k;
  a.v = (uint8_t *)kv->v;
  a.ks = kv->k_scale;
  a.vs = kv->v_scale;
  a.table = kv->table;
  a.pages = kv->pages;
  a.P = kv->page_size;
  a.lgP = kv->page_size == 16 ? 4 : kv->page_size == 32 ? 5 : kv->page_size == 64 ? 6 : 7;
  a.KVH = kv->kv_heads;
  a.hd = kv->head_dim;
  a.R = kv_row(kv->head_dim);
  a.max_pages = kv->max_pages;
  return GN_OK;
}

int batch_check(gn_ctx *c, KvArgs &a, const int32_t *starts, const int32_t *lens, int B, int N, int max_new, int max_len,
                int heads, int dtype, int32_t *bad) {
  if (dtype != GN_DTYPE_F32 && dtype != GN_DTYPE_BF16) return set_err(c, GN_ERR_INVALID, "unknown dtype %d", dtype);
  if (!starts || !lens) return set_err(c, GN_ERR_INVALID, "null pointer");
  if (B < 0 || N < 0 || max_new < 0 || max_len < 0 || heads < 1 || heads % a.KVH)
    return set_err(c, GN_ERR_INVALID, "B %d, N %d, max_new %d, max_len %d, %d heads over %d", B, N, max_new, max_len,
                   heads, a.KVH);
  if (B > 65535 || N > kMaxRows || heads > 65535 || (int64_t)B * max_new > kMaxRows || too_many_rows(B, max_new, heads))
    return set_err(c, GN_ERR_UNSUPPORTED, "B %d, N %d, max_new %d or %d heads beyond the launch limits", B, N, max_new, heads);
  a.starts = starts;
  a.lens = lens;
  a.B = B;
  a.N = N;
  a.max_new = max_new;
  a.max_len = max_len;
  a.limit = std::min(max_len, a.max_pages * a.P);
  a.bad = bad;
  return GN_OK;
}

// a call without rows: its sequences are still looked at
int no_rows(gn_ctx *c, const KvArgs &a) {
  if (a.B > 0 && a.bad) HIP_OK(c, launch_kv_check(a, c->stream));
  return GN_OK;
}

int row_check(gn_ctx *c, const char *what, const void *p, int64_t stride, int64_t width, int dtype) {
  if (!p) return set_err(c, GN_ERR_INVALID, "%s is null", what);
  if (stride < width)
    return set_err(c, GN_ERR_INVALID, "%s: stride %lld is less than a row of %lld", what, (long long)stride,
                   (long long)width);
  if ((uintptr_t)p & (dtype == GN_DTYPE_F32 ? 3 : 1)) return set_err(c, GN_ERR_INVALID, "%s is misaligned", what);
  return GN_OK;
}

bool aligned4(const void *p, int64_t stride, int dtype) {
  return ((uintptr_t)p & (dtype == GN_DTYPE_F32 ? 15 : 7)) == 0 && stride % 4 == 0;
}

int append_impl(gn_ctx *c, const KvArgs &kv, const void *q, const void *k, const void *v, void *q_out, int64_t q_stride,
                int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos, const float *sin, int heads,
                int dtype) {
  KvAppendArgs a{};
  a.c = kv;
  a.c.max_new = std::min(kv.max_new, kv.N);  // no sequence has more, whatever the bound
  a.q = q;
  a.x[0] = k;
  a.x[1] = v;
  a.qo = q_out;
  a.qs = q_stride;
  a.xs[0] = k_stride;
  a.xs[1] = v_stride;
  a.qos = q_out_stride;
  a.cs = cos;
  a.sn = sin;
  a.H = heads;
  a.vec = kv.hd % 8 == 0 && aligned4(k, k_stride, dtype) && aligned4(v, v_stride, dtype) &&
          (!q || (aligned4(q, q_stride, dtype) && aligned4(q_out, q_out_stride, dtype))) &&
          (!cos || (((uintptr_t)cos | (uintptr_t)sin) & 15) == 0);
  const double e = dtype == GN_DTYPE_F32 ? 4 : 2;
  KTimer kt(c, GN_KCLASS_OTHER, "kv_append", kv.N * (double)kv.hd * (kv.KVH * 2 * (e + 1) + (q ? 2 * e * heads : 0)));
  HIP_OK(c, launch_kv_append(a, dtype, c->stream));
  return GN_OK;
}

int attn_impl(gn_ctx *c, const KvArgs &kv, const void *q, void *out, int64_t qs, int64_t os, int heads, float scale,
              int causal, int dtype, float *work) {
  KvAttnArgs a{};
  a.c = kv;
  a.q = q;
  a.out = out;
  a.qs = qs;
  a.os = os;
  a.H = heads;
  a.G = heads / kv.KVH;
  a.scale = scale;
  a.causal = causal != 0;
  a.vec = kv.hd % 8 == 0 && aligned4(q, qs, dtype) && aligned4(out, os, dtype);
  a.work = work;
  // the cache's lengths are on the device: the bound stands for them
  KTimer kt(c, GN_KCLASS_OTHER, "kv_attention", 2.0 * kv.B * kv.max_len * (double)kv.KVH * kv.hd);
  HIP_OK(c, launch_kv_attn(a, dtype, c->scratch, (int64_t)c->scratch_floats, c->stream));
  return GN_OK;
}

}  // namespace

extern "C" int gn_kv_cache_bytes(int32_t pages, int32_t page_size, int32_t kv_heads, int32_t head_dim, int64_t *bytes,
                                 int32_t *row) {
  if (!bytes || pages < 1 || kv_heads < 1 || head_dim < 1 || head_dim > KV_MAX_HEAD ||
      (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128))
    return GN_ERR_INVALID;
  const int r = kv_row(head_dim);
  *bytes = (int64_t)pages * page_size * kv_heads * r;
  if (row) *row = r;
  return GN_OK;
}

extern "C" int gn_rope_tables(gn_ctx *c, float *cos, float *sin, int32_t positions, int32_t head_dim) {
  ENTRY(c);
  if (!cos || !sin || positions < 1 || head_dim < 1 || head_dim > 65536 || positions > kMaxRows)
    return set_err(c, GN_ERR_INVALID, "bad rope_tables args");
  if (head_dim < 2) return GN_OK;
  const int half = head_dim / 2;
  try {
    // in parts, so that host memory does not follow the context's length
    const int part = std::max(1, (1 << 20) / half);
    std::vector<float> cs, sn;
    for (int p0 = 0; p0 < positions; p0 += part) {
      const int n = std::min(part, positions - p0);
      rope_tables(n, head_dim, cs, sn, p0);
      const size_t bytes = (size_t)n * half * sizeof(float);
      HIP_OK(c, hipMemcpyAsync(cos + (size_t)p0 * half, cs.data(), bytes, hipMemcpyHostToDevice, c->stream));
      HIP_OK(c, hipMemcpyAsync(sin + (size_t)p0 * half, sn.data(), bytes, hipMemcpyHostToDevice, c->stream));
      HIP_OK(c, hipStreamSynchronize(c->stream));  // the host tables are filled again
    }
  } catch (const std::bad_alloc &) {
    return set_err(c, GN_ERR_OOM, "rope_tables: no host memory");
  }
  return GN_OK;
}

extern "C" int gn_kv_append(gn_ctx *c, const gn_kv_cache *kv, const void *q, const void *k, const void *v, void *q_out,
                            int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos,
                            const float *sin, int32_t rope_len, const int32_t *starts, const int32_t *lens, int32_t B,
                            int32_t N, int32_t max_new, int32_t heads, int32_t dtype, int32_t *bad) {
  ENTRY(c);
  KvArgs a{};
  int rc = cache_check(c, kv, a);
  if (rc) return rc;
  rc = batch_check(c, a, starts, lens, B, N, max_new, a.max_pages * a.P, heads, dtype, bad);
  if (rc) return rc;
  if (!cos != !sin || (cos && rope_len < 0)) return set_err(c, GN_ERR_INVALID, "cos and sin come together");
  if (!q != !q_out) return set_err(c, GN_ERR_INVALID, "q and q_out come together");
  if (cos) a.limit = std::min(a.limit, rope_len);
  if (B == 0 || N == 0 || max_new == 0) return no_rows(c, a);
  const int64_t kw = (int64_t)a.KVH * a.hd, qw = (int64_t)heads * a.hd;
  if ((rc = row_check(c, "k", k, k_stride, kw, dtype)) || (rc = row_check(c, "v", v, v_stride, kw, dtype))) return rc;
  if (q && ((rc = row_check(c, "q", q, q_stride, qw, dtype)) || (rc = row_check(c, "q_out", q_out, q_out_stride, qw, dtype))))
    return rc;
  if (q == q_out && q && q_stride != q_out_stride)
    return set_err(c, GN_ERR_INVALID, "q_out in place of q needs q's stride");
  return append_impl(c, a, q, k, v, q_out, q_stride, k_stride, v_stride, q_out_stride, cos, sin, heads, dtype);
}

extern "C" int gn_kv_attention_workspace(int32_t B, int32_t max_new, int32_t max_len, int32_t heads, int32_t kv_heads,
                                         int32_t head_dim, int64_t *floats) {
  if (!floats || B < 0 || max_new < 0 || max_len < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 ||
      head_dim > KV_MAX_HEAD || too_many_rows(B, max_new, heads))
    return GN_ERR_INVALID;
  *floats = kv_attn_work_floats(B, max_new, max_len, heads, kv_heads, head_dim);
  return GN_OK;
}

extern "C" int gn_kv_attention(gn_ctx *c, const gn_kv_cache *kv, const void *q, void *out, int64_t q_stride,
                               int64_t out_stride, const int32_t *starts, const int32_t *lens, int32_t B, int32_t N,
                               int32_t max_new, int32_t max_len, int32_t heads, float scale, int32_t causal,
                               int32_t dtype, float *work, int32_t *bad) {
  ENTRY(c);
  KvArgs a{};
  int rc = cache_check(c, kv, a);
  if (rc) return rc;
  rc = batch_check(c, a, starts, lens, B, N, max_new, max_len, heads, dtype, bad);
  if (rc) return rc;
  if (!isfinite(scale)) return set_err(c, GN_ERR_INVALID, "scale is not finite");
  if (B == 0 || N == 0 || max_new == 0) return no_rows(c, a);
  const int64_t w = (int64_t)heads * a.hd;
  if ((rc = row_check(c, "q", q, q_stride, w, dtype)) || (rc = row_check(c, "out", out, out_stride, w, dtype))) return rc;
  if (!work && kv_attn_uses_work(a, heads, dtype))
    return set_err(c, GN_ERR_INVALID, "kv_attention needs its workspace");
  if ((uintptr_t)work & 15) return set_err(c, GN_ERR_INVALID, "kv_attention: work must be 16-byte aligned");
  return attn_impl(c, a, q, out, q_stride, out_stride, heads, scale, causal, dtype, work);
}

// ---------------------------------------------------------------------------
// MultiHeadAttention.ForwardWithArena (transformer.go:405-529) for new tokens:
// the layer's projections of the new rows alone, the cache in place of the
// other tokens' keys and values.  work: Q | K | V | O rows, then attention's.
// ---------------------------------------------------------------------------
extern "C" int gn_mha_cached_workspace(int32_t B, int32_t N, int32_t max_new, int32_t max_len, int32_t D, int32_t heads,
                                       int64_t *floats) {
  if (!floats || B < 0 || N < 0 || max_new < 0 || max_len < 0 || D < 1 || heads < 1 || D % heads ||
      D / heads > KV_MAX_HEAD || too_many_rows(B, max_new, heads))
    return GN_ERR_INVALID;
  *floats = 4 * (((int64_t)N * D + 63) / 64 * 64) +
            kv_attn_work_floats(B, max_new, max_len, heads, heads, D / heads);
  return GN_OK;
}

extern "C" int gn_mha_cached_forward(gn_ctx *c, const gn_kv_cache *kv, const float *x, const float *params, float *out,
                                     const float *cos, const float *sin, int32_t rope_len, const int32_t *starts,
                                     const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t max_len, int32_t D,
                                     float *work, int32_t *bad) {
  ENTRY(c);
  KvArgs a{};
  int rc = cache_check(c, kv, a);
  if (rc) return rc;
  rc = batch_check(c, a, starts, lens, B, N, max_new, max_len, a.KVH, GN_DTYPE_F32, bad);
  if (rc) return rc;
  // one limit for both halves: what is not appended is not attended to, nor the other way
  if (cos) a.limit = std::min(a.limit, rope_len);
  if ((int64_t)a.KVH * a.hd != D) return set_err(c, GN_ERR_SHAPE, "%d heads of %d are not D = %d", a.KVH, a.hd, D);
  if (!cos != !sin || (cos && rope_len < 0)) return set_err(c, GN_ERR_INVALID, "cos and sin come together");
  const bool some = B > 0 && N > 0 && max_new > 0;
  if (!some && (rc = no_rows(c, a))) return rc;
  if (N == 0) return GN_OK;
  if (!x || !params || !out || !work) return set_err(c, GN_ERR_INVALID, "null pointer");
  if ((uintptr_t)work & 15) return set_err(c, GN_ERR_INVALID, "mha_cached: work must be 16-byte aligned");
  const int64_t nd = (int64_t)D * D + D, rows = ((int64_t)N * D + 63) / 64 * 64;
  float *qkv = work, *o = work + 3 * rows;
  if (some) {
    GemmArgs g{};
    g.M = N; g.N = D; g.K = D;
    g.A = x; g.lda = D; g.B = params; g.ldb = D;
    g.C = qkv; g.ldc = D; g.alpha = 1.f; g.bias = params + (int64_t)D * D; g.act = F_IDENTITY;
    g.ws = c->scratch; g.ws_cap = c->scratch_floats;
    g.nbatch = 3;
    g.bstride_B = nd; g.bstride_bias = nd; g.bstride_C = rows;
    KTimer kt(c, GN_KCLASS_GEMM, "gemm_fwd", gemm_flops(g));
    HIP_OK(c, launch_gemm('N', 'T', EPI_BIAS_ACT, g, c->stream));
    rc = append_impl(c, a, qkv, qkv + rows, qkv + 2 * rows, qkv, D, D, D, D, cos, sin, a.KVH, GN_DTYPE_F32);
    if (rc) return rc;
  }
  // rows outside every sequence are not attention's to write, but wOut reads them
  HIP_OK(c, launch_fill(o, 0.f, (int64_t)N * D, c->stream));
  if (some) {
    rc = attn_impl(c, a, qkv, o, D, D, a.KVH, (float)(1.0 / sqrt((double)a.hd)), 1, GN_DTYPE_F32, work + 4 * rows);
    if (rc) return rc;
  }
  GemmArgs g{};
  g.M = N; g.N = D; g.K = D;
  g.A = o; g.lda = D; g.B = params + 3 * nd; g.ldb = D;
  g.C = out; g.ldc = D; g.alpha = 1.f; g.bias = params + 3 * nd + (int64_t)D * D; g.act = F_IDENTITY;
  g.ws = c->scratch; g.ws_cap = c->scratch_floats;
  KTimer kt(c, GN_KCLASS_GEMM, "gemm_fwd", gemm_flops(g));
  HIP_OK(c, launch_gemm('N', 'T', EPI_BIAS_ACT, g, c->stream));
  return GN_OK;
}

// ---------------------------------------------------------------- sampling
extern "C" int gn_sample_workspace(int32_t B, int32_t V, int64_t *floats) {
  if (!floats || B < 0 || V < 1 || V > SAMPLE_MAX_V) return GN_ERR_INVALID;
  *floats = sample_work_floats(B, V);
  return GN_OK;
}

extern "C" int gn_sample(gn_ctx *c, const void *logits, int64_t stride, int32_t dtype, const float *temperature,
                         const int32_t *top_k, const float *top_p, const float *min_p, const float *u, int32_t *ids,
                         int32_t B, int32_t V, float *work) {
  ENTRY(c);
  if (dtype != GN_DTYPE_F32 && dtype != GN_DTYPE_BF16) return set_err(c, GN_ERR_INVALID, "unknown dtype %d", dtype);
  if (B < 0 || V < 1) return set_err(c, GN_ERR_INVALID, "B %d, V %d", B, V);
  if (B > 65535 || V > SAMPLE_MAX_V)
    return set_err(c, GN_ERR_UNSUPPORTED, "sample: B %d or V %d beyond 65535 rows of %d", B, V, SAMPLE_MAX_V);
  if (B == 0) return GN_OK;
  if (!u || !ids || !work) return set_err(c, GN_ERR_INVALID, "null pointer");
  if ((uintptr_t)work & 7) return set_err(c, GN_ERR_INVALID, "sample: work must be 8-byte aligned");
  int rc = row_check(c, "logits", logits, stride, V, dtype);
  if (rc) return rc;
  SampleArgs a{};
  a.z = logits;
  a.stride = stride;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.u = u;
  a.ids = ids;
  a.B = B;
  a.V = V;
  a.work = work;
  KTimer kt(c, GN_KCLASS_OTHER, "sample", (double)B * V * (dtype == GN_DTYPE_F32 ? 4 : 2));
  HIP_OK(c, launch_sample(a, dtype, c->stream));
  return GN_OK;
}
