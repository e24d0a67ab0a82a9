// Entry points of the operators that answer token by token: the paged 8-bit
// cache, attention over it, the MultiHeadAttention layer on such a cache,
// rules on logits and sampling.  Arguments are checked here; what lies in device memory (starts,
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
                int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos, const float *sin,
                const int32_t *positions, int rope_len, int heads, int dtype) {
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
  a.at = cos ? positions : nullptr;
  a.rope_len = rope_len;
  a.H = heads;
  a.vec = kv.hd % 8 == 0 && aligned4(k, k_stride, dtype) && aligned4(v, v_stride, dtype) &&
          (!q || (aligned4(q, q_stride, dtype) && aligned4(q_out, q_out_stride, dtype))) &&
          (!cos || (((uintptr_t)cos | (uintptr_t)sin) & 15) == 0);
  const double e = dtype == GN_DTYPE_F32 ? 4 : 2;
  KTimer kt(c, GN_KCLASS_OTHER, "kv_append", kv.N * (double)kv.hd * (kv.KVH * 2 * (e + 1) + (q ? 2 * e * heads : 0)));
  HIP_OK(c, a.at ? launch_kv_append_at(a, dtype, c->stream) : launch_kv_append(a, dtype, c->stream));
  return GN_OK;
}

KvAttnArgs attn_args(const KvArgs &kv, const void *q, void *out, int64_t qs, int64_t os, int heads, float scale, int causal,
                     int dtype, float *work) {
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
  a.view = KV_PREFIX;
  return a;
}

int attn_impl(gn_ctx *c, const KvAttnArgs &a, int dtype) {
  const KvArgs &kv = a.c;
  // the cache's lengths are on the device: the bound stands for them
  const double len = a.view == KV_WINDOW ? std::min((double)kv.max_len, (double)a.sinks + a.window + kv.max_new) : kv.max_len;
  KTimer kt(c, GN_KCLASS_OTHER, a.view == KV_WINDOW ? "kv_window" : a.view == KV_TREE ? "kv_tree" : "kv_attention",
            2.0 * kv.B * len * (double)kv.KVH * kv.hd);
  HIP_OK(c, launch_kv_attn(a, dtype, c->scratch, (int64_t)c->scratch_floats, c->stream));
  return GN_OK;
}

// what the attention calls check alike, and the call
int attention(gn_ctx *c, KvAttnArgs &a, int dtype, const char *what) {
  const int64_t w = (int64_t)a.H * a.c.hd;
  int rc;
  if ((rc = row_check(c, "q", a.q, a.qs, w, dtype)) || (rc = row_check(c, "out", a.out, a.os, w, dtype))) return rc;
  if (!a.work && kv_attn_need_floats(a, dtype) > 0) return set_err(c, GN_ERR_INVALID, "%s needs its workspace", what);
  if ((uintptr_t)a.work & 15) return set_err(c, GN_ERR_INVALID, "%s: work must be 16-byte aligned", what);
  return attn_impl(c, a, dtype);
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

namespace {
int append(gn_ctx *c, const gn_kv_cache *kv, const void *q, const void *k, const void *v, void *q_out, int64_t q_stride,
           int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos, const float *sin, int rope_len,
           const int32_t *positions, bool by_positions, const int32_t *starts, const int32_t *lens, int B, int N, int max_new,
           int heads, int dtype, int32_t *bad) {
  KvArgs a{};
  int rc = cache_check(c, kv, a);
  if (rc) return rc;
  rc = batch_check(c, a, starts, lens, B, N, max_new, a.max_pages * a.P, heads, dtype, bad);
  if (rc) return rc;
  if (!cos != !sin || (cos && rope_len < 0)) return set_err(c, GN_ERR_INVALID, "cos and sin come together");
  if (!q != !q_out) return set_err(c, GN_ERR_INVALID, "q and q_out come together");
  if (cos && !by_positions) a.limit = std::min(a.limit, rope_len);
  if (B == 0 || N == 0 || max_new == 0) return no_rows(c, a);
  if (by_positions && cos && (!positions || rope_len < 1))
    return set_err(c, GN_ERR_INVALID, "rotation needs positions and tables");
  const int64_t kw = (int64_t)a.KVH * a.hd, qw = (int64_t)heads * a.hd;
  if ((rc = row_check(c, "k", k, k_stride, kw, dtype)) || (rc = row_check(c, "v", v, v_stride, kw, dtype))) return rc;
  if (q && ((rc = row_check(c, "q", q, q_stride, qw, dtype)) || (rc = row_check(c, "q_out", q_out, q_out_stride, qw, dtype))))
    return rc;
  if (q == q_out && q && q_stride != q_out_stride)
    return set_err(c, GN_ERR_INVALID, "q_out in place of q needs q's stride");
  return append_impl(c, a, q, k, v, q_out, q_stride, k_stride, v_stride, q_out_stride, cos, sin, by_positions ? positions : nullptr,
                     rope_len, heads, dtype);
}
}  // namespace

extern "C" int gn_kv_append(gn_ctx *c, const gn_kv_cache *kv, const void *q, const void *k, const void *v, void *q_out,
                            int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos,
                            const float *sin, int32_t rope_len, const int32_t *starts, const int32_t *lens, int32_t B,
                            int32_t N, int32_t max_new, int32_t heads, int32_t dtype, int32_t *bad) {
  ENTRY(c);
  return append(c, kv, q, k, v, q_out, q_stride, k_stride, v_stride, q_out_stride, cos, sin, rope_len, nullptr, false, starts,
                lens, B, N, max_new, heads, dtype, bad);
}

extern "C" int gn_kv_append_at(gn_ctx *c, const gn_kv_cache *kv, const void *q, const void *k, const void *v, void *q_out,
                               int64_t q_stride, int64_t k_stride, int64_t v_stride, int64_t q_out_stride, const float *cos,
                               const float *sin, int32_t rope_len, const int32_t *positions, const int32_t *starts,
                               const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t heads, int32_t dtype,
                               int32_t *bad) {
  ENTRY(c);
  return append(c, kv, q, k, v, q_out, q_stride, k_stride, v_stride, q_out_stride, cos, sin, rope_len, positions, true, starts,
                lens, B, N, max_new, heads, dtype, bad);
}

extern "C" int gn_kv_keep(gn_ctx *c, const gn_kv_cache *kv, const int32_t *keep, const int32_t *counts, const int32_t *starts,
                          const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t *bad) {
  ENTRY(c);
  KvArgs a{};
  int rc = cache_check(c, kv, a);
  if (rc) return rc;
  rc = batch_check(c, a, starts, lens, B, N, max_new, a.max_pages * a.P, a.KVH, GN_DTYPE_F32, bad);
  if (rc) return rc;
  if (B == 0 || N == 0 || max_new == 0) return no_rows(c, a);
  if (!keep || !counts) return set_err(c, GN_ERR_INVALID, "null pointer");
  KTimer kt(c, GN_KCLASS_OTHER, "kv_keep", 4.0 * N * (double)a.KVH * a.hd);
  HIP_OK(c, launch_kv_keep(a, keep, counts, c->stream));
  return GN_OK;
}

extern "C" int gn_kv_attention_workspace(int32_t B, int32_t max_new, int32_t max_len, int32_t heads, int32_t kv_heads,
                                         int32_t head_dim, int64_t *floats) {
  if (!floats || B < 0 || max_new < 0 || max_len < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || head_dim < 1 ||
      head_dim > KV_MAX_HEAD || too_many_rows(B, max_new, heads))
    return GN_ERR_INVALID;
  *floats = kv_attn_work_floats(B, max_new, max_len, heads, kv_heads, head_dim, true);
  return GN_OK;
}

// Not of the public interface: what a call of these sizes would take of its workspace
// (view: KvView; -1 for sizes that no call has), for the test that holds it against
// gn_kv_attention_workspace.
extern "C" int64_t gn_kv_attention_need(int32_t view, int32_t B, int32_t max_new, int32_t max_len, int32_t heads,
                                        int32_t kv_heads, int32_t head_dim, int32_t sinks, int32_t window, int32_t dtype) {
  if (view < KV_PREFIX || view > KV_TREE || B < 1 || max_new < 1 || max_len < 0 || heads < 1 || kv_heads < 1 ||
      heads % kv_heads || head_dim < 1 || head_dim > KV_MAX_HEAD || sinks < 0 || window < 0 || too_many_rows(B, max_new, heads))
    return -1;
  KvAttnArgs a{};
  a.c.B = B;
  a.c.max_new = max_new;
  a.c.max_len = max_len;
  a.c.KVH = kv_heads;
  a.c.R = kv_row(head_dim);
  a.H = heads;
  a.G = heads / kv_heads;
  a.view = view;
  a.sinks = sinks;
  a.window = window;
  return kv_attn_need_floats(a, dtype);
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
  KvAttnArgs t = attn_args(a, q, out, q_stride, out_stride, heads, scale, causal, dtype, work);
  return attention(c, t, dtype, "kv_attention");
}

extern "C" int gn_kv_attention_window(gn_ctx *c, const gn_kv_cache *kv, const void *q, void *out, int64_t q_stride,
                                      int64_t out_stride, const int32_t *starts, const int32_t *lens, int32_t B, int32_t N,
                                      int32_t max_new, int32_t max_len, int32_t heads, float scale, int32_t sinks,
                                      int32_t window, int32_t dtype, float *work, int32_t *bad) {
  ENTRY(c);
  KvArgs a{};
  int rc = cache_check(c, kv, a);
  if (rc) return rc;
  rc = batch_check(c, a, starts, lens, B, N, max_new, max_len, heads, dtype, bad);
  if (rc) return rc;
  if (!isfinite(scale)) return set_err(c, GN_ERR_INVALID, "scale is not finite");
  if (sinks < 0 || window < 0) return set_err(c, GN_ERR_INVALID, "%d first tokens, a window of %d", sinks, window);
  if (B == 0 || N == 0 || max_new == 0) return no_rows(c, a);
  KvAttnArgs t = attn_args(a, q, out, q_stride, out_stride, heads, scale, 1, dtype, work);
  t.view = KV_WINDOW;
  t.sinks = sinks;
  t.window = window;
  return attention(c, t, dtype, "kv_attention_window");
}

extern "C" int gn_kv_attention_tree(gn_ctx *c, const gn_kv_cache *kv, const void *q, void *out, int64_t q_stride,
                                    int64_t out_stride, const uint32_t *mask, int64_t mask_stride, const int32_t *starts,
                                    const int32_t *lens, int32_t B, int32_t N, int32_t max_new, int32_t max_len, int32_t heads,
                                    float scale, int32_t dtype, float *work, int32_t *bad) {
  ENTRY(c);
  KvArgs a{};
  int rc = cache_check(c, kv, a);
  if (rc) return rc;
  rc = batch_check(c, a, starts, lens, B, N, max_new, max_len, heads, dtype, bad);
  if (rc) return rc;
  if (!isfinite(scale)) return set_err(c, GN_ERR_INVALID, "scale is not finite");
  if (B == 0 || N == 0 || max_new == 0) return no_rows(c, a);
  if (!mask) return set_err(c, GN_ERR_INVALID, "mask is null");
  if ((uintptr_t)mask & 3) return set_err(c, GN_ERR_INVALID, "mask is misaligned");
  if (mask_stride < (std::min(max_new, N) + 31) / 32)
    return set_err(c, GN_ERR_INVALID, "mask: %lld words do not hold %d bits", (long long)mask_stride, std::min(max_new, N));
  KvAttnArgs t = attn_args(a, q, out, q_stride, out_stride, heads, scale, 0, dtype, work);
  t.view = KV_TREE;
  t.mask = mask;
  t.ms = mask_stride;
  return attention(c, t, dtype, "kv_attention_tree");
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
            kv_attn_work_floats(B, max_new, max_len, heads, heads, D / heads, false);  // it calls no other view
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
    rc = append_impl(c, a, qkv, qkv + rows, qkv + 2 * rows, qkv, D, D, D, D, cos, sin, nullptr, rope_len, a.KVH, GN_DTYPE_F32);
    if (rc) return rc;
  }
  // rows outside every sequence are not attention's to write, but wOut reads them
  HIP_OK(c, launch_fill(o, 0.f, (int64_t)N * D, c->stream));
  if (some) {
    rc = attn_impl(c, attn_args(a, qkv, o, D, D, a.KVH, (float)(1.0 / sqrt((double)a.hd)), 1, GN_DTYPE_F32, work + 4 * rows),
                   GN_DTYPE_F32);
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

// ---------------------------------------------------------------- rules on logits
extern "C" int gn_logits_adjust(gn_ctx *c, const void *logits, int64_t stride, void *out, int64_t out_stride, int32_t dtype,
                                const gn_logit_rules *rules, int32_t B, int32_t V) {
  ENTRY(c);
  if (dtype != GN_DTYPE_F32 && dtype != GN_DTYPE_BF16) return set_err(c, GN_ERR_INVALID, "unknown dtype %d", dtype);
  if (B < 0 || V < 1) return set_err(c, GN_ERR_INVALID, "B %d, V %d", B, V);
  if (!rules) return set_err(c, GN_ERR_INVALID, "rules are null");
  const gn_logit_rules &r = *rules;
  const bool past = r.repetition || r.frequency || r.presence;
  if (r.tokens_stride < 0 || r.bias_stride < 0) return set_err(c, GN_ERR_INVALID, "rules: a negative stride");
  if (past && r.tokens_stride > 0 && !r.tokens) return set_err(c, GN_ERR_INVALID, "penalties need the rows' tokens");
  if (r.bias_stride > 0 && (!r.bias != !r.bias_ids)) return set_err(c, GN_ERR_INVALID, "bias and bias_ids come together");
  if (r.allowed && (r.allowed_stride < (V + 31) / 32 || r.allowed_rows < 1 || (!r.allowed_row && r.allowed_rows < B)))
    return set_err(c, GN_ERR_INVALID, "allowed: %d rows of %lld words for B %d, V %d", r.allowed_rows,
                   (long long)r.allowed_stride, B, V);
  if (B > 65535 || V > SAMPLE_MAX_V || r.tokens_stride > LOGITS_MAX_LIST || r.bias_stride > LOGITS_MAX_LIST)
    return set_err(c, GN_ERR_UNSUPPORTED, "logits_adjust: B %d, V %d or lists beyond 65535 rows of %d", B, V, SAMPLE_MAX_V);
  if (B == 0) return GN_OK;
  int rc = row_check(c, "logits", logits, stride, V, dtype);
  if (rc || (rc = row_check(c, "out", out, out_stride, V, dtype))) return rc;
  if (((uintptr_t)r.repetition | (uintptr_t)r.frequency | (uintptr_t)r.presence | (uintptr_t)r.tokens | (uintptr_t)r.token_lens |
       (uintptr_t)r.prompt_lens | (uintptr_t)r.bias_ids | (uintptr_t)r.bias | (uintptr_t)r.bias_lens | (uintptr_t)r.allowed |
       (uintptr_t)r.allowed_row) & 3)
    return set_err(c, GN_ERR_INVALID, "rules: a misaligned array");
  if (logits == out && stride != out_stride) return set_err(c, GN_ERR_INVALID, "out in place of logits needs their stride");
  LogitArgs a{};
  a.z = logits;
  a.out = out;
  a.zs = stride;
  a.os = out_stride;
  a.r = r;
  if (!past) a.r.tokens_stride = 0;  // a history that nothing is taken from
  if (!r.bias) a.r.bias_stride = 0;
  a.B = B;
  a.V = V;
  KTimer kt(c, GN_KCLASS_OTHER, "logits_adjust", 2.0 * B * V * (dtype == GN_DTYPE_F32 ? 4 : 2));
  HIP_OK(c, launch_logits_adjust(a, dtype, c->stream));
  return GN_OK;
}
