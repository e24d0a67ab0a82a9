// Library-private: the operators that answer token by token (paged 8-bit
// cache, attention over it, sampling), kernels in k_kv.hip and k_sample.hip,
// entry points in gn_serve.hip.
#pragma once
#include "gn_common.h"

namespace gn {

constexpr int KV_MAX_HEAD = 256;
constexpr int KV_MAX_TOKENS = 0x7fffffff - 4096;  // of a sequence; of a call's (token, head) rows
constexpr int KV_MAX_SCALE_EXP = -100;  // smallest block scale: 2^-100
// the padded row of a head: what the kernels are built for
inline int kv_row(int hd) {
  return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 96 ? 96 : hd <= 128 ? 128 : hd <= 192 ? 192 : 256;
}

// one call's view of the cache and of the packed sequences
struct KvArgs {
  uint8_t *k, *v;
  float *ks, *vs;
  const int32_t *table, *starts, *lens;
  int32_t *bad;
  int pages, P, lgP, KVH, hd, R, max_pages;
  int B, N, max_new, max_len;
  int limit;  // tokens that a sequence may have, its new ones among them
};

struct KvAppendArgs {
  KvArgs c;
  const void *q, *x[2];  // queries, (keys, values)
  void *qo;
  int64_t qs, xs[2], qos;
  const float *cs, *sn;  // null: no rotation
  int H;
  int touch;             // pages a sequence's new tokens can lie in
  int qtiles;            // rotation blocks a sequence
  uint32_t per_inv, group_inv, pair_inv;  // inverses of a query head's groups, a row's, a key head's pairs of them
  int vec;               // rows, tables and halves allow 4-value accesses
};
hipError_t launch_kv_append(const KvAppendArgs &a, int dtype, hipStream_t s);
hipError_t launch_kv_check(const KvArgs &c, hipStream_t s);

struct KvAttnArgs {
  KvArgs c;
  const void *q;
  void *out;
  int64_t qs, os;
  int H, G;  // query heads, query heads a key head
  float scale;
  int causal;
  int vec;  // queries and outputs allow 4-value accesses, heads are whole eights
  float *work;
};
// how a call's work is split
struct KvPlan {
  int chunk, splits;  // keys of a split, splits of the longest sequence
  int rt, rows_wg;    // 16-row tiles of a wave, rows of a workgroup
  bool by_rows;       // the workgroup's waves take rows of their own (else keys)
  int tiles;
  bool work;          // the splits meet in the caller's workspace (else, if any, in the context's scratch)
};
// Single tokens of sequences of up to this length need no workspace of the caller's: their
// splits are few enough for the context's scratch.
constexpr int KV_SHORT = 4096;
// padded heads up to this size leave registers for two 16-row tiles a wave
constexpr int kv_two_tiles(int bytes) { return bytes == 4 ? 64 : 128; }
// the workspace: (maximum, sum) of every split's rows, then their outputs
__host__ __device__ inline int64_t kv_part_at(int splits, int64_t slots) { return (splits * slots * 2 + 3) / 4 * 4; }
int64_t kv_attn_work_floats(int B, int max_new, int max_len, int H, int KVH, int hd);
bool kv_attn_uses_work(const KvArgs &c, int H, int dtype);  // whether a call of these very sizes does
hipError_t launch_kv_attn(const KvAttnArgs &a, int dtype, float *scratch, int64_t scratch_floats, hipStream_t s);
hipError_t launch_kv_attn_bf16(const KvAttnArgs &a, const KvPlan &p, hipStream_t s);

struct SampleArgs {
  const void *z;
  int64_t stride;
  const float *temperature, *top_p, *min_p, *u;
  const int32_t *top_k;
  int32_t *ids;
  int B, V;
  float *work;
};
constexpr int SAMPLE_MAX_V = 1 << 20;
int64_t sample_work_floats(int B, int V);
hipError_t launch_sample(const SampleArgs &a, int dtype, hipStream_t s);

}  // namespace gn
