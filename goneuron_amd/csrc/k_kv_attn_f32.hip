// Attention over the paged 8-bit cache: the split of the work, and the kernels for
// float32 queries.
#include <algorithm>

#include "k_kv_attn.h"

namespace gn {

static KvPlan kv_plan(int B, int max_new, int max_len, int H, int KVH, int R, int bytes) {
  KvPlan p{};
  const int64_t rows = (int64_t)max_new * (H / KVH);
  // up to one tile of rows the waves share it and split the keys; beyond, every
  // further tile would read all keys again
  p.by_rows = rows > 16;
  // two tiles a wave use a K or V operand twice: 241 us for two prompts of 2048 tokens
  // behind 2048, one tile 338; larger heads and float32's parts leave no registers
  p.rt = rows > 64 && R <= kv_two_tiles(bytes) ? 2 : 1;
  p.rows_wg = 16 * p.rt * (p.by_rows ? 4 : 1);
  p.tiles = (int)((rows + p.rows_wg - 1) / p.rows_wg);
  // Keys are split until every CU has work to change over to.  Single tokens: 4096
  // workgroups for sequences of unlike length (64 of up to 8192 tokens, 8 heads: 122 us;
  // 8192 workgroups 137, 2048 128), but 32 splits at most, or 64 while a workgroup a
  // CU is not reached: the join reads them all (one sequence of 131072, 8 heads: 58 us
  // with 32 splits, 61 with 64; one head: 36 and 27).  Prompts: 512 workgroups (24.8 us
  // for the five float32 prompts, 1024: 33.2), 128 keys a split at least.
  const int64_t items = (int64_t)B * KVH * p.tiles, unit = p.by_rows ? 64 : 256;
  int64_t splits = p.by_rows ? 512 / items : std::min<int64_t>(4096 / items, std::clamp<int64_t>(256 / items, 32, 64));
  const int64_t len = std::min(std::max(max_len, 1), KV_MAX_TOKENS);  // no table holds more
  splits = std::min(splits, len / (p.by_rows ? 128 : 512));
  splits = std::max<int64_t>(splits, 1);
  const int64_t chunk = (len + splits - 1) / splits;
  p.chunk = (int)((chunk + unit - 1) / unit * unit);
  p.splits = (int)((len + p.chunk - 1) / p.chunk);
  return p;
}

int64_t kv_attn_work_floats(int B, int max_new, int max_len, int H, int KVH, int hd) {
  if (B == 0 || max_new == 0 || max_len == 0) return 0;
  const int R = kv_row(hd);
  const int64_t slots = (int64_t)B * max_new * H;
  int64_t most = 0;
  for (int bytes = 2; bytes <= 4; bytes += 2) {  // whichever type the queries have
    const KvPlan p = kv_plan(B, max_new, max_len, H, KVH, R, bytes);
    if (p.splits > 1) most = std::max(most, kv_part_at(p.splits, slots) + p.splits * slots * R);
  }
  return most;
}

hipError_t launch_kv_attn(const KvAttnArgs &a, int dtype, hipStream_t s) {
  const KvArgs &c = a.c;
  const KvPlan p = kv_plan(c.B, c.max_new, c.max_len, a.H, c.KVH, c.R, dtype == GN_DTYPE_F32 ? 4 : 2);
  return dtype == GN_DTYPE_F32 ? kv_attn_typed<float>(a, p, s) : launch_kv_attn_bf16(a, p, s);
}

}  // namespace gn
