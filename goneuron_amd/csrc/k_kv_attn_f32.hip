// Attention over the paged 8-bit cache: the split of the work, and the kernels for
// float32 queries.
#include <algorithm>

#include "k_kv_attn.h"

namespace gn {

// Keys are split until every CU has work to change over to; items: workgroups without a
// split.  Single tokens: 4096 workgroups for sequences of unlike length (64 of up to 8192
// tokens, 8 heads: 121 us; 8192 workgroups 137, 2048 128), but 32 splits at most, or 64
// while a workgroup a CU is not reached: the join reads them all (one sequence of 131072,
// 8 heads: 57 us with 32 splits, 61 with 64; one head: 36 and 27).  Prompts: 512
// workgroups (24.8 us for the five float32 prompts, 1024: 33.2), 128 keys a split at
// least.
static int64_t kv_splits(bool by_rows, int64_t items, int64_t len) {
  int64_t splits = by_rows ? 512 / items : std::min<int64_t>(4096 / items, std::clamp<int64_t>(256 / items, 32, 64));
  splits = std::min(splits, len / (by_rows ? 128 : 512));
  return std::max<int64_t>(splits, 1);
}

static KvPlan kv_plan(int B, int max_new, int max_len, int H, int KVH, int R, int bytes) {
  KvPlan p{};
  const int64_t rows = (int64_t)max_new * (H / KVH);
  // up to one tile of rows the waves share it and split the keys; beyond, every
  // further tile would read all keys again
  p.by_rows = rows > 16;
  // two tiles a wave use a K or V operand twice: 310 us for two prompts of 2048 tokens
  // behind 2048, one tile 376; larger heads and float32's parts leave no registers
  p.rt = rows > 64 && R <= kv_two_tiles(bytes) ? 2 : 1;
  p.rows_wg = 16 * p.rt * (p.by_rows ? 4 : 1);
  p.tiles = (int)((rows + p.rows_wg - 1) / p.rows_wg);
  const int64_t items = (int64_t)B * KVH * p.tiles, unit = p.by_rows ? 64 : 256;
  const int64_t len = std::min(std::max(max_len, 1), KV_MAX_TOKENS);  // no table holds more
  const int64_t splits = kv_splits(p.by_rows, items, len), chunk = (len + splits - 1) / splits;
  p.chunk = (int)((chunk + unit - 1) / unit * unit);
  p.splits = (int)((len + p.chunk - 1) / p.chunk);  // no more than kv_splits: chunks only grow
  p.work = p.splits > 1 && (p.by_rows || len > KV_SHORT);
  return p;
}

// what `rows` (split, token, head) rows of outputs take
static int64_t kv_part_floats(int64_t rows, int R) { return kv_part_at(1, rows) + rows * R; }

// Enough for every call with no more sequences, new tokens or tokens.  One with fewer of
// the first two is split further, and a shorter bound may round to more splits, so the
// most that splits x rows reaches is looked for over all numbers of workgroups that are
// split at all, with as many rows as their tiles hold.
int64_t kv_attn_work_floats(int B, int max_new, int max_len, int H, int KVH, int hd) {
  if (B == 0 || max_new == 0 || max_len == 0) return 0;
  const int R = kv_row(hd), G = H / KVH;
  const int64_t len = std::min(max_len, KV_MAX_TOKENS);
  int64_t most = 0;
  const auto look = [&](bool by_rows, int64_t tiles, int64_t rows) {  // rows: of a key head
    const int64_t n = std::min<int64_t>(max_new, rows / G);
    if (n == 0 || (n * G > 16) != by_rows) return;
    for (int64_t b = 1; b <= B && b * KVH * tiles <= (by_rows ? 256 : 2048); ++b) {
      const int64_t s = kv_splits(by_rows, b * KVH * tiles, len);
      if (s > 1) most = std::max(most, s * b * n * H);
    }
  };
  if (len > KV_SHORT) look(false, 1, 16);
  for (int64_t tiles = 1; tiles * KVH <= 256; ++tiles) {  // of one 16-row tile a wave, of two
    look(true, tiles, tiles * 64);
    look(true, tiles, tiles * 128);
  }
  return most ? kv_part_floats(most, R) : 0;
}

bool kv_attn_uses_work(const KvArgs &c, int H, int dtype) {
  return kv_plan(c.B, c.max_new, c.max_len, H, c.KVH, c.R, dtype == GN_DTYPE_F32 ? 4 : 2).work;
}

hipError_t launch_kv_attn(const KvAttnArgs &a0, int dtype, float *scratch, int64_t scratch_floats, hipStream_t s) {
  KvAttnArgs a = a0;
  const KvArgs &c = a.c;
  KvPlan p = kv_plan(c.B, c.max_new, c.max_len, a.H, c.KVH, c.R, dtype == GN_DTYPE_F32 ? 4 : 2);
  if (p.splits > 1 && !p.work) {
    a.work = scratch;
    if (kv_part_floats((int64_t)p.splits * c.B * c.max_new * a.H, c.R) > scratch_floats) {
      p.splits = 1;
      p.chunk = c.max_len;
    }
  }
  return dtype == GN_DTYPE_F32 ? kv_attn_typed<float>(a, p, s) : launch_kv_attn_bf16(a, p, s);
}

}  // namespace gn
