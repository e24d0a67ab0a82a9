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
// Windows make sequences alike: a workgroup a CU and no more (64 tokens with windows of 4096,
// 32 heads of 128 over 8, bfloat16: 91 us, 512 workgroups 102, 4096 111; 16 of them: 31
// us, 34 with 384; 24: 39, 48; one of 40 with 8192, 8 heads, float32: 21, 29 with 512), and
// 64 splits at most as well (a window of 131072, 8 heads of 128 over one, bfloat16: 27
// us, 31 with 256; of 65536: 21.6, 20.8 with 128; float32: 29, 32 and 23.4, 22.3).
// Trees whose waves share their rows: 512 workgroups (64 trees of four tokens behind 8000,
// 32 heads of 64 over 8: 60 us, 69 with 1024 or 4096), or 1024 of 2048 keys at least while
// there are few without a split (three trees of 37 behind up to 33333, 12 heads of 80 over
// 4, float32: 35 us, 54 with 512).
// Trees whose waves take rows of their own have few tiles of sequences of unlike length: up
// to 2048 workgroups as long as a split has 1024 keys (16 trees of up to 64 tokens behind up
// to 8000, 32 heads of 128 over 8, bfloat16: 140 us; 512 workgroups: 215), or 1024 of 512
// keys (16 trees of 24 behind up to 3000, 8 heads of 128: 32 us, 36 without; two trees of
// 40 behind 8000, 48 workgroups a split, float32: 54, with 1024 63).
static int64_t kv_splits(bool by_rows, int view, int64_t items, int64_t len) {
  int64_t splits;
  if (!by_rows) {
    splits = std::min<int64_t>(4096 / items, std::clamp<int64_t>(256 / items, 32, 64));
    if (view == KV_WINDOW) splits = std::min(splits, 256 / items);
    if (view == KV_TREE)
      splits = std::min(splits, std::max(512 / items, items < 256 ? std::min(1024 / items, len / 2048) : 0));
    return std::max<int64_t>(std::min(splits, len / 512), 1);
  }
  splits = std::min<int64_t>(512 / items, len / 128);
  if (view == KV_TREE)
    splits = std::max({splits, items >= 64 ? std::min(1024 / items, len / 512) : 0, std::min(2048 / items, len / 1024)});
  return std::max<int64_t>(splits, 1);
}

// Whether a workgroup's waves take rows of their own, through LDS, or else the same 16 rows
// and every fourth step of keys, which other tiles read again.  For windows and trees the
// second has no barrier and no idle waves; it loses where its workgroups (`shared`) are many
// and, for long rows, which every tile turns into bf16 again, the rows.  Both sides, shared
// rows first, in us (32 query heads over 8; B trees of n tokens behind a history, or windows):
//   heads of up to 96 share: of 64, bfloat16, 1 of 50 behind 200: 6.1, 12.9; 4 of 250 behind
//     12000: 228, 271; of 96, float32, 1 of 2000 (8 heads) behind 12000: 250, 305 (but 4 of
//     250 behind 200: 40, 29);
//   more than 128, and 128 in float32, share up to 1024 rows, but for many of a short history:
//     of 256, bfloat16, 4 of 128 behind 3000: 183, 204; 4 of 250 behind 200: 138, 67; 128,
//     float32, 4 of 50 behind 3000: 51, 68; 4 of 250 behind 200: 85, 33 (3000: 217, 182);
//     4 of 250, a window of 1000: 119, 58;
//   128 in bfloat16, of which waves hold two tiles of their own: 1 of 60 behind 700: 11, 23; 4
//     of 128 behind 3000: 77, 90; but 1 of 60 behind 12000: 52, 43; 4 of 100 behind 6000:
//     137, 118; 12 of 60 behind 1: 23, 13; 12 of 128 behind 700: 80, 54; a window of 512, 1
//     of 128: 12, 26, 12 of 128: 75, 46.  Histories are bounds of unlike lengths, for which
//     rows of their own take more splits than for windows (of 8192, 1 of 128: 53, 59; not
//     for all the best, 4 of 128: 183, 143).
// With enough workgroups for the card rows of their own are as fast or faster (64 trees of 32
// behind 100, 8 heads of 64, float32: 12, 9).  On 110 sizes at random where limits on the
// rows alone (1024; for the last kind 160 in trees, 512 in windows) say otherwise this takes 0.61
// of their time, 1.09 at worst.  items: sequences times key heads; keys: that a tile sees.
constexpr int SHARED_ROWS = 8192;  // at most
static bool by_rows(int view, int64_t items, int64_t rows, int64_t keys, int R, int bytes) {
  if (rows <= 16 || view == KV_PREFIX) return rows > 16;
  if (rows > SHARED_ROWS || items * ((rows + 127) / 128) >= 512) return true;
  const int64_t shared = items * ((rows + 15) / 16);
  if (R <= 96) return false;
  if (rows > 1024) return true;
  if (R > 128 || bytes == 4) return shared > 1024 && keys < (view == KV_TREE ? 768 : 1280);
  if (rows <= 160) return false;
  if (rows > 512 || (shared > 1536 && keys < 1024) || (shared > 1024 && keys < 256) || (shared > 768 && keys < 128)) return true;
  return view == KV_TREE && (shared > 1536 || keys > 4096 || shared * keys > 4000000);
}

static KvPlan kv_plan(const KvAttnArgs &a, int dtype) {
  const int B = a.c.B, max_new = a.c.max_new, H = a.H, KVH = a.c.KVH, R = a.c.R;
  const int bytes = dtype == GN_DTYPE_F32 ? 4 : 2;
  KvPlan p{};
  const int64_t rows = (int64_t)max_new * (H / KVH);
  // what the rows of a workgroup see at most: in a window whole steps of the first tokens, and
  // from its first row's window, rounded to a step, to its last row
  const auto keys = [&](int rows_wg) {
    const int64_t len = std::min(std::max(a.c.max_len, 1), KV_MAX_TOKENS);  // no table holds more
    if (a.view != KV_WINDOW) return len;
    const int64_t tokens = std::min<int64_t>(max_new, (rows_wg - 1) / a.G + 2);
    return std::min(len, ((int64_t)a.sinks + 63) / 64 * 64 + a.window + tokens + 63);
  };
  // up to one tile of rows the waves share it and split the keys; beyond, every further
  // tile would read all keys again, which windows and trees often still gain by
  p.by_rows = by_rows(a.view, (int64_t)B * KVH, rows, keys(16), R, bytes);
  // two tiles a wave use a K or V operand twice: 310 us for two prompts of 2048 tokens
  // behind 2048, one tile 376; larger heads and float32's parts leave no registers
  p.rt = p.by_rows && rows > 64 && R <= kv_two_tiles(bytes) ? 2 : 1;
  p.rows_wg = 16 * p.rt * (p.by_rows ? 4 : 1);
  p.tiles = (int)((rows + p.rows_wg - 1) / p.rows_wg);
  const int64_t items = (int64_t)B * KVH * p.tiles, unit = p.by_rows ? 64 : 256;
  const int64_t len = keys(p.rows_wg);
  const int64_t splits = kv_splits(p.by_rows, a.view, items, len), chunk = (len + splits - 1) / splits;
  p.chunk = (int)((chunk + unit - 1) / unit * unit);
  p.splits = (int)((len + p.chunk - 1) / p.chunk);  // no more than kv_splits: chunks only grow
  p.work = p.splits > 1 && (rows > 16 || len > KV_SHORT);
  return p;
}

// what `rows` (split, token, head) rows of outputs take
static int64_t kv_part_floats(int64_t rows, int R) { return kv_part_at(1, rows) + rows * R; }

// Enough for every call of every view, or of prefixes alone, with no more sequences, new
// tokens or tokens.  One with fewer of the first two is split further, and a shorter bound
// may round to more splits, so the most that splits x rows reaches is looked for over all
// numbers of workgroups that a view splits at all, with as many rows as their tiles hold.
int64_t kv_attn_work_floats(int B, int max_new, int max_len, int H, int KVH, int hd, bool every_view) {
  if (B == 0 || max_new == 0 || max_len == 0) return 0;
  const int R = kv_row(hd), G = H / KVH;
  const int64_t len = std::min(max_len, KV_MAX_TOKENS);
  int64_t most = 0;
  const auto look = [&](bool own, int64_t tiles, int64_t rows) {  // own: rows of a wave's own; rows: of a key head
    const int64_t n = std::min<int64_t>(max_new, rows / G);
    if (n == 0 || (own && n * G <= 16)) return;
    const int first = !own && tiles > 1 ? KV_WINDOW : KV_PREFIX;  // prefixes share one tile alone
    for (int64_t b = 1; b <= B && b * KVH * tiles <= (own ? 1024 : 2048); ++b) {
      // heads of up to 96 go by rows and sequences alone
      const bool views = every_view && (!own || R > 96 || by_rows(KV_TREE, b * KVH, n * G, len, R, 4));
      int64_t s = 0;
      for (int view = first; view <= (views ? KV_TREE : KV_PREFIX); ++view)
        s = std::max(s, kv_splits(own, view, b * KVH * tiles, len));
      if (s > 1) most = std::max(most, s * b * n * H);
    }
  };
  if (len > KV_SHORT) look(false, 1, 16);
  for (int64_t tiles = 1; tiles * KVH <= 1024; ++tiles) {  // of one 16-row tile a wave, of two
    look(true, tiles, tiles * 64);
    look(true, tiles, tiles * 128);
  }
  if (every_view && max_new * (int64_t)G > 16)  // windows and trees whose rows all waves share
    for (int64_t tiles = 1; tiles * KVH <= 2048 && tiles * 16 <= SHARED_ROWS; ++tiles) look(false, tiles, tiles * 16);
  return most ? kv_part_floats(most, R) : 0;
}

int64_t kv_attn_need_floats(const KvAttnArgs &a, int dtype) {
  const KvPlan p = kv_plan(a, dtype);
  return p.work ? kv_part_floats((int64_t)p.splits * a.c.B * a.c.max_new * a.H, a.c.R) : 0;
}

hipError_t launch_kv_attn(const KvAttnArgs &a0, int dtype, float *scratch, int64_t scratch_floats, hipStream_t s) {
  KvAttnArgs a = a0;
  const KvArgs &c = a.c;
  KvPlan p = kv_plan(a, dtype);
  if (p.splits > 1 && !p.work) {
    a.work = scratch;
    if (kv_part_floats((int64_t)p.splits * c.B * c.max_new * a.H, c.R) > scratch_floats) {
      p.splits = 1;
      p.chunk = c.max_len;
    }
  }
  const bool f32 = dtype == GN_DTYPE_F32;
  if (a.view == KV_WINDOW) return f32 ? launch_kv_window_f32(a, p, s) : launch_kv_window_bf16(a, p, s);
  if (a.view == KV_TREE) return f32 ? launch_kv_tree_f32(a, p, s) : launch_kv_tree_bf16(a, p, s);
  return f32 ? kv_attn_typed<float, KV_PREFIX>(a, p, s) : launch_kv_attn_bf16(a, p, s);
}

}  // namespace gn
