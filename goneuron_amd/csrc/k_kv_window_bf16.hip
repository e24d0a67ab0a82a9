// Attention over the paged 8-bit cache for bfloat16 queries that see a sliding window and the first tokens.
#include "k_kv_attn.h"

namespace gn {
hipError_t launch_kv_window_bf16(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  return kv_attn_typed<uint16_t, KV_WINDOW>(a, p, s);
}
}  // namespace gn
