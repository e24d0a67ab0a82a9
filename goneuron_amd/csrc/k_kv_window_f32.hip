// Attention over the paged 8-bit cache for float32 queries that see a sliding window and the first tokens.
#include "k_kv_attn.h"

namespace gn {
hipError_t launch_kv_window_f32(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  return kv_attn_typed<float, KV_WINDOW>(a, p, s);
}
}  // namespace gn
