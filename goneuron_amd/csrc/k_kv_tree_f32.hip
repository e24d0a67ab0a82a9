// Attention over the paged 8-bit cache for float32 queries that see the cached tokens and those that a mask names.
#include "k_kv_attn.h"

namespace gn {
hipError_t launch_kv_tree_f32(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  return kv_attn_typed<float, KV_TREE>(a, p, s);
}
}  // namespace gn
