// Attention over the paged 8-bit cache for bfloat16 queries.
#include "k_kv_attn.h"

namespace gn {
hipError_t launch_kv_attn_bf16(const KvAttnArgs &a, const KvPlan &p, hipStream_t s) {
  return kv_attn_typed<uint16_t>(a, p, s);
}
}  // namespace gn
