// Masked attention forward for bf16 storage.
#include "masked_attn_fwd.h"

namespace dmf {
int mattn_fwd_bf16(const AtArgs& a, AtPlan p, hipStream_t stream) { return mattn_fwd_t<bf16_t>(a, p, stream); }
}  // namespace dmf
