// Masked attention forward for f32 storage.
#include "masked_attn_fwd.h"

namespace dmf {
int mattn_fwd_f32(const AtArgs& a, AtPlan p, hipStream_t stream) { return mattn_fwd_t<float>(a, p, stream); }
}  // namespace dmf
