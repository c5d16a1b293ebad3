// Masked attention forward for f16 storage.
#include "masked_attn_fwd.h"

namespace dmf {
int mattn_fwd_f16(const AtArgs& a, AtPlan p, hipStream_t stream) { return mattn_fwd_t<f16_t>(a, p, stream); }
}  // namespace dmf
