// Masked attention backward for f16 storage.
#include "masked_attn_bwd.h"

namespace dmf {
int mattn_bwd_f16(const AtArgs& a, hipStream_t stream) { return mattn_bwd_t<f16_t>(a, stream); }
}  // namespace dmf
