// Masked attention backward for f32 storage.
#include "masked_attn_bwd.h"

namespace dmf {
int mattn_bwd_f32(const AtArgs& a, hipStream_t stream) { return mattn_bwd_t<float>(a, stream); }
}  // namespace dmf
