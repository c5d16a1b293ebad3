// Masked attention backward for bf16 storage.
#include "masked_attn_bwd.h"

namespace dmf {
int mattn_bwd_bf16(const AtArgs& a, hipStream_t stream) { return mattn_bwd_t<bf16_t>(a, stream); }
}  // namespace dmf
