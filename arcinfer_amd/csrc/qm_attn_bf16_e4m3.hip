// Attention over a paged cache: q of bf16, an e4m3 cache (qm_attn_impl.h)
#include "qm_attn_launch.h"

namespace qm {
hipError_t attn_bf16_e4m3(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) { return attn_types<__bf16, uint8_t>(a, mt, grid, s); }
}  // namespace qm
