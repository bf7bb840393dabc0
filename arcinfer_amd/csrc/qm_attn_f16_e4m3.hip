// Attention over a paged cache: q of f16, an e4m3 cache (qm_attn_impl.h)
#include "qm_attn_launch.h"

namespace qm {
hipError_t attn_f16_e4m3(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) { return attn_types<_Float16, uint8_t>(a, mt, grid, s); }
}  // namespace qm
