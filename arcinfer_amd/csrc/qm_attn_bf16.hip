// Attention over a paged cache: q of bf16, the cache too (qm_attn_impl.h)
#include "qm_attn_launch.h"

namespace qm {
hipError_t attn_bf16(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) { return attn_types<__bf16, __bf16>(a, mt, grid, s); }
}  // namespace qm
