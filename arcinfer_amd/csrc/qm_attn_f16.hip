// Attention over a paged cache: q of f16, the cache too (qm_attn_impl.h)
#include "qm_attn_launch.h"

namespace qm {
hipError_t attn_f16(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) { return attn_types<_Float16, _Float16>(a, mt, grid, s); }
}  // namespace qm
