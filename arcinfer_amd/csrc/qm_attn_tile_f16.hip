// Attention of many rows over a paged cache: q of f16, the cache too (qm_attn_tile.h)
#include "qm_attn_tile_launch.h"

namespace qm {
hipError_t attn_tile_f16(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) { return tile_types<_Float16, _Float16>(a, mt, grid, s); }
}  // namespace qm
