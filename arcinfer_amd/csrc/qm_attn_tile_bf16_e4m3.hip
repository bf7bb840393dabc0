// Attention of many rows over a paged cache: q of bf16, an e4m3 cache (qm_attn_tile.h)
#include "qm_attn_tile_launch.h"

namespace qm {
hipError_t attn_tile_bf16_e4m3(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) { return tile_types<__bf16, uint8_t>(a, mt, grid, s); }
}  // namespace qm
