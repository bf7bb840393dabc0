// Launches of attn_tile_kernel for one pair of types (each pair is compiled in a file of its own)
#pragma once
#include "qm_attn_tile.h"

namespace qm {

template <typename TQ, typename TC, int DC, int MT, int PARTS>
hipError_t tile_mode(const AttnArgs& a, unsigned grid, hipStream_t s) {
  if (a.kv.D == DC) attn_tile_kernel<TQ, TC, DC, true, MT, PARTS><<<grid, 256, 0, s>>>(a);
  else attn_tile_kernel<TQ, TC, DC, false, MT, PARTS><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

template <typename TQ, typename TC, int PARTS>
hipError_t tile_parts(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) {
  // (behind 8-bit caches, tiles of 64 rows are of heads beyond 128 only)
  if constexpr (sizeof(TC) == 1) {
    if (a.kv.D <= 64) return tile_mode<TQ, TC, 64, 2, PARTS>(a, grid, s);
    if (a.kv.D <= 128) return tile_mode<TQ, TC, 128, 2, PARTS>(a, grid, s);
    return tile_mode<TQ, TC, 256, 1, PARTS>(a, grid, s);
  } else {
    if (a.kv.D <= 64) return mt == 1 ? tile_mode<TQ, TC, 64, 1, PARTS>(a, grid, s) : tile_mode<TQ, TC, 64, 2, PARTS>(a, grid, s);
    if (a.kv.D <= 128) return mt == 1 ? tile_mode<TQ, TC, 128, 1, PARTS>(a, grid, s) : tile_mode<TQ, TC, 128, 2, PARTS>(a, grid, s);
    return tile_mode<TQ, TC, 256, 1, PARTS>(a, grid, s);
  }
}

// Parts of P by the bits that the result keeps: f16 behind an 8-bit cache (P is bf16 there) two; f32 two of f16, three of bf16 (two would
// leave 2^-18 of a weight: 2.4e-6 of the result, where f32 sums leave 1e-6)
template <typename TQ, typename TC>
hipError_t tile_types(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) {
  if constexpr (sizeof(TC) == 1 && __is_same(TQ, _Float16)) return a.otype == DT_F32 ? tile_parts<TQ, TC, 3>(a, mt, grid, s) : tile_parts<TQ, TC, 2>(a, mt, grid, s);
  else return a.otype == DT_F32 ? tile_parts<TQ, TC, sizeof(TC) == 2 && __is_same(TQ, _Float16) ? 2 : 3>(a, mt, grid, s) : tile_parts<TQ, TC, 1>(a, mt, grid, s);
}

}  // namespace qm
