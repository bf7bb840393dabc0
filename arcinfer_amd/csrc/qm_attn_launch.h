// Launches of attn_kernel for one pair of types (each pair is compiled in a file of its own)
#pragma once
#include "qm_attn_impl.h"

namespace qm {

template <typename TQ, typename TC, int DC, bool FULL, int MT, int PARTS>
void attn_full(const AttnArgs& a, unsigned grid, hipStream_t s) {
  if (a.sel) attn_kernel<TQ, TC, DC, FULL, MT, PARTS, true><<<grid, 256, 0, s>>>(a);
  else attn_kernel<TQ, TC, DC, FULL, MT, PARTS, false><<<grid, 256, 0, s>>>(a);
}

template <typename TQ, typename TC, int DC, int MT, int PARTS>
hipError_t attn_mode(const AttnArgs& a, unsigned grid, hipStream_t s) {
  if (a.kv.D == DC) attn_full<TQ, TC, DC, true, MT, PARTS>(a, grid, s);
  else attn_full<TQ, TC, DC, false, MT, PARTS>(a, grid, s);
  return hipGetLastError();
}

template <typename TQ, typename TC, int PARTS>
hipError_t attn_parts(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) {
  // (row tiles: what the registers hold, as few_rows has it)
  if (a.kv.D <= 64) return mt == 1 ? attn_mode<TQ, TC, 64, 1, PARTS>(a, grid, s) : mt == 2 ? attn_mode<TQ, TC, 64, 2, PARTS>(a, grid, s) : attn_mode<TQ, TC, 64, 4, PARTS>(a, grid, s);
  if (a.kv.D <= 128) return mt == 1 ? attn_mode<TQ, TC, 128, 1, PARTS>(a, grid, s) : attn_mode<TQ, TC, 128, 2, PARTS>(a, grid, s);
  return attn_mode<TQ, TC, 256, 1, PARTS>(a, grid, s);
}

// Parts of P by the bits that the result keeps: f16 behind an 8-bit cache (P is bf16 there) two; f32 two of f16, three of bf16 (two would
// leave 2^-18 of a weight: 2.4e-6 of the result, where f32 sums leave 1e-6)
template <typename TQ, typename TC>
hipError_t attn_types(const AttnArgs& a, int mt, unsigned grid, hipStream_t s) {
  if constexpr (sizeof(TC) == 1 && __is_same(TQ, _Float16)) return a.otype == DT_F32 ? attn_parts<TQ, TC, 3>(a, mt, grid, s) : attn_parts<TQ, TC, 2>(a, mt, grid, s);
  else return a.otype == DT_F32 ? attn_parts<TQ, TC, sizeof(TC) == 2 && __is_same(TQ, _Float16) ? 2 : 3>(a, mt, grid, s) : attn_parts<TQ, TC, 1>(a, mt, grid, s);
}

}  // namespace qm
