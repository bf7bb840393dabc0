// Which work-group of an attention call takes which rows and keys: worked out on the device, from the lengths as they are when the
// call runs (a captured graph's sequences grow). Every work-group adds up the batch's blocks for itself: for a few hundred sequences
// that is one load a thread and two sums, about a microsecond, where a launch before this one would be two.
#pragma once
#include "qm_kv.h"

namespace qm {

constexpr int kWaves = 4;   // of a work-group
constexpr int kBlock = 32;  // keys of a wave's step

// Rows of a sequence, clamped to the call's (device lists are not trusted with memory)
__device__ __forceinline__ int row_from(const Seqs& s, int b) {
  if (!s.start) return b < s.T ? b : s.T;
  const int r = s.start[b];
  return r < 0 ? 0 : r < s.T ? r : s.T;
}
__device__ __forceinline__ int rows_of(const Seqs& s, int b) {
  const int n = (s.start ? row_from(s, b + 1) : (b < s.T ? b + 1 : s.T)) - row_from(s, b);
  return n > 0 ? n : 0;
}

// The sequence of row t (-1: none)
__device__ __forceinline__ int sequence_of(const Seqs& s, int t) {
  if (!s.start) return t < s.B ? t : -1;
  int lo = 0, hi = s.B;  // the last b with start[b] <= t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.start[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo < s.B && t - row_from(s, lo) < rows_of(s, lo) && t >= row_from(s, lo) ? lo : -1;
}

// The item of a work-group: a row tile rt of sequence b, and piece c of its blocks
struct Item {
  int b, rt, c, blocks;  // blocks of 128 keys of a piece
  int unit;              // the first piece's number of the sequence
};

// Blocks of 128 keys of sequence b, the prefix in front of them
__device__ __forceinline__ long long blocks_of(const AttnArgs& a, int b) {
  const long long most = (long long)a.s.W << a.kv.lg;
  long long n = a.s.len[b];
  n = n < 0 ? 0 : n < most ? n : most;
  return ((n + 31) / 32 + (a.prefix_len + 31) / 32 + 3) >> 2;
}

// Sum over a work-group of 256 (every thread gets it)
__device__ __forceinline__ long long sum256(long long v, long long* red) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// Blocks of a piece: the batch's (row tile, block) pairs of all heads over the pieces aimed at
__device__ __forceinline__ int piece_blocks(const AttnArgs& a, int RT, long long* red) {
  if (!a.target) return 0x7fffffff;
  long long all = 0;
  for (int b = threadIdx.x; b < a.s.B; b += 256) all += (long long)((rows_of(a.s, b) * a.G + RT - 1) / RT) * blocks_of(a, b);
  all = sum256(all, red) * a.kv.HK;
  const long long n = (all + a.target - 1) / a.target;
  return n > 1 ? (int)n : 1;
}

// Pieces of one row tile of sequence b
__device__ __forceinline__ int pieces_of(const AttnArgs& a, int b, int blocks) {
  const long long n = (blocks_of(a, b) + blocks - 1) / blocks;
  return n > 1 ? (int)n : 1;
}

// The item of piece number `unit` (piece c of row tile rt is number first + c * row tiles + rt of its sequence); false: there is none
template <int RT>
__device__ __forceinline__ bool find_item(const AttnArgs& a, int unit, Item* out, long long* red) {
  const int blocks = piece_blocks(a, RT, red);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) out->b = -1;
  long long base = 0;
  for (int b0 = 0; b0 < a.s.B && base <= unit; b0 += 256) {
    const int b = b0 + threadIdx.x;
    const int rts = b < a.s.B ? (rows_of(a.s, b) * a.G + RT - 1) / RT : 0;
    const long long units = rts ? (long long)rts * pieces_of(a, b, blocks) : 0;
    long long end = units;  // inclusive sums: of the wave's lanes, then of the waves before
    for (int o = 1; o < 64; o <<= 1) {
      const long long v = __shfl_up(end, o);
      if (lane >= o) end += v;
    }
    __syncthreads();
    if (lane == 63) red[wave] = end;
    __syncthreads();
    long long all = 0;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) end += red[w];
      all += red[w];
    }
    const long long first = base + end - units;
    if (units && unit >= first && unit < first + units) {
      const int at = (int)(unit - first);
      out->b = b;
      out->rt = at % rts;
      out->c = at / rts;
      out->blocks = blocks;
      out->unit = (int)first;
    }
    base += all;
  }
  __syncthreads();
  return out->b >= 0;
}

}  // namespace qm
