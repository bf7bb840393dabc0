// Which work-group of an attention call takes which rows and keys: worked out on the device, from the lengths as they are when the
// call runs (a captured graph's sequences grow). Every work-group adds up the batch's blocks for itself: for a few hundred sequences
// that is one load a thread and two sums, about a microsecond, where a launch before this one would be two.
#pragma once
#include "qm_kv.h"

namespace qm {

constexpr int kWaves = 4;   // of a work-group
constexpr int kBlock = 32;  // keys of a wave's step
constexpr int kLeast = 1;   // blocks of 128 keys of a piece at least
constexpr int kWhole = 1 << 30;  // and of one that is not cut (a row tile sees fewer than 2^25)

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

// Tokens of a sequence (lengths below zero are zero: sums of them stay within 32 bits)
__device__ __forceinline__ int length_of(const Seqs& s, int b) { return max(s.len[b], 0); }

// Blocks of 128 keys of sequence b, the prefix in front of them (below 2^25: a prefix and a table hold 2^30 keys each)
__device__ __forceinline__ int blocks_of(const AttnArgs& a, int b) {
  const int most = a.s.W << a.kv.lg, n = min(length_of(a.s, b), most);
  return (int)(((unsigned)(n + 31) / 32 + (a.shared ? 0u : (unsigned)(a.prefix_len + 31) / 32) + 3) / 4);
}

// The place of the result of row tile rt's first piece among the slots (of a head): row tiles of RT rows, of a sequence whose rows begin at
// row0. Known without the other sequences' lengths: the tiles of the rows before are at most row0 G / RT and one for each sequence.
__device__ __forceinline__ int first_slot(const AttnArgs& a, int RT, int b, int row0, int rt) {
  return a.s.start ? row0 * a.G / RT + b + rt : b * ((a.G + RT - 1) / RT) + rt;
}

// What a work-group does: row tile rt of key head h of sequence b, piece c of its keys. Pieces behind the first have their results behind all
// first ones: number `more` and on, `rts` from one to the next.
struct Item {
  int b, h, rt, c, rts;
  int blocks;  // blocks of 128 keys of a piece
  int more;
  int parts, slot;  // of a row tile behind the last whole round: its pieces at most, and the place of this one's result (-1: not such a one)
};

// Row tiles of attn_tile_kernel that fill the GPU more than once are whole, but for those behind the last whole round of a.tail work-groups: they
// would leave most CUs idle, and are cut into as many pieces as there is room for, which fill up what the round before them leaves.
struct Tail {
  int whole, tail, parts;
};
constexpr int kMostParts = 32;
// Blocks of 128 keys of such a piece at least: it has its start and a result to be joined (576 row tiles of 1300 to 2800 keys, 128 rows of 128 elements: 168 us;
// by 8 blocks 173, by 16 191, uncut 186)
constexpr int kLeastPart = 4;

// The sequence's row tiles and those of all
__device__ __forceinline__ int tiles_of(const AttnArgs& a, int RT, int b) { return b < a.s.B ? (rows_of(a.s, b) * a.G + RT - 1) / RT : 0; }

// Inclusive sums over the lanes of a wave, by moves within rows of 16 and from one row's end to the next (no LDS)
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false); }
__device__ __forceinline__ int scan64(int v) {
  v += moved<0x111, 0xF>(v);
  v += moved<0x112, 0xF>(v);
  v += moved<0x114, 0xF>(v);
  v += moved<0x118, 0xF>(v);
  v += moved<0x142, 0xA>(v);  // (a row's last lane to the row behind it, of the second and fourth rows)
  return v + moved<0x143, 0xC>(v);  // (the second row's last lane to the third and fourth)
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved_f(float v) { return __builtin_bit_cast(float, moved<CTRL, ROWS>(__builtin_bit_cast(int, v))); }
__device__ __forceinline__ float sum64(float v) {
  v += moved_f<0x111, 0xF>(v);
  v += moved_f<0x112, 0xF>(v);
  v += moved_f<0x114, 0xF>(v);
  v += moved_f<0x118, 0xF>(v);
  v += moved_f<0x142, 0xA>(v);
  v += moved_f<0x143, 0xC>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

__device__ __forceinline__ Tail tail_of(const AttnArgs& a, int RT) {
  float all = 0.0f;  // (below 2^24: exact)
  for (int b = threadIdx.x & 63; b < a.s.B; b += 64) all += (float)tiles_of(a, RT, b);
  const int n = (int)sum64(all) * a.kv.HK, left = n % a.tail;
  Tail t{n, 0, 1};
  if (left && a.tail / left > 1) t = {n - left, left, min(a.tail / left, kMostParts)};
  return t;
}
// Blocks of 128 keys that a row tile's last row sees (the prefix's among them, if it reads them), and of a piece of them
__device__ __forceinline__ int tile_blocks(const AttnArgs& a, int RT, int b, int rt, int rows) {
  const int last = min((rt + 1) * RT, rows * a.G) - 1, most = (int)min((long long)a.s.W << a.kv.lg, 0x7fffffffLL);
  const int seen = min(max(length_of(a.s, b) - rows + last / a.G + 1, 0), most);
  return (int)(((unsigned)(seen + kBlock - 1) / kBlock + (a.shared ? 0u : (unsigned)(a.prefix_len + kBlock - 1) / kBlock) + kWaves - 1) / kWaves);
}
__device__ __forceinline__ int part_blocks(int blocks, int parts) { return parts > 1 ? max((blocks + parts - 1) / parts, kLeastPart) : kWhole; }

// Sequences are looked at 64 at a time by each wave for itself (no wave waits for another): the sum over all of them, then the scan that says
// whose unit number this is. (A call's units and row tiles are below 2^24, as its grid is; sums over lists that are none may wrap.)
__device__ __forceinline__ bool find_item(const AttnArgs& a, int RT, int unit, Item& out) {
  const int lane = threadIdx.x & 63, HK = a.kv.HK;
  out.slot = -1;
  out.parts = 1;
  // Many sequences whose row tiles are whole: unit numbers are those of the tiles' first slots, whose sequence is known or a search finds, where adding up 64
  // at a time would take longer (1024 sequences of 200 tokens, 8 heads of 128: 171 us against 235; of 100, two rows each: 151 against 294). With a list of rows
  // some numbers are no tile's, which leaves CUs idle (100 sequences of 16 rows, tiles of 64: 56 us against 37): there from many more sequences on.
  if (a.s.B > (a.s.start ? 16 * RT : 64) && !a.target && !a.tail) {
    const int f = unit / HK;
    int lo = 0, hi = a.s.B - 1;  // the last b whose first tile's number is not above f
    if (a.s.start) {
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_slot(a, RT, mid, row_from(a.s, mid), 0) <= f) lo = mid;
        else hi = mid - 1;
      }
    } else {
      lo = min(f / ((a.G + RT - 1) / RT), hi);
    }
    out.b = lo;
    out.rts = tiles_of(a, RT, lo);
    const int rt = f - first_slot(a, RT, lo, row_from(a.s, lo), 0);
    if (rt < 0 || rt >= out.rts) return false;
    out.rt = out.rts - 1 - rt;
    out.h = unit % HK;
    out.c = 0;
    out.blocks = kWhole;
    out.more = 0;
    return true;
  }
  // (the first 64 sequences are held: most batches are no larger)
  const int rts0 = tiles_of(a, RT, lane), blocks0 = rts0 ? blocks_of(a, lane) : 0;
  int blocks = kWhole, c = 0;
  if (a.tail) {
    const Tail t = tail_of(a, RT);
    if (unit >= t.whole) {
      const int u = unit - t.whole;
      if (u >= t.tail * t.parts) return false;
      c = u / t.tail;
      unit = t.whole + u % t.tail;
      out.slot = u;
      out.parts = t.parts;
    }
  } else if (a.target) {
    float all = (float)rts0 * (float)blocks0;  // (a few parts in a million more or less do not matter)
    for (int b = lane + 64; b < a.s.B; b += 64) {
      const int n = tiles_of(a, RT, b);
      if (n) all += (float)n * (float)blocks_of(a, b);
    }
    all = sum64(all);
    blocks = max((int)ceilf(all * (float)HK / (float)a.target * 1.00001f), kLeast);
  }
  int units0 = 0, tiles0 = 0;
  for (int b0 = 0; b0 < a.s.B; b0 += 64) {
    const int rts = b0 ? tiles_of(a, RT, b0 + lane) : rts0, n = b0 ? (rts ? blocks_of(a, b0 + lane) : 0) : blocks0;
    const int pieces = max((n + blocks - 1) / blocks, 1), mine = rts * pieces * HK;
    const int units = scan64(mine), tiles = scan64(rts);
    const unsigned long long past = __ballot(units0 + units > unit);
    if (past) {
      const int at = __ffsll(past) - 1;
      out.b = b0 + at;
      out.rts = __builtin_amdgcn_readlane(rts, at);
      out.blocks = blocks;
      const int np = __builtin_amdgcn_readlane(pieces, at) * HK;
      units0 += __builtin_amdgcn_readlane(units - mine, at);
      tiles0 += __builtin_amdgcn_readlane(tiles - rts, at);
      // The row tiles of one piece and head lie 8 work-groups apart: on one XCD, whose L2 then reads the piece once. The last rows' tiles, which
      // see the most keys, begin.
      const int j = unit - units0, whole = np / 8 * 8, rest = np - whole;
      int pair = j, rt = 0;
      if (out.rts > 1) {
        if (j < whole * out.rts) {
          pair = j / (8 * out.rts) * 8 + j % 8;
          rt = j % (8 * out.rts) / 8;
        } else {
          pair = whole + (j - whole * out.rts) % rest;
          rt = (j - whole * out.rts) / rest;
        }
      }
      out.rt = out.rts - 1 - rt;
      out.h = pair % HK;
      out.c = c ? c : pair / HK;
      out.more = units0 / HK - tiles0;
      return true;
    }
    units0 += __builtin_amdgcn_readlane(units, 63);
    tiles0 += __builtin_amdgcn_readlane(tiles, 63);
  }
  return false;
}

// The slots: partial results of row tiles. A slot is four words, the RT rows' maxima and sums, and their results; the words of a row tile's
// first one are how many pieces there are, and the places of the others (the second one's, and from one to the next).
__device__ __forceinline__ size_t slot_floats(int RT, int D) { return 4 + (size_t)RT * (D + 2); }

}  // namespace qm
