// Attention over a paged cache, few rows: tokens that are being decoded, chosen pages, and a prefix that a small batch shares. Rows of q against
// the keys and values of one key head:
//
//   S = K q^T, x = scale * S, o = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m)
//
// in one pass over the keys with the running maximum m and sum l of each row. A work-group takes a row tile: 16 MT rows, a row
// being one query head of one token, all of one key head (so that G query heads share each key and value). Its four waves take blocks of
// 32 keys in turn, each with a maximum, a sum and a result of its own, and join them at the end; nothing is shared before, and no
// wave waits for another.
//
// A block in a wave: two MFMAs' worth of 16 keys are the rows of S^T (A operand: 16 bytes of a key a lane, as the cache holds them), the
// tile's rows its columns. In the result layout a lane has four neighbouring keys of each 16 for one row: as the B operand of
// the second product, o^T = V^T P^T, it gives the same eight keys, so P never leaves its lane. V's operand needs eight keys of
// one element a lane: each lane loads 16 bytes (8 elements) of its eight keys and v_perm transposes the 8 x 8 in registers (one
// instruction a register), which makes row r of the j-th MFMA element 8 r + j. Keys and values are thus read straight from the cache, once,
// with no LDS; the page of 16 keys is the same for the whole wave and its address is kept in scalar registers.
//
// P is rounded to V's 16-bit type (bf16 for an 8-bit cache) for the matrix pipe, relative to each weight, where the result is of a type that
// keeps no more bits than that; in two or three parts (each what the ones before left) where it keeps more. The sum l is f32 and unrounded.
//
// What bounds it: long caches, HBM (16 sequences of 4096 tokens, 8 heads of 128, bf16: 50 us, 5.4 TB/s; a large copy reaches 5.1); few short ones, latency: the
// split worked out 1.6 us, q and the first keys 3, the waves' join and the result 2. Chosen pages of prompt tokens (151 of 768 keys of 256, e4m3): 39 us,
// of which a wave spends a third on 8-bit values on their way to the second product.
#pragma once
#include <type_traits>

#include "qm_attn_plan.h"
#include "qm_fp8_dev.h"

namespace qm {

typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

constexpr float kSlack = 8.0f;     // a row's maximum is renewed when it is passed by 2^8: the weights stay below that
constexpr float kMinusInf = -__builtin_inff();

// A value and the one that the lane 16 (32) away holds, in this order or the other
template <int N>
__device__ __forceinline__ void with_other(float v, float& a, float& b) {
  const unsigned x = __builtin_bit_cast(unsigned, v);
  const auto r = N == 16 ? __builtin_amdgcn_permlane16_swap(x, x, false, false) : __builtin_amdgcn_permlane32_swap(x, x, false, false);
  const unsigned r0 = r[0], r1 = r[1];  // (a bit cast of an element itself takes the first one)
  a = __builtin_bit_cast(float, r0);
  b = __builtin_bit_cast(float, r1);
}
// The larger one (NaN if one is: its row's result is)
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max_groups(float v) {  // of the four lanes that hold a row
  float a, b;
  with_other<16>(v, a, b);
  with_other<32>(larger(a, b), a, b);
  return larger(a, b);
}
__device__ __forceinline__ float sum_groups(float v) {
  float a, b;
  with_other<16>(v, a, b);
  with_other<32>(a + b, a, b);
  return a + b;
}

template <typename T>
__device__ __forceinline__ v4f mfma16(v4i a, v4i b, v4f c) {
  if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ int pack2(float x, float y) {
  typedef T v2t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(int, v2t{(T)x, (T)y});
}
template <typename T>
__device__ __forceinline__ float part_of(int w, int i) {
  if constexpr (__is_same(T, _Float16)) return (float)__builtin_bit_cast(v2h, w)[i];
  else return __builtin_bit_cast(float, i ? w & (int)0xFFFF0000 : w << 16);
}
// Two weights as PARTS words of two values: rounded, and what each rounding left
template <typename T, int PARTS, typename F>
__device__ __forceinline__ void in_parts(float x, float y, F put) {
#pragma unroll
  for (int n = 0; n < PARTS; ++n) {
    const int w = pack2<T>(x, y);
    put(n, w);
    x -= part_of<T>(w, 0);
    y -= part_of<T>(w, 1);
  }
}
// Two e4m3 values (bytes 2 HI, 2 HI + 1 of w) as T, exact
template <typename T, bool HI>
__device__ __forceinline__ int widen2(int w) {
  if constexpr (__is_same(T, _Float16)) return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  else return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
}
template <typename T>
__device__ __forceinline__ v4i widen8(int lo, int hi) {
  return v4i{widen2<T, false>(lo), widen2<T, true>(lo), widen2<T, false>(hi), widen2<T, true>(hi)};
}

// p[i] by the scalar unit (i is the same for the whole wave): a vector load would have to be waited for behind the keys' and values'
__device__ __forceinline__ int scalar(const int32_t* p, size_t i) { return ((const __attribute__((address_space(4))) int32_t*)p)[i]; }

// N results to a row of any alignment, 16 bytes at a time where it is aligned to them (N values)
template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, const float* y) {
  constexpr int V = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  typedef T vt __attribute__((ext_vector_type(V)));
  if (((uintptr_t)p & (V * sizeof(T) - 1)) == 0) {
#pragma unroll
    for (int i = 0; i < N; i += V) {
      vt t;
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] = (T)y[i + j];
      *(vt*)(p + i) = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = (T)y[i];
  }
}

// Whether a word of the cache's type holds a value that is not finite
template <typename T>
__device__ __forceinline__ bool odd_word(int w) {
  if constexpr (sizeof(T) == 1) {
    const unsigned x = (unsigned)w & 0x7f7f7f7fu;  // (0x7f and 0xff are NaN: a byte that 1 carries out of)
    return ((x + 0x01010101u) & 0x80808080u) != 0;
  } else {
    constexpr int e = __is_same(T, _Float16) ? 0x7C00 : 0x7F80;
    return ((w & e) == e) | ((w >> 16 & e) == e);
  }
}

// Values that are not finite, in a word of two 16-bit values: as ones where they are of a kind (0 NaN, 1 plus and 2 minus infinity), else zeros
template <typename T>
__device__ __forceinline__ constexpr int one16() { return __is_same(T, _Float16) ? 0x3C00 : 0x3F80; }
template <typename T>
__device__ __forceinline__ int odd_ones(int w, int kind) {
  constexpr int e = __is_same(T, _Float16) ? 0x7C00 : 0x7F80;
  const auto one = [&](int v) {
    const bool is = kind == 0 ? (v & 0x7FFF) > e : kind == 1 ? v == e : v == (e | 0x8000);
    return is ? one16<T>() : 0;
  };
  return one(w & 0xFFFF) | one(w >> 16 & 0xFFFF) << 16;
}
// The word with zeros in their place
template <typename T>
__device__ __forceinline__ int without_odd(int w) {
  if constexpr (sizeof(T) == 1) {
    const unsigned at = (((unsigned)w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return w & ~(int)((at >> 7) * 255u);
  } else {
    constexpr int e = __is_same(T, _Float16) ? 0x7C00 : 0x7F80;
    return w & ~(((w & e) == e ? 0xFFFF : 0) | ((w >> 16 & e) == e ? (int)0xFFFF0000 : 0));
  }
}

// TQ: q's type. TC: the cache's, TQ or uint8_t (e4m3). DC: D rounded up to 64, 128 or 256 (FULL: it is that). MT: row tiles of 16. PARTS: of P. CHOSEN: chosen pages of
// each token; else each sequence's own keys, and in the first work-groups those of the prefix for the rows of the whole batch.

template <typename TQ, typename TC, int DC, bool FULL, int MT, int PARTS, bool CHOSEN>
__global__ __launch_bounds__(256, 2) void attn_kernel(AttnArgs a) {
  constexpr bool E8 = sizeof(TC) == 1;
  typedef std::conditional_t<E8, __bf16, TQ> TP;           // of P and V on the matrix pipe
  constexpr float kBias = __is_same(TP, _Float16) ? 6.0f : 0.0f;  // f16 weights are held times 2^6: with kSlack below 2^14, and small ones longer
  constexpr int RT = 16 * MT, KS = DC / 32;                // rows, k steps of the first product
  constexpr int VB = DC > 128 ? 2 : 1, VE = DC / 16 / VB;  // V: vectors of VE elements a lane and key, VB of them
  constexpr int KL = E8 ? KS / 2 : KS;                     // loads of a key's 16 bytes
  typedef int kvec __attribute__((ext_vector_type(4)));
  typedef int vvec __attribute__((ext_vector_type(VE * (E8 ? 1 : 2) / 4)));
  constexpr int VW = VE * (E8 ? 1 : 2) / 4;                // 32-bit words of a V vector
  constexpr int NO = VB * VE * MT;                         // results of four values
  constexpr bool QL = MT * DC >= 256;                      // q in LDS
  constexpr bool LATE = MT * DC >= 256;                    // the next keys are asked for after the softmax: before it their registers are its own
  constexpr int kJoin = (kWaves - 1) * NO / 4 * 64, kQs = QL ? MT * KS * 64 : 0, kLds = kJoin > kQs ? kJoin : kQs;  // (q's place is free when the waves join)
  __shared__ v4f lds[kLds];
  __shared__ float stat[kWaves][2][RT];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const KvView& kv = a.kv;
  int h, b = 0, rt, c = 0, blocks = kWhole, row0 = 0, rows, after = 0;  // (after: tokens of the sequence behind these rows)
  int rts = 1, more = 0;
  const bool shared = !CHOSEN && (int)blockIdx.x < a.shared_grid;
  if constexpr (CHOSEN) {
    // (each token's pages are its own: the tile is of one token, and every token has the same number of pieces)
    const int unit = blockIdx.x / kv.HK;
    h = blockIdx.x % kv.HK;
    rts = (a.G + RT - 1) / RT;
    row0 = unit / (rts * a.pieces);
    rt = unit % rts;
    c = unit / rts % a.pieces;
    blocks = a.blocks;
    b = sequence_of(a.s, row0);
    if (b < 0) return;  // (a row of no sequence)
    rows = 1;
    after = row_from(a.s, b) + rows_of(a.s, b) - 1 - row0;
  } else if (shared) {
    // the row tiles of one piece and head lie 8 work-groups apart: on one XCD, whose L2 then reads the piece once
    const unsigned w = blockIdx.x, at = w >> 3, pc = (at / a.shared_tiles) * 8 + (w & 7);
    rt = at % a.shared_tiles;
    h = pc % kv.HK;
    c = pc / kv.HK;
    if (c >= a.shared) return;
    blocks = a.shared_blocks;
    rows = a.s.T;
  } else {
    Item it;
    if (!find_item(a, RT, blockIdx.x - a.shared_grid, it)) return;
    b = __builtin_amdgcn_readfirstlane(it.b);
    h = __builtin_amdgcn_readfirstlane(it.h);
    rt = __builtin_amdgcn_readfirstlane(it.rt);
    c = __builtin_amdgcn_readfirstlane(it.c);
    rts = __builtin_amdgcn_readfirstlane(it.rts);
    blocks = __builtin_amdgcn_readfirstlane(it.blocks);
    more = __builtin_amdgcn_readfirstlane(it.more);
    row0 = __builtin_amdgcn_readfirstlane(row_from(a.s, b));
    rows = __builtin_amdgcn_readfirstlane(rows_of(a.s, b));
  }
  // (rows: tokens; a row of the tile is token r / G, query head h G + r % G)
  const int nrows = rows * a.G, first = rt * RT, last = min(first + RT, nrows) - 1;
  const int capacity = shared ? 0 : (int)min((long long)a.s.W << kv.lg, 0x7fffffffLL);
  const int len = shared ? 0 : __builtin_amdgcn_readfirstlane(length_of(a.s, b)) - after;
  // keys that the tile's first and last tokens see of their own
  const int lo_lim = min(max(len - rows + first / a.G + 1, 0), capacity);
  const int hi_lim = min(max(len - rows + last / a.G + 1, 0), capacity);
  int lim[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = first + 16 * m + col;
    lim[m] = min(max(len - rows + r / a.G + 1, 0), capacity);
  }

  // blocks of 32 keys: of the prefix, then of the sequence's own (or of the chosen pages)
  const int shared_blocks32 = CHOSEN || (a.shared && !shared) ? 0 : (a.prefix_len + kBlock - 1) / kBlock;
  const int own_blocks = CHOSEN ? (int)(((long long)a.k * kv.page + kBlock - 1) / kBlock) : (int)(((long long)hi_lim + kBlock - 1) / kBlock);
  const int all_blocks = shared_blocks32 + own_blocks;
  const int begin = (int)min((long long)c * blocks * kWaves, (long long)all_blocks);
  const int end = (int)min((long long)begin + (long long)blocks * kWaves, (long long)all_blocks);
  if (!shared && c > 0 && begin >= all_blocks) return;  // (a piece that this tile's rows do not see)

  // q: k step t of row col holds elements 32 t + 8 g .. + 7 (8-bit keys: 64 (t / 2) + 16 g + 8 (t % 2), as their loads lie). Of larger
  // tiles it stays in LDS, in operand order: the registers are the result's.
  v4i* qs = (v4i*)lds;
  v4i q[QL ? 1 : MT][QL ? 1 : KS];
  const bool qvec = ((uintptr_t)a.q & 15) == 0 && (a.ldq & 7) == 0;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (QL && m % kWaves != wave) continue;
    const int r = min(first + 16 * m + col, nrows - 1);
    const TQ* p = (const TQ*)a.q + (size_t)(row0 + r / a.G) * a.ldq + (size_t)(h * a.G + r % a.G) * kv.D;
    v4i f[KS];
    if (qvec) {
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const int d = E8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g;
        f[t] = *(const v4i*)(p + (FULL || d < kv.D ? d : 0));
      }
    } else {
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const int d = E8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g;
        typedef TQ v8t __attribute__((ext_vector_type(8)));
        v8t e;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[(FULL || d < kv.D ? d : 0) + i];
        f[t] = __builtin_bit_cast(v4i, e);
      }
    }
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int d = E8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g;
      if (!FULL && d >= kv.D) f[t] = v4i(0);
      if constexpr (QL) qs[(m * KS + t) * 64 + lane] = f[t];
      else q[m][t] = f[t];
    }
  }
  if constexpr (QL) __syncthreads();
  const auto query = [&](int m, int t) -> v4i {
    if constexpr (QL) return qs[(m * KS + t) * 64 + lane];
    else return q[m][t];
  };

  v4f o[VB][VE][MT];
  float mx[MT], sum[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    mx[m] = kMinusInf;
    sum[m] = 0.0f;
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int j = 0; j < VE; ++j) o[vb][j][m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }

  // Where the 16 keys of each half of a block lie. The numbers of pages come by scalar loads, asked for one block ahead of the address that
  // they make, and of chosen pages the places in the list one more: nothing waits for them.
  struct Place {
    long long base;  // bytes from the cache's first key (value) to the first of them (a masked page's: of the first page)
    size_t scale;    // and of their scales, in elements
    int pos, limit;  // the first one's place among the prefix's keys, of which `limit` are seen, or (limit -1) in the sequence
    bool dead;       // masked
    __device__ __forceinline__ int sees(int lim) const { return dead ? 0 : (limit >= 0 ? limit : lim) - pos; }  // how many of them a row of limit lim sees
  };
  const int32_t* table = a.s.table + (size_t)b * a.s.W;
  const int32_t* sel = a.sel + ((size_t)row0 * kv.HK + h) * a.k;
  struct Asked {
    int page[2], pos[2], limit;
  };
  const auto chosen = [&](int i, int s) {  // the entry of the list of chosen pages
    const int e = (i * kBlock + 16 * s) >> kv.lg;
    return scalar(sel, e < a.k ? e : 0);
  };
  const auto ask = [&](int i, const int* pick) {
    Asked r;
    const bool pre = !CHOSEN && i < shared_blocks32;
    r.limit = pre ? a.prefix_len : -1;
    const int32_t* list = pre ? a.prefix : table;
    const int most = pre ? a.prefix_len : hi_lim;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      int pos = i < end ? (pre ? i : i - shared_blocks32) * kBlock + 16 * s : 0x7fffffff;
      if constexpr (CHOSEN) {
        const int in = (i * kBlock + 16 * s) & (kv.page - 1), n = pick[s];
        pos = i < end && (i * kBlock + 16 * s) >> kv.lg < a.k && n >= 0 && n < a.s.W ? (n << kv.lg) + in : 0x7fffffff;
      }
      r.pos[s] = pos;
      r.page[s] = scalar(list, pos < most ? pos >> kv.lg : 0);  // (without a branch: one would wait; `placed` looks at the place)
    }
    return r;
  };
  const auto placed = [&](const Asked& q, int s) {
    Place r;
    r.pos = q.pos[s];
    r.limit = q.limit;
    const int page = q.page[s];
    r.dead = (unsigned)page >= (unsigned)kv.pages || r.pos >= (q.limit >= 0 ? q.limit : hi_lim);
    const int pg = r.dead ? 0 : page, in = r.dead ? 0 : r.pos & (kv.page - 1);  // (16 rows from there are the page's: place 0 of page 0 always is)
    r.base = (pg * kv.ps + h * kv.hs + in * kv.ts) * (long long)sizeof(TC);
    r.scale = ((size_t)pg * kv.HK + h) * kv.page + in;
    return r;
  };

  // a lane's places in 16 keys (token_stride is below 2^26 elements)
  const unsigned k_row = (unsigned)col * (unsigned)kv.ts * (unsigned)sizeof(TC), v_row = 4u * (unsigned)g * (unsigned)kv.ts * (unsigned)sizeof(TC);
  kvec kr[2][KL];
  vvec vr[VB][2][4];
  v4f ks[2], vs[2];
  const auto load_k = [&](int s, const Place& at) {
#pragma unroll
    for (int t = 0; t < KL; ++t) {
      const int d = (E8 ? 64 * t + 16 * g : 32 * t + 8 * g);
      kr[s][t] = *(const kvec*)((const char*)kv.k + at.base + (k_row + (FULL || d < kv.D ? d : 0) * (unsigned)sizeof(TC)));
    }
    if constexpr (E8) ks[s] = *(const v4f*)(kv.ksc + at.scale + 4 * g);
  };
  // Elements of V vector vb of lane c of 16: of 8 bits two of a lane lie next to each other, one load of 16 bytes
  constexpr bool PAIR = E8 && VB == 2;
  const auto element = [&](int vb, int c) { return PAIR ? 2 * VE * c + VE * vb : vb * 128 + VE * c; };
  const auto load_v = [&](int vb, int s, const Place& at) {
    const int d = element(vb, col);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const char* p = (const char*)kv.v + at.base + e * kv.ts * (long long)sizeof(TC) + (v_row + (FULL || d < kv.D ? d : 0) * (unsigned)sizeof(TC));
      if constexpr (PAIR) {
        if (vb) continue;
        const kvec w = *(const kvec*)p;
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          vr[0][s][e][i] = w[i];
          vr[VB - 1][s][e][i] = w[VW + i];
        }
      } else {
        vr[vb][s][e] = *(const vvec*)p;
      }
    }
    if (E8 && vb == 0) vs[s] = *(const v4f*)(kv.vsc + at.scale + 4 * g);
  };
  // Registers of K and of V are loaded for the next block as soon as this one's products have taken them: what a block waits for was asked
  // for nearly a block before.
  Place now[2], next[2];
  int pick[2] = {0, 0};
  const auto list = [&](int i) {
    if constexpr (CHOSEN) {
      pick[0] = chosen(i, 0);
      pick[1] = chosen(i, 1);
    }
  };
  list(begin + wave);
  Asked asked = ask(begin + wave, pick);
  list(begin + wave + kWaves);
#pragma unroll
  for (int s = 0; s < 2; ++s) now[s] = placed(asked, s);
  asked = ask(begin + wave + kWaves, pick);
  list(begin + wave + 2 * kWaves);
#pragma unroll
  for (int s = 0; s < 2; ++s) load_k(s, now[s]);
#pragma unroll
  for (int vb = 0; vb < VB; ++vb)
#pragma unroll
    for (int s = 0; s < 2; ++s) load_v(vb, s, now[s]);
  for (int i = begin + wave; i < end; i += kWaves) {
    asm volatile("" ::: "memory");  // (q is read from LDS for each block: kept in registers it would not leave room for the rest)
#pragma unroll
    for (int s = 0; s < 2; ++s) next[s] = placed(asked, s);

    // S^T: lane (col, g) has keys 4 g .. + 3 of each half for row col
    v4f x[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < MT; ++m) x[s][m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      v4i k[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if constexpr (E8) k[s] = widen8<TQ>(kr[s][t / 2][2 * (t & 1)], kr[s][t / 2][2 * (t & 1) + 1]);
        else k[s] = kr[s][t];
        if constexpr (!FULL) {  // (what was read in place of elements behind the head must not meet q's zeros: it may be infinite)
          const int d = E8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g;
          if (d >= kv.D) k[s] = v4i(0);
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const v4i f = query(m, t);
#pragma unroll
        for (int s = 0; s < 2; ++s) x[s][m] = mfma16<TQ>(k[s], f, x[s][m]);
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[s][m][e] *= E8 ? a.c * ks[s][e] : a.c;
      if (!LATE) load_k(s, next[s]);
    }

    asked = ask(i + 2 * kWaves, pick);  // (here: a wait for q from LDS would be one for these too)
    list(i + 3 * kWaves);

    // mask; values of keys that no row sees become zeros (they may hold anything)
    bool partial = false, odd = false;
#pragma unroll
    for (int s = 0; s < 2; ++s) partial |= now[s].dead | (now[s].sees(lo_lim) < 16);
    if (__builtin_expect(partial, 0)) {
      bool bad = false;  // a value that is not finite, of a key that some rows see and others may not
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int edge = now[s].sees(hi_lim);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int l = now[s].sees(lim[m]) - 4 * g;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[s][m][e] = e < l ? x[s][m][e] : kMinusInf;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int vb = 0; vb < VB; ++vb)
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              if (4 * g + e >= edge) vr[vb][s][e][w] = 0;
              if (!CHOSEN) bad |= odd_word<TC>(vr[vb][s][e][w]);
            }
      }
      odd = !CHOSEN && lo_lim != hi_lim && __builtin_amdgcn_ballot_w64(bad) != 0;
    }

    // the rows' maxima: renewed when one is passed by more than kSlack (rarely, after the first blocks)
    float top[MT];
    bool renew = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float t = fmaxf(fmaxf(x[0][m][0], x[0][m][1]), fmaxf(x[0][m][2], x[0][m][3]));
      t = fmaxf(t, fmaxf(fmaxf(x[1][m][0], x[1][m][1]), fmaxf(x[1][m][2], x[1][m][3])));
      top[m] = max_groups(t);
      renew = renew || top[m] > mx[m] + kSlack;
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(renew) != 0, 0)) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const bool up = top[m] > mx[m] + kSlack;
        const float f = up ? __builtin_amdgcn_exp2f(mx[m] - top[m]) : 1.0f;
        if (up) mx[m] = top[m];
        sum[m] *= f;
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
#pragma unroll
          for (int j = 0; j < VE; ++j) o[vb][j][m] *= f;
      }
    }

    // P, in V's operand order: the four keys of each half
    v4i p[PARTS][MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const float from = (mx[m] == kMinusInf ? 0.0f : mx[m]) - kBias;
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = __builtin_amdgcn_exp2f(x[e >> 2][m][e & 3] - from);
        sum[m] += w[e];
        if constexpr (E8) w[e] = x[e >> 2][m][e & 3] == kMinusInf ? 0.0f : w[e] * vs[e >> 2][e & 3];  // (a masked key's scale may be anything)
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) in_parts<TP, PARTS>(w[2 * e], w[2 * e + 1], [&](int n, int v) { p[n][m][e] = v; });
    }

    // V^T: the operands of results (vb, 2 w) and (vb, 2 w + 1)
    const auto operands = [&](int vb, int w, v4i& even, v4i& odd_one) {
      int x8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const vvec& r = vr[vb][e >> 2][e & 3];
        if constexpr (E8) x8[e] = w & 1 ? widen2<TP, true>(r[w / 2]) : widen2<TP, false>(r[w / 2]);
        else x8[e] = r[w];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        even[e] = __builtin_amdgcn_perm(x8[2 * e + 1], x8[2 * e], 0x05040100);
        odd_one[e] = __builtin_amdgcn_perm(x8[2 * e + 1], x8[2 * e], 0x07060302);
      }
    };
    if (LATE) {
#pragma unroll
      for (int s = 0; s < 2; ++s) load_k(s, next[s]);
    }
    if (__builtin_expect(odd, 0)) {
      // Zero times infinity would reach the rows that do not see the key. How many NaN and infinities of either sign each row sees is a product
      // of ones and zeros; then they are zeros in V.
      v4i seen[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int l = now[e >> 1].sees(lim[m]) - 4 * g - 2 * (e & 1);
          seen[m][e] = (l > 0 ? one16<TP>() : 0) | (l > 1 ? one16<TP>() << 16 : 0);
        }
#pragma unroll 1
      for (int kind = 0; kind < (E8 ? 1 : 3); ++kind)
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
#pragma unroll
          for (int w = 0; w < VE / 2; ++w) {
            v4i v[2];
            operands(vb, w, v[0], v[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
              for (int e = 0; e < 4; ++e) v[j][e] = odd_ones<TP>(v[j][e], kind);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const v4f n = mfma16<TP>(v[j], seen[m], v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (n[e] > 0.0f) o[vb][2 * w + j][m][e] += kind == 0 ? __builtin_nanf("") : kind == 1 ? -kMinusInf : kMinusInf;
              }
            }
          }
#pragma unroll
      for (int vb = 0; vb < VB; ++vb)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[vb][s][e][w] = without_odd<TC>(vr[vb][s][e][w]);
    }
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int w = 0; w < VE / 2; ++w) {
        v4i v[2];
        operands(vb, w, v[0], v[1]);
#pragma unroll
        for (int n = 0; n < PARTS; ++n)  // (parts outermost: no product waits for the one before)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int m = 0; m < MT; ++m) o[vb][2 * w + j][m] = mfma16<TP>(v[j], p[n][m], o[vb][2 * w + j][m]);
      }
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int s = 0; s < 2; ++s) load_v(vb, s, next[s]);
#pragma unroll
    for (int s = 0; s < 2; ++s) now[s] = next[s];
  }

  // Join the waves: each result relative to the largest maximum of its row, then the sums, two waves at a time through LDS
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    sum[m] = sum_groups(sum[m]);
    if (g == 0) {
      stat[wave][0][16 * m + col] = mx[m];
      stat[wave][1][16 * m + col] = sum[m];
    }
  }
  __syncthreads();
  float top[MT], all[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = kMinusInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top[m] = fmaxf(top[m], stat[w][0][16 * m + col]);
    const float from = top[m] == kMinusInf ? 0.0f : top[m];
    all[m] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all[m] += stat[w][1][16 * m + col] * __builtin_amdgcn_exp2f(stat[w][0][16 * m + col] - from);
    const float f = __builtin_amdgcn_exp2f(mx[m] - from);
#pragma unroll
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int j = 0; j < VE; ++j) o[vb][j][m] *= f;
  }
  // wave i ends with value i of each four: row col of each tile, elements VE (4 g + i) + j of each 128
  float y[VB][VE][MT];
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    __syncthreads();
    if (wave != i) {
      const int at = (wave < i ? wave : wave - 1) * (NO / 4);
#pragma unroll
      for (int n = 0; n < NO; n += 4) {
        v4f t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = o[(n + e) / (VE * MT)][(n + e) / MT % VE][(n + e) % MT][i];
        lds[(at + n / 4) * 64 + lane] = t;
      }
    } else {
#pragma unroll
      for (int n = 0; n < NO; ++n) y[n / (VE * MT)][n / MT % VE][n % MT] = o[n / (VE * MT)][n / MT % VE][n % MT][i];
    }
    __syncthreads();
    if (wave == i) {
#pragma unroll
      for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
        for (int n = 0; n < NO; n += 4) {
          const v4f t = lds[(w * (NO / 4) + n / 4) * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[(n + e) / (VE * MT)][(n + e) / MT % VE][(n + e) % MT] += t[e];
        }
    }
  }

  const int all_pieces = CHOSEN ? a.pieces : ((all_blocks + kWaves - 1) / kWaves + blocks - 1) / blocks;
  const bool split = a.shared > 0 || all_pieces > 1;
  float* slot = nullptr;
  if (shared) {
    slot = a.shared_part + ((size_t)(h * a.shared_tiles + rt) * a.shared + c) * slot_floats(RT, kv.D);
  } else if (a.slots) {
    const int at = CHOSEN ? row0 * rts + rt : first_slot(a, RT, b, row0, rt);
    const int others = a.firsts + (CHOSEN ? row0 * rts * (a.pieces - 1) : more) + rt;
    const long long n = ((long long)(c ? others + (c - 1) * rts : at)) * kv.HK + h;
    if (n >= a.slots) return;  // (rows of lists that are none)
    slot = a.part + (size_t)n * slot_floats(RT, kv.D);
    if (c == 0 && threadIdx.x == 0) *(int4*)slot = int4{all_pieces > 1 ? all_pieces : 1, others, rts, 0};
  }
  if (split) {
    slot += 4;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = 16 * m + col;
      if (first + r > last) continue;
      if (g == 0 && wave == 0) {
        slot[r] = top[m] - kBias;
        slot[RT + r] = all[m];
      }
#pragma unroll
      for (int vb = 0; vb < VB; ++vb) {
        const int d = element(vb, 4 * g + wave);
        if (!FULL && d >= kv.D) continue;
#pragma unroll
        for (int j = 0; j < VE; j += 4) *(v4f*)(slot + 2 * RT + (size_t)r * kv.D + d + j) = v4f{y[vb][j][m], y[vb][j + 1][m], y[vb][j + 2][m], y[vb][j + 3][m]};
      }
    }
    return;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = first + 16 * m + col;
    if (r > last) continue;
    const float inv = all[m] > 0.0f || all[m] != all[m] ? 1.0f / all[m] : 0.0f;  // (a row that sees no key is zeros)
    const size_t at = (size_t)(row0 + r / a.G) * a.ldo + (size_t)(h * a.G + r % a.G) * kv.D;
#pragma unroll
    for (int vb = 0; vb < VB; ++vb) {
      const int d = element(vb, 4 * g + wave);
      if (!FULL && d >= kv.D) continue;
      float z[VE];
#pragma unroll
      for (int j = 0; j < VE; ++j) z[j] = y[vb][j][m] * inv;
      if (a.otype == DT_F32) store_row<float, VE>((float*)a.o + at + d, z);
      else store_row<TQ, VE>((TQ*)a.o + at + d, z);
    }
  }
}

}  // namespace qm
