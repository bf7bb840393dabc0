// Attention over a paged cache, one kernel for every call: rows of q against the keys and values of one key head.
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
// keeps no more bits than that; in two parts (the second what the first left) where it keeps more. The sum l is f32 and unrounded.
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
__device__ __forceinline__ float max_groups(float v) {  // of the four lanes that hold a row
  float a, b;
  with_other<16>(v, a, b);
  with_other<32>(fmaxf(a, b), a, b);
  return fmaxf(a, b);
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
  typedef T v2t __attribute__((ext_vector_type(2)));
  return (float)__builtin_bit_cast(v2t, w)[i];
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

// Whether a 16-bit word holds a value that is not finite in either half
template <typename T>
__device__ __forceinline__ bool odd_half(int w) {
  constexpr int e = __is_same(T, _Float16) ? 0x7C00 : 0x7F80;
  return (w & e) == e || (w >> 16 & e) == e;
}

// TQ: q's type. TC: the cache's, TQ or uint8_t (e4m3). DC: D rounded up to 64, 128 or 256. MT: row tiles of 16. PARTS: of P. MODE: the keys of
// each sequence (OWN), of the prefix for the rows of the whole batch (SHARED), or of chosen pages (CHOSEN).
enum : int { OWN = 0, SHARED = 1, CHOSEN = 2 };

template <typename TQ, typename TC, int DC, int MT, int PARTS, int MODE>
__global__ __launch_bounds__(256) void attn_kernel(AttnArgs a) {
  constexpr bool E8 = sizeof(TC) == 1;
  typedef std::conditional_t<E8, __bf16, TQ> TP;           // of P and V on the matrix pipe
  constexpr float kBias = __is_same(TP, _Float16) ? 6.0f : 0.0f;  // f16 weights are held times 2^6: with kSlack below 2^14, and small ones longer
  constexpr int RT = 16 * MT, KS = DC / 32;                // rows, k steps of the first product
  constexpr int VB = DC > 128 ? 2 : 1, VE = DC / 16 / VB;  // V: vectors of VE elements a lane and key, VB of them
  constexpr int KL = E8 ? KS / 2 : KS;                     // loads of a key's 16 bytes
  typedef int kvec __attribute__((ext_vector_type(4)));
  typedef int vvec __attribute__((ext_vector_type(VE * (E8 ? 1 : 2) / 4)));
  constexpr int NO = VB * VE * MT;                         // results of four values
  __shared__ float xo[2 * NO * 4 * 64];
  __shared__ float stat[kWaves][2][RT];
  __shared__ long long red[4];
  __shared__ Item found;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const KvView& kv = a.kv;
  int h, b = 0, rt, c = 0, blocks = 0x7fffffff, row0 = 0, rows, unit = 0, after = 0;  // (after: tokens of the sequence behind these rows)
  if constexpr (MODE == SHARED) {
    // the row tiles of one piece and head lie 8 work-groups apart: on one XCD, whose L2 then reads the piece once
    const unsigned w = blockIdx.x, at = w >> 3, pc = (at / a.shared_tiles) * 8 + (w & 7);
    rt = at % a.shared_tiles;
    h = pc % kv.HK;
    c = pc / kv.HK;
    if (c >= a.shared) return;
    blocks = a.shared_blocks;
    rows = a.s.T;
  } else if constexpr (MODE == CHOSEN) {
    // (each token's pages are its own: the tile is of one token, and every token has the same number of pieces)
    h = blockIdx.x % kv.HK;
    unit = blockIdx.x / kv.HK;
    const int rts = (a.G + RT - 1) / RT;
    const int t = unit / (rts * a.pieces);
    rt = unit % rts;
    c = unit / rts % a.pieces;
    blocks = a.blocks;
    b = sequence_of(a.s, t);
    if (b < 0) return;  // (a row of no sequence)
    row0 = t;
    rows = 1;
    after = row_from(a.s, b) + rows_of(a.s, b) - 1 - t;
  } else {
    h = blockIdx.x % kv.HK;
    unit = blockIdx.x / kv.HK;
    if (!find_item<RT>(a, unit, &found, red)) return;
    b = __builtin_amdgcn_readfirstlane(found.b);
    rt = __builtin_amdgcn_readfirstlane(found.rt);
    c = __builtin_amdgcn_readfirstlane(found.c);
    blocks = __builtin_amdgcn_readfirstlane(found.blocks);
    row0 = __builtin_amdgcn_readfirstlane(row_from(a.s, b));
    rows = __builtin_amdgcn_readfirstlane(rows_of(a.s, b));
  }
  // (rows: tokens; a row of the tile is token r / G, query head h G + r % G)
  const int nrows = rows * a.G, first = rt * RT, last = min(first + RT, nrows) - 1;
  const int capacity = MODE == SHARED ? 0 : (int)min((long long)a.s.W << kv.lg, 0x7fffffffLL);
  const int len = MODE == SHARED ? 0 : __builtin_amdgcn_readfirstlane(a.s.len[b]) - after;
  // keys that the tile's first and last tokens see of their own
  const int lo_lim = MODE == SHARED ? 0 : min(max(len - rows + first / a.G + 1, 0), capacity);
  const int hi_lim = MODE == SHARED ? 0 : min(max(len - rows + last / a.G + 1, 0), capacity);
  int lim[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = first + 16 * m + col;
    lim[m] = MODE == SHARED ? 0 : min(max(len - rows + r / a.G + 1, 0), capacity);
  }

  // blocks of 32 keys: of the prefix, then of the sequence's own (or of the chosen pages)
  const int shared_blocks32 = MODE == CHOSEN ? 0 : (a.prefix_len + kBlock - 1) / kBlock;
    const int own_blocks = MODE == SHARED ? 0 : MODE == CHOSEN ? (int)(((long long)a.k * kv.page + kBlock - 1) / kBlock) : (int)(((long long)hi_lim + kBlock - 1) / kBlock);
  const int all_blocks = shared_blocks32 + own_blocks;
  const int begin = (int)min((long long)c * blocks * kWaves, (long long)all_blocks);
  const int end = (int)min((long long)begin + (long long)blocks * kWaves, (long long)all_blocks);
  if (MODE != SHARED && c > 0 && begin >= all_blocks) return;  // (a piece that this tile's rows do not see)

  // q: k step t of row col holds elements 32 t + 8 g .. + 7 (8-bit keys: 64 (t / 2) + 16 g + 8 (t % 2), as their loads lie)
  v4i q[MT][KS];
  const bool qvec = ((uintptr_t)a.q & 15) == 0 && (a.ldq & 7) == 0;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = first + 16 * m + col;
    const TQ* p = (const TQ*)a.q + (size_t)(row0 + r / a.G) * a.ldq + (size_t)(h * a.G + r % a.G) * kv.D;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int d = E8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g;
      q[m][t] = v4i(0);
      if (r < nrows && d < kv.D) {
        if (qvec) {
          q[m][t] = *(const v4i*)(p + d);
        } else {
          typedef TQ v8t __attribute__((ext_vector_type(8)));
          v8t e;
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = p[d + i];
          q[m][t] = __builtin_bit_cast(v4i, e);
        }
      }
    }
  }

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

  // Where the 16 keys of half s of block i lie: the page (-1: masked) and the first one's place in it, and in the sequence
  const auto place = [&](int i, int s, int& page, int& in, int& pos, int& limit) {
    page = -1;
    limit = 0;
    if (MODE != CHOSEN && i < shared_blocks32) {
      pos = i * kBlock + 16 * s;
      limit = a.prefix_len;
      if (pos < limit) page = a.prefix[pos >> kv.lg];
    } else {
      pos = (i - shared_blocks32) * kBlock + 16 * s;
      limit = -1;  // each row's own
      if constexpr (MODE == CHOSEN) {
        const int e = pos >> kv.lg;
        const int n = e < a.k ? a.sel[((size_t)row0 * kv.HK + h) * a.k + e] : -1;
        in = pos & (kv.page - 1);
        pos = n >= 0 && n < a.s.W ? (int)min(((long long)n << kv.lg) + in, 0x7fffffffLL) : 0x7fffffff;
      }
      if (MODE != SHARED && pos < hi_lim) page = a.s.table[(size_t)b * a.s.W + (pos >> kv.lg)];
    }
    in = pos & (kv.page - 1);
    if ((unsigned)page >= (unsigned)kv.pages) page = -1;
    page = __builtin_amdgcn_readfirstlane(page);
    pos = __builtin_amdgcn_readfirstlane(pos);
    in = __builtin_amdgcn_readfirstlane(in);
  };

  const bool ragged = kv.D < DC;
  for (int i = begin + wave; i < end; i += kWaves) {
    kvec kr[2][KL];
    vvec vr[2][4][VB];
    v4f ks[2], vs[2];
    int page[2], in[2], pos[2], limit[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      place(i, s, page[s], in[s], pos[s], limit[s]);
      const int pg = page[s] < 0 ? 0 : page[s], at = page[s] < 0 ? 0 : in[s];  // (a masked page's place is read from the first one)
      const long long base = pg * kv.ps + h * kv.hs + at * kv.ts;
      const TC* kp = (const TC*)kv.k + base + col * kv.ts;
      const TC* vp = (const TC*)kv.v + base + 4 * g * kv.ts;
#pragma unroll
      for (int t = 0; t < KL; ++t) {
        const int d = (E8 ? 64 * t + 16 * g : 32 * t + 8 * g);
        kr[s][t] = *(const kvec*)(kp + (d < kv.D ? d : 0));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) {
          const int d = vb * 128 + VE * col;
          vr[s][e][vb] = *(const vvec*)(vp + e * kv.ts + (d < kv.D ? d : 0));
        }
      if constexpr (E8) {
        const size_t at4 = ((size_t)pg * kv.HK + h) * kv.page + at + 4 * g;
        ks[s] = *(const v4f*)(kv.ksc + at4);
        vs[s] = *(const v4f*)(kv.vsc + at4);
      }
    }

    // S^T: lane (col, g) has keys 4 g .. + 3 of each half for row col
    v4f x[2][MT];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int m = 0; m < MT; ++m) x[s][m] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        v4i k;
        if constexpr (E8) k = widen8<TQ>(kr[s][t / 2][2 * (t & 1)], kr[s][t / 2][2 * (t & 1) + 1]);
        else k = kr[s][t];
        if (ragged) {  // (what was read in place of elements behind the head must not meet q's zeros: it may be infinite)
          const int d = E8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g;
          if (d >= kv.D) k = v4i(0);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) x[s][m] = mfma16<TQ>(k, q[m][t], x[s][m]);
      }
    }

    // scale and mask
    bool partial = false, dead[2];
    int edge[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      // keys that some row sees, and whether all rows see all 16
      const int most = limit[s] >= 0 ? limit[s] : hi_lim, least = limit[s] >= 0 ? limit[s] : lo_lim;
      dead[s] = page[s] < 0;
      edge[s] = dead[s] ? 0 : most - pos[s];
      partial = partial || dead[s] || pos[s] > least - 16;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[s][m][e] *= E8 ? a.c * ks[s][e] : a.c;
    }
    if (partial) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int l = dead[s] ? 0 : (limit[s] >= 0 ? limit[s] : lim[m]) - pos[s] - 4 * g;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[s][m][e] = e < l ? x[s][m][e] : kMinusInf;
        }
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
    if (__builtin_amdgcn_ballot_w64(renew)) {
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
      for (int e = 0; e < 4; ++e) {
        p[0][m][e] = pack2<TP>(w[2 * e], w[2 * e + 1]);
        if constexpr (PARTS == 2) p[1][m][e] = pack2<TP>(w[2 * e] - part_of<TP>(p[0][m][e], 0), w[2 * e + 1] - part_of<TP>(p[0][m][e], 1));
      }
    }

    // V^T: the operand of result (vb, j), keys masked for every row as zeros (they may hold anything)
    int vw[2][4][VB][VE / 2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int vb = 0; vb < VB; ++vb) {
#pragma unroll
          for (int w = 0; w < VE / 2; ++w) {
            if constexpr (E8) vw[s][e][vb][w] = w & 1 ? widen2<TP, true>(vr[s][e][vb][w / 2]) : widen2<TP, false>(vr[s][e][vb][w / 2]);
            else vw[s][e][vb][w] = vr[s][e][vb][w];
          }
          if (partial && 4 * g + e >= edge[s]) {
#pragma unroll
            for (int w = 0; w < VE / 2; ++w) vw[s][e][vb][w] = 0;
          }
        }
    const auto operand = [&](int vb, int j) {
      v4i r;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[e] = __builtin_amdgcn_perm(vw[e >> 1][2 * (e & 1) + 1][vb][j / 2], vw[e >> 1][2 * (e & 1)][vb][j / 2], j & 1 ? 0x07060302 : 0x05040100);
      return r;
    };
    bool odd = false;
    if (partial && MODE != SHARED) {  // a value that is not finite, of a key that some rows see and others do not
      bool bad = false;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int vb = 0; vb < VB; ++vb)
#pragma unroll
            for (int w = 0; w < VE / 2; ++w) bad = bad || odd_half<TP>(vw[s][e][vb][w]);
      odd = __builtin_amdgcn_ballot_w64(bad) != 0;
    }
    if (!odd) {
#pragma unroll
      for (int vb = 0; vb < VB; ++vb)
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const v4i v = operand(vb, j);
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < PARTS; ++n) o[vb][j][m] = mfma16<TP>(v, p[n][m], o[vb][j][m]);
        }
    } else {
      // One key at a time, added to the rows that see it (zero times infinity would reach the others)
#pragma unroll 1
      for (int key = 0; key < kBlock; ++key) {
        const int s = key >> 4, mine = (key & 15) - 4 * g, word = 2 * s + ((mine & 3) >> 1);
        const bool here = mine >= 0 && mine < 4;
        const unsigned half = mine & 1 ? 0xffff0000u : 0xffffu;
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            v4i v = operand(vb, j);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = here && e == word ? (int)(v[e] & half) : 0;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const bool sees = !dead[s] && (key & 15) + pos[s] < (limit[s] >= 0 ? limit[s] : lim[m]);
              v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int n = 0; n < PARTS; ++n) y = mfma16<TP>(v, p[n][m], y);
              if (sees) o[vb][j][m] += y;
            }
          }
      }
    }
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
  v4f* buf = (v4f*)xo;
  const auto give = [&](int at) {
#pragma unroll
    for (int n = 0; n < NO; ++n) buf[(at * NO + n) * 64 + lane] = o[n / (VE * MT)][n / MT % VE][n % MT];
  };
  const auto take = [&](int at) {
#pragma unroll
    for (int n = 0; n < NO; ++n) o[n / (VE * MT)][n / MT % VE][n % MT] += buf[(at * NO + n) * 64 + lane];
  };
  if (wave >= 2) give(wave - 2);
  __syncthreads();
  if (wave < 2) take(wave);
  __syncthreads();
  if (wave == 1) give(0);
  __syncthreads();
  if (wave > 0) return;
  take(0);

  // lane (col, g): row col of each tile, elements VE (4 g + i) + j of each 128
  const bool split = MODE == SHARED || (MODE == OWN && a.shared > 0) || (all_blocks + kWaves - 1) / kWaves > blocks;
  if (split) {
    float* slot = MODE == SHARED ? a.shared_part + ((size_t)(h * a.shared_tiles + rt) * a.shared + c) * (RT * (kv.D + 2))
                                 : a.part + ((size_t)unit * kv.HK + h) * (RT * (kv.D + 2));
    if (MODE != SHARED && (long long)unit * kv.HK + h >= a.slots) return;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = 16 * m + col;
      if (first + r > last) continue;
      if (g == 0) {
        slot[r] = top[m] - kBias;
        slot[RT + r] = all[m];
      }
#pragma unroll
      for (int vb = 0; vb < VB; ++vb)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = vb * 128 + VE * (4 * g + i);
          if (d >= kv.D) continue;
#pragma unroll
          for (int j = 0; j < VE; j += 4)
            *(v4f*)(slot + 2 * RT + (size_t)r * kv.D + d + j) = v4f{o[vb][j][m][i], o[vb][j + 1][m][i], o[vb][j + 2][m][i], o[vb][j + 3][m][i]};
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
    for (int vb = 0; vb < VB; ++vb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = vb * 128 + VE * (4 * g + i);
        if (d >= kv.D) continue;
        float y[VE];
#pragma unroll
        for (int j = 0; j < VE; ++j) y[j] = o[vb][j][m][i] * inv;
        if (a.otype == DT_F32) store_row<float, VE>((float*)a.o + at + d, y);
        else store_row<TQ, VE>((TQ*)a.o + at + d, y);
      }
  }
}

}  // namespace qm
