// Attention of many rows over a paged cache: attn_kernel (qm_attn_impl.h) has four waves take keys in turn for the same few rows; here each of
// the four has rows of its own, 16 MT of them, and all take the same keys, from LDS. A work-group's 64 MT rows then read a key once, where row tiles
// of attn_kernel read it once for 16 or 32: prompts, drafted tokens, and a prefix's keys for the rows of a large batch.
//
// 64 keys a step (32 of heads beyond 128), two steps' places in turn: while a step is worked on the next one's loads are on their way, and there is one
// barrier a step. A 16-bit cache's keys and values go straight to LDS, keys in operand order (a lane's 16 bytes are one operand), values as they lie, their
// chunks exchanged within a row so that the reads, which transpose, meet no bank twice; what no row sees and what is behind the head is out of the
// buffer's range, zeros. 8-bit ones go through registers, widened and transposed on the way: once, for all rows. A step's places in memory are worked out during
// the step before (scalar instructions, between matrix instructions).
//
// The logits stay unscaled: e^(scale (s - m)) is one fma and one v_exp, the maximum is that of s (for a scale below zero -q is taken). What bounds it: the
// matrix pipe (64 keys of 128 by a wave's 32 rows: 1024 cycles, 46 % of the time at the full clock) with the vector instructions (160, and 32 exponentials of
// four times an instruction's time) beside it. Measured, 32 heads of 128 over 8, bf16, at best and on average over a long run, whose clock is lower: the last 4096 of
// 16384 tokens 838 and 907 us (1150 and 1060 Tflop/s of what they see), 4096 of 4096 141 and 161; f32 results, three parts of each weight, 1405 and 1508; a large
// library product reaches 1250.
// Tried and not kept: the next scores' products between this block's exponentials (as fast with three parts, 5 % slower with one), values through
// registers for 16-bit caches too (1016 us).
#pragma once
#include "qm_attn_impl.h"

namespace qm {

constexpr int kAheadOps = 4;  // operands that are read from LDS ahead of their products
typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p, unsigned bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00020000); }
// 16 bytes a lane from there to LDS, a wave's 1 KB in lane order
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t from, v4i* to, unsigned off) { __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_void*)to, 16, off, 0, 0, 0); }
// Of each 16 lanes, lane i names four 16-bit values of row i / 4, columns 4 (i % 4) on; it gets column i of the four rows
typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
__device__ __forceinline__ v2i transposed(const void* p) { return __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p)); }
constexpr int kBetween = 4;  // vector instructions between two matrix instructions: as long as one takes
constexpr int kNoLoads = 0x0F70;  // (s_waitcnt: no vector load under way)
constexpr int kFree = 6;      // vector and scalar arithmetic, that the compiler may move past these reads

template <typename TQ, typename TC, int DC, bool FULL, int MT, int PARTS>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(AttnArgs a) {
  constexpr bool E8 = sizeof(TC) == 1;
  typedef std::conditional_t<E8, __bf16, TQ> TP;
  constexpr float kBias = __is_same(TP, _Float16) ? 6.0f : 0.0f;
  constexpr int RT = 64 * MT, KS = DC / 32;
  constexpr int VB = DC > 128 ? 2 : 1, VE = DC / 16 / VB;
  constexpr int NB = DC > 128 ? 1 : 2;        // blocks of 32 keys of a step: four groups of 16 keys (two), one (half) a wave's to load
  constexpr int KT = KS / (2 / NB);           // operands of K that a wave loads
  constexpr int KL = E8 ? KT / 2 : KT;        // in loads of 16 bytes
  constexpr int VW = VE * (E8 ? 1 : 2) / 4;
  constexpr int kOps = NB * 2 * KS * 64;      // operands of K (V) of a step, in 16 bytes
  constexpr bool DIRECT = !E8;                // the cache's own values go straight to LDS; 8-bit ones through registers, widened on the way
  typedef int vvec __attribute__((ext_vector_type(VW)));
  struct Step {
    v4i k[kOps], v[kOps];
  };
  struct Notes {
    int flags[4];                             // of each wave's group of 16 keys: 1 its page is none, 2 (8-bit) a value is not finite
    float scales[2][E8 ? 64 : 4];             // 8-bit: of keys and of values
  };
  __shared__ Step step0, step1;               // (variables, no arrays: the compiler can tell loads into one from reads of the others)
  __shared__ Notes notes0, notes1;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const KvView& kv = a.kv;
  int h, b = 0, rt, c = 0, blocks = kWhole, row0 = 0, rows, rts = 1, more = 0, tail_slot = -1;
  const bool shared = (int)blockIdx.x < a.shared_grid;
  if (shared) {
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
    tail_slot = __builtin_amdgcn_readfirstlane(it.slot);
    const int parts = __builtin_amdgcn_readfirstlane(it.parts);
    if (tail_slot >= 0) blocks = part_blocks(__builtin_amdgcn_readfirstlane(tile_blocks(a, RT, b, rt, rows)), parts);
  }
  const int nrows = rows * a.G, first = rt * RT, last = min(first + RT, nrows) - 1;
  const int capacity = shared ? 0 : (int)min((long long)a.s.W << kv.lg, 0x7fffffffLL);
  const int len = shared ? 0 : __builtin_amdgcn_readfirstlane(length_of(a.s, b));
  const auto limit_of = [&](int r) { return min(max(len - rows + r / a.G + 1, 0), capacity); };  // keys that row r sees of its own
  const int lo_lim = limit_of(first), hi_lim = limit_of(last);
  int lim[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) lim[m] = limit_of(first + 16 * (MT * wave + m) + col);

  // blocks of 32 keys: of the prefix, then of the sequence's own; steps of NB of them
  const int pre_blocks = a.shared && !shared ? 0 : (a.prefix_len + kBlock - 1) / kBlock;
  const int all_blocks = pre_blocks + (int)(((long long)hi_lim + kBlock - 1) / kBlock);
  const int begin = (int)min((long long)c * blocks * kWaves, (long long)all_blocks);
  const int end = (int)min((long long)begin + (long long)blocks * kWaves, (long long)all_blocks);
  if (!shared && c > 0 && begin >= all_blocks) return;  // (a piece that this tile's rows do not see)

  // q as attn_kernel holds it
  // (a scale below zero is its negative's with -q: the maximum is that of the products then. None of zero comes here: masked logits would be NaN.)
  const float scale = __builtin_fabsf(a.c);
  const int q_xor = a.c < 0.0f ? 0x80008000 : 0;
  v4i q[MT][KS];
  const bool qvec = ((uintptr_t)a.q & 15) == 0 && (a.ldq & 7) == 0;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = min(first + 16 * (MT * wave + m) + col, nrows - 1);
    const TQ* p = (const TQ*)a.q + (size_t)(row0 + r / a.G) * a.ldq + (size_t)(h * a.G + r % a.G) * kv.D;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int d = E8 ? 64 * (t / 2) + 16 * g + 8 * (t & 1) : 32 * t + 8 * g, at = FULL || d < kv.D ? d : 0;
      if (qvec) {
        q[m][t] = *(const v4i*)(p + at);
      } else {
        typedef TQ v8t __attribute__((ext_vector_type(8)));
        v8t e;
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[at + i];
        q[m][t] = __builtin_bit_cast(v4i, e);
      }
      q[m][t] ^= q_xor;
      if (!FULL && d >= kv.D) q[m][t] = v4i(0);
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

  // Steps of keys that every row sees: blocks below seen_pre, and those from pre_blocks on below seen_own
  const int seen_pre = min(a.prefix_len / kBlock, pre_blocks), seen_own = pre_blocks + lo_lim / kBlock;
  // This wave's group of 16 keys of a step (NB 1: waves 0, 1 the first one, each half of its K operands and of its V vectors)
  const int mine = NB == 2 ? wave : wave >> 1, half = NB == 2 ? 0 : wave & 1;
  const int32_t* table = a.s.table + (size_t)b * a.s.W;
  // Where it lies: its page's number is asked for a step before the place is worked out, and that a step before the loads (between the
  // matrix instructions: scalar instructions one after the other would take longer than a quarter of the step)
  struct Group {
    int page, pos, most;
    bool pre;
  };
  const auto ask = [&](int i) {  // (without a branch, as in attn_kernel; asked behind the end too, and not used then)
    Group r;
    const int block = i + (mine >> 1);
    r.pre = block < pre_blocks;
    r.pos = (r.pre ? block : block - pre_blocks) * kBlock + 16 * (mine & 1);
    r.most = r.pre ? a.prefix_len : hi_lim;
    r.page = scalar(r.pre ? a.prefix : table, r.pos < r.most ? r.pos >> kv.lg : 0);
    return r;
  };
  struct Place {
    long long base;  // bytes from the cache's first key (value) to the group's first
    size_t scale;    // and of its scales, in elements
    int edge;        // keys of the group that some row sees
    bool dead, mixed;  // its page is none or it is behind the end; there are rows that do not see all of it
  };
  const long long ps = kv.ps * (long long)sizeof(TC), ts = kv.ts * (long long)sizeof(TC), head = h * kv.hs * (long long)sizeof(TC);
  const auto place = [&](const Group& r) {
    Place p;
    p.dead = (unsigned)r.page >= (unsigned)kv.pages || r.pos >= r.most;
    p.edge = p.dead ? 0 : r.most - r.pos;
    p.mixed = !r.pre && lo_lim - r.pos < 16;
    const int pg = p.dead ? 0 : r.page, in = p.dead ? 0 : r.pos & (kv.page - 1);  // (16 keys from there are the page's)
    p.base = head + pg * ps + in * ts;
    if constexpr (E8) p.scale = ((size_t)pg * kv.HK + h) * kv.page + in;
    return p;
  };

  // Loads of a 16-bit cache: by 1 KB a wave's instruction to LDS, K in operand order, V key by key: chunk x (16 bytes) of key r at x ^ twist(r), so
  // that the reads below take different banks. What lies behind the last key that a row sees, or behind the head, is out of the buffer's
  // range: zeros.
  constexpr int CR = DC / 8;  // chunks of a key
  const auto twist = [](int r) { return CR == 8 ? 2 * (r >> 1 & 3) : 2 * (r & 7); };
  constexpr unsigned kNowhere = 0xFFFFFF00u;
  unsigned k_off[DIRECT ? KT : 1], v_off[DIRECT ? KT : 1];
  if constexpr (DIRECT) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int d = 32 * (half * KT + t) + 8 * g, at = (half * KT + t) * 64 + lane, r = at / CR, x = at % CR ^ twist(r);
      k_off[t] = FULL || d < kv.D ? (unsigned)col * (unsigned)ts + 2u * d : kNowhere;
      v_off[t] = FULL || 8 * x < kv.D ? (unsigned)r * (unsigned)ts + 16u * x : kNowhere;
    }
  }
  // Of an 8-bit one: through registers
  const unsigned k_row = (unsigned)col * (unsigned)ts, v_row = 4u * (unsigned)g * (unsigned)ts;
  v4i kr[DIRECT ? 1 : KL];
  vvec vr[4];
  v4f ks, vs;
  // (16-bit) the group's keys and values as buffers; nothing of them is in range where there is no such step
  struct Aim {
    __amdgpu_buffer_rsrc_t k, v;
  };
  const auto aim = [&](const Place& at, bool there) {
    const unsigned range = !there ? 0 : at.edge < 16 ? (unsigned)at.edge * (unsigned)ts : 15u * (unsigned)ts + 2u * kv.D;
    return Aim{buffer_at((const char*)kv.k + at.base, range), buffer_at((const char*)kv.v + at.base, range)};
  };
  const auto fetch = [&](const Aim& from, Step& to, int t) {  // t of KT loads of each
    const int n = (mine * KS + half * KT + t) * 64;
    to_lds(from.k, to.k + n, k_off[t]);
    to_lds(from.v, to.v + n, v_off[t]);
  };
  const auto load = [&](const Place& at, Step& to, Notes& note) {
    if constexpr (DIRECT) {
      const Aim from = aim(at, true);
#pragma unroll
      for (int t = 0; t < KT; ++t) fetch(from, to, t);
      if (lane == 0) note.flags[wave] = at.dead;
    } else {
#pragma unroll
      for (int t = 0; t < KL; ++t) {
        const int d = 64 * (half * KL + t) + 16 * g;
        kr[t] = *(const v4i*)((const char*)kv.k + at.base + (k_row + (FULL || d < kv.D ? d : 0)));
      }
      const int d = half * 128 + VE * col;
#pragma unroll
      for (int e = 0; e < 4; ++e) vr[e] = *(const vvec*)((const char*)kv.v + at.base + e * ts + (v_row + (FULL || d < kv.D ? d : 0)));
      ks = *(const v4f*)(kv.ksc + at.scale + 4 * g);
      vs = *(const v4f*)(kv.vsc + at.scale + 4 * g);
    }
  };
  // What has come: registers to LDS, widened, four keys of VE elements -> VE elements of four keys, half of an operand each
  const auto keep = [&](const Place& at, Step& to, Notes& note) {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int t = 0; t < KL; ++t) {
        const int u = half * KL + t;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          v4i w = widen8<TQ>(kr[t][2 * e], kr[t][2 * e + 1]);
          if (!FULL && 64 * u + 16 * g + 8 * e >= kv.D) w = v4i(0);
          to.k[(mine * KS + 2 * u + e) * 64 + lane] = w;
        }
      }
      // values behind the last key that a row sees may be anything: zeros; those of keys that some rows see and others do not are looked at
      bool bad = false;
      if (__builtin_expect(at.edge < 16 || at.mixed, 0)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!(__builtin_fabsf(vs[e]) < -kMinusInf)) {  // (a scale that is not finite, of a key that some rows see: their results are not either)
            vr[e] = vvec(0x7F7F7F7F);
            vs[e] = 1.0f;
          }
          if (4 * g + e >= at.edge) {
            vr[e] = vvec(0);
            vs[e] = 0.0f;
          }
#pragma unroll
          for (int w = 0; w < VW; ++w) bad |= odd_word<TC>(vr[e][w]);
        }
      }
      int w4[4][VE / 2];
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int w = 0; w < VE / 2; ++w) w4[e][w] = w & 1 ? widen2<TP, true>(vr[e][w / 2]) : widen2<TP, false>(vr[e][w / 2]);
      v2i* at2 = (v2i*)(to.v + (((mine >> 1) * VB + half) * VE) * 64 + lane) + (mine & 1);
#pragma unroll
      for (int w = 0; w < VE / 2; ++w) {
        at2[(2 * w) * 128] = v2i{(int)__builtin_amdgcn_perm(w4[1][w], w4[0][w], 0x05040100), (int)__builtin_amdgcn_perm(w4[3][w], w4[2][w], 0x05040100)};
        at2[(2 * w + 1) * 128] = v2i{(int)__builtin_amdgcn_perm(w4[1][w], w4[0][w], 0x07060302), (int)__builtin_amdgcn_perm(w4[3][w], w4[2][w], 0x07060302)};
      }
      if (col == 0 && half == 0) {
        *(v4f*)&note.scales[0][16 * mine + 4 * g] = ks;
        *(v4f*)&note.scales[1][16 * mine + 4 * g] = vs;
      }
      const bool any = __builtin_amdgcn_ballot_w64(bad) != 0;
      if (lane == 0) note.flags[wave] = (at.dead ? 1 : 0) | (any ? 2 : 0);
    }
  };
  // V's operand of elements 16 n and on (8-bit: VB, VE as the loads lie) of block nb. From keys as they lie: the transposing read gives lane (col, g)
  // element col of the four keys whose places lanes 16 g .. + 15 name.
  unsigned v_at[DIRECT ? (CR == 8 ? 4 : 8) : 1];
  if constexpr (DIRECT) {
    const int r = 4 * g + (col >> 2);
#pragma unroll
    for (int n = 0; n < (CR == 8 ? 4 : 8); ++n) v_at[n] = (unsigned)((r * CR + (2 * n ^ twist(r)) + (col >> 1 & 1)) * 16 + 8 * (col & 1));
  }
  const auto value = [&](Step& from, int nb, int n) {
    if constexpr (DIRECT) {
      v2i w[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) w[s] = transposed((const char*)(from.v + (2 * nb + s) * KS * 64) + v_at[n & 7] + (n >> 3) * 256);
      return v4i{w[0][0], w[0][1], w[1][0], w[1][1]};
    } else {
      return from.v[(nb * VB * VE + n) * 64 + lane];
    }
  };

  Place now = place(ask(begin)), next;
  Group asked = ask(begin + NB);
  load(now, step0, notes0);
  next = place(asked);
  keep(now, step0, notes0);
  __builtin_amdgcn_s_waitcnt(kNoLoads);
  __syncthreads();
  const auto work = [&](int i, Step& cur, Step& other, const Notes& note, Notes& other_note) __attribute__((always_inline)) {
    // (16-bit: between the first product's matrix instructions: a work-group's 32 KB at once would keep each wave for 580 cycles)
    if constexpr (!DIRECT)
      if (i + NB < end) load(next, other, other_note);
    const Place coming = next;
    Aim from;
    if constexpr (DIRECT) {
      from = aim(next, i + NB < end);
      if (lane == 0) other_note.flags[wave] = next.dead;
    }
    // S^T. Operands are read from LDS four ahead of the products that take them (the compiler would read each and wait for it).
    v4i op[2][kAheadOps];
    constexpr int NK = NB * 2 * KS, NV = NB * VB * VE, VC = VB * VE / kAheadOps;
    const auto read_k = [&](int n) {
#pragma unroll
      for (int u = 0; u < kAheadOps; ++u) {
        const int at = n * kAheadOps + u, nb = at / (2 * KS), t = at % (2 * KS) / 2;  // (both halves of a block in turn: no product waits for the one before)
        op[n & 1][u] = cur.k[((nb * 2 + (u & 1)) * KS + t) * 64 + lane];
      }
      __builtin_amdgcn_sched_barrier(kFree);
    };
    const auto read_v = [&](int n) {
#pragma unroll
      for (int u = 0; u < kAheadOps; ++u) op[n & 1][u] = value(cur, (n * kAheadOps + u) / (VB * VE), (n * kAheadOps + u) % (VB * VE));
    };
    v4f x[NB][2][MT];
    read_k(0);
    const v4i raised = *(const v4i*)note.flags;
#pragma unroll
    for (int n = 0; n < NK / kAheadOps; ++n) {
      if ((n + 1) * kAheadOps < NK) read_k(n + 1);
      if constexpr (DIRECT) {
        static_assert(NK / kAheadOps == KT, "a load of each beside every four operands");
        fetch(from, other, n);
        __builtin_amdgcn_sched_barrier(kFree);
      }
#pragma unroll
      for (int u = 0; u < kAheadOps; ++u) {
        const int nb = (n * kAheadOps + u) / (2 * KS), t = (n * kAheadOps + u) % (2 * KS) / 2, s = u & 1;
#pragma unroll
        for (int m = 0; m < MT; ++m) x[nb][s][m] = mfma16<TQ>(op[n & 1][u], q[m][t], t ? x[nb][s][m] : v4f{0.0f, 0.0f, 0.0f, 0.0f});
      }
      __builtin_amdgcn_sched_barrier(kFree);
    }
    v4f vsc[NB][2];
    if constexpr (E8) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const v4f f = *(const v4f*)&note.scales[0][16 * (2 * nb + s) + 4 * g];
          vsc[nb][s] = *(const v4f*)&note.scales[1][16 * (2 * nb + s) + 4 * g];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[nb][s][m][e] *= f[e];
        }
    }
    __builtin_amdgcn_sched_barrier(0);  // (a scalar load on its way makes each wait for LDS one for it)
    asked = ask(i + 2 * NB);
    read_v(0);
    // masks
    const int raise = __builtin_amdgcn_readfirstlane(raised[0] | raised[1] | raised[2] | raised[3]);
    const bool partial = (raise & 1) | !(i + NB <= seen_pre || (i >= pre_blocks && i + NB <= seen_own));
    int dead_groups = 0;
    // Of a lane's four keys of group n, those that its row of tile m sees
    const auto seen_of = [&](int n, int m) {
      const int block = i + (n >> 1);
      const bool pre = block < pre_blocks;
      const int l = (pre ? a.prefix_len : lim[m]) - (pre ? block : block - pre_blocks) * kBlock - 16 * (n & 1);
      return (dead_groups >> n & 1 ? 0 : l) - 4 * g;
    };
    bool odd = false;
    if (__builtin_expect(partial, 0)) {
#pragma unroll
      for (int n = 0; n < 4; ++n) dead_groups |= (__builtin_amdgcn_readfirstlane(raised[n]) & 1) << (NB == 2 ? n : n >> 1);
#pragma unroll
      for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int l = seen_of(n, m);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[n >> 1][n & 1][m][e] = e < l ? x[n >> 1][n & 1][m][e] : kMinusInf;
        }
      if (lo_lim != hi_lim) {
        bool bad = raise & 2;
        if constexpr (DIRECT) {
#pragma unroll 1
          for (int u = lane; u < kOps; u += 64) {
            const v4i w = cur.v[u];
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= odd_word<TC>(w[e]);
          }
        }
        odd = __builtin_amdgcn_ballot_w64(bad) != 0;
      }
    }
    float top[MT];
    bool renew = false;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float t = kMinusInf;
#pragma unroll
      for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
        for (int e = 0; e < 4; e += 2) t = larger(t, larger(x[n >> 1][n & 1][m][e], x[n >> 1][n & 1][m][e + 1]));
      top[m] = max_groups(t);
      renew = renew || fmaf(top[m], scale, -mx[m]) > kSlack;
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(renew) != 0, 0)) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const bool up = fmaf(top[m], scale, -mx[m]) > kSlack;
        const float to = top[m] * scale, f = up ? __builtin_amdgcn_exp2f(mx[m] - to) : 1.0f;
        if (up) mx[m] = to;
        sum[m] *= f;
#pragma unroll
        for (int vb = 0; vb < VB; ++vb)
#pragma unroll
          for (int j = 0; j < VE; ++j) o[vb][j][m] *= f;
      }
    }
    float w[NB][MT][8];
    const auto weights = [&](int nb) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float from = (mx[m] == kMinusInf ? 0.0f : mx[m]) - kBias;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          w[nb][m][e] = __builtin_amdgcn_exp2f(fmaf(x[nb][e >> 2][m][e & 3], scale, -from));
          sum[m] += w[nb][m][e];
          if constexpr (E8) w[nb][m][e] *= vsc[nb][e >> 2][e & 3];
        }
      }
    };
    weights(0);
    // Values that are not finite, of keys that some rows see and others do not: as in attn_kernel, counted apart, and zeros in the product (in LDS:
    // the work-group's waves all come here, or none does)
    if (__builtin_expect(odd, 0)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        v4i sees[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int l = seen_of(2 * nb + (e >> 1), m) - 2 * (e & 1);
            sees[m][e] = (l > 0 ? one16<TP>() : 0) | (l > 1 ? one16<TP>() << 16 : 0);
          }
#pragma unroll 1
        for (int kind = 0; kind < (E8 ? 1 : 3); ++kind)
#pragma unroll
          for (int n = 0; n < VB * VE; ++n) {
            v4i v = value(cur, nb, n);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = odd_ones<TP>(v[e], kind);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              const v4f c = mfma16<TP>(v, sees[m], v4f{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (c[e] > 0.0f) o[n / VE][n % VE][m][e] += kind == 0 ? __builtin_nanf("") : kind == 1 ? -kMinusInf : kMinusInf;
            }
            asm volatile("" ::: "memory");  // (no registers for more than one at once)
            __builtin_amdgcn_sched_barrier(0);
          }
      }
      __syncthreads();
      for (int u = threadIdx.x; u < kOps; u += 256) {
        v4i v = cur.v[u];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = without_odd<TP>(v[e]);
        cur.v[u] = v;
      }
      __syncthreads();
      read_v(0);
    }
    // (of two waves on a SIMD, the one that has its weights goes first: the last 4096 of 16384 tokens 907 us against 943, f32 1533 against 1600, as
    // this was then; both products: 941)
    __builtin_amdgcn_s_setprio(1);
    v4i p[PARTS][MT];
#pragma unroll
    for (int n = 0; n < NV / kAheadOps; ++n) {
      if (n * kAheadOps % (VE * VB) == 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float* y = &w[n * kAheadOps / (VE * VB)][m][2 * e];
            in_parts<TP, PARTS>(y[0], y[1], [&](int r, int v) { p[r][m][e] = v; });
          }
      }
      if ((n + 1) * kAheadOps < NV) read_v(n + 1);
      // (the second block's weights between the first one's products: 838 us against 843, f32 1405 against 1421)
      if (NB == 2 && n == 0) weights(NB - 1);
      if (n == 0) next = place(asked);
      if (NB == 1 || n >= VC) __builtin_amdgcn_sched_barrier(kFree);
#pragma unroll
      for (int r = 0; r < PARTS; ++r)
#pragma unroll
        for (int u = 0; u < kAheadOps; ++u) {
          const int j = (n * kAheadOps + u) % VE, vb = (n * kAheadOps + u) / VE % VB;
#pragma unroll
          for (int m = 0; m < MT; ++m) o[vb][j][m] = mfma16<TP>(op[n & 1][u], p[r][m], o[vb][j][m]);
        }
      if (NB == 1 || n >= VC) __builtin_amdgcn_sched_barrier(kFree);
      if (NB == 2 && n == VC - 1) {
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          __builtin_amdgcn_sched_group_barrier(0x100, (DIRECT ? 2 : 1) * kAheadOps, 0);
#pragma unroll
          for (int u = 0; u < kAheadOps * MT * PARTS; ++u) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, kBetween, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (i + NB < end) keep(coming, other, other_note);
    __builtin_amdgcn_s_waitcnt(kNoLoads);
    __syncthreads();
  };
  for (int i = begin; i < end; i += 2 * NB) {
    work(i, step0, step1, notes0, notes1);
    if (i + NB < end) work(i + NB, step1, step0, notes1, notes0);
  }

  // lane (col, g): row col of each of the wave's tiles
  const int all_pieces = ((all_blocks + kWaves - 1) / kWaves + blocks - 1) / blocks;
  const bool split = a.shared > 0 || all_pieces > 1;
  float* slot = nullptr;
  if (shared) {
    slot = a.shared_part + ((size_t)(h * a.shared_tiles + rt) * a.shared + c) * slot_floats(RT, kv.D);
  } else if (a.tail) {
    if (all_pieces > 1) slot = a.part + (size_t)tail_slot * slot_floats(RT, kv.D);
  } else if (a.slots) {
    const int at = first_slot(a, RT, b, row0, rt), others = a.firsts + more + rt;
    const long long n = ((long long)(c ? others + (c - 1) * rts : at)) * kv.HK + h;
    if (n >= a.slots) return;  // (rows of lists that are none)
    slot = a.part + (size_t)n * slot_floats(RT, kv.D);
    if (c == 0 && threadIdx.x == 0) *(int4*)slot = int4{all_pieces > 1 ? all_pieces : 1, others, rts, 0};
  }
  if (split) slot += 4;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = 16 * (MT * wave + m) + col;
    const float all = sum_groups(sum[m]);
    if (first + r > last) continue;
    if (split && g == 0) {
      slot[r] = mx[m] - kBias;
      slot[RT + r] = all;
    }
    const float inv = split ? 1.0f : all > 0.0f || all != all ? 1.0f / all : 0.0f;  // (a row that sees no key is zeros)
    const size_t at = (size_t)(row0 + (first + r) / a.G) * a.ldo + (size_t)(h * a.G + (first + r) % a.G) * kv.D;
    const auto put = [&](int d, auto& y) {
      constexpr int N = sizeof(y) / sizeof(float);
      if (!FULL && d >= kv.D) return;
      if (split) store_row<float, N>(slot + 2 * RT + (size_t)r * kv.D + d, y);
      else if (a.otype == DT_F32) store_row<float, N>((float*)a.o + at + d, y);
      else store_row<TQ, N>((TQ*)a.o + at + d, y);
    };
#pragma unroll
    for (int vb = 0; vb < VB; ++vb) {
      if constexpr (DIRECT) {  // four elements of each 16
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = o[vb][j][m][e] * inv;
          put(16 * (vb * VE + j) + 4 * g, y);
        }
      } else {  // VE of each 4 VE
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y[VE];
#pragma unroll
          for (int j = 0; j < VE; ++j) y[j] = o[vb][j][m][e] * inv;
          put(vb * 128 + VE * (4 * g + e), y);
        }
      }
    }
  }
}

}  // namespace qm
