// Prompt products of e4m3 activations and weights: tiles of 256 rows x 16 MT tokens.
//
// Four waves, each 64 rows (a prepared group) by all tokens of the tile. A wave loads its own weight fragments straight into
// registers, one block of K ahead (no other wave needs them); the tokens, which all four share, go to LDS by asynchronous
// loads up to three blocks ahead, 16-byte pieces exchanged within a row (piece ^ row % 8) so that the fragment reads meet no bank
// twice. One barrier a block.
#include "qm_fp8_dev.h"

namespace qm {

namespace {

template <int MT>
struct Tokens {
  uint4 v[MT * 128];                   // [token][8 pieces]
  float sc[(MT * 16 + 63) / 64 * 64];  // (loaded 64 at a time)
};

typedef __attribute__((address_space(3))) void lds_void;

// A buffer of `bytes` from p on: loads take a lane's offset and a uniform one, both 32 bits
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, 0x00027000);
}
__device__ __forceinline__ v4i load16(__amdgpu_buffer_rsrc_t b, uint32_t lane_off, uint32_t off) {
  return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(b, lane_off, off, 0));
}

// The scheduler moves nothing across: the order of the source is the order of issue
__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }
// Waits until at most n vector loads are under way
constexpr int wait_loads(int n) { return 0x0F70 | (n & 15) | (n >> 4 << 14); }
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// What this wave's lanes wrote to LDS before it, its lanes read behind it. (The hardware keeps a wave's LDS accesses in order; this
// tells the compiler to.)
__device__ __forceinline__ void exchange() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

struct Frags {
  v4i lo[4], hi[4];
};

template <int MT, bool EXACT>
struct TileWave {
  static constexpr int kLoads = (MT + 1) / 2 + 1;  // asynchronous loads of a block's tokens by one wave (every wave issues as many)
  // Where a block's token loads are issued. Large tiles: behind the barrier, for three blocks ahead (work-groups that share a CU
  // cover each other: 4096 x 5120 -> 17408 1.5 % faster). Small ones: between the next block's matrix instructions, for two
  // ahead, so that the fragments do not queue behind them (777 x 17408 -> 5120 uncut, MT 6, a work-group a CU: 100 us against 111).
  static constexpr bool kBehind = MT >= 7;
  static constexpr int kAhead = kBehind ? 3 : 2;
  static_assert(kLoads < MT, "every token load is issued before the block's barrier, as its wait counts");

  __amdgpu_buffer_rsrc_t wbuf, rows, asc;  // the group's fragments, the tile's token rows and scales, all from the first block on
  uint32_t frag_stride, lane16, off[(MT + 1) / 2], sc_off;  // off, sc_off: this thread's token pieces and scale
  int wave, M_stride, last, r, at0, at1;
  v4f acc[4][MT], p[4];  // p: the sums of the token tile before this one, added while this one's are on the matrix pipe
  float s;               // p's scale
  v4i a0, a1;            // the next token tile, and its token scale
  float sc;

  __device__ __forceinline__ void load_frags(Frags& f, int b) {
    const uint32_t at = (uint32_t)min(b, last) * kFragBytes;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f.lo[t] = load16(wbuf, lane16, at + t * frag_stride);
      f.hi[t] = load16(wbuf, lane16 + 1024, at + t * frag_stride);
    }
  }
  __device__ __forceinline__ void load_tokens(Tokens<MT>& to, int b, int i) {
    const uint32_t bb = (uint32_t)min(b, last);
    if (i < kLoads - 1) __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (lds_void*)(to.v + dst(i)), 16, off[i], 128 * bb, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(asc, (lds_void*)(to.sc + sc_dst()), 4, sc_off, bb * M_stride * 4, 0, 0);
  }
  // (an odd MT: the upper two waves load the lower two's pieces of the last round again)
  __device__ __forceinline__ int dst(int i) const { return 64 * (2 * i + 1 < MT ? wave : wave & 1) + 256 * i; }
  __device__ __forceinline__ int sc_dst() const { return 64 * min(wave, (MT * 16 + 63) / 64 - 1); }

  __device__ __forceinline__ void first_tile(const Tokens<MT>& tk) {
    a0 = *(const v4i*)(tk.v + at0);
    a1 = *(const v4i*)(tk.v + at1);
    sc = tk.sc[r];
  }
  __device__ __forceinline__ void add_last(int t, v4f& c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = fmaf(s, p[t][i], c[i]);
  }

  // Block b: tokens tk, fragments w; wn takes the next fragments (EXACT: w itself, once widened), tn are the next tokens, to takes
  // those kAhead blocks on.
  __device__ __forceinline__ void block(int b, Frags& w, const Tokens<MT>& tk, float ws, Frags& wn, const Tokens<MT>& tn, Tokens<MT>& to) {
    v8h wide[EXACT ? 4 : 1][4];
    if constexpr (EXACT) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        wide[t][0] = widen(w.lo[t][0], w.lo[t][1]);
        wide[t][1] = widen(w.lo[t][2], w.lo[t][3]);
        wide[t][2] = widen(w.hi[t][0], w.hi[t][1]);
        wide[t][3] = widen(w.hi[t][2], w.hi[t][3]);
      }
      keep_order();
    }
    load_frags(wn, b + 1);
    // (of two waves on a SIMD, the one that has its operands goes first: 4096 x 5120 -> 17408 327 us against 330, f32 633 against 641)
    __builtin_amdgcn_s_setprio(1);
    keep_order();
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const v4i x0 = a0, x1 = a1;
      const float sn = sc * ws;
      if (j + 1 < MT) {
        a0 = *(const v4i*)(tk.v + 128 * (j + 1) + at0);
        a1 = *(const v4i*)(tk.v + 128 * (j + 1) + at1);
        sc = tk.sc[16 * (j + 1) + r];
      } else {
        // This wave's tokens b + 1 have come (what was issued since are the next fragments and one block's tokens), and every other
        // wave's beyond the barrier, which also says that block b - 1's have been read.
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_s_waitcnt(wait_loads(8 + kLoads));
        meet();
        if (kBehind)
#pragma unroll
          for (int i = 0; i < kLoads; ++i) load_tokens(to, b + kAhead, i);
        first_tile(tn);
      }
      if (!kBehind && j < kLoads) load_tokens(to, b + kAhead, j);
      keep_order();
      if constexpr (EXACT) {
        const v8h x[4] = {widen(x0[0], x0[1]), widen(x0[2], x0[3]), widen(x1[0], x1[1]), widen(x1[2], x1[3])};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          add_last(t, acc[t][j ? j - 1 : MT - 1]);
          p[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wide[t][0], x[0], v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
          keep_order();
        }
#pragma unroll
        for (int c = 1; c < 4; ++c)
#pragma unroll
          for (int t = 0; t < 4; ++t) p[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wide[t][c], x[c], p[t], 0, 0, 0);
        keep_order();
      } else {
        const v8i x = join(x0, x1);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          add_last(t, acc[t][j ? j - 1 : MT - 1]);
          p[t] = dot_block<false>(join(w.lo[t], w.hi[t]), x);
          keep_order();
        }
      }
      s = sn;
    }
  }
};

}  // namespace

// splits > 1: each tile's blocks are cut into that many pieces, whose sums go to part [splits][M][64 groups] in f32
template <int MT, bool EXACT>
__global__ __launch_bounds__(256, 2) void fp8_tile_kernel(Fp8GemmArgs a, int tn, int tm, int splits) {
  __shared__ Tokens<MT> t0, t1, t2, t3;  // (four variables: the compiler can tell loads into one from reads of another)
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4;
  // neighbouring work-groups go to the XCDs in turn: each XCD takes a run of tiles, in bands of 8 token tiles (4096 x 5120 -> 17408: 329 us;
  // bands of 4 333, of 16 335, of 32 353)
  const int tiles = tn * tm, total = tiles * splits, per = (total + 7) / 8;
  const int item = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || item >= total) return;
  const int piece = item / tiles, idx = item - piece * tiles;
  const int band = idx / (8 * tn), in = idx - band * 8 * tn, bm = min(8, tm - band * 8);
  const int tile_n = in / bm, tile_m = band * 8 + in - tile_n * bm;
  const int groups = (a.w.rows + 63) / 64, m0 = tile_m * 16 * MT;
  const int group = min(tile_n * 4 + wave, groups - 1);
  const int b0 = (int)((long long)a.w.kb * piece / splits), kb = (int)((long long)a.w.kb * (piece + 1) / splits) - b0;
  TileWave<MT, EXACT> w;
  w.wave = wave;
  w.r = lane & 15;
  w.lane16 = 16 * lane;
  w.M_stride = a.M_stride;
  w.last = kb - 1;
  w.frag_stride = (uint32_t)a.w.kb * kFragBytes;
  w.wbuf = buffer_of(a.w.q + (size_t)group * 4 * w.frag_stride + (size_t)b0 * kFragBytes, 4 * w.frag_stride - (uint32_t)b0 * kFragBytes);
  const float* wsc = a.w.sc + (size_t)(group >> 1) * a.w.kb + b0;
  const int left = a.M - 1 - m0;  // (rows behind the last token: the last one again, their results are not stored)
  const uint32_t row_bytes = (uint32_t)a.w.kb * 128, rows = (uint32_t)min(16 * MT, left + 1);
#pragma unroll
  for (int i = 0; i < (MT + 1) / 2; ++i) {
    const int piece16 = w.dst(i) + lane, row = piece16 >> 3;
    w.off[i] = (uint32_t)min(row, left) * row_bytes + 16 * ((piece16 & 7) ^ (row & 7));
  }
  w.sc_off = 4 * (uint32_t)min(w.sc_dst() + lane, left);
  w.rows = buffer_of(a.a8 + (size_t)m0 * row_bytes + 128 * (size_t)b0, rows * row_bytes - 128 * (uint32_t)b0);
  w.asc = buffer_of(a.asc + (size_t)b0 * a.M_stride + m0, ((uint32_t)(kb - 1) * (uint32_t)a.M_stride + rows) * 4);
  w.at0 = 8 * w.r + (g ^ (w.r & 7));
  w.at1 = 8 * w.r + ((4 + g) ^ (w.r & 7));
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    w.p[t] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < MT; ++j) w.acc[t][j] = {0.0f, 0.0f, 0.0f, 0.0f};
  }
  w.s = 0.0f;
  constexpr int kLoads = TileWave<MT, EXACT>::kLoads, kAhead = TileWave<MT, EXACT>::kAhead;
  Frags w0, w1;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) w.load_tokens(t0, 0, i);
#pragma unroll
  for (int i = 0; i < kLoads; ++i) w.load_tokens(t1, 1, i);
  asm volatile("" ::: "memory");
  w.load_frags(w0, 0);
  asm volatile("" ::: "memory");
  if (kAhead == 3)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) w.load_tokens(t2, 2, i);
  float ws64 = wsc[min(lane, w.last)];  // the scales of 64 blocks, one a lane (a scalar load would make every LDS wait whole)
  __builtin_amdgcn_s_waitcnt(wait_loads(8 + kLoads));
  meet();
  w.first_tile(t0);
#define QM_WS(B) __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, ws64), (B) & 63))
#define QM_STEP(B, T, T1, T2, T3, W, WN) w.block(B, W, T, QM_WS(B), EXACT ? W : WN, T1, kAhead == 3 ? T3 : T2)
  int b = 0;
  for (; b + 4 <= kb; b += 4) {
    if (b && (b & 63) == 0) ws64 = wsc[min(b + lane, w.last)];
    QM_STEP(b, t0, t1, t2, t3, w0, w1);
    QM_STEP(b + 1, t1, t2, t3, t0, (EXACT ? w0 : w1), w0);
    QM_STEP(b + 2, t2, t3, t0, t1, w0, w1);
    QM_STEP(b + 3, t3, t0, t1, t2, (EXACT ? w0 : w1), w0);
  }
  if (b && (b & 63) == 0) ws64 = wsc[min(b + lane, w.last)];
  if (b < kb) QM_STEP(b, t0, t1, t2, t3, w0, w1);
  if (b + 1 < kb) QM_STEP(b + 1, t1, t2, t3, t0, (EXACT ? w0 : w1), w0);
  if (b + 2 < kb) QM_STEP(b + 2, t2, t3, t0, t1, w0, w1);
#undef QM_STEP
#undef QM_WS
  __builtin_amdgcn_s_waitcnt(wait_loads(0));  // (no load into LDS outlives the work-group)
#pragma unroll
  for (int t = 0; t < 4; ++t) w.add_last(t, w.acc[t][MT - 1]);
  // Stores: a result lane holds 16 n of one token, a token's 64 n lie over four lanes. Each token tile goes through LDS (the wave's
  // own part of the token buffers, which every wave has read by now), so that eight lanes store one token's 64 n: stored from
  // where they lie (8 bytes a lane) they took a quarter of the kernel's time.
  __syncthreads();
  if (tile_n * 4 + wave >= groups) return;
  constexpr int kRow = 68;  // floats of a token's row, with padding
  float* lds = (float*)(wave == 0 ? t0.v : wave == 1 ? t1.v : wave == 2 ? t2.v : t3.v);
  static_assert(sizeof(t0.v) >= 16 * kRow * sizeof(float), "a token tile");
  constexpr bool kTwo = sizeof(t0.v) >= 2 * 16 * kRow * sizeof(float);
  const int n = 64 * group + 8 * (lane & 7), mr = lane >> 3;
  // (token, its eight sums) for both halves of a token tile at a time, to `put`
  const auto rows_out = [&](auto put) {
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      float* pj = lds + (kTwo ? (j & 1) * 16 * kRow : 0);
#pragma unroll
      for (int t = 0; t < 4; ++t) *(v4f*)(pj + w.r * kRow + 16 * g + 4 * t) = w.acc[t][j];
      exchange();
      v4f lo[2], hi[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        lo[h] = *(const v4f*)(pj + (8 * h + mr) * kRow + 8 * (lane & 7));
        hi[h] = *(const v4f*)(pj + (8 * h + mr) * kRow + 8 * (lane & 7) + 4);
      }
      exchange();
#pragma unroll
      for (int h = 0; h < 2; ++h) put(m0 + 16 * j + 8 * h + mr, lo[h], hi[h]);
    }
  };
  const bool whole = left + 1 >= 16 * MT && 64 * group + 64 <= a.w.rows;  // (no test between the stores: they are all under way at once)
  const bool vec = vec_stores8(a);
  if (splits > 1) {
    float* to = a.part + (size_t)piece * a.M * (64 * (size_t)groups) + n;
    rows_out([&](int m, v4f lo, v4f hi) {
      if (m >= a.M) return;
      v4f* at = (v4f*)(to + (size_t)m * (64 * (size_t)groups));
      at[0] = lo;
      at[1] = hi;
    });
  } else if (!EXACT && whole && vec && a.accumulate == 0) {
    if (a.ctype == DT_F16) rows_out([&](int m, v4f lo, v4f hi) { put8_whole((_Float16*)a.C + (size_t)m * a.ldc + a.c_off + n, lo, hi); });
    else rows_out([&](int m, v4f lo, v4f hi) { put8_whole((__bf16*)a.C + (size_t)m * a.ldc + a.c_off + n, lo, hi); });
  } else if (EXACT && whole && vec && a.accumulate == 0) {
    rows_out([&](int m, v4f lo, v4f hi) {
      v4f* at = (v4f*)((float*)a.C + (size_t)m * a.ldc + a.c_off + n);
      at[0] = lo;
      at[1] = hi;
    });
  } else {
    rows_out([&](int m, v4f lo, v4f hi) {
      if (m < a.M) store8(a, m, n, lo, hi, vec);
    });
  }
}

// C (op)= the sum of the pieces, in their order; eight n a thread. Four pieces are on their way at once: one after the other they
// cost a memory latency each.
__global__ __launch_bounds__(256) void fp8_sum_kernel(Fp8GemmArgs a, int splits, int width) {
  const int n = 8 * (blockIdx.y * 256 + threadIdx.x), m = blockIdx.x;
  if (n >= a.w.rows) return;
  const size_t next = (size_t)a.M * width;
  const float* at = a.part + (size_t)m * width + n;
  v4f lo = {0.0f, 0.0f, 0.0f, 0.0f}, hi = lo;
  for (int p = 0; p < splits; p += 4) {
    v4f l[4], h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float* q = at + (size_t)min(p + i, splits - 1) * next;
      l[i] = *(const v4f*)q;
      h[i] = *(const v4f*)(q + 4);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p + i < splits) {
        lo += l[i];
        hi += h[i];
      }
    }
  }
  store8(a, m, n, lo, hi, vec_stores8(a));
}

namespace {

template <int MT>
hipError_t tile_of(const Fp8GemmArgs& a, int splits, hipStream_t s) {
  const int tn = (a.w.rows + 255) / 256, tm = (a.M + 16 * MT - 1) / (16 * MT);
  const unsigned grid = (unsigned)((tn * tm * splits + 7) / 8 * 8);
  if (a.ctype != DT_F32) {
    fp8_tile_kernel<MT, false><<<grid, 256, 0, s>>>(a, tn, tm, splits);
  } else if constexpr (MT <= 6) {
    fp8_tile_kernel<MT, true><<<grid, 256, 0, s>>>(a, tn, tm, splits);
  } else {
    return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_tile(const Fp8GemmArgs& a, int mt, int splits, hipStream_t s) {
  const hipError_t e = mt == 4 ? tile_of<4>(a, splits, s) : mt == 5 ? tile_of<5>(a, splits, s) : mt == 6 ? tile_of<6>(a, splits, s)
                     : mt == 7 ? tile_of<7>(a, splits, s) : mt == 8 ? tile_of<8>(a, splits, s) : hipErrorInvalidValue;
  if (e != hipSuccess || splits == 1) return e;
  const int width = (a.w.rows + 63) / 64 * 64;
  fp8_sum_kernel<<<dim3(a.M, (width + 2047) / 2048), 256, 0, s>>>(a, splits, width);
  return hipGetLastError();
}

}  // namespace qm
