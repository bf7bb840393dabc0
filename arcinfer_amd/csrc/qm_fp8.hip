// Products of e4m3 activations and weights with block scales.
//   C[m][n] = sum_b asc[b][m] * wsc[n / 128][b] * S_b,   S_b = sum over the 128 values of block b of a8[m][k] * w8[n][k]
// S_b comes off the matrix pipe with a zero accumulator, and an f32 FMA adds it to the result with the product of both scales.
// The weight is the A operand (result rows), the tokens are the B operand (result columns), so a lane's four results belong to
// one token and one weight block: one scale product serves them.
//
// Which pipe. One v_mfma_f32_16x16x128_f8f6f4 is exactly one block of K, at twice the f16 rate. But every fp8 MFMA adds
// the products of eight neighbouring k on a common exponent and drops what lies 2^-13 below the largest of them (measured;
// between the eights the sum is f32): 1.3e-5 of the result for normal values, whichever fp8 instruction it is. Under a C of 16 bits
// (rounded by 2^-9 or 2^-12) that is nothing. A C of f32 gets the f16 pipe: e4m3 values are f16 values, their products exact
// there and the sums f32 (1e-8), for four v_mfma_f32_16x16x32_f16 a block and the conversions.
#include "qm_fp8_dev.h"

namespace qm {

// e4m3 rows -> the prepared layout, 16 bytes a thread
__global__ __launch_bounds__(256) void fp8_repack_kernel(const uint8_t* __restrict__ w, int rows, int K, int kb, size_t n,
                                                         bool vec, uint8_t* __restrict__ q) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int lane = (int)(i & 63), half = (int)(i >> 6) & 1;
  const size_t fb = i >> 7;
  const int b = (int)(fb % kb), tile = (int)(fb / kb), r = lane & 15;
  const int row = 64 * (tile >> 2) + 16 * (r >> 2) + 4 * (tile & 3) + (r & 3), k0 = 128 * b + 64 * half + 16 * (lane >> 4);
  uint4 v = make_uint4(0, 0, 0, 0);
  if (row < rows) {
    const uint8_t* src = w + (size_t)row * K;
    if (vec && k0 + 16 <= K) {
      v = *(const uint4*)(src + k0);
    } else {
      uint32_t t[4] = {0, 0, 0, 0};
      for (int j = 0; j < 16; ++j)
        if (k0 + j < K) t[j >> 2] |= (uint32_t)src[k0 + j] << (8 * (j & 3));
      v = make_uint4(t[0], t[1], t[2], t[3]);
    }
  }
  *(uint4*)(q + 16 * i) = v;
}

hipError_t launch_fp8_repack(const uint8_t* w8, int rows, int K, uint8_t* q, hipStream_t s) {
  const int kb = (K + 127) / 128;
  const size_t n = (size_t)((rows + 63) / 64) * 4 * kb * 128;  // 16-byte pieces
  const bool vec = K % 16 == 0 && (uintptr_t)w8 % 16 == 0;
  fp8_repack_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(w8, rows, K, kb, n, vec, q);
  return hipGetLastError();
}

// Few tokens: RT fragments of 16 rows against 16 MT tokens. The W waves of a work-group take the blocks of K in turn, so that
// it streams its rows from one end to the other, and add their sums in wave order.
template <int MT, int RT, int W, bool EXACT>
__global__ __launch_bounds__(64 * W) void fp8_few_kernel(Fp8GemmArgs a) {
  __shared__ v4f red[W][RT * MT][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const unsigned units = (unsigned)((a.w.rows + 63) / 64 * 4 / RT);  // (neighbouring work-groups take neighbouring rows)
  const int tile = RT * (int)(blockIdx.x % units), m0 = (int)(blockIdx.x / units) * 16 * MT, kb = a.w.kb;
  const size_t frag_stride = (size_t)kb * kFragBytes;
  const uint8_t* wp = a.w.q + (size_t)tile * frag_stride + 16 * lane;
  const float* wsc = a.w.sc + (size_t)(tile >> 3) * kb;
  const size_t Kp = (size_t)kb * 128;
  const uint8_t* ap = a.a8 + (size_t)(m0 + r) * Kp + 16 * g;
  const float* asc = a.asc + m0 + r;
  v4f acc[RT][MT];
#pragma unroll
  for (int f = 0; f < RT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[f][t] = {0.0f, 0.0f, 0.0f, 0.0f};
  const auto block = [&](int b, const v4i (&w)[RT][2]) {
    const float ws = wsc[b];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      v4i a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
      float s = 0.0f;
      if (m0 + 16 * t + r < a.M) {
        const uint8_t* p = ap + 16 * t * Kp + 128 * (size_t)b;
        a0 = *(const v4i*)p;
        a1 = *(const v4i*)(p + 64);
        s = asc[(size_t)b * a.M_stride + 16 * t] * ws;
      }
#pragma unroll
      for (int f = 0; f < RT; ++f) {
        const v4f p = dot_block<EXACT>(join(w[f][0], w[f][1]), join(a0, a1));
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][t][i] = fmaf(s, p[i], acc[f][t][i]);
      }
    }
  };
  const auto load = [&](int b, v4i (&w)[RT][2]) {
#pragma unroll
    for (int f = 0; f < RT; ++f) {
      const uint8_t* p = wp + f * frag_stride + (size_t)b * kFragBytes;
      // (streaming loads are 5 % faster where nothing is cached, 8 weights of 17408 x 5120 in turn 20.1 us against 21.4, and 10 to 20 %
      //  slower where the last-level cache holds part of them, 2 in turn 21.5 against 19.4)
      w[f][0] = *(const v4i*)p;
      w[f][1] = *(const v4i*)(p + 1024);
    }
  };
  // U blocks' weights are under way at once
  constexpr int U = RT == 1 ? 4 : 2;
  int b = wave;
  for (; b + (U - 1) * W < kb; b += U * W) {
    v4i w[U][RT][2];
#pragma unroll
    for (int u = 0; u < U; ++u) load(b + u * W, w[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) block(b + u * W, w[u]);
  }
  for (; b < kb; b += W) {
    v4i w[RT][2];
    load(b, w);
    block(b, w);
  }
#pragma unroll
  for (int f = 0; f < RT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[wave][f * MT + t][lane] = acc[f][t];
  __syncthreads();
  const bool vec = vec_stores(a);
  for (int i = wave; i < RT * MT; i += W) {
    const int f = i / MT, t = i - f * MT, m = m0 + 16 * t + r;
    v4f v = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[w][i][lane];
    if (m < a.M) store4(a, m, 64 * (tile >> 2) + 16 * g + 4 * ((tile & 3) + f), v, vec);
  }
}

namespace {

template <int MT, int RT, int W>
void launch_few(const Fp8GemmArgs& a, hipStream_t s) {
  const unsigned grid = (unsigned)((a.w.rows + 63) / 64 * 4 / RT) * (((unsigned)a.M + 16 * MT - 1) / (16 * MT));
  if (a.ctype == DT_F32) fp8_few_kernel<MT, RT, W, true><<<grid, 64 * W, 0, s>>>(a);
  else fp8_few_kernel<MT, RT, W, false><<<grid, 64 * W, 0, s>>>(a);
}

// The few-token kernel's shape. Two fragments a work-group once one would put more than a work-group on every CU (the token
// reads halve: 5 x 17408 -> 5120 20 us against 24), and as many waves as keep a CU busy and have blocks to take (1 x 4096 -> 4096, 256
// fragments: 16 waves 5.3 us, 8 6.1, 4 7.2; with more than one work-group a CU 8: 16 x 5120 -> 17408 22.2 against 23.8).
struct FewShape {
  int rt, waves;
};
FewShape few_shape(int M, int rows, int kb) {
  const int tiles = (rows + 63) / 64 * 4, rt = tiles > 256 ? 2 : 1, wg = tiles / rt;
  int w = 8;
  if (kb < 8 || (M > 16 && wg > 512)) w = 4;
  else if (kb >= 16 && wg <= 256 && (M <= 16 || (M <= 32 && rt == 1))) w = 16;
  return {rt, w};
}

// Whether its work-groups fit a grid (those of up to 16 tokens do: a weight is below 64 GiB)
bool few_fits(int M, int rows, FewShape f) {
  const long long mt = M > 48 ? 4 : (M + 15) / 16, turns = (M + 16 * mt - 1) / (16 * mt), units = (rows + 63) / 64 * 4 / f.rt;
  return units * turns * 64 * f.waves <= kMostThreads;
}

hipError_t launch_few_tokens(const Fp8GemmArgs& a, const Fp8Plan& f, hipStream_t s) {
  // (only products that the tile kernel cannot take, of activations beyond 128 GiB, come to that many)
  if (!few_fits(a.M, a.w.rows, {f.rt, f.waves})) return hipErrorInvalidConfiguration;
#define QM_FEW(MT, RT) (f.waves == 8 ? launch_few<MT, RT, 8>(a, s) : launch_few<MT, RT, 4>(a, s))
  if (a.M <= 16) {
    if (f.waves == 16) f.rt == 1 ? launch_few<1, 1, 16>(a, s) : launch_few<1, 2, 16>(a, s);
    else f.rt == 1 ? QM_FEW(1, 1) : QM_FEW(1, 2);
  } else if (a.M <= 32) {
    if (f.waves == 16) launch_few<2, 1, 16>(a, s);
    else f.rt == 1 ? QM_FEW(2, 1) : QM_FEW(2, 2);
  } else if (a.M <= 48) {
    f.rt == 1 ? QM_FEW(3, 1) : QM_FEW(3, 2);
  } else {
    f.rt == 1 ? QM_FEW(4, 1) : QM_FEW(4, 2);
  }
#undef QM_FEW
  return hipGetLastError();
}

// Times in microseconds, fitted to those of profiles/fp8_variants.txt: 7300 (C of 16 bits) and 4460 (f32) of 200 products of 20 to 4096
// tokens and ten weights from 512 x 1024 to 17408 x 5120 (rms 9 and 7 %). The choice by them loses 3.0 and 1.6 % on average against the
// fastest variant, 37 and 28 % at most (64 x 5120 -> 17408, 64 x 4096 -> 4096).
// Tile kernel: `call`; a work-group's blocks and `more` (its prologue and store), each block one + one_mt * MT where work-groups have
// their CU to themselves (`crowd` of it more with every CU taken), two + two_mt * MT where two share it, a last round behind
// others `tail` of that; never less than the weight's bytes at `stream` a microsecond; cut: `sum`, and the pieces written and read at `part`.
// Few-token kernel: few_call; bytes of weight and of tokens (read once a work-group) at few_w and few_t; few_mt a block, token tile and fragment.
struct Rates {
  float call, more, one, one_mt, crowd, two, two_mt, tail, stream, sum, part;
  float few_call, few_w, few_t, few_mt;
};
constexpr Rates kRates16 = {2.9f, 3.8f, 0.18f, 0.072f, 0.31f, 0.53f, 0.12f, 0.74f, 4.6e6f, 2.45f, 6.9e6f, 3.8f, 11.1e6f, 7.9e6f, 0.071f};
constexpr Rates kRates32 = {3.1f, 2.4f, 0.0f, 0.248f, 0.19f, 0.03f, 0.41f, 0.75f, 4.5e6f, 2.6f, 8.1e6f, 4.0f, 8.5e6f, 7.4e6f, 0.094f};
constexpr float kFewBlock16 = 0.19f;  // (few-token kernel, fp8 pipe: a block of a wave; nothing measurable on the f16 pipe)

float tile_us(const Rates& r, int M, int rows, int kb, int mt, int splits) {
  const int n = (rows + 255) / 256 * ((M + 16 * mt - 1) / (16 * mt)) * splits, full = n / kFp8Slots, rem = n % kFp8Slots;
  const float two = r.two + r.two_mt * mt;
  float rounds = full * two;
  if (rem) rounds += (rem > kFp8Slots / 2 ? two : (r.one + r.one_mt * mt) * (1.0f + r.crowd * rem / (kFp8Slots / 2))) * (full ? r.tail : 1.0f);
  const float run = rounds * ((kb + splits - 1) / splits + r.more), read = (float)rows * kb * 128.0f / r.stream;
  const float run2 = run * run, read2 = read * read;
  float t = r.call + sqrtf(sqrtf(run2 * run2 + read2 * read2));  // (the larger, and both where they are alike)
  if (splits > 1) t += r.sum + 8.0f * splits * M * ((rows + 63) / 64 * 64.0f) / r.part;
  return t;
}

float few_us(const Rates& r, float block, int M, int rows, int kb) {
  const FewShape f = few_shape(M, rows, kb);
  const int tiles = (rows + 63) / 64 * 4, mt = M > 48 ? 4 : (M + 15) / 16, turns = (M + 63) / 64;
  const float bytes = tiles * 2048.0f * kb;
  return r.few_call + bytes / r.few_w + bytes / f.rt * mt * turns / r.few_t + (block + r.few_mt * mt * f.rt) * kb / f.waves;
}

}  // namespace

// Up to 16 tokens: the few-token kernel. Beyond, what the times above say: that kernel (mt = 0), or tiles of mt token tiles, each
// in `splits` pieces of at least three blocks, as many as part_bytes of workspace hold the sums of.
Fp8Plan fp8_plan(int M, int M_stride, int rows, int kb, bool exact, size_t part_bytes) {
  const FewShape f = few_shape(M, rows, kb);
  Fp8Plan p{0, 1, f.rt, f.waves};
  if (part_bytes > kFp8PartBytes) part_bytes = kFp8PartBytes;
  // (the tile kernel's token scales are a buffer of 32-bit offsets)
  if (M <= 16 || (size_t)kb * M_stride >= (size_t)1 << 30) return p;
  const Rates& r = exact ? kRates32 : kRates16;
  float best = M <= 1024 && few_fits(M, rows, f) ? few_us(r, exact ? 0.0f : kFewBlock16, M, rows, kb) : 1e30f;
  constexpr int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16};
  for (int mt = exact ? 6 : 8; mt >= 4; --mt) {
    for (int s : kSplits) {
      if (s > 1 && (kb / s < 3 || fp8_part_bytes(M, rows, s) > part_bytes)) break;
      const float t = tile_us(r, M, rows, kb, mt, s);
      // (a smaller tile only for 2 %: what the times cannot tell apart is faster with the larger one, 4096 x 5120 -> 17408 329 us against
      //  342; it reads less)
      if (t < best * (p.mt > mt ? 0.98f : 1.0f)) {
        best = t;
        p = {mt, s, 0, 0};
      }
    }
  }
  return p;
}

size_t fp8_workspace_bytes(int M, int rows, int kb) {
  // (the larger of both output types': the call's is not known yet)
  size_t most = 0;
  for (int exact = 0; exact < 2; ++exact) {
    const Fp8Plan p = fp8_plan(M, M, rows, kb, exact != 0, kFp8PartBytes);
    if (p.splits > 1 && fp8_part_bytes(M, rows, p.splits) > most) most = fp8_part_bytes(M, rows, p.splits);
  }
  return most;
}

hipError_t launch_gemm_fp8(const Fp8GemmArgs& a, const Fp8Plan& p, hipStream_t s) {
  return p.mt ? launch_fp8_tile(a, p.mt, p.splits, s) : launch_few_tokens(a, p, s);
}

}  // namespace qm
