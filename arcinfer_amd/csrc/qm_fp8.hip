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
#include "qm_fp8.h"

namespace qm {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kFragBytes = 2048;

__device__ __forceinline__ v8i join(v4i lo, v4i hi) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); }

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// Eight e4m3 values as f16 (exact; NaN stays NaN)
__device__ __forceinline__ v8h widen(int lo, int hi) {
  const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// S of one block: 16 rows by 16 tokens, 32 bytes of each a lane. (The builtin without scales is the unscaled instruction.)
template <bool EXACT>
__device__ __forceinline__ v4f dot_block(v8i w, v8i a) {
  v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
  if constexpr (EXACT) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(widen(w[i], w[i + 1]), widen(a[i], a[i + 1]), s, 0, 0, 0);
    return s;
  } else {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, s, 0, 0, 0, 0, 0, 0);
  }
}

// C[i] (op)= v for elements of type T, computed in f32 and rounded once
template <typename T>
__device__ __forceinline__ void put(T* C, float v, int accumulate) {
  if (accumulate == 1) {
    v += (float)*C;
  } else if (accumulate == 2) {
    const float g = (float)*C;
    v = g / (1.0f + expf(-g)) * v;
  }
  *C = (T)v;
}

// Four neighbouring results n .. n + 3 of token m (n % 4 == 0; rows: the weight's)
template <typename T>
__device__ __forceinline__ void put4(T* C, size_t at, v4f v, int left, int accumulate, bool vec) {
  typedef T v4t __attribute__((ext_vector_type(4)));
  if (vec && left >= 4) {
    if (accumulate) {
      const v4t o = *(const v4t*)(C + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float c = (float)o[i];
        v[i] = accumulate == 1 ? v[i] + c : c / (1.0f + expf(-c)) * v[i];
      }
    }
    v4t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (T)v[i];
    *(v4t*)(C + at) = r;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) put(C + at + i, v[i], accumulate);
}

__device__ __forceinline__ void store4(const Fp8GemmArgs& a, int m, int n, v4f v, bool vec) {
  const size_t at = (size_t)m * a.ldc + a.c_off + n;
  const int left = a.w.rows - n;
  if (left <= 0) return;
  if (a.ctype == DT_F32) put4((float*)a.C, at, v, left, a.accumulate, vec);
  else if (a.ctype == DT_F16) put4((_Float16*)a.C, at, v, left, a.accumulate, vec);
  else put4((__bf16*)a.C, at, v, left, a.accumulate, vec);
}

// whether every group of four results lies on its own alignment
__device__ __forceinline__ bool vec_stores(const Fp8GemmArgs& a) {
  const uintptr_t size = a.ctype == DT_F32 ? 4 : 2;
  return ((((uintptr_t)a.C / size) | (uintptr_t)a.ldc | (uintptr_t)a.c_off) & 3) == 0;
}

}  // namespace

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

// One fragment of 16 rows against 16 MT tokens: four waves take every fourth block of K, and add their sums in wave order.
template <int MT, bool EXACT>
__global__ __launch_bounds__(256) void fp8_few_kernel(Fp8GemmArgs a) {
  __shared__ v4f red[4][MT][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int tile = blockIdx.x, m0 = blockIdx.y * 16 * MT, kb = a.w.kb;
  const uint8_t* wp = a.w.q + (size_t)tile * kb * kFragBytes + 16 * lane;
  const float* wsc = a.w.sc + (size_t)(tile >> 3) * kb;
  const size_t Kp = (size_t)kb * 128;
  v4f acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int b = wave; b < kb; b += 4) {
    const v4i w0 = *(const v4i*)(wp + (size_t)b * kFragBytes), w1 = *(const v4i*)(wp + (size_t)b * kFragBytes + 1024);
    const float ws = wsc[b];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int m = m0 + 16 * t + r;
      v4i a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
      float s = 0.0f;
      if (m < a.M) {
        const uint8_t* ap = a.a8 + m * Kp + 128 * (size_t)b + 16 * g;
        a0 = *(const v4i*)ap;
        a1 = *(const v4i*)(ap + 64);
        s = a.asc[(size_t)b * a.M_stride + m] * ws;
      }
      const v4f p = dot_block<EXACT>(join(w0, w1), join(a0, a1));
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(s, p[i], acc[t][i]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  const bool vec = vec_stores(a);
  for (int t = wave; t < MT; t += 4) {
    const int m = m0 + 16 * t + r;
    v4f v = red[0][t][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += red[w][t][lane][i];
    }
    if (m < a.M) store4(a, m, 64 * (tile >> 2) + 16 * g + 4 * (tile & 3), v, vec);
  }
}

size_t fp8_workspace_bytes(int M, int rows, int kb) {
  (void)M;
  (void)rows;
  (void)kb;
  return 0;
}

namespace {

template <bool EXACT>
void launch_few(const Fp8GemmArgs& a, hipStream_t s) {
  const unsigned tiles = (unsigned)((a.w.rows + 63) / 64 * 4);
  if (a.M <= 16) fp8_few_kernel<1, EXACT><<<tiles, 256, 0, s>>>(a);
  else if (a.M <= 32) fp8_few_kernel<2, EXACT><<<tiles, 256, 0, s>>>(a);
  else fp8_few_kernel<4, EXACT><<<dim3(tiles, (a.M + 63) / 64), 256, 0, s>>>(a);
}

}  // namespace

hipError_t launch_gemm_fp8(const Fp8GemmArgs& a, hipStream_t s) {
  if (a.ctype == DT_F32) launch_few<true>(a, s);
  else launch_few<false>(a, s);
  return hipGetLastError();
}

}  // namespace qm
