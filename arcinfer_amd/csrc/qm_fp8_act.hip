// Producers of e4m3 activations: rows, RMS-normed rows or gated rows, with one f32 scale per 128 values. HBM-bound: each
// input is read once, each output written once. A block of 128 values is 16 lanes of 8 values, its amax a reduction over them.
#include "qm_fp8.h"

namespace qm {

namespace {

constexpr float kTop = 448.0f;        // the largest e4m3 value
constexpr float kTiny = 0x1p-100f;    // blocks below it are zeros: 448 / amax stays finite and amax / 448 normal

// The largest of 16 neighbouring lanes, in each of them (rotations within a row of 16 lanes: no LDS)
template <int N>
__device__ __forceinline__ float rotated16(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xF, 0xF, false));
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, rotated16<8>(v));
  v = fmaxf(v, rotated16<4>(v));
  v = fmaxf(v, rotated16<2>(v));
  return fmaxf(v, rotated16<1>(v));
}

// Eight elements of a row from element i on; those past K are zero. VEC: K % 8 == 0 and 16-byte aligned rows.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ r, int i, int K, float v[8]) {
  if constexpr (VEC) {
    constexpr int N = 16 / sizeof(T);
    typedef T vt __attribute__((ext_vector_type(N)));
    if (i < K) {
#pragma unroll
      for (int j = 0; j < 8; j += N) {
        const vt t = *(const vt*)(r + i + j);
#pragma unroll
        for (int e = 0; e < N; ++e) v[j + e] = (float)t[e];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = i + j < K ? (float)r[i + j] : 0.0f;
  }
}

// Quantizes a block of 128 held by 16 neighbouring lanes, 8 values each, `at` the element of this lane's first. Every lane of the
// 16 calls it; store masks the writes.
__device__ __forceinline__ void quant16(const float v[8], bool store, int m, int at, int M_stride, size_t Kp,
                                        uint8_t* __restrict__ a8, float* __restrict__ asc) {
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(v[j]));
  amax = max16(amax);
  const float inv = amax >= kTiny ? kTop / amax : 0.0f;
  if (!store) return;
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
  *(int2*)(a8 + m * Kp + at) = make_int2(lo, hi);
  if ((threadIdx.x & 15) == 0) asc[(size_t)(at >> 7) * M_stride + m] = amax >= kTiny ? amax / kTop : 0.0f;
}

// e^x = 2^(x log2 e), the product in two parts: the exponent's rounding would cost |x| / 2 steps of the result. Within 2 steps.
__device__ __forceinline__ float exp_fast(float x) {
  constexpr float kHi = 1.44269502f, kLo = 1.92596303e-8f;  // log2 e
  const float h = x * kHi, l = fmaf(x, kLo, fmaf(x, kHi, -h));
  const float e = __builtin_amdgcn_exp2f(h);
  return fmaf(e, l * 0.693147181f, e);
}
// x / (1 + e^-z): silu for z = x. The quotient by a reciprocal and one correction, within 2 steps (the correctly rounded division and expf
// took more of the vector pipe than the rows take of HBM: 2048 rows of 17408 in bf16 45.9 us against 40.2). The exponent is kept where
// e and the sum are finite; what lies beyond is far_gated's. A NaN of x stays one, an infinite x becomes one.
constexpr float kFar = -83.0f;  // (e^83 is over 2^119)
__device__ __forceinline__ float gated(float x, float z) {
  const float d = 1.0f + exp_fast(fminf(fmaxf(-z, -104.0f), -kFar));
  const float r = __builtin_amdgcn_rcpf(d), q = x * r;
  return fmaf(fmaf(-d, q, x), r, q);
}
// The same for z below kFar, where the sum is its exponential: x e^z, of which what is below 2^-126 may be zero
__device__ __forceinline__ float far_gated(float x, float z) { return x * exp_fast(fmaxf(z, -104.0f)); }
// gelu: 0.5 x (1 + tanh y), y = sqrt(2 / pi) (x + 0.044715 x^3): 1 + tanh y is 2 / (1 + e^-2y)
__device__ __forceinline__ float gelu_z(float x) { return 1.59576912f * fmaf(0.044715f * x * x, x, x); }

enum : int { ROWS = 0, SILU = 1, GELU = 2 };

}  // namespace

// One work-group per row and 2048 values, a row's work-groups next to each other.
template <typename T, bool VEC, int OP>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T* __restrict__ x, int ldx, int K, int M, int M_stride,
                                                       uint8_t* __restrict__ a8, float* __restrict__ asc) {
  const unsigned chunks = (unsigned)(K + 2047) / 2048;
  const int m = (int)(blockIdx.x / chunks), kp = (K + 127) / 128 * 128, at = 2048 * (int)(blockIdx.x % chunks) + 8 * threadIdx.x;
  const T* r = x + (size_t)m * ldx;
  float v[8] = {};
  if (m < M) {
    load8<T, VEC>(r, at, K, v);
    if constexpr (OP != ROWS) {
      float u[8];
      load8<T, VEC>(r + K, at, K, u);
      float z[8], low = 0.0f, g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        z[j] = OP == SILU ? v[j] : gelu_z(v[j]);
        g[j] = v[j];
        low = fminf(low, z[j]);
        v[j] = gated(g[j], z[j]) * u[j];
      }
      if (low < kFar) {  // (hardly ever: a branch for eight values)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (z[j] < kFar) v[j] = far_gated(g[j], z[j]) * u[j];
      }
    }
  }
  quant16(v, at < kp, m, at, M_stride, kp, a8, asc);
}

// y = x * r * w, r = 1 / sqrt(mean(x^2) + eps). One work-group per row (and, of few rows, per every gridDim.y-th pass of 2048
// values: each reads the row for its mean square). PASSES > 0: the row stays in registers; 0: it is read again.
template <typename T, bool VEC, int PASSES>
__global__ __launch_bounds__(256) void fp8_rmsnorm_kernel(const T* __restrict__ x, int ldx, const float* __restrict__ w,
                                                          int K, int M, int M_stride, float eps, uint8_t* __restrict__ a8,
                                                          float* __restrict__ asc, float* __restrict__ h, int ldh) {
  __shared__ float red[4];
  const int m = blockIdx.x, kp = (K + 127) / 128 * 128;
  const bool valid = m < M;
  const T* r = x + (size_t)m * ldx;
  float xv[PASSES ? PASSES : 1][8];
  float ss = 0.0f;
  const auto square = [&](const float v[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
  };
  if (valid) {
    if constexpr (PASSES > 0) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) load8<T, VEC>(r, 2048 * p + 8 * threadIdx.x, K, xv[p]);
#pragma unroll
      for (int p = 0; p < PASSES; ++p) square(xv[p]);
    } else {
      for (int i = 8 * threadIdx.x; i < K; i += 2048) {
        load8<T, VEC>(r, i, K, xv[0]);
        square(xv[0]);
      }
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) ss += __shfl_xor(ss, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
  __syncthreads();
  ss = ((red[0] + red[1]) + red[2]) + red[3];
  const float n = 1.0f / sqrtf(ss / (float)K + eps);
  const bool h_vec = VEC && h && (((uintptr_t)h >> 2 | (uintptr_t)ldh) & 3) == 0;
  const auto finish = [&](const float xr[8], int p) {
    const int at = 2048 * p + 8 * threadIdx.x;
    float v[8] = {};
    if (valid) {
      float wv[8];
      load8<float, VEC>(w, at, K, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = xr[j] * n * wv[j];
      float* hr = h + (size_t)m * ldh + at;
      if (h_vec) {
        if (at < K) {
          *(float4*)hr = make_float4(v[0], v[1], v[2], v[3]);
          *(float4*)(hr + 4) = make_float4(v[4], v[5], v[6], v[7]);
        }
      } else if (h) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at + j < K) hr[j] = v[j];
      }
    }
    quant16(v, at < kp, m, at, M_stride, kp, a8, asc);
  };
  if constexpr (PASSES > 0) {
#pragma unroll
    for (int p = 0; p < PASSES; ++p)
      if (p % (int)gridDim.y == (int)blockIdx.y) finish(xv[p], p);
  } else {
    for (int p = blockIdx.y; 2048 * p < kp; p += gridDim.y) {
      if (valid) load8<T, VEC>(r, 2048 * p + 8 * threadIdx.x, K, xv[0]);
      finish(xv[0], p);
    }
  }
}

namespace {

// whether rows of `size`-byte elements can be read 16 bytes at a time
bool rows_aligned(const void* p, int ld, int K, int size) {
  return K % 8 == 0 && (uintptr_t)p % 16 == 0 && (size_t)ld * size % 16 == 0;
}

template <typename T>
hipError_t rows_of(const T* x, int ldx, int K, int M, int rows, int M_stride, int op, uint8_t* a8, float* asc, hipStream_t s) {
  const unsigned grid = (unsigned)rows * ((K + 2047) / 2048);
  const bool vec = rows_aligned(x, ldx, K, sizeof(T)) && (op == ROWS || (size_t)K * sizeof(T) % 16 == 0);
#define QM_F8R(OP) \
  if (vec) fp8_rows_kernel<T, true, OP><<<grid, 256, 0, s>>>(x, ldx, K, M, M_stride, a8, asc); \
  else fp8_rows_kernel<T, false, OP><<<grid, 256, 0, s>>>(x, ldx, K, M, M_stride, a8, asc)
  if (op == ROWS) { QM_F8R(ROWS); }
  else if (op == SILU) { QM_F8R(SILU); }
  else { QM_F8R(GELU); }
#undef QM_F8R
  return hipGetLastError();
}

template <typename T, bool VEC>
hipError_t norm_of(const T* x, int ldx, const float* w, int K, int M, int rows, int M_stride, float eps, uint8_t* a8, float* asc,
                   float* h, int ldh, hipStream_t s) {
  const int passes = (K + 2047) / 2048;
  const dim3 grid(rows, M_stride < 256 ? passes : 1);  // (few rows: the GPU would be nearly idle)
#define QM_F8N(P) fp8_rmsnorm_kernel<T, VEC, P><<<grid, 256, 0, s>>>(x, ldx, w, K, M, M_stride, eps, a8, asc, h, ldh)
  if (passes <= 1) QM_F8N(1);
  else if (passes <= 2) QM_F8N(2);
  else if (passes <= 4) QM_F8N(4);
  else if (passes <= 8) QM_F8N(8);
  else QM_F8N(0);
#undef QM_F8N
  return hipGetLastError();
}

// A launch for as many rows as a grid holds, of `groups` work-groups each: f(first row, rows)
template <typename F>
hipError_t by_grids(int M_stride, int groups, F f) {
  const int most = (int)(kMostThreads / 256 / groups);
  for (int m0 = 0;; m0 += most) {
    const int rows = M_stride - m0 < most ? M_stride - m0 : most;
    const hipError_t e = f(m0, rows);
    if (e != hipSuccess || m0 + rows == M_stride) return e;
  }
}

template <typename T>
hipError_t norm_any(const T* x, int ldx, const float* w, int K, int M, int M_stride, float eps, uint8_t* a8, float* asc,
                    float* h, int ldh, hipStream_t s) {
  const size_t kp = ((size_t)K + 127) / 128 * 128;
  const bool vec = rows_aligned(x, ldx, K, sizeof(T)) && (uintptr_t)w % 16 == 0;
  return by_grids(M_stride, 1, [&](int m0, int rows) {
    const T* xr = x + (size_t)m0 * ldx;
    float* hr = h ? h + (size_t)m0 * ldh : nullptr;
    return vec ? norm_of<T, true>(xr, ldx, w, K, M - m0, rows, M_stride, eps, a8 + m0 * kp, asc + m0, hr, ldh, s)
               : norm_of<T, false>(xr, ldx, w, K, M - m0, rows, M_stride, eps, a8 + m0 * kp, asc + m0, hr, ldh, s);
  });
}

hipError_t rows_any(const void* x, int xtype, int ldx, int K, int M, int M_stride, int op, uint8_t* a8, float* asc,
                    hipStream_t s) {
  const size_t kp = ((size_t)K + 127) / 128 * 128;
  return by_grids(M_stride, (K + 2047) / 2048, [&](int m0, int rows) {
    const size_t at = (size_t)m0 * ldx;
    uint8_t* qr = a8 + m0 * kp;
    float* sr = asc + m0;
    if (xtype == DT_F32) return rows_of((const float*)x + at, ldx, K, M - m0, rows, M_stride, op, qr, sr, s);
    if (xtype == DT_F16) return rows_of((const _Float16*)x + at, ldx, K, M - m0, rows, M_stride, op, qr, sr, s);
    return rows_of((const __bf16*)x + at, ldx, K, M - m0, rows, M_stride, op, qr, sr, s);
  });
}

}  // namespace

hipError_t launch_quantize_fp8(const void* x, int xtype, int ldx, int M, int M_stride, int K, uint8_t* a8, float* asc,
                               hipStream_t s) {
  return rows_any(x, xtype, ldx, K, M, M_stride, ROWS, a8, asc, s);
}

hipError_t launch_swiglu_fp8(const void* gu, int xtype, int ldg, int F, int M, int M_stride, int gelu, uint8_t* a8,
                             float* asc, hipStream_t s) {
  return rows_any(gu, xtype, ldg, F, M, M_stride, gelu ? GELU : SILU, a8, asc, s);
}

hipError_t launch_rmsnorm_fp8(const void* x, int xtype, int ldx, const float* w, int K, int M, int M_stride, float eps,
                              uint8_t* a8, float* asc, float* h, int ldh, hipStream_t s) {
  if (xtype == DT_F32) return norm_any((const float*)x, ldx, w, K, M, M_stride, eps, a8, asc, h, ldh, s);
  if (xtype == DT_F16) return norm_any((const _Float16*)x, ldx, w, K, M, M_stride, eps, a8, asc, h, ldh, s);
  return norm_any((const __bf16*)x, ldx, w, K, M, M_stride, eps, a8, asc, h, ldh, s);
}

}  // namespace qm
