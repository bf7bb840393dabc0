// Device-side building blocks of the e4m3 products (qm_fp8.hip, qm_fp8_tile.hip).
#pragma once
#include "qm_fp8.h"

namespace qm {

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

// Eight neighbouring results, rounded to T, as one store of 16 bytes
template <typename T>
__device__ __forceinline__ void put8_whole(T* C, v4f lo, v4f hi) {
  typedef T v8t __attribute__((ext_vector_type(8)));
  v8t r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (T)(i < 4 ? lo[i & 3] : hi[i & 3]);
  *(v8t*)C = r;
}

// Eight neighbouring results of token m from n on (n % 8 == 0), 16 bytes of C at a time where vec
template <typename T>
__device__ __forceinline__ void put8(T* C, size_t at, v4f lo, v4f hi, int left, int accumulate, bool vec) {
  typedef T v8t __attribute__((ext_vector_type(8)));
  if (vec && left >= 8) {
    if (accumulate) {
      const v8t o = *(const v8t*)(C + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = (float)o[i];
        const float f = i < 4 ? lo[i & 3] : hi[i & 3], v = accumulate == 1 ? f + c : c / (1.0f + expf(-c)) * f;
        if (i < 4) lo[i & 3] = v;
        else hi[i & 3] = v;
      }
    }
    put8_whole(C + at, lo, hi);
    return;
  }
  put4(C, at, lo, left, accumulate, false);
  put4(C, at + 4, hi, left - 4, accumulate, false);
}
__device__ __forceinline__ void store8(const Fp8GemmArgs& a, int m, int n, v4f lo, v4f hi, bool vec) {
  const size_t at = (size_t)m * a.ldc + a.c_off + n;
  const int left = a.w.rows - n;
  if (a.ctype == DT_F32) put8((float*)a.C, at, lo, hi, left, a.accumulate, vec);
  else if (a.ctype == DT_F16) put8((_Float16*)a.C, at, lo, hi, left, a.accumulate, vec);
  else put8((__bf16*)a.C, at, lo, hi, left, a.accumulate, vec);
}
// whether every group of eight results lies on 16 bytes
__device__ __forceinline__ bool vec_stores8(const Fp8GemmArgs& a) {
  const int bits = a.ctype == DT_F32 ? 2 : 1;
  const uintptr_t at = (uintptr_t)a.C | (uintptr_t)a.ldc << bits | (uintptr_t)a.c_off << bits;
  return (at & (a.ctype == DT_F32 ? 31 : 15)) == 0;
}

// whether every group of four results lies on its own alignment
__device__ __forceinline__ bool vec_stores(const Fp8GemmArgs& a) {
  const uintptr_t size = a.ctype == DT_F32 ? 4 : 2;
  return ((((uintptr_t)a.C / size) | (uintptr_t)a.ldc | (uintptr_t)a.c_off) & 3) == 0;
}

}  // namespace qm
