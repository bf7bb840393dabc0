// Device-side building blocks of the head norm + rotation (qm_rope.hip) and of appending to a cache (qm_kv.hip).
#pragma once
#include "qm_fp8.h"

namespace qm {

constexpr int kTable = 1024;  // cosine / sine pairs of a work-group

__device__ __forceinline__ int axis_of(const RopeArgs& a, int i) {
  if (a.axes == 1) return 0;
  if (a.turns) {
    const int x = i % a.axes;
    return i < a.axes * a.sections[x] ? x : 0;
  }
  int x = 0, end = a.sections[0];
  while (i >= end && x < a.axes - 1) end += a.sections[++x];
  return x;
}

template <typename T, int V>
__device__ __forceinline__ void loadv(const T* p, float* v) {
  typedef T vt __attribute__((ext_vector_type(V)));
  const vt t = *(const vt*)p;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (float)t[i];
}
template <typename T, int V>
__device__ __forceinline__ void storev(T* p, const float* v) {
  typedef T vt __attribute__((ext_vector_type(V)));
  vt t;
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = (T)v[i];
  *(vt*)p = t;
}

}  // namespace qm
