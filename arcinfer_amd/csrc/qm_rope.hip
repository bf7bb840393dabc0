// RMS norm of each query and key head and the rotation by the token's position, in one pass over the heads. HBM-bound:
// each element is read once and written once.
//
// A head is D / (2 V) chunks of two vectors of V elements: chunk c of the first rot / (2 V) is V whole pairs (vectors at V c
// and rot/2 + V c, or, with adjacent pairs, 2 V c and 2 V c + V), the rest pass (two neighbouring vectors). A pair never
// crosses a lane: a group of L lanes holds one head, the mean square is a reduction over them.
// The cosines and sines of a token are computed once for all its heads, into LDS.
#include "qm_fp8.h"

namespace qm {

namespace {

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

}  // namespace

// U: chunks of a lane (1 but for V = 1). tokens: of a work-group. lanes: of a head.
template <typename TI, typename TO, int V, int U>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a, int tokens, int lanes) {
  __shared__ float2 table[kTable];
  const int half = a.rot >> 1, t0 = blockIdx.x * tokens, nt = min(tokens, a.T - t0);
  for (int e = threadIdx.x; e < nt * half; e += 256) {
    const int t = e / half, i = e - t * half;
    // the product of a 31-bit position and a 24-bit frequency is (nearly) exact in f64, and so is what is left of whole turns
    const double turns = (double)a.pos[(size_t)axis_of(a, i) * a.pos_stride + t0 + t] * (double)a.inv_freq[i] * 0.15915494309189535;
    float sn, cs;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    table[e] = make_float2(cs * a.scale, sn * a.scale);
  }
  __syncthreads();
  const int H = a.HQ + a.HK, group = threadIdx.x / lanes, sub = threadIdx.x & (lanes - 1), groups = 256 / lanes;
  const int chunks = a.D / (2 * V), turned = half / V;
  const int units = nt * H, step = groups * gridDim.y;
  for (int u0 = blockIdx.y * groups; u0 < units; u0 += step) {
    const int u = u0 + group;
    const bool live = u < units;
    const int t = live ? u / H : 0, hh = live ? u - t * H : 0;
    const bool is_q = hh < a.HQ;
    const int h = is_q ? hh : hh - a.HQ;
    const float* w = is_q ? a.wq : a.wk;
    const TI* x = (const TI*)a.x + (size_t)(t0 + t) * a.ldx + (is_q ? a.q_off + (size_t)h * a.q_hs : a.k_off + (size_t)h * a.k_hs);
    TO* y = is_q ? (TO*)a.q + (size_t)(t0 + t) * a.ldq + (size_t)h * a.D : (TO*)a.k + (size_t)(t0 + t) * a.ldk + (size_t)h * a.D;
    float v[U][2 * V];
    int lo[U], hi[U];
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < U; ++c) {
      const int k = sub + c * lanes;
      const bool on = live && k < chunks;
      lo[c] = k < turned && !a.adjacent ? V * k : 2 * V * k;
      hi[c] = k < turned && !a.adjacent ? half + V * k : 2 * V * k + V;
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) v[c][i] = 0.0f;
      if (on) {
        loadv<TI, V>(x + lo[c], v[c]);
        loadv<TI, V>(x + hi[c], v[c] + V);
      }
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) ss = fmaf(v[c][i], v[c][i], ss);
    }
    float n = 1.0f;
    if (w) {  // (one head's lanes take the same way; the reduction stays within them)
      for (int o = lanes >> 1; o; o >>= 1) ss += __shfl_xor(ss, o);
      n = 1.0f / sqrtf(ss / (float)a.D + a.eps);
    }
#pragma unroll
    for (int c = 0; c < U; ++c) {
      const int k = sub + c * lanes;
      if (!live || k >= chunks) continue;
      if (w) {
        float wv[2 * V];
        loadv<float, V>(w + lo[c], wv);
        loadv<float, V>(w + hi[c], wv + V);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) v[c][i] = v[c][i] * n * wv[i];
      }
      float r[2 * V];
      if (k < turned) {
        const float2* cs = table + t * half + V * k;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int p = a.adjacent ? 2 * i : i, q = a.adjacent ? 2 * i + 1 : V + i;
          r[p] = v[c][p] * cs[i].x - v[c][q] * cs[i].y;
          r[q] = v[c][q] * cs[i].x + v[c][p] * cs[i].y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) r[i] = v[c][i];
      }
      storev<TO, V>(y + lo[c], r);
      storev<TO, V>(y + hi[c], r + V);
    }
  }
}

namespace {

template <typename TI, typename TO>
hipError_t rope_of(const RopeArgs& a, hipStream_t s) {
  // four elements at a time where the pairs' vectors and every row, offset and stride allow it
  const uintptr_t vi = 4 * sizeof(TI), vo = 4 * sizeof(TO);
  bool vec = a.D % 8 == 0 && a.rot % 8 == 0 && (uintptr_t)a.x % vi == 0 && a.ldx % 4 == 0;
  if (a.HQ) vec = vec && a.q_off % 4 == 0 && a.q_hs % 4 == 0 && a.ldq % 4 == 0 && (uintptr_t)a.q % vo == 0 && (uintptr_t)a.wq % 16 == 0;
  if (a.HK) vec = vec && a.k_off % 4 == 0 && a.k_hs % 4 == 0 && a.ldk % 4 == 0 && (uintptr_t)a.k % vo == 0 && (uintptr_t)a.wk % 16 == 0;
  const int chunks = a.D / (vec ? 8 : 2), half = a.rot / 2 > 0 ? a.rot / 2 : 1;
  int lanes = 1;
  while (lanes < chunks && lanes < 64) lanes *= 2;
  int tokens = kTable / half < 4 ? kTable / half : 4;
  if (a.T < 1024) tokens = 1;
  const unsigned gx = (unsigned)((a.T + tokens - 1) / tokens);
  const unsigned iters = (unsigned)((tokens * (a.HQ + a.HK) * lanes + 255) / 256);
  unsigned gy = gx >= 512 ? 1 : (512 + gx - 1) / gx;  // few tokens: their heads over several work-groups
  if (gy > iters) gy = iters;
  if (vec) qk_norm_rope_kernel<TI, TO, 4, 1><<<dim3(gx, gy), 256, 0, s>>>(a, tokens, lanes);
  else if (chunks <= 64) qk_norm_rope_kernel<TI, TO, 1, 1><<<dim3(gx, gy), 256, 0, s>>>(a, tokens, lanes);
  else qk_norm_rope_kernel<TI, TO, 1, 4><<<dim3(gx, gy), 256, 0, s>>>(a, tokens, lanes);
  return hipGetLastError();
}

template <typename TI>
hipError_t rope_to(const RopeArgs& a, hipStream_t s) {
  if (a.otype == DT_F32) return rope_of<TI, float>(a, s);
  if (a.otype == DT_F16) return rope_of<TI, _Float16>(a, s);
  return rope_of<TI, __bf16>(a, s);
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeArgs& a, hipStream_t s) {
  if (a.xtype == DT_F32) return rope_to<float>(a, s);
  if (a.xtype == DT_F16) return rope_to<_Float16>(a, s);
  return rope_to<__bf16>(a, s);
}

}  // namespace qm
