// RMS norm of each query and key head and the rotation by the token's position, in one pass over the heads. HBM-bound:
// each element is read once and written once.
//
// A head is D / (2 V) chunks of two vectors of V elements: chunk c of the first rot / (2 V) is V whole pairs (vectors at V c
// and rot/2 + V c, or, with adjacent pairs, 2 V c and 2 V c + V), the rest pass (two neighbouring vectors). A pair never
// crosses a lane: a group of L lanes holds one head, the mean square is a reduction over them.
// The cosines and sines of a token are computed once for all its heads, into LDS.
#include "qm_rope_dev.h"

namespace qm {

// One head of one token, as the lanes of a group hold it: U chunks of 2 V elements a lane
template <typename TI, typename TO, int V, int U>
struct Head {
  typedef TI vt __attribute__((ext_vector_type(V)));
  vt x0[U], x1[U];  // (as loaded: a head on its way costs half the registers that its f32 values would)
  const float* w;
  TO* y;
  int t;  // the token, from the work-group's first on
  bool live;

  __device__ __forceinline__ static int lo_at(const RopeArgs& a, int k, int turned) { return k < turned && !a.adjacent ? V * k : 2 * V * k; }
  __device__ __forceinline__ static int hi_at(const RopeArgs& a, int k, int turned) {
    return k < turned && !a.adjacent ? (a.rot >> 1) + V * k : 2 * V * k + V;
  }

  __device__ __forceinline__ void load(const RopeArgs& a, int u, int units, int t0, int sub, int lanes, int chunks, int turned) {
    const int H = a.HQ + a.HK;
    live = u < units;
    t = live ? u / H : 0;
    const int hh = live ? u - t * H : 0, h = hh < a.HQ ? hh : hh - a.HQ;
    const bool is_q = hh < a.HQ;
    const size_t row = (size_t)(t0 + t);
    w = is_q ? a.wq : a.wk;
    const TI* x = (const TI*)a.x + row * a.ldx + (is_q ? a.q_off + (size_t)h * a.q_hs : a.k_off + (size_t)h * a.k_hs);
    y = (is_q ? (TO*)a.q + row * a.ldq : (TO*)a.k + row * a.ldk) + (size_t)h * a.D;
#pragma unroll
    for (int c = 0; c < U; ++c) {
      const int k = sub + c * lanes;
      x0[c] = x1[c] = vt(0);
      if (live && k < chunks) {
        x0[c] = *(const vt*)(x + lo_at(a, k, turned));
        x1[c] = *(const vt*)(x + hi_at(a, k, turned));
      }
    }
  }

  __device__ __forceinline__ void finish(const RopeArgs& a, const float2* table, int sub, int lanes, int chunks, int turned) {
    float v[U][2 * V];
#pragma unroll
    for (int c = 0; c < U; ++c)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[c][i] = (float)x0[c][i];
        v[c][V + i] = (float)x1[c][i];
      }
    float n = 1.0f;
    if (w) {  // (one head's lanes take the same way; the reduction stays within them)
      float ss = 0.0f;
#pragma unroll
      for (int c = 0; c < U; ++c)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) ss = fmaf(v[c][i], v[c][i], ss);
      for (int o = lanes >> 1; o; o >>= 1) ss += __shfl_xor(ss, o);
      n = 1.0f / sqrtf(ss / (float)a.D + a.eps);
    }
#pragma unroll
    for (int c = 0; c < U; ++c) {
      const int k = sub + c * lanes;
      if (!live || k >= chunks) continue;
      const int lo = lo_at(a, k, turned), hi = hi_at(a, k, turned);
      if (w) {
        float wv[2 * V];
        loadv<float, V>(w + lo, wv);
        loadv<float, V>(w + hi, wv + V);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) v[c][i] = v[c][i] * n * wv[i];
      }
      float r[2 * V];
      if (k < turned) {
        const float2* cs = table + t * (a.rot >> 1) + V * k;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // (both ways are written out: the pairing is the launch's, an index of it would put v into memory)
          const float e = a.adjacent ? v[c][2 * i] : v[c][i], f = a.adjacent ? v[c][2 * i + 1] : v[c][V + i];
          const float y0 = e * cs[i].x - f * cs[i].y, y1 = f * cs[i].x + e * cs[i].y;
          r[i] = y0;
          r[V + i] = y1;
        }
        if (a.adjacent) {
          float z[2 * V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            z[2 * i] = r[i];
            z[2 * i + 1] = r[V + i];
          }
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) r[i] = z[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) r[i] = v[c][i];
      }
      storev<TO, V>(y + lo, r);
      storev<TO, V>(y + hi, r + V);
    }
  }
};

// tokens: of a work-group. lanes: of a head. A group of lanes holds two batches of B heads: one is on its way while the other is
// finished, and the first while the table is computed.
template <typename TI, typename TO, int V, int U, int B>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a, int tokens, int lanes) {
  __shared__ float2 table[kTable];
  const int half = a.rot >> 1, t0 = blockIdx.x * tokens, nt = min(tokens, a.T - t0);
  const int group = threadIdx.x / lanes, sub = threadIdx.x & (lanes - 1), groups = 256 / lanes;
  const int chunks = a.D / (2 * V), turned = half / V;
  const int units = nt * (a.HQ + a.HK), step = groups * (int)gridDim.y;
  Head<TI, TO, V, U> now[B], next[B];
  int u = (int)blockIdx.y * groups;
#pragma unroll
  for (int i = 0; i < B; ++i) now[i].load(a, u + i * step + group, units, t0, sub, lanes, chunks, turned);
  for (int e = threadIdx.x; e < nt * half; e += 256) {
    const int t = e / half, i = e - t * half;
    // the product of a 31-bit position and a 24-bit frequency is (nearly) exact in f64, and so is what is left of whole turns
    const double turns = (double)a.pos[(size_t)axis_of(a, i) * a.pos_stride + t0 + t] * (double)a.inv_freq[i] * 0.15915494309189535;
    float sn, cs;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    table[e] = make_float2(cs * a.scale, sn * a.scale);
  }
  __syncthreads();
  while (u < units) {
    u += B * step;
    if (u < units) {
#pragma unroll
      for (int i = 0; i < B; ++i) next[i].load(a, u + i * step + group, units, t0, sub, lanes, chunks, turned);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) now[i].finish(a, table, sub, lanes, chunks, turned);
    if (u < units) {
#pragma unroll
      for (int i = 0; i < B; ++i) now[i] = next[i];
    }
  }
}

namespace {

// eight at a time where both sides are of 16 bits (16 bytes a load and store)
template <typename TI, typename TO>
constexpr bool kRopeV8 = sizeof(TI) == 2 && sizeof(TO) == 2;

template <typename TI, typename TO>
hipError_t rope_of(const RopeArgs& a, hipStream_t s) {
  // V elements at a time where the pairs' vectors and every row, offset and stride allow it
  const auto fits = [&](int v) {
    const uintptr_t vi = v * sizeof(TI) < 16 ? v * sizeof(TI) : 16, vo = v * sizeof(TO) < 16 ? v * sizeof(TO) : 16;
    bool ok = a.D % (2 * v) == 0 && a.rot % (2 * v) == 0 && (uintptr_t)a.x % vi == 0 && a.ldx % v == 0;
    if (a.HQ) ok = ok && a.q_off % v == 0 && a.q_hs % v == 0 && a.ldq % v == 0 && (uintptr_t)a.q % vo == 0 && (uintptr_t)a.wq % 16 == 0;
    if (a.HK) ok = ok && a.k_off % v == 0 && a.k_hs % v == 0 && a.ldk % v == 0 && (uintptr_t)a.k % vo == 0 && (uintptr_t)a.wk % 16 == 0;
    return ok;
  };
  const int v = kRopeV8<TI, TO> && fits(8) ? 8 : fits(4) ? 4 : 1;
  const int chunks = a.D / (2 * v), half = a.rot / 2 > 0 ? a.rot / 2 : 1;
  int lanes = 1;
  while (lanes < chunks && lanes < 64) lanes *= 2;
  int tokens = kTable / half < 4 ? kTable / half : 4;
  if (a.T < 1024) tokens = 1;
  const unsigned gx = (unsigned)((a.T + tokens - 1) / tokens);
  const unsigned iters = (unsigned)((tokens * (a.HQ + a.HK) * lanes + 255) / 256);
  unsigned gy = gx >= 1024 ? 1 : (1024 + gx - 1) / gx;  // few tokens: their heads over several work-groups
  if (gy > iters) gy = iters;
  const dim3 grid(gx, gy);
  if (v == 8) {
    if constexpr (kRopeV8<TI, TO>) qk_norm_rope_kernel<TI, TO, 8, 1, 2><<<grid, 256, 0, s>>>(a, tokens, lanes);
  } else if (v == 4) {
    qk_norm_rope_kernel<TI, TO, 4, 1, 2><<<grid, 256, 0, s>>>(a, tokens, lanes);
  } else if (chunks <= 64) {
    qk_norm_rope_kernel<TI, TO, 1, 1, 1><<<grid, 256, 0, s>>>(a, tokens, lanes);
  } else {
    qk_norm_rope_kernel<TI, TO, 1, 4, 1><<<grid, 256, 0, s>>>(a, tokens, lanes);
  }
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
  // a launch for as many tokens as a grid holds for certain
  constexpr int kMost = (int)(kMostThreads / 256);
  const size_t si = a.xtype == DT_F32 ? 4 : 2, so = a.otype == DT_F32 ? 4 : 2;
  RopeArgs b = a;
  for (int t0 = 0;; t0 += kMost) {
    b.T = a.T - t0 < kMost ? a.T - t0 : kMost;
    const hipError_t e = a.xtype == DT_F32 ? rope_to<float>(b, s) : a.xtype == DT_F16 ? rope_to<_Float16>(b, s) : rope_to<__bf16>(b, s);
    if (e != hipSuccess || t0 + b.T == a.T) return e;
    b.x = (const char*)b.x + kMost * si * (size_t)a.ldx;
    if (b.q) b.q = (char*)b.q + kMost * so * (size_t)a.ldq;
    if (b.k) b.k = (char*)b.k + kMost * so * (size_t)a.ldk;
    if (b.pos) b.pos += kMost;
  }
}

}  // namespace qm
