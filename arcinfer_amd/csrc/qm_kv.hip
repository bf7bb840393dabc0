// Appending to a paged cache of keys and values: RMS norm of each query and key head and its rotation by the token's position, as
// qm_rope.hip does it, with the keys and values going to their tokens' places in the cache on the way. HBM-bound: each element
// is read once and written once.
//
// A group of lanes holds a head (see qm_rope.hip for its chunks), so the largest value of a head, which an 8-bit cache scales by, is a
// reduction over the group like the mean square. Values are heads that are neither normed nor turned.
#include "qm_kv.h"
#include "qm_rope_dev.h"

namespace qm {

namespace {

constexpr float kTop = 448.0f;      // the largest e4m3 value
constexpr float kTiny = 0x1p-100f;  // heads below it are zeros: 448 / amax stays finite and amax / 448 normal

// V values as e4m3, in V bytes
template <int V>
__device__ __forceinline__ void store8(uint8_t* p, const float* v) {
  if constexpr (V == 1) {
    *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[0], 0, false);
  } else {
    int w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], w[i], true);
    }
    if constexpr (V == 8) *(int2*)p = make_int2(w[0], w[1]);
    else *(int*)p = w[0];
  }
}

}  // namespace

// One head of one token, as the lanes of a group hold it: U chunks of 2 V elements a lane
template <typename TI, int V, int U>
struct CacheHead {
  typedef TI vt __attribute__((ext_vector_type(V)));
  vt x0[U], x1[U];
  const float* w;
  int t, h, slot, kind;  // the token, from the work-group's first on; the head of its kind: 0 query, 1 key, 2 value
  bool live;

  __device__ __forceinline__ static int lo_at(const RopeArgs& a, int k, int turned) { return k < turned && !a.adjacent ? V * k : 2 * V * k; }
  __device__ __forceinline__ static int hi_at(const RopeArgs& a, int k, int turned) {
    return k < turned && !a.adjacent ? (a.rot >> 1) + V * k : 2 * V * k + V;
  }

  __device__ __forceinline__ void load(const AppendArgs& a, int u, int units, int t0, int sub, int lanes, int chunks, int turned) {
    const RopeArgs& r = a.r;
    const int H = r.HQ + 2 * r.HK;
    live = u < units;
    t = live ? u / H : 0;
    h = live ? u - t * H : 0;
    kind = h < r.HQ ? 0 : h < r.HQ + r.HK ? 1 : 2;
    h -= kind == 0 ? 0 : kind == 1 ? r.HQ : r.HQ + r.HK;
    const size_t row = (size_t)(t0 + t);
    w = kind == 0 ? r.wq : kind == 1 ? r.wk : nullptr;
    slot = live && kind ? a.slots[row] : -1;
    const size_t off = kind == 0 ? r.q_off + (size_t)h * r.q_hs : kind == 1 ? r.k_off + (size_t)h * r.k_hs : a.v_off + (size_t)h * a.v_hs;
    const TI* x = (const TI*)r.x + row * r.ldx + off;
    if (kind == 2) turned = 0;
#pragma unroll
    for (int c = 0; c < U; ++c) {
      const int k = sub + c * lanes;
      x0[c] = x1[c] = vt(0);
      if (live && k < chunks) {
        x0[c] = *(const vt*)(x + lo_at(r, k, turned));
        x1[c] = *(const vt*)(x + hi_at(r, k, turned));
      }
    }
  }

  __device__ __forceinline__ void finish(const AppendArgs& a, const float2* table, int t0, int sub, int lanes, int chunks, int turned) {
    const RopeArgs& r = a.r;
    if (kind == 2) turned = 0;
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
      n = 1.0f / sqrtf(ss / (float)r.D + r.eps);
    }
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < U; ++c) {
      const int k = sub + c * lanes;
      const bool in = k < chunks;
      const int lo = lo_at(r, k, turned), hi = hi_at(r, k, turned);
      if (w && in) {
        float wv[2 * V];
        loadv<float, V>(w + lo, wv);
        loadv<float, V>(w + hi, wv + V);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) v[c][i] = v[c][i] * n * wv[i];
      }
      if (live && k < turned) {
        const float2* cs = table + t * (r.rot >> 1) + V * k;
        float y[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // (both ways are written out: the pairing is the launch's, an index of it would put v into memory)
          const float e = r.adjacent ? v[c][2 * i] : v[c][i], f = r.adjacent ? v[c][2 * i + 1] : v[c][V + i];
          const float y0 = e * cs[i].x - f * cs[i].y, y1 = f * cs[i].x + e * cs[i].y;
          y[i] = y0;
          y[V + i] = y1;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[c][2 * i] = r.adjacent ? y[i] : y[2 * i];
          v[c][2 * i + 1] = r.adjacent ? y[V + i] : y[2 * i + 1];
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) amax = fmaxf(amax, fabsf(v[c][i]));
    }
    if (kind == 0) {
      if (!live) return;
      const size_t at = (size_t)(t0 + t) * r.ldq + (size_t)h * r.D;
      if (r.otype == DT_F32) put<float>((float*)r.q + at, v, r, sub, lanes, chunks, turned);
      else if (r.otype == DT_F16) put<_Float16>((_Float16*)r.q + at, v, r, sub, lanes, chunks, turned);
      else put<__bf16>((__bf16*)r.q + at, v, r, sub, lanes, chunks, turned);
      return;
    }
    const KvView& kv = a.kv;
    if (kv.type == DT_E4M3)
      for (int o = lanes >> 1; o; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
    if (slot < 0 || slot >> kv.lg >= kv.pages) return;  // (a token without a place, or with one that there is not)
    const int page = slot >> kv.lg, i = slot & (kv.page - 1);
    const size_t at = (size_t)(page * kv.ps + h * kv.hs + i * kv.ts);
    void* base = kind == 1 ? kv.k : kv.v;
    if (kv.type == DT_F16) {
      put<_Float16>((_Float16*)base + at, v, r, sub, lanes, chunks, turned);
    } else if (kv.type == DT_BF16) {
      put<__bf16>((__bf16*)base + at, v, r, sub, lanes, chunks, turned);
    } else {
      const float inv = amax >= kTiny ? kTop / amax : 0.0f;
      uint8_t* y = (uint8_t*)base + at;
#pragma unroll
      for (int c = 0; c < U; ++c) {
        const int k = sub + c * lanes;
        if (k >= chunks) continue;
#pragma unroll
        for (int j = 0; j < 2 * V; ++j) v[c][j] *= inv;
        store8<V>(y + lo_at(r, k, turned), v[c]);
        store8<V>(y + hi_at(r, k, turned), v[c] + V);
      }
      if (sub == 0) (kind == 1 ? kv.ksc : kv.vsc)[((size_t)page * kv.HK + h) * kv.page + i] = amax >= kTiny ? amax / kTop : 0.0f;
    }
  }

  template <typename TO>
  __device__ __forceinline__ static void put(TO* y, const float (*v)[2 * V], const RopeArgs& r, int sub, int lanes, int chunks, int turned) {
#pragma unroll
    for (int c = 0; c < U; ++c) {
      const int k = sub + c * lanes;
      if (k >= chunks) continue;
      storev<TO, V>(y + lo_at(r, k, turned), v[c]);
      storev<TO, V>(y + hi_at(r, k, turned), v[c] + V);
    }
  }
};

// tokens: of a work-group. lanes: of a head. A group of lanes holds two batches of B heads: one is on its way while the other is
// finished, and the first while the table is computed.
template <typename TI, int V, int U, int B>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a, int tokens, int lanes) {
  __shared__ float2 table[kTable];
  const RopeArgs& r = a.r;
  const int half = r.rot >> 1, t0 = blockIdx.x * tokens, nt = min(tokens, r.T - t0);
  const int group = threadIdx.x / lanes, sub = threadIdx.x & (lanes - 1), groups = 256 / lanes;
  const int chunks = r.D / (2 * V), turned = half / V;
  const int units = nt * (r.HQ + 2 * r.HK), step = groups * (int)gridDim.y;
  CacheHead<TI, V, U> now[B], next[B];
  int u = (int)blockIdx.y * groups;
#pragma unroll
  for (int i = 0; i < B; ++i) now[i].load(a, u + i * step + group, units, t0, sub, lanes, chunks, turned);
  for (int e = threadIdx.x; e < nt * half; e += 256) {
    const int t = e / half, i = e - t * half;
    // the product of a 31-bit position and a 24-bit frequency is (nearly) exact in f64, and so is what is left of whole turns
    const double turns = (double)r.pos[(size_t)axis_of(r, i) * r.pos_stride + t0 + t] * (double)r.inv_freq[i] * 0.15915494309189535;
    float sn, cs;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
    table[e] = make_float2(cs * r.scale, sn * r.scale);
  }
  __syncthreads();
  while (u < units) {
    u += B * step;
    if (u < units) {
#pragma unroll
      for (int i = 0; i < B; ++i) next[i].load(a, u + i * step + group, units, t0, sub, lanes, chunks, turned);
    }
#pragma unroll
    for (int i = 0; i < B; ++i) now[i].finish(a, table, t0, sub, lanes, chunks, turned);
    if (u < units) {
#pragma unroll
      for (int i = 0; i < B; ++i) now[i] = next[i];
    }
  }
}

// The mean key of each page that a token of the call completes (its last place), from the keys as the cache holds them: a second
// launch, since a page's other tokens may be other work-groups'. A work-group looks at 64 tokens for one head: 256 / (D / 8) rows at
// a time, 8 elements a lane, the rows' sums joined in one order.
constexpr int kMeanTokens = 64;
template <typename TC>
__global__ __launch_bounds__(256) void page_mean_kernel(AppendArgs a) {
  __shared__ float red[256 * 8];
  const KvView& kv = a.kv;
  const int h = blockIdx.y, lanes = kv.D / 8, rows = 256 / lanes, d = (int)threadIdx.x % lanes, row = (int)threadIdx.x / lanes;
  const long long t = (long long)blockIdx.x * kMeanTokens + (threadIdx.x & 63);
  const int mine = t < a.r.T ? a.slots[t] : -1;  // (each wave sees all of them)
  unsigned long long full = __ballot(mine >= 0 && mine >> kv.lg < kv.pages && (mine & (kv.page - 1)) == kv.page - 1);
  for (; full; full &= full - 1) {
    const int page = __builtin_amdgcn_readlane(mine, __ffsll(full) - 1) >> kv.lg;
    float sum[8] = {};
    if (row < rows)
      for (int i = row; i < kv.page; i += rows) {
        const TC* p = (const TC*)kv.k + (page * kv.ps + h * kv.hs + i * kv.ts) + 8 * d;
        if constexpr (sizeof(TC) == 1) {
          const int2 w = *(const int2*)p;
          const float s = kv.ksc[((size_t)page * kv.HK + h) * kv.page + i];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(j < 2 ? w.x : w.y, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(j < 2 ? w.x : w.y, true);
            sum[2 * j] = fmaf(j & 1 ? hi[0] : lo[0], s, sum[2 * j]);
            sum[2 * j + 1] = fmaf(j & 1 ? hi[1] : lo[1], s, sum[2 * j + 1]);
          }
        } else {
          float v[8];
          loadv<TC, 8>(p, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[j] += v[j];
        }
      }
#pragma unroll
    for (int j = 0; j < 8; ++j) red[j * 256 + threadIdx.x] = sum[j];
    __syncthreads();
    for (int c = threadIdx.x; c < kv.D; c += 256) {
      float s = 0.0f;
      for (int i = 0; i < rows; ++i) s += red[(c & 7) * 256 + i * lanes + (c >> 3)];
      ((__bf16*)kv.mean)[((size_t)page * kv.HK + h) * kv.D + c] = (__bf16)(s / (float)kv.page);
    }
    __syncthreads();
  }
}

namespace {

template <typename TI>
hipError_t append_of(const AppendArgs& a, hipStream_t s) {
  const RopeArgs& r = a.r;
  // V elements at a time where the pairs' vectors and every row, offset and stride allow it (a cache's always do)
  const auto fits = [&](int v) {
    const uintptr_t vi = v * sizeof(TI) < 16 ? v * sizeof(TI) : 16, so = r.otype == DT_F32 ? 4 : 2, vo = v * so < 16 ? v * so : 16;
    bool ok = r.rot % (2 * v) == 0 && (uintptr_t)r.x % vi == 0 && r.ldx % v == 0;
    if (r.HQ) ok = ok && r.q_off % v == 0 && r.q_hs % v == 0 && r.ldq % v == 0 && (uintptr_t)r.q % vo == 0 && (uintptr_t)r.wq % 16 == 0;
    return ok && r.k_off % v == 0 && r.k_hs % v == 0 && a.v_off % v == 0 && a.v_hs % v == 0 && (uintptr_t)r.wk % 16 == 0;
  };
  const int v = sizeof(TI) == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
  const int chunks = r.D / (2 * v), half = r.rot / 2 > 0 ? r.rot / 2 : 1, H = r.HQ + 2 * r.HK;
  int lanes = 1;
  while (lanes < chunks && lanes < 64) lanes *= 2;
  int tokens = kTable / half < 4 ? kTable / half : 4;
  if (r.T < 1024) tokens = 1;
  const unsigned gx = (unsigned)((r.T + tokens - 1) / tokens);
  const unsigned iters = (unsigned)(((long long)tokens * H * lanes + 255) / 256);
  unsigned gy = gx >= 1024 ? 1 : (1024 + gx - 1) / gx;  // few tokens: their heads over several work-groups
  if (gy > iters) gy = iters;
  const dim3 grid(gx, gy);
  if (v == 8) {
    if constexpr (sizeof(TI) == 2) kv_append_kernel<TI, 8, 1, 2><<<grid, 256, 0, s>>>(a, tokens, lanes);
  } else if (v == 4) {
    kv_append_kernel<TI, 4, 1, 2><<<grid, 256, 0, s>>>(a, tokens, lanes);
  } else {
    kv_append_kernel<TI, 1, 2, 1><<<grid, 256, 0, s>>>(a, tokens, lanes);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append(const AppendArgs& a, hipStream_t s) {
  const hipError_t e = a.r.xtype == DT_F32 ? append_of<float>(a, s) : a.r.xtype == DT_F16 ? append_of<_Float16>(a, s) : append_of<__bf16>(a, s);
  if (e != hipSuccess || !a.kv.mean) return e;
  const dim3 grid((unsigned)((a.r.T + kMeanTokens - 1) / kMeanTokens), (unsigned)a.kv.HK);
  if (a.kv.type == DT_F16) page_mean_kernel<_Float16><<<grid, 256, 0, s>>>(a);
  else if (a.kv.type == DT_BF16) page_mean_kernel<__bf16><<<grid, 256, 0, s>>>(a);
  else page_mean_kernel<uint8_t><<<grid, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace qm
