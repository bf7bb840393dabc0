// The choice of pages for attention over a part of a cache: each token's query heads of a key head score the pages of its sequence
// against the pages' mean keys, score = max over the heads of q . mean, and the k best are taken (ties to the lower page).
//
// Scores are sums in f64: the products of 16-bit values are exact there and so, but for the last bits of sums over very different
// magnitudes, are the sums, whatever their order. Which page is the k-th best is then a property of the inputs and not of the kernel.
#include "qm_attn_plan.h"
#include "qm_rope_dev.h"

namespace qm {

namespace {

constexpr int kHeads = 8;  // query heads at a time

// Pages that row t of q sees (0: it is of no sequence, or sees nothing)
__device__ __forceinline__ int pages_seen(const SelectArgs& a, int t, int& b) {
  b = sequence_of(a.s, t);
  if (b < 0) return 0;
  const int at = a.s.len[b] - (row_from(a.s, b) + rows_of(a.s, b) - t);  // the token's place
  return at < 0 ? 0 : min((at >> a.kv.lg) + 1, a.s.W);
}

__device__ __forceinline__ unsigned long long ordered(double s) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, s + 0.0);  // (one zero)
  return u >> 63 ? ~u : u | 1ull << 63;
}

}  // namespace

// A thread a page, 256 pages a work-group; the query heads in LDS
template <typename TQ>
__global__ __launch_bounds__(256) void page_score_kernel(SelectArgs a, int chunks) {
  __shared__ double q[kHeads * 256];
  const int item = blockIdx.x / chunks, h = item % a.kv.HK, t = item / a.kv.HK, D = a.kv.D;
  const int j = (int)(blockIdx.x % chunks) * 256 + (int)threadIdx.x;
  int b;
  const int n = pages_seen(a, t, b);
  if (n <= a.k || j - (int)threadIdx.x >= n) return;
  const int page = j < n ? a.s.table[(size_t)b * a.s.W + j] : -1;
  const bool there = (unsigned)page < (unsigned)a.kv.pages;
  const __bf16* m = (const __bf16*)a.kv.mean + ((size_t)(there ? page : 0) * a.kv.HK + h) * D;
  double best = -__builtin_inf();
  for (int g0 = 0; g0 < a.G; g0 += kHeads) {
    const int heads = min(kHeads, a.G - g0);
    __syncthreads();
    for (int i = threadIdx.x; i < kHeads * D; i += 256) {
      const int g = i / D, d = i - g * D;
      q[i] = g < heads ? (double)(float)((const TQ*)a.q)[(size_t)t * a.ldq + (size_t)(h * a.G + g0 + g) * D + d] : 0.0;
    }
    __syncthreads();
    double s[kHeads] = {};
    for (int d = 0; d < D; d += 8) {
      float v[8];
      loadv<__bf16, 8>(m + d, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double x = (double)v[i];
#pragma unroll
        for (int g = 0; g < kHeads; ++g) s[g] = fma(q[g * D + d + i], x, s[g]);
      }
    }
#pragma unroll
    for (int g = 0; g < kHeads; ++g)
      if (g < heads) best = fmax(best, s[g]);  // (a NaN is passed over)
  }
  if (j < n) a.scores[(size_t)item * a.s.W + j] = there ? best : -__builtin_inf();
}

// A work-group a token and key head: the k-th largest score eight bits at a time, then the pages above it in their order
__global__ __launch_bounds__(256) void page_pick_kernel(SelectArgs a) {
  __shared__ int hist[256], part[4], pick[3];
  const int item = blockIdx.x, t = item / a.kv.HK, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int b;
  const int n = pages_seen(a, t, b);
  if (b < 0) return;  // (a row of no sequence: left as it is)
  int32_t* sel = a.sel + (size_t)item * a.k;
  if (n <= a.k) {
    for (int i = tid; i < a.k; i += 256) sel[i] = i < n ? i : -1;
    return;
  }
  const double* s = a.scores + (size_t)item * a.s.W;
  const int lo = a.first, hi = n - a.last;
  int need = a.k - a.first - a.last;  // of the pages lo .. hi - 1
  for (int i = tid; i < a.first; i += 256) sel[i] = i;
  for (int i = tid; i < a.last; i += 256) sel[a.k - a.last + i] = hi + i;
  if (need == 0) return;
  unsigned long long known = 0, mask = 0;
  for (int shift = 56; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += 256) {
      const unsigned long long u = ordered(s[j]);
      if ((u & mask) == known) atomicAdd(&hist[(u >> shift) & 255], 1);
    }
    __syncthreads();
    // how many lie in digits above this thread's (digit 255 - tid), and in it
    const int mine = hist[255 - tid];
    int up = mine;
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(up, o);
      if (lane >= o) up += v;
    }
    if (lane == 63) part[wave] = up;
    __syncthreads();
    for (int w = 0; w < wave; ++w) up += part[w];
    if (up >= need && up - mine < need) {
      pick[0] = 255 - tid;
      pick[1] = need - (up - mine);
      pick[2] = mine;
    }
    __syncthreads();
    known |= (unsigned long long)pick[0] << shift;
    mask |= 255ull << shift;
    need = pick[1];
    if (pick[2] == need) break;  // (all that share these bits are taken)
    __syncthreads();
  }
  // those above, and of those that share the bits the first `need`
  int out = a.first, equal = 0;
  for (int j0 = lo; j0 < hi; j0 += 256) {
    const int j = j0 + tid;
    const unsigned long long u = j < hi ? ordered(s[j]) & mask : 0;
    const bool gt = j < hi && u > known, eq = j < hi && u == known;
    const unsigned long long below = (1ull << lane) - 1, e = __ballot(eq);
    __syncthreads();
    if (lane == 0) part[wave] = __popcll(e);
    __syncthreads();
    int before = equal + __popcll(e & below);
    for (int w = 0; w < wave; ++w) before += part[w];
    equal += part[0] + part[1] + part[2] + part[3];
    const bool take = gt || (eq && before < need);
    const unsigned long long k = __ballot(take);
    __syncthreads();
    if (lane == 0) part[wave] = __popcll(k);
    __syncthreads();
    int at = out + __popcll(k & below);
    for (int w = 0; w < wave; ++w) at += part[w];
    if (take) sel[at] = j;
    out += part[0] + part[1] + part[2] + part[3];
  }
}

hipError_t launch_select(const SelectArgs& a, hipStream_t s) {
  const unsigned items = (unsigned)(a.s.T * a.kv.HK), chunks = (unsigned)((a.s.W + 255) / 256);
  if (a.s.W > a.k) {
    if (a.qtype == DT_F16) page_score_kernel<_Float16><<<items * chunks, 256, 0, s>>>(a, (int)chunks);
    else page_score_kernel<__bf16><<<items * chunks, 256, 0, s>>>(a, (int)chunks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  page_pick_kernel<<<items, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace qm
