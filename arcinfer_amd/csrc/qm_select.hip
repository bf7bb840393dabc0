// The choice of pages for attention over a part of a cache: each token's query heads of a key head score the pages of its sequence
// against the pages' mean keys, score = max over the heads of q . mean, and the k best are taken (ties to the lower page).
//
// Scores are sums in f64: the products of 16-bit values are exact there and so, but for the last bits of sums over very different
// magnitudes, are the sums, whatever their order. Which page is the k-th best is then a property of the inputs and not of the kernel.
#include "qm_attn_plan.h"
#include "qm_rope_dev.h"

namespace qm {

namespace {

// Pages that row t of q sees (0: it is of no sequence, or sees nothing)
__device__ __forceinline__ int pages_seen(const SelectArgs& a, int t, int& b) {
  b = sequence_of(a.s, t);
  if (b < 0) return 0;
  const int at = length_of(a.s, b) - (row_from(a.s, b) + rows_of(a.s, b) - t);  // the token's place
  return at < 0 ? 0 : min((at >> a.kv.lg) + 1, a.s.W);
}

__device__ __forceinline__ unsigned long long ordered(double s) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, s + 0.0);  // (one zero)
  return u >> 63 ? ~u : u | 1ull << 63;
}

}  // namespace

typedef double v4d __attribute__((ext_vector_type(4)));

// Scores of the pages of one token and key head, every chunks-th 64 of them a work-group, 16 at a time a wave: a product of 16 pages by 16 query heads on the f64 matrix
// pipe, four elements of the heads at a time. Lane (c, g) holds elements g D / 4 .. of page c and of head c (the sum does not depend on which four
// meet), four of them a load; the next pages' means are asked for before this product. The result's rows, in the order g + 4 i, are
// the pages, its columns the heads. Few pages: latency-bound; many: bound by the pipe, 64 cycles an instruction (16 pages of 128 elements
// 2048 cycles, for 16 heads or for one), about as long as the means take from HBM.
constexpr int kChunks = 16;  // of four elements a lane, at most: D 256

// The largest of 16 neighbouring lanes, in each of them
template <int N>
__device__ __forceinline__ double rotated(double v) {
  const long long u = __builtin_bit_cast(long long, v);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)u, 0x120 + N, 0xF, 0xF, false), hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), 0x120 + N, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (long long)(unsigned)lo | (long long)hi << 32);
}
__device__ __forceinline__ double max16(double v) {
  v = fmax(v, rotated<8>(v));
  v = fmax(v, rotated<4>(v));
  v = fmax(v, rotated<2>(v));
  return fmax(v, rotated<1>(v));
}

template <typename TQ>
__global__ __launch_bounds__(256) void page_score_kernel(SelectArgs a, int chunks) {
  typedef __bf16 v4b __attribute__((ext_vector_type(4)));
  typedef TQ v4q __attribute__((ext_vector_type(4)));
  const int item = blockIdx.x / chunks, h = item % a.kv.HK, t = item / a.kv.HK, D = a.kv.D;
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, first = (int)(blockIdx.x % chunks) * 64 + 16 * (threadIdx.x >> 6), step = 64 * chunks;
  int b;
  const int n = pages_seen(a, t, b);
  if (n <= a.k || first >= n) return;
  const int steps = D / 16;
  const bool qvec = ((uintptr_t)a.q & 7) == 0 && (a.ldq & 3) == 0;
  v4b m[kChunks];
  v4q q[kChunks];
  const auto page_of = [&](int j) { return j < n ? a.s.table[(size_t)b * a.s.W + j] : -1; };
  const auto load_means = [&](int page) {
    const __bf16* p = (const __bf16*)a.kv.mean + ((size_t)((unsigned)page < (unsigned)a.kv.pages ? page : 0) * a.kv.HK + h) * D + g * (D / 4);
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      if (i < steps) m[i] = *(const v4b*)(p + 4 * i);
  };
  const auto load_heads = [&](int g0) {  // (columns behind the last head are the last head)
    const TQ* p = (const TQ*)a.q + (size_t)t * a.ldq + (size_t)(h * a.G + min(g0 + c, a.G - 1)) * D + g * (D / 4);
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      if (i < steps) {
        if (qvec) q[i] = *(const v4q*)(p + 4 * i);
        else q[i] = v4q{p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]};
      }
  };
  int page = page_of(first + c), next = page_of(first + step + c);
  load_heads(0);
  load_means(page);
  for (int j0 = first; j0 < n; j0 += step) {
    const int after = page_of(j0 + 2 * step + c);
    v4d best = -__builtin_inf();
    for (int g0 = 0; g0 < a.G; g0 += 16) {
      if (g0 || (j0 > first && a.G > 16)) load_heads(g0);
      v4d s = 0.0;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        if (i < steps) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)m[i][e], (double)(float)q[i][e], s, 0, 0, 0);
        }
      if (g0 + 16 >= a.G) load_means(next);
#pragma unroll
      for (int i = 0; i < 4; ++i) best[i] = fmax(best[i], max16(fmax(s[i], -__builtin_inf())));  // (a NaN is passed over)
    }
    // lane (i, g) writes page g + 4 i (of a page that is none: minus infinity)
    const double mine = c == 0 ? best[0] : c == 1 ? best[1] : c == 2 ? best[2] : best[3];
    const int row = g + 4 * (c & 3);
    const bool is = (unsigned)__shfl(page, row) < (unsigned)a.kv.pages;
    if (c < 4 && j0 + row < n) a.scores[(size_t)item * a.s.W + j0 + row] = is ? mine : -__builtin_inf();
    page = next;
    next = after;
  }
}

// A work-group a token and key head. The k-th largest score, eleven bits at a time from the first one that the scores differ in (by counts in LDS, whole
// numbers: their order does not matter); as soon as all that share the known bits are taken, it is found. Scores are held in registers (K a
// thread; K = 0: read again each time, for tables beyond 256 kMostKept pages). Latency-bound.
constexpr int kMostKept = 32;
constexpr int kBits = 11, kBins = 1 << kBits;  // of scores that are told apart at a time: 3 times at most for most batches

template <int K>
__global__ __launch_bounds__(256) void page_pick_kernel(SelectArgs a) {
  typedef unsigned long long u64;
  constexpr int N = K ? K : 1;
  __shared__ int hist[kBins], before[4], found[3];
  __shared__ int counts[N][4];  // (K > 0) of each round and wave
  __shared__ u64 bits[2][4];
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
  const int need = a.k - a.first - a.last;  // of the pages lo .. hi - 1
  u64 key[N], any = 0, all = ~0ull;
  const auto key_of = [&](int j) { return j < hi ? ordered(s[j]) : 0; };  // (0 is below every score's)
  const int rounds = (hi - lo + 255) / 256;
  const auto take_key = [&](int r) {
    const int j = lo + r * 256 + tid;
    const u64 u = key_of(j);
    if constexpr (K > 0) key[r] = u;
    if (j < hi) {
      any |= u;
      all &= u;
    }
  };
  if constexpr (K > 0) {
#pragma unroll
    for (int r = 0; r < K; ++r) take_key(r);
  } else {
    for (int r = 0; r < rounds; ++r) take_key(r);
  }
  for (int i = tid; i < a.first; i += 256) sel[i] = i;
  for (int i = tid; i < a.last; i += 256) sel[a.k - a.last + i] = hi + i;
  if (need == 0) return;
  for (int o = 32; o; o >>= 1) {
    any |= __shfl_xor(any, o);
    all &= __shfl_xor(all, o);
  }
  if (lane == 0) {
    bits[0][wave] = any;
    bits[1][wave] = all;
  }
  __syncthreads();
  any = bits[0][0] | bits[0][1] | bits[0][2] | bits[0][3];
  all = bits[1][0] & bits[1][1] & bits[1][2] & bits[1][3];
  // (all: the bits that every score has, of those above the first one that they differ in)
  const u64 differ = any & ~all;
  // The threshold: kBits at a time, from the first one that they differ in, by how many scores have each value of them
  int top = differ ? 64 - __clzll(differ) : 0;  // bits that are not known yet
  u64 from = top == 64 ? 0 : all >> top << top;
  bool exact = false;  // whether those from `from` on are as many as are needed
  int left = need;     // of those that share the known bits
  while (top > 0 && !exact) {
    const int low = top > kBits ? top - kBits : 0;
    const u64 known = top == 64 ? 0 : ~0ull << top;
#pragma unroll
    for (int i = 0; i < kBins; i += 256) hist[i + tid] = 0;
    __syncthreads();
    const auto count = [&](int r, u64 u) {
      if (lo + r * 256 + tid < hi && (u & known) == from) atomicAdd(&hist[(int)(u >> low) & ((1 << (top - low)) - 1)], 1);
    };
    if constexpr (K > 0) {
#pragma unroll
      for (int r = 0; r < K; ++r)
        if (r < rounds) count(r, key[r]);
    } else {
      for (int r = 0; r < rounds; ++r) count(r, key_of(lo + r * 256 + tid));
    }
    __syncthreads();
    // how many have a larger value of these bits than the last of thread tid's bins (kBins / 256 from the top), or it
    constexpr int B = kBins / 256;
    int bin[B], here = 0;
#pragma unroll
    for (int i = 0; i < B; ++i) here += bin[i] = hist[kBins - 1 - B * tid - i];
    int up = here;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(up, o);
      if (lane >= o) up += v;
    }
    if (lane == 63) before[wave] = up;
    __syncthreads();
    for (int w = 0; w < wave; ++w) up += before[w];
    if (up >= left && up - here < left) {
      int over = up - here;  // larger ones
      bool is = false;
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (!is && over + bin[i] >= left) {
          is = true;
          found[0] = kBins - 1 - B * tid - i;
          found[1] = left - over;
          found[2] = bin[i];
        }
        over += bin[i];
      }
    }
    __syncthreads();
    from |= (u64)found[0] << low;
    left = found[1];
    exact = found[2] == left;
    top = low;
  }
  // Those above `from`, and of those that are equal to it the first that are needed still; in their order
  const u64 below = (1ull << lane) - 1;
  if constexpr (K > 0) {
    // (counts of all rounds at once: two barriers each for those of equals and of those taken)
    const auto ranks = [&](auto is, int (&at)[N]) {
#pragma unroll
      for (int r = 0; r < K; ++r) {
        const u64 m = r < rounds ? __ballot(is(r)) : 0;
        at[r] = __popcll(m & below);
        if (lane == 0) counts[r][wave] = __popcll(m);
      }
      __syncthreads();
      int sum = 0;
#pragma unroll
      for (int r = 0; r < K; ++r) {
        if (r >= rounds) break;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if (w == wave) at[r] += sum;
          sum += counts[r][w];
        }
      }
      __syncthreads();
    };
    const auto in = [&](int r) { return lo + r * 256 + tid < hi; };
    int equal[N], at[N];
    if (!exact) ranks([&](int r) { return in(r) && key[r] == from; }, equal);
    const auto take = [&](int r) { return in(r) && key[r] >= from && (exact || key[r] != from || equal[r] < left); };
    ranks(take, at);
#pragma unroll
    for (int r = 0; r < K; ++r)
      if (r < rounds && take(r)) sel[a.first + at[r]] = lo + r * 256 + tid;
  } else {
    int equal = 0, out = a.first;
    for (int r = 0; r < rounds; ++r) {
      const int j = lo + r * 256 + tid;
      const u64 u = key_of(j);
      bool take = j < hi && u >= from;
      if (!exact) {
        const bool eq = j < hi && u == from;
        const u64 e = __ballot(eq);
        __syncthreads();
        if (lane == 0) before[wave] = __popcll(e);
        __syncthreads();
        int at = equal + __popcll(e & below);
        for (int w = 0; w < wave; ++w) at += before[w];
        equal += before[0] + before[1] + before[2] + before[3];
        take = take && (!eq || at < left);
      }
      const u64 k = __ballot(take);
      __syncthreads();
      if (lane == 0) before[wave] = __popcll(k);
      __syncthreads();
      int at = out + __popcll(k & below);
      for (int w = 0; w < wave; ++w) at += before[w];
      if (take) sel[at] = j;
      out += before[0] + before[1] + before[2] + before[3];
    }
  }
}

// Work-groups of all tokens and key heads, as many as the chip holds (four a CU) and some: each takes its pages in turn, as many as the sequence has (sequences of
// 60000 tokens, 8 heads of 128: 32 of them 44 us, with a work-group for every 64 pages 51; 128 116 against 127; 64 of them with 4 heads of 256 69 against 95)
constexpr int kScoreTarget = 1280;
static int score_chunks(long long items, int W) {
  const long long most = (W + 63) / 64, n = kScoreTarget / items;
  return (int)(n < 1 ? 1 : n < most ? n : most);
}
long long select_grid(int T, int HK, int W) { return (long long)T * HK * score_chunks((long long)T * HK, W); }

hipError_t launch_select(const SelectArgs& a, hipStream_t s) {
  const unsigned items = (unsigned)(a.s.T * a.kv.HK);
  if (a.s.W > a.k) {
    const int chunks = score_chunks(items, a.s.W);
    if (a.qtype == DT_F16) page_score_kernel<_Float16><<<items * chunks, 256, 0, s>>>(a, chunks);
    else page_score_kernel<__bf16><<<items * chunks, 256, 0, s>>>(a, chunks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (a.s.W <= 256 * 8) page_pick_kernel<8><<<items, 256, 0, s>>>(a);
  else if (a.s.W <= 256 * kMostKept) page_pick_kernel<kMostKept><<<items, 256, 0, s>>>(a);
  else page_pick_kernel<0><<<items, 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace qm
