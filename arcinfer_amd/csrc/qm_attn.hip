// Attention over a paged cache: how a call is cut into pieces, its launches, and the kernel that joins the pieces.
#include "qm_attn_plan.h"

namespace qm {

hipError_t attn_bf16(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);
hipError_t attn_f16(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);
hipError_t attn_bf16_e4m3(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);
hipError_t attn_f16_e4m3(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);
hipError_t attn_tile_bf16(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);
hipError_t attn_tile_f16(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);
hipError_t attn_tile_bf16_e4m3(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);
hipError_t attn_tile_f16_e4m3(const AttnArgs& a, int mt, unsigned grid, hipStream_t s);

// Joins the pieces of one row: o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p. A work-group a row (a query head of a token): D / 4 lanes of four
// elements, the pieces dealt to 1024 / D groups of lanes, whose sums are joined in their order. Every partial result is read once; rows
// of a single piece are left as attn_kernel wrote them. What a row needs to know of the split stands in its tile's first slot.
// Latency-bound: a launch, that slot's words, then the pieces' maxima and sums and kAhead results of each group at once.
constexpr int kAhead = 8;
__device__ __forceinline__ void store4(const AttnArgs& a, size_t to, const float (&y)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (a.otype == DT_F32) ((float*)a.o)[to + i] = y[i];
    else if (a.otype == DT_F16) ((_Float16*)a.o)[to + i] = (_Float16)y[i];
    else ((__bf16*)a.o)[to + i] = (__bf16)y[i];
  }
}
template <int THREADS>
__global__ __launch_bounds__(THREADS) void attn_join_kernel(AttnArgs a, int RT, int chosen) {
  constexpr int kWavesHere = THREADS / 64;
  __shared__ float wave_max[kWavesHere], weight[THREADS], wsum[kWavesHere];
  __shared__ float4 osum[THREADS];
  const int hq = blockIdx.x % a.HQ, t = blockIdx.x / a.HQ, h = hq / a.G, g = hq % a.G, D = a.kv.D, tid = threadIdx.x;
  const int b = sequence_of(a.s, t);
  if (b < 0) return;
  const int row0 = chosen ? t : row_from(a.s, b), r0 = (t - row0) * a.G + g, rt = r0 / RT;
  const long long n0 = (long long)(chosen ? t * ((a.G + RT - 1) / RT) + rt : first_slot(a, RT, b, row0, rt)) * a.kv.HK + h;
  if (n0 >= a.slots) return;
  const size_t size = slot_floats(RT, D);
  const float* first = a.part + (size_t)n0 * size;
  int4 head = *(const int4*)first;
  // (lists that are no batch leave slots unwritten: their words may be anything, and stay within the slots)
  head = {min(max(head.x, 1), a.slots), max(head.y, 0), max(head.z, 0), 0};
  const long long srow = (long long)t * a.G + g;
  // the partial result of piece p: of its row, the maximum; the sum lies a tile's rows behind it, the elements from two on. (The prefix's pieces and the
  // first one are known without the slot's words.)
  const int srt = a.shared_rt;
  const size_t ssize = slot_floats(srt, D);
  const float* sfirst = a.shared_part + (size_t)(h * a.shared_tiles + srow / srt) * a.shared * ssize + 4;
  const auto slot = [&](int p) -> const float* {
    if (p < a.shared) return sfirst + (size_t)p * ssize;
    if (p == a.shared) return first + 4;
    const long long n = ((long long)head.y + (long long)(p - a.shared - 1) * head.z) * a.kv.HK + h;
    return (n < a.slots ? a.part + (size_t)n * size : first) + 4;
  };
  const auto row_of = [&](int p) { return p < a.shared ? (int)(srow % srt) : r0 % RT; };
  const auto tile_of = [&](int p) { return p < a.shared ? srt : RT; };
  const int lanes = D / 4, groups = THREADS / lanes, group = tid / lanes, d = 4 * (tid % lanes);
  float l = 0.0f, top = -__builtin_inff();
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  int all = a.shared + 1;
  if (!a.shared) {
    if (head.x == 1) return;  // (attn_kernel wrote the result)
    all = head.x;
  }
  for (int p0 = 0; p0 < all;) {
    // up to THREADS pieces at a time: their maxima and sums, and the first results of each group, are asked for together
    const int n = min(THREADS, all - p0);
    float4 v[kAhead];
    const auto ask = [&](int i, int from) {
      const int p = p0 + min(group + (from + i) * groups, n - 1);
      v[i] = *(const float4*)(slot(p) + 2 * tile_of(p) + (size_t)row_of(p) * D + d);
    };
    const bool in = tid < n;
    const float* s = slot(p0 + (in ? tid : 0)) + row_of(p0 + (in ? tid : 0));
    const float m = s[0], w = in ? s[tile_of(p0 + tid)] : 0.0f;
    if (group < groups) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i * groups < n) ask(i, 0);
    }
    all = a.shared + head.x;
    // (a piece that the row sees nothing of has the sum 0)
    float most = w != 0.0f ? m : -__builtin_inff();
    for (int k = 32; k; k >>= 1) most = fmaxf(most, __shfl_xor(most, k));
    __syncthreads();
    if ((tid & 63) == 0) wave_max[tid >> 6] = most;
    __syncthreads();
    most = top;
#pragma unroll
    for (int i = 0; i < kWavesHere; ++i) most = fmaxf(most, wave_max[i]);
    if (most != top) {
      const float f = __builtin_amdgcn_exp2f(top - most);
      l *= f;
      o.x *= f;
      o.y *= f;
      o.z *= f;
      o.w *= f;
      top = most;
    }
    const float f = w != 0.0f ? __builtin_amdgcn_exp2f(m - top) : 0.0f;
    weight[tid] = w != 0.0f ? f : -1.0f;  // (a weight that vanishes counts: its result may not be finite)
    if (w != 0.0f) l = fmaf(f, w, l);
    __syncthreads();
    if (group < groups) {
      for (int from = 0; group + from * groups < n; from += kAhead) {
        if (from) {
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
            if ((from + i) * groups < n) ask(i, from);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int p = group + (from + i) * groups;
          if (p >= n) continue;
          const float k = weight[p];
          if (k < 0.0f) continue;  // (nothing seen: the slot may hold anything)
          o.x = fmaf(k, v[i].x, o.x);
          o.y = fmaf(k, v[i].y, o.y);
          o.z = fmaf(k, v[i].z, o.z);
          o.w = fmaf(k, v[i].w, o.w);
        }
      }
    }
    p0 += n;
  }
  for (int k = 32; k; k >>= 1) l += __shfl_xor(l, k);
  osum[tid] = o;
  if ((tid & 63) == 0) wsum[tid >> 6] = l;
  __syncthreads();
  if (group) return;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < kWavesHere; ++i) l += wsum[i];
  for (int i = 1; i < groups; ++i) {
    const float4 v = osum[i * lanes + tid];
    o.x += v.x;
    o.y += v.y;
    o.z += v.z;
    o.w += v.w;
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // (a row that sees no key is zeros)
  const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  store4(a, (size_t)t * a.ldo + (size_t)hq * D + d, y);
}

// Joins the pieces of the row tiles that were cut behind the last whole round: 16 rows a work-group, D / 4 lanes of four elements a row. Pieces are
// few (2 to 32): their maxima first, then results and sums.
constexpr int kTailRows = 16;
__global__ __launch_bounds__(256) void attn_tail_join_kernel(AttnArgs a, int RT) {
  const int chunks = RT / kTailRows, j = blockIdx.x / chunks, D = a.kv.D;
  const Tail t = tail_of(a, RT);
  Item it;
  if (j >= t.tail || !find_item(a, RT, t.whole + j, it)) return;
  const int row0 = row_from(a.s, it.b), rows = rows_of(a.s, it.b), blocks = tile_blocks(a, RT, it.b, it.rt, rows);
  const int size = part_blocks(blocks, t.parts), pieces = (blocks + size - 1) / size;
  if (pieces <= 1) return;  // (attn_tile_kernel wrote the result)
  const int lanes = D / 4, per = 256 / lanes, d = 4 * (threadIdx.x % lanes), from = blockIdx.x % chunks * kTailRows;
  if ((int)threadIdx.x / lanes >= per) return;
  const size_t floats = slot_floats(RT, D);
  for (int r = from + threadIdx.x / lanes; r < from + kTailRows; r += per) {
    const int row = it.rt * RT + r;
    if (row >= rows * a.G) return;
    const float* s = a.part + (size_t)j * floats + 4 + r;
    const size_t step = (size_t)t.tail * floats;
    float top = -__builtin_inff();
    for (int p = 0; p < pieces; ++p)
      if (s[p * step + RT] != 0.0f) top = fmaxf(top, s[p * step]);  // (a piece that the row sees nothing of has the sum 0)
    float l = 0.0f;
    float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < pieces; ++p) {
      const float w = s[p * step + RT];
      if (w == 0.0f) continue;
      const float f = __builtin_amdgcn_exp2f(s[p * step] - top);
      const float4 v = *(const float4*)(s + p * step - r + 2 * RT + (size_t)r * D + d);
      l = fmaf(f, w, l);
      o.x = fmaf(f, v.x, o.x);
      o.y = fmaf(f, v.y, o.y);
      o.z = fmaf(f, v.z, o.z);
      o.w = fmaf(f, v.w, o.w);
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    const size_t to = (size_t)(row0 + row / a.G) * a.ldo + (size_t)(it.h * a.G + row % a.G) * D + d;
    store4(a, to, y);
  }
}

namespace {

// Pieces that a call is cut into: two work-groups a CU. attn_kernel's may be as many more as there are row tiles; attn_tile_kernel's, which take longer to
// start and end, are kept to one round (12 sequences of 580 to 17200 tokens, 24 heads of 256 over 4: 64 us against 77; attn_kernel 74 against 71).
constexpr int kTarget = 512;  // (attn_tile_kernel's 64 us: 80 by 256 pieces, 78 by 1024)
// Pieces of the shared prefix: one work-group a CU beside the sequences' own keys (48 sequences behind 8192 tokens 46 us, 16 behind 65000 60; 128 pieces
// 59 and 96; 512 51 and 59). In a launch of its own as many as any call's (768 rows behind 16384: 92 us, 105 by 256 pieces).
constexpr int kSharedTarget = 256;
// Bytes of a prefix, read once more for each further sequence, from which it is read once for all: below, the pieces' join takes longer than that.
// 8 heads of 128, bf16, 500 tokens of their own, us: 8 sequences x 256 tokens 16.9 against 14.7, x 1024 17.3 against 16.9; 48 x 256 27.8 against 32.0,
// x 1024 32 against 48; 2 x 1024 15.2 against 13.6.
constexpr double kSharedBytes = 3.2e7;
constexpr int kTailMost = 2;        // rounds of work-groups from which the last one is not cut (6656 tokens, 3.3 rounds: 362 us cut, 359 not)
constexpr int kSharedRows = 64;     // rows of the batch from which attn_tile_kernel may take a prefix
// Products of a prefix (rows of all heads times keys times D) from which it does, in a launch of its own: below, attn_kernel's tiles in the
// sequences' own launch take less. 8 heads of 128, rows of a head x keys, us: 192 x 2048 31 against 21, 192 x 16384 47 against 44, 384 x 16384
// 63 against 85, 768 x 16384 92 against 158; D 256, 384 x 8192: 67 against 99. Behind 8-bit caches 192 x 16384 53 against 46, 512 x 16384 79 against 92.
constexpr double kSharedFrom16 = 4e9, kSharedFrom8 = 6e9;

long long div_up(long long a, long long b) { return (a + b - 1) / b; }
// Rows of attn_kernel's tile: what its registers hold
int few_rows(long long rows, int D) {
  const int most = D <= 64 ? 64 : D <= 128 ? 32 : 16, want = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  return want < most ? want : most;
}
// Rows of a sequence from which attn_tile_kernel takes them. 16 sequences of 4096 tokens, us: D 128, 8 heads: 48 rows 57 against 65, 20 rows 51.3
// against 52.3 (but of 1000 tokens 18 against 16.7); D 256, 4 heads: 18 rows 53 against 64, 12 rows 51 against 53. Behind 8-bit caches, which
// it widens on the way: D 128: 128 rows 72 against 77, 64 rows 56 against 54; D 256: 36 rows 52 against 65, 18 rows 49 against 44.
int tile_from(int D, bool e8) { return e8 ? (D > 128 ? 33 : 65) : (D > 128 ? 17 : 33); }
// Of its tile: 64 where that is all there is (64 rows of one sequence of 16384 tokens: 26.6 us against 30.5; 80 rows of 16 of 4096: 72 against 65), or all
// that the registers hold
int many_rows(long long rows, int D, bool e8) { return D <= 128 && (rows > 64 || e8) ? 128 : 64; }
// Row tiles of all sequences at most
long long row_tiles(int T, int B, bool start, int G, int rt) {
  return start ? (long long)T * G / rt + B : B * div_up(G, rt);  // (as first_slot counts them)
}

}  // namespace

static size_t slot_bytes(int rt, int D) { return (4 + (size_t)rt * (D + 2)) * sizeof(float); }
static size_t shared_bytes(const AttnPlan& p, int HK, int D) { return p.shared ? (size_t)HK * p.shared_tiles * p.shared * slot_bytes(p.shared_rt, D) : 0; }
static unsigned shared_grid(const AttnPlan& p, int HK) { return (unsigned)(div_up((long long)HK * p.shared, 8) * 8 * p.shared_tiles); }

size_t attn_used_bytes(const AttnPlan& p, int HK, int D) { return shared_bytes(p, HK, D) + p.slots * slot_bytes(p.rt, D); }

AttnPlan attn_plan(int T, int B, bool start, bool few, bool e8, int HQ, int HK, int D, int prefix_len, size_t ws_bytes) {
  const int G = HQ / HK;
  const long long rows = start ? div_up(T, B < T ? B : T) * G : G;  // of a sequence, on average
  const size_t have = ws_bytes / 256 * 256;
  AttnPlan p{};
  p.tile = !few && rows >= tile_from(D, e8);
  p.rt = p.tile ? many_rows(rows, D, e8) : few_rows(rows, D);
  const AttnPlan alone = p;
  if ((double)(B - 1) * prefix_len * HK * D * (e8 ? 2 : 4) >= kSharedBytes && T > 1 && rows < kSharedRows) {
    const long long all = (long long)T * G;
    p.shared_tile = !few && all >= kSharedRows && (double)T * HQ * prefix_len * D >= (e8 ? kSharedFrom8 : kSharedFrom16);
    p.shared_rt = p.shared_tile ? many_rows(all, D, e8) : few_rows(all, D);
    // (one launch for both: the batch's rows fill the tile, and a sequence's own keys take no longer for it)
    if (!p.shared_tile) {
      p.tile = 0;
      p.rt = p.shared_rt;
    }
    p.shared_tiles = (int)div_up((long long)T * G, p.shared_rt);
    const int blocks = (int)div_up(prefix_len, 128);
    long long n = (p.shared_tile ? kTarget : kSharedTarget) / ((long long)HK * p.shared_tiles);
    if (n > blocks) n = blocks;
    if (n < 1) n = 1;
    p.shared_blocks = (int)div_up(blocks, n);
    p.shared = (int)div_up(blocks, p.shared_blocks);
    if (shared_bytes(p, HK, D) + row_tiles(T, B, start, G, p.rt) * HK * slot_bytes(p.rt, D) > have) p = alone;
  }
  const long long items = row_tiles(T, B, start, G, p.rt) * HK;
  const long long left = ((long long)have - (long long)shared_bytes(p, HK, D)) / (long long)slot_bytes(p.rt, D) - items;
  // (pieces of all row tiles are at most the target and one more for each of them; more row tiles than fill the chip are left whole. Lengths are not looked at for that, and are not known
  // here: 43 sequences of 500 to 20000 tokens, five rows each, 24 heads of 256 over 4, take 228 us, 44 of them 443.)
  if (left > 0 && items < (p.tile ? kTarget / 2 : 2 * kTarget)) {
    // (beside a prefix's work-groups half as many: 32 sequences of 300 tokens behind 4096 24 us against 31, 4 of 4000 behind 16384 31 against 36; 48 of 16 to 1500
    // behind 8192 47 against 46)
    const long long want = p.tile ? kTarget - items : p.shared && !p.shared_tile ? kTarget / 2 : kTarget;
    p.target = (int)(left < want ? left : want);
  }
  p.slots = p.target || p.shared ? (int)(items + p.target) : 0;
  if (p.tile && !p.slots && items < kTailMost * kTarget && kTarget * slot_bytes(p.rt, D) <= have) p.slots = p.tail = kTarget;
  p.firsts = (int)(items / HK);
  return p;
}

size_t attn_workspace_bytes(int T, int B, bool e8, int HQ, int HK, int D, int prefix_len) {
  size_t most = 0;
  for (int mode = 0; mode < 3; ++mode) {  // a row a sequence, rows of the caller's, chosen pages
    const size_t n = attn_used_bytes(attn_plan(T, mode == 2 ? T : B, mode == 1, mode == 2, e8, HQ, HK, D, mode == 2 ? 0 : prefix_len, (size_t)1 << 60), HK, D);
    if (n > most) most = n;
  }
  return (most + 255) / 256 * 256;
}

long long attn_grid(const AttnPlan& p, int T, int B, bool start, int HQ, int HK) {
  const long long own = p.slots && !p.tail ? p.slots : row_tiles(T, B, start, HQ / HK, p.rt) * HK + p.tail;
  const long long grid = own + (p.shared ? shared_grid(p, HK) : 0), join = p.slots ? (long long)T * HQ : 0;
  const long long most = grid > join ? grid : join;
  return most * 256 <= kMostThreads ? most : 0;
}

namespace {

hipError_t attn_any(const AttnArgs& a, int rt, int tile, unsigned grid, hipStream_t s) {
  if (tile) {
    const int mt = rt / 64;
    if (a.kv.type == DT_E4M3) return a.qtype == DT_F16 ? attn_tile_f16_e4m3(a, mt, grid, s) : attn_tile_bf16_e4m3(a, mt, grid, s);
    return a.qtype == DT_F16 ? attn_tile_f16(a, mt, grid, s) : attn_tile_bf16(a, mt, grid, s);
  }
  const int mt = rt / 16;
  if (a.kv.type == DT_E4M3) return a.qtype == DT_F16 ? attn_f16_e4m3(a, mt, grid, s) : attn_bf16_e4m3(a, mt, grid, s);
  return a.qtype == DT_F16 ? attn_f16(a, mt, grid, s) : attn_bf16(a, mt, grid, s);
}

}  // namespace

hipError_t launch_attn(const AttnArgs& args, const AttnPlan& p, hipStream_t s) {
  AttnArgs a = args;
  a.target = p.target;
  a.slots = p.slots;
  a.firsts = p.firsts;
  a.shared_grid = a.shared = 0;
  a.shared_rt = p.rt;
  int tile = p.tile;
  a.tail = p.tail;
  long long grid = p.slots && !p.tail ? p.slots : row_tiles(a.s.T, a.s.B, a.s.start != nullptr, a.G, p.rt) * a.kv.HK + p.tail;
  if (a.sel) {  // as many pieces for every token: the target's, within the slots
    const long long items = (long long)a.s.T * div_up(a.G, p.rt) * a.kv.HK, blocks = div_up((long long)a.k * a.kv.page, 128);
    long long n = p.slots / items;
    if (n > blocks) n = blocks;
    if (n < 1) n = 1;
    a.blocks = (int)div_up(blocks, n);
    a.pieces = (int)div_up(blocks, a.blocks);
    grid = items * a.pieces;
    if (a.pieces == 1) a.slots = 0;
  } else if (p.shared) {
    a.shared_grid = (int)shared_grid(p, a.kv.HK);
    a.shared = p.shared;
    a.shared_rt = p.shared_rt;
    a.shared_tiles = p.shared_tiles;
    a.shared_blocks = p.shared_blocks;
    a.shared_part = a.part;
    a.part += shared_bytes(p, a.kv.HK, a.kv.D) / sizeof(float);
    if (p.shared_tile) {
      const hipError_t e = attn_any(a, p.shared_rt, 1, (unsigned)a.shared_grid, s);
      if (e != hipSuccess) return e;
      a.shared_grid = 0;
    } else {
      grid += a.shared_grid;
    }
  }
  const hipError_t e = attn_any(a, p.rt, tile, (unsigned)grid, s);
  if (e != hipSuccess || !a.slots) return e;
  if (a.tail) {
    attn_tail_join_kernel<<<(unsigned)(a.tail / 2 * (p.rt / kTailRows)), 256, 0, s>>>(a, p.rt);
    return hipGetLastError();
  }
  // A wave a row where there are rows enough: work-groups of four waves, most of which have nothing to do, take longer to start than that (1536 rows:
  // the call 57 us against 60). Sixteen waves where there are few rows, and so many pieces of each (24 rows of 40 pieces of D 256: 17.3 us
  // against 17.9; 512 rows of 32: 67 against 59).
  const long long rows = (long long)a.s.T * a.HQ;
  if (rows >= 1024) attn_join_kernel<64><<<(unsigned)rows, 64, 0, s>>>(a, p.rt, a.sel ? 1 : 0);
  else if (rows >= 128) attn_join_kernel<256><<<(unsigned)rows, 256, 0, s>>>(a, p.rt, a.sel ? 1 : 0);
  else attn_join_kernel<1024><<<(unsigned)rows, 1024, 0, s>>>(a, p.rt, a.sel ? 1 : 0);
  return hipGetLastError();
}

}  // namespace qm
