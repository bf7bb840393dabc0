// Attention over a paged cache: how a call is cut into pieces, its launches, and the kernel that joins the pieces.
#include "qm_attn_plan.h"

namespace qm {

hipError_t attn_bf16(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);
hipError_t attn_f16(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);
hipError_t attn_bf16_e4m3(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);
hipError_t attn_f16_e4m3(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);

// Joins the pieces of one row: o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p, in one pass over them with the running maximum. A
// work-group a row (a query head of a token): D / 4 lanes of four elements, the pieces dealt to 1024 / D groups of lanes, the groups joined
// in their order. Every partial result is read once; rows of a single piece are left as attn_kernel wrote them. What a row needs to
// know of the split stands in its tile's first slot. Latency-bound: a launch, that slot's words, the partial results.
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int RT, int chosen) {
  __shared__ float gmax[256], gsum[256];
  __shared__ float4 osum[256];
  const int hq = blockIdx.x % a.HQ, t = blockIdx.x / a.HQ, h = hq / a.G, g = hq % a.G, D = a.kv.D;
  const int b = sequence_of(a.s, t);
  if (b < 0) return;
  const int row0 = chosen ? t : row_from(a.s, b), r0 = (t - row0) * a.G + g, rt = r0 / RT;
  const long long n0 = (long long)(chosen ? t * ((a.G + RT - 1) / RT) + rt : first_slot(a, RT, b, row0, rt)) * a.kv.HK + h;
  if (n0 >= a.slots) return;
  const size_t size = slot_floats(RT, D);
  const float* first = a.part + (size_t)n0 * size;
  const int4 head = *(const int4*)first;
  if (!a.shared && head.x == 1) return;
  const int all = a.shared + head.x;
  const long long srow = (long long)t * a.G + g;
  const size_t ssize = slot_floats(a.shared_rt, D);
  const int lanes = D / 4, groups = 256 / lanes, group = (int)threadIdx.x / lanes, d = 4 * ((int)threadIdx.x % lanes);
  float top = -__builtin_inff(), l = 0.0f;
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (group < groups) {
#pragma unroll 4
    for (int p = group; p < all; p += groups) {
      const float* s;
      int rows = RT, r = r0 % RT;
      if (p < a.shared) {
        rows = a.shared_rt;
        r = (int)(srow % rows);
        s = a.shared_part + ((size_t)(h * a.shared_tiles + srow / rows) * a.shared + p) * ssize;
      } else if (p == a.shared) {
        s = first;
      } else {
        const long long n = ((long long)head.y + (long long)(p - a.shared - 1) * head.z) * a.kv.HK + h;
        if (n >= a.slots) continue;
        s = a.part + (size_t)n * size;
      }
      s += 4;
      const float m = s[r], w = s[rows + r];
      const float4 v = *(const float4*)(s + 2 * rows + (size_t)r * D + d);
      if (w == 0.0f) continue;  // (a piece that the row sees nothing of)
      const float now = fmaxf(top, m), f0 = top == now ? 1.0f : __builtin_amdgcn_exp2f(top - now), f = __builtin_amdgcn_exp2f(m - now);
      top = now;
      l = fmaf(f, w, l * f0);
      o.x = fmaf(f, v.x, o.x * f0);
      o.y = fmaf(f, v.y, o.y * f0);
      o.z = fmaf(f, v.z, o.z * f0);
      o.w = fmaf(f, v.w, o.w * f0);
    }
  }
  gmax[threadIdx.x] = top;
  gsum[threadIdx.x] = l;
  osum[threadIdx.x] = o;
  __syncthreads();
  if (group) return;
  float most = top;
  for (int i = 1; i < groups; ++i) most = fmaxf(most, gmax[i * lanes + threadIdx.x]);
  l = 0.0f;
  o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < groups; ++i) {
    const int at = i * lanes + threadIdx.x;
    if (gsum[at] == 0.0f) continue;
    const float f = __builtin_amdgcn_exp2f(gmax[at] - most);
    const float4 v = osum[at];
    l = fmaf(f, gsum[at], l);
    o.x = fmaf(f, v.x, o.x);
    o.y = fmaf(f, v.y, o.y);
    o.z = fmaf(f, v.z, o.z);
    o.w = fmaf(f, v.w, o.w);
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // (a row that sees no key is zeros)
  const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  const size_t to = (size_t)t * a.ldo + (size_t)hq * D + d;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (a.otype == DT_F32) ((float*)a.o)[to + i] = y[i];
    else if (a.otype == DT_F16) ((_Float16*)a.o)[to + i] = (_Float16)y[i];
    else ((__bf16*)a.o)[to + i] = (__bf16)y[i];
  }
}

namespace {

constexpr int kTarget = 1024;        // pieces that a call is cut into
constexpr int kSharedTarget = 512;   // pieces of the shared prefix
constexpr int kSharedFrom = 256;     // a shorter prefix is read with each sequence's own keys

// Row tiles of 16 a work-group: what its registers hold
int tiles_for(long long rows, int D) {
  const int most = D <= 64 ? 4 : D <= 128 ? 2 : 1;
  const int want = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  return want < most ? want : most;
}
long long div_up(long long a, long long b) { return (a + b - 1) / b; }
// Row tiles of all sequences at most
long long row_tiles(int T, int B, bool start, int G, int rt) {
  return start ? (long long)T * G / rt + B : B * div_up(G, rt);  // (as first_slot counts them)
}

}  // namespace

size_t attn_slot_bytes(int mt, int D) { return (4 + (size_t)16 * mt * (D + 2)) * sizeof(float); }

AttnPlan attn_plan(int T, int B, bool start, int HQ, int HK, int D, int prefix_len, size_t ws_bytes) {
  AttnPlan p{};
  const int G = HQ / HK;
  const long long rows = start ? div_up(T, B < T ? B : T) * G : G;  // of a sequence, on average
  p.mt = tiles_for(rows, D);
  const long long items = row_tiles(T, B, start, G, 16 * p.mt) * HK;
  const size_t slot = attn_slot_bytes(p.mt, D);
  const size_t have = ws_bytes / 256 * 256;
  if (prefix_len >= kSharedFrom && B > 1 && T > 1 && rows < 64) {
    p.shared_mt = tiles_for((long long)T * G, D);
    p.shared_tiles = (int)div_up((long long)T * G, 16 * p.shared_mt);
    const int blocks = (int)div_up(prefix_len, 128);
    long long n = kSharedTarget / ((long long)HK * p.shared_tiles);
    if (n > blocks) n = blocks;
    if (n < 1) n = 1;
    p.shared_blocks = (int)div_up(blocks, n);
    p.shared = (int)div_up(blocks, p.shared_blocks);
    const size_t need = (size_t)HK * p.shared_tiles * p.shared * attn_slot_bytes(p.shared_mt, D) + items * slot;
    if (need > have) p.shared = 0;
  }
  const size_t left = have - (p.shared ? (size_t)HK * p.shared_tiles * p.shared * attn_slot_bytes(p.shared_mt, D) : 0);
  // (pieces of all row tiles are at most the target and one more for each of them)
  if (items < 2 * kTarget && left / slot > (size_t)items) {
    const long long n = (long long)(left / slot) - items;
    p.target = (int)(n < kTarget ? n : kTarget);
  }
  p.slots = p.target || p.shared ? (int)(items + p.target) : 0;
  p.firsts = (int)(items / HK);
  return p;
}

size_t attn_workspace_bytes(int T, int B, int HQ, int HK, int D, int prefix_len) {
  size_t most = 0;
  for (int start = 0; start < 2; ++start) {
    const AttnPlan p = attn_plan(T, B, start, HQ, HK, D, prefix_len, (size_t)1 << 62);
    size_t n = (size_t)p.slots * attn_slot_bytes(p.mt, D);
    if (p.shared) n += (size_t)HK * p.shared_tiles * p.shared * attn_slot_bytes(p.shared_mt, D);
    if (n > most) most = n;
  }
  return (most + 255) / 256 * 256;
}

long long attn_grid(const AttnPlan& p, int T, int B, bool start, int HQ, int HK) {
  const long long own = p.slots ? p.slots : row_tiles(T, B, start, HQ / HK, 16 * p.mt) * HK;
  const long long shared = p.shared ? div_up((long long)HK * p.shared, 8) * 8 * p.shared_tiles : 0;
  const long long join = p.slots ? (long long)T * HQ : 0;
  const long long most = own > shared ? own > join ? own : join : shared > join ? shared : join;
  return most * 256 <= kMostThreads ? most : 0;
}

namespace {

hipError_t attn_any(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s) {
  if (a.kv.type == DT_E4M3) return a.qtype == DT_F16 ? attn_f16_e4m3(a, mt, mode, grid, s) : attn_bf16_e4m3(a, mt, mode, grid, s);
  return a.qtype == DT_F16 ? attn_f16(a, mt, mode, grid, s) : attn_bf16(a, mt, mode, grid, s);
}

}  // namespace

hipError_t launch_attn(const AttnArgs& args, const AttnPlan& p, hipStream_t s) {
  AttnArgs a = args;
  float* ws = a.part;
  a.target = p.target;
  a.slots = p.slots;
  a.firsts = p.firsts;
  a.shared = 0;
  a.shared_rt = 16;
  if (a.sel) {  // as many pieces for every token: the target's, within the slots
    const long long items = row_tiles(a.s.T, a.s.T, false, a.G, 16 * p.mt) * a.kv.HK, blocks = div_up((long long)a.k * a.kv.page, 128);
    long long n = p.slots / items;  // (as all first pieces, and as many more)
    if (n > blocks) n = blocks;
    if (n < 1) n = 1;
    a.blocks = (int)div_up(blocks, n);
    a.pieces = (int)div_up(blocks, a.blocks);
    hipError_t e = attn_any(a, p.mt, 2, (unsigned)(items * a.pieces), s);
    if (e != hipSuccess || a.pieces == 1) return e;
    attn_join_kernel<<<(unsigned)((long long)a.s.T * a.HQ), 256, 0, s>>>(a, 16 * p.mt, 1);
    return hipGetLastError();
  }
  if (p.shared) {
    a.shared = p.shared;
    a.shared_rt = 16 * p.shared_mt;
    a.shared_tiles = p.shared_tiles;
    a.shared_blocks = p.shared_blocks;
    a.shared_part = ws;
    a.part = ws + (size_t)a.kv.HK * p.shared_tiles * p.shared * (attn_slot_bytes(p.shared_mt, a.kv.D) / sizeof(float));
    const hipError_t e = attn_any(a, p.shared_mt, 1, (unsigned)(div_up((long long)a.kv.HK * p.shared, 8) * 8 * p.shared_tiles), s);
    if (e != hipSuccess) return e;
    a.prefix_len = 0;
  }
  const long long grid = p.slots ? p.slots : row_tiles(a.s.T, a.s.B, a.s.start != nullptr, a.G, 16 * p.mt) * a.kv.HK;
  const hipError_t e = attn_any(a, p.mt, 0, (unsigned)grid, s);
  if (e != hipSuccess || !p.slots) return e;
  attn_join_kernel<<<(unsigned)((long long)a.s.T * a.HQ), 256, 0, s>>>(a, 16 * p.mt, 0);
  return hipGetLastError();
}

}  // namespace qm
