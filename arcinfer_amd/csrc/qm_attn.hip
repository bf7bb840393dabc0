// Attention over a paged cache: how a call is cut into pieces, its launches, and the kernel that joins the pieces.
#include "qm_attn_plan.h"

namespace qm {

hipError_t attn_bf16(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);
hipError_t attn_f16(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);
hipError_t attn_bf16_e4m3(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);
hipError_t attn_f16_e4m3(const AttnArgs& a, int mt, int mode, unsigned grid, hipStream_t s);

// Joins the pieces of one row: o = sum_p 2^(m_p - m) o_p / sum_p 2^(m_p - m) l_p, in the order of the pieces, the prefix's first. A
// work-group a row (a query head of a token): D / 4 lanes of four elements, the pieces dealt to 1024 / D groups of lanes. Every
// partial result is read once; rows of a single piece are left as attn_kernel wrote them.
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int RT, int chosen) {
  __shared__ long long red[4];
  __shared__ float wave_max[4], lsum[256];
  __shared__ float4 osum[256];
  const int hq = blockIdx.x % a.HQ, t = blockIdx.x / a.HQ, h = hq / a.G, D = a.kv.D;
  const int b = sequence_of(a.s, t);
  if (b < 0) return;
  const int row0 = row_from(a.s, b), rows = rows_of(a.s, b);
  long long unit, step;  // the slot of this row tile's first piece, and from one piece to the next
  int own, at;           // own pieces, and the row's place in its tile
  if (chosen) {
    const int rts = (a.G + RT - 1) / RT, rt = hq % a.G / RT;
    own = a.pieces;
    at = hq % a.G % RT;
    unit = (long long)t * rts * a.pieces + rt;
    step = rts;
  } else {
    const int blocks = piece_blocks(a, RT, red);
    const int r = (t - row0) * a.G + hq % a.G, rt = r / RT, rts = (rows * a.G + RT - 1) / RT;
    at = r % RT;
    long long before = 0;
    for (int i = threadIdx.x; i < b; i += 256) {
      const int n = (rows_of(a.s, i) * a.G + RT - 1) / RT;
      before += n ? (long long)n * pieces_of(a, i, blocks) : 0;
    }
    unit = sum256(before, red) + rt;
    step = rts;
    // (the keys that the tile's last row sees, as attn_kernel counts them)
    const int last = min(rt * RT + RT, rows * a.G) - 1;
    const long long most = (long long)a.s.W << a.kv.lg;
    const int lim = (int)min((long long)max(a.s.len[b] - rows + last / a.G + 1, 0), min(most, 0x7fffffffLL));
    const int n = (a.prefix_len + kBlock - 1) / kBlock + (int)(((long long)lim + kBlock - 1) / kBlock);
    own = (int)(((n + kWaves - 1) / kWaves + (long long)blocks - 1) / blocks);
    if (own < 1) own = 1;
    if (!a.shared && own == 1) return;
  }
  const int all = a.shared + own;
  const long long srow = (long long)t * a.G + hq % a.G;
  const auto slot = [&](int p, int& rt, int& r) -> const float* {
    if (p < a.shared) {
      rt = a.shared_rt;
      r = (int)(srow % rt);
      return a.shared_part + ((size_t)(h * a.shared_tiles + srow / rt) * a.shared + p) * ((size_t)rt * (D + 2));
    }
    rt = RT;
    r = at;
    const long long i = (unit + (p - a.shared) * step) * a.kv.HK + h;
    return i < a.slots ? a.part + (size_t)i * ((size_t)rt * (D + 2)) : nullptr;
  };
  float top = -__builtin_inff();
  for (int p = threadIdx.x; p < all; p += 256) {
    int rt, r;
    const float* s = slot(p, rt, r);
    // (a piece whose rows saw nothing has the sum 0, whatever its maximum says)
    if (s && s[rt + r] != 0.0f) top = fmaxf(top, s[r]);
  }
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  const int lanes = D / 4, groups = 256 / lanes, group = (int)threadIdx.x / lanes, d = 4 * ((int)threadIdx.x % lanes);
  float l = 0.0f;
  float4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (group < groups)
    for (int p = group; p < all; p += groups) {
      int rt, r;
      const float* s = slot(p, rt, r);
      if (!s || s[rt + r] == 0.0f) continue;
      const float f = __builtin_amdgcn_exp2f(s[r] - top);
      const float4 v = *(const float4*)(s + 2 * rt + (size_t)r * D + d);
      l = fmaf(f, s[rt + r], l);
      o.x = fmaf(f, v.x, o.x);
      o.y = fmaf(f, v.y, o.y);
      o.z = fmaf(f, v.z, o.z);
      o.w = fmaf(f, v.w, o.w);
    }
  lsum[threadIdx.x] = l;
  osum[threadIdx.x] = o;
  __syncthreads();
  if (group) return;
  for (int i = 1; i < groups; ++i) {
    const float4 v = osum[i * lanes + threadIdx.x];
    l += lsum[i * lanes + threadIdx.x];
    o.x += v.x;
    o.y += v.y;
    o.z += v.z;
    o.w += v.w;
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
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

int tiles_for(long long rows, int D) { return rows <= 16 ? 1 : rows <= 32 || D > 128 ? 2 : 4; }
long long div_up(long long a, long long b) { return (a + b - 1) / b; }
// Row tiles of all sequences at most
long long row_tiles(int T, int B, bool start, int G, int rt) {
  return start ? (long long)T * G / rt + (B < T ? B : T) : (B < T ? B : T) * div_up(G, rt);
}

}  // namespace

size_t attn_slot_bytes(int mt, int D) { return (size_t)16 * mt * (D + 2) * sizeof(float); }

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
  a.shared = 0;
  if (a.sel) {  // as many pieces for every token: the target's, within the slots
    const long long items = row_tiles(a.s.T, a.s.T, false, a.G, 16 * p.mt) * a.kv.HK, blocks = div_up((long long)a.k * a.kv.page, 128);
    long long n = p.slots / items;
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
