// Host-side launchers of the paged cache of keys and values: appending, attention over it, and the choice of pages. Shapes are
// checked by the C-ABI layer (qm_api.hip) beforehand.
#pragma once
#include "qm_fp8.h"

namespace qm {

enum : int { DT_E4M3 = 256 };

// The cache. Element d of the head h of token i of page p: p * ps + h * hs + i * ts + d, in keys and in values.
struct KvView {
  int type, D, HK, page, lg, pages;  // page = 1 << lg tokens
  long long ps, hs, ts;
  void *k, *v;
  float *ksc, *vsc;  // e4m3: [pages][HK][page]
  uint16_t* mean;    // bf16 [pages][HK][D], or null
};

struct AppendArgs {
  RopeArgs r;  // (q, otype, ldq: the queries' result; k, ldk are not used)
  int v_off, v_hs;
  const int32_t* slots;
  KvView kv;
};
hipError_t launch_kv_append(const AppendArgs& a, hipStream_t s);

// The sequences of a batch: rows start[b] .. start[b + 1] of q (start null: row b), the last of its len[b] tokens
struct Seqs {
  int B, T;
  const int32_t *start, *len, *table;
  int W;  // the table's row stride: pages of a sequence at most
};

struct AttnArgs {
  const void* q;
  int qtype, ldq, HQ, G;
  KvView kv;
  Seqs s;
  const int32_t* prefix;
  int prefix_len;       // keys in front of each sequence's own
  const int32_t* sel;   // pages of each row and key head [T][HK][k] (null: all)
  int k;
  float c;              // scale * log2 e
  void* o;
  int otype, ldo;
  // The split. A piece is a run of blocks of 128 keys of one row tile and head; its partial result goes to the slot of its number.
  float* part;          // null: nothing is split, each row tile writes its result
  int target, slots;    // pieces that are aimed at (0: whole row tiles), and partial results that `part` holds, those of
  int firsts;           // first pieces (of a head) in front
  int pieces, blocks;   // chosen pages: pieces of a row tile, and blocks of 128 keys of one
  int tail;             // work-groups at a time: the row tiles that are left behind the last whole round of them are cut (0: none)
  // The prefix for the rows of the whole batch (shared pieces; 0: it is read with each sequence's own keys), by shared_grid work-groups in front
  // of the launch's others: pieces of shared_blocks blocks of 128 keys for each of shared_tiles tiles of shared_rt rows of a key head; slot
  // (head * shared_tiles + tile) * shared + piece
  float* shared_part;
  int shared_grid, shared, shared_rt, shared_tiles, shared_blocks;
};

// How a call runs: tiles of rt rows (16 to 64: attn_kernel; more, or `tile`: attn_tile_kernel); pieces and blocks as in AttnArgs
struct AttnPlan {
  int rt, tile, target, slots, firsts;                              // target 0: nothing is split,
  int tail;                                                         // or (not 0) the last row tiles alone
  int shared, shared_rt, shared_tile, shared_tiles, shared_blocks;  // shared 0: the prefix is read with each sequence's own keys
};
// few: attn_kernel alone. Chosen pages are a row's own, never many rows; and a scale of zero, which attn_tile_kernel cannot have in front of its masks.
AttnPlan attn_plan(int T, int B, bool start, bool few, bool e8, int HQ, int HK, int D, int prefix_len, size_t ws_bytes);
size_t attn_used_bytes(const AttnPlan& p, int HK, int D);
size_t attn_workspace_bytes(int T, int B, bool e8, int HQ, int HK, int D, int prefix_len);
// Work-groups of the calls's launches at most (0: more than a grid holds)
long long attn_grid(const AttnPlan& p, int T, int B, bool start, int HQ, int HK);
hipError_t launch_attn(const AttnArgs& a, const AttnPlan& p, hipStream_t s);

struct SelectArgs {
  const void* q;
  int qtype, ldq, HQ, G;
  KvView kv;
  Seqs s;
  int k, first, last;
  double* scores;  // [T][HK][W]
  int32_t* sel;    // [T][HK][k]
};
long long select_grid(int T, int HK, int W);  // work-groups
hipError_t launch_select(const SelectArgs& a, hipStream_t s);

}  // namespace qm
