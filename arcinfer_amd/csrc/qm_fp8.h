// Host-side launchers of the e4m3 products, their activation producers and the q/k norm + rotation. Shapes are checked by
// the C-ABI layer (qm_api.hip) beforehand.
//
// Prepared e4m3 weight. The rows are padded to whole groups of 64, K to whole blocks of 128, with zeros. A fragment is what
// one v_mfma_f32_16x16x128_f8f6f4 takes of 16 rows and one block: 2 KB, in two halves of 64 lanes x 16 bytes, so that a
// wave loads it with two fully coalesced 16-byte loads and no staging:
//   [rows/64 groups][4 fragments][K/128][2 halves][64 lanes][16 bytes]
// Lane l of half h holds k = 64 h + 16 (l / 16) .. + 15 of the fragment's row l % 16 (the token operand is read with the same
// k order, so the sum does not depend on it). Row r of fragment t is n = 64 group + 16 (r / 4) + 4 t + r % 4: a result lane
// (rows 4 (l / 16) .. + 3 of one token) then holds 16 neighbouring n over the four fragments of a group.
// Scales: float [ceil(rows / 128)][K / 128], as given.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qm {

constexpr long long kMostThreads = (1LL << 32) - 1;  // of one dimension of a grid

enum : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 30 };

struct Fp8View {
  const uint8_t* q;
  const float* sc;
  int rows, kb;  // kb: blocks of 128 in a row
};

struct Fp8GemmArgs {
  Fp8View w;
  const uint8_t* a8;
  const float* asc;
  int M, M_stride;
  void* C;
  int ctype, ldc, c_off, accumulate;
  float* part;  // partial results of calls whose K is cut
};
hipError_t launch_fp8_repack(const uint8_t* w8, int rows, int K, uint8_t* q, hipStream_t s);
// Workspace for the pieces of cut products (0: the call is not cut)
size_t fp8_workspace_bytes(int M, int rows, int kb);
// How a product runs: tiles of mt token tiles with K in `splits` pieces, or (mt 0) the few-token kernel, rt fragments a work-group of
// `waves` waves
struct Fp8Plan {
  int mt, splits, rt, waves;
};
// part_bytes: the workspace at hand (less than the call would use: fewer pieces)
Fp8Plan fp8_plan(int M, int M_stride, int rows, int kb, bool exact, size_t part_bytes);
hipError_t launch_gemm_fp8(const Fp8GemmArgs& a, const Fp8Plan& plan, hipStream_t s);

// The tile kernel (qm_fp8_tile.hip): tiles of 256 rows x 16 mt tokens (mt 4..8, 4..6 for a C of f32), K in `splits` pieces
constexpr int kFp8Slots = 512;                    // its work-groups that the chip holds at once (two per CU)
constexpr size_t kFp8PartBytes = (size_t)64 << 20;  // most partial results of one call
inline size_t fp8_part_bytes(int M, int rows, int splits) { return (size_t)splits * M * ((rows + 63) / 64 * 64) * sizeof(float); }
hipError_t launch_fp8_tile(const Fp8GemmArgs& a, int mt, int splits, hipStream_t s);

hipError_t launch_quantize_fp8(const void* x, int xtype, int ldx, int M, int M_stride, int K, uint8_t* a8, float* asc,
                               hipStream_t s);
hipError_t launch_rmsnorm_fp8(const void* x, int xtype, int ldx, const float* w, int K, int M, int M_stride, float eps,
                              uint8_t* a8, float* asc, float* h, int ldh, hipStream_t s);
hipError_t launch_swiglu_fp8(const void* gu, int xtype, int ldg, int F, int M, int M_stride, int gelu, uint8_t* a8,
                             float* asc, hipStream_t s);

struct RopeArgs {
  const void* x;
  int xtype, ldx, T, D, q_off, q_hs, HQ, k_off, k_hs, HK;
  const float *wq, *wk;
  float eps;
  int rot, adjacent, axes, turns, sections[4];
  float scale;
  const int32_t* pos;
  int pos_stride;
  const float* inv_freq;
  void *q, *k;
  int otype, ldq, ldk;
};
hipError_t launch_qk_norm_rope(const RopeArgs& a, hipStream_t s);

}  // namespace qm
