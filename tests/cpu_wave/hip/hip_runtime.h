// What csrc/qm_attn_plan.h needs of a GPU, for g++: a wave of 64 lanes as fibers that take turns. Each cross-lane operation is a place where all of them
// meet; threadIdx.x is the running lane.
#pragma once
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#include <algorithm>
#include <cmath>

#define __device__
#define __forceinline__ inline
typedef int hipError_t;
typedef void* hipStream_t;
using std::max;
using std::min;

struct Wave {
  ucontext_t home, lane[64];
  int at, ops[64], word[2][64];  // (a lane may be one operation ahead: words of two)
  bool ended[64];
  void (*work)();
};
inline Wave wave;
inline struct {
  int x;
} threadIdx;

inline void next_lane() {
  const int from = wave.at;
  wave.at = threadIdx.x = (from + 1) & 63;
  swapcontext(&wave.lane[from], &wave.lane[wave.at]);
}
// All lanes' values of one operation
inline const int* exchanged(int v) {
  const int lane = wave.at;
  int* words = wave.word[wave.ops[lane]++ & 1];
  words[lane] = v;
  next_lane();
  return words;
}
inline void lane_main() {
  wave.work();
  wave.ended[wave.at] = true;
  if (wave.at == 63) swapcontext(&wave.lane[63], &wave.home);
  next_lane();
  abort();  // (nobody comes back to a lane that has ended)
}
// Runs `work` in 64 lanes. False: they did not all take the same way.
inline bool run_wave(void (*work)()) {
  static char stack[64][32768];
  wave.work = work;
  memset(wave.ops, 0, sizeof(wave.ops));
  memset(wave.ended, 0, sizeof(wave.ended));
  for (int i = 0; i < 64; ++i) {
    getcontext(&wave.lane[i]);
    wave.lane[i].uc_stack.ss_sp = stack[i];
    wave.lane[i].uc_stack.ss_size = sizeof(stack[i]);
    wave.lane[i].uc_link = nullptr;
    makecontext(&wave.lane[i], lane_main, 0);
  }
  wave.at = threadIdx.x = 0;
  swapcontext(&wave.home, &wave.lane[0]);
  for (int i = 0; i < 64; ++i)
    if (!wave.ended[i] || wave.ops[i] != wave.ops[0]) return false;
  return true;
}

inline unsigned long long __ballot(int p) {
  const int* w = exchanged(p);
  unsigned long long r = 0;
  for (int i = 0; i < 64; ++i) r |= (unsigned long long)(w[i] != 0) << i;
  return r;
}
inline int __ffsll(unsigned long long v) { return __builtin_ffsll((long long)v); }
inline int read_lane(int v, int lane) { return exchanged(v)[lane & 63]; }
// row_shr:n (0x110 + n), row_bcast:15 (0x142) and row_bcast:31 (0x143); what has no source, or is of another row, keeps `old`
inline int moved_by(int old, int v, int ctrl, int rows) {
  const int* w = exchanged(v);
  const int lane = (wave.at), row = lane >> 4;
  if (!(rows >> row & 1)) return old;
  if (ctrl == 0x142) return row ? w[16 * row - 1] : old;
  if (ctrl == 0x143) return lane >= 32 ? w[31] : old;
  const int n = ctrl - 0x110;
  return (lane & 15) >= n ? w[lane - n] : old;
}
#define __builtin_amdgcn_readlane read_lane
#define __builtin_amdgcn_update_dpp(old, v, ctrl, rows, banks, bound) moved_by(old, v, ctrl, rows)
