// The split of an attention call (csrc/qm_attn_plan.h, device code) on a wave that exists on paper. stdin: a batch; stdout: what each of the units asked for does.
#include <stdio.h>

#include <vector>

#include "qm_attn_plan.h"

static qm::AttnArgs a;
static int RT, unit;
static bool found[64];
static qm::Item item[64];
static std::vector<int> start, len;

int main() {
  int HK, B, T, has_start, page_lg, units, first, step;
  while (scanf("%d %d %d %d %d %d %d %d %d %d %d %d %d", &RT, &HK, &a.G, &B, &T, &has_start, &a.s.W, &page_lg, &a.target, &a.tail, &units, &first, &step) == 13) {
    start.resize(B + 1);
    len.resize(B);
    if (has_start)
      for (int& v : start) if (scanf("%d", &v) != 1) return 2;
    for (int& v : len) if (scanf("%d", &v) != 1) return 2;
    a.kv.HK = HK;
    a.kv.lg = page_lg;
    a.s.B = B;
    a.s.T = T;
    a.s.start = has_start ? start.data() : nullptr;
    a.s.len = len.data();
    for (unit = first; unit < units; unit += step) {
      if (!run_wave([] { const int l = threadIdx.x; item[l] = {}; found[l] = qm::find_item(a, RT, unit, item[l]); })) return 3;
      for (int l = 1; l < 64; ++l)
        if (found[l] != found[0] || (found[0] && memcmp(&item[l], &item[0], sizeof(item[0])))) return 4;
      const qm::Item& i = item[0];
      if (found[0]) printf("%d %d %d %d %d %d %d %d %d %d\n", unit, i.b, i.h, i.rt, i.c, i.rts, i.blocks, i.more, i.parts, i.slot);
    }
    printf("-1\n");
    fflush(stdout);
  }
  return 0;
}
