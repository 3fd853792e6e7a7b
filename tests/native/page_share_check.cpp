// Host-only check of how the attention over pages shares out its list of units (units_per_group, share_begin in
// iq_paged.h): for every (total, grid) given on stdin, the workgroups' shares follow one another from 0 to total, and a
// share's first and last unit name their workgroup.  Input lines: total grid.  Prints "ok" or "FAIL <reason>" per line.
#include <cstdio>

#include "../../innerq_amd/csrc/iq_paged.h"

int main() {
  int total, grid;
  while (std::scanf("%d %d", &total, &grid) == 2) {
    const int per = iq::units_per_group(total, grid);
    const char* err = per < iq::SHARE_LEAST ? "a share of too few units" : nullptr;
    int at = 0;
    for (int g = 0; g < grid && !err; ++g) {
      const int u = iq::share_begin(g, per, total), u1 = iq::share_begin(g + 1, per, total);
      if (u != at || u1 < u || u1 - u > per) err = "shares do not follow one another";
      else if (u1 > u && (u / per != g || (u1 - 1) / per != g)) err = "a unit names another workgroup";
      at = u1;
    }
    if (!err && at != total) err = "units are left out";
    if (err) std::printf("FAIL %s\n", err);
    else std::printf("ok\n");
  }
  return 0;
}
