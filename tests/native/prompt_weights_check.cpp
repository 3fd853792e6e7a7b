// Host-only view of how a prompt's keys are weighed (iq_prompt_weights.h).  Input lines: S N Nk Hq H.  Prints, per line, whether
// the call counts as few rows over many keys, the steps of a workgroup there, the workgroups that share a key, and the rows of
// a chunk.
#include <cstdio>

#include "../../innerq_amd/csrc/iq_prompt_weights.h"

int main() {
  int S, N, Nk, Hq, H;
  while (std::scanf("%d %d %d %d %d", &S, &N, &Nk, &Hq, &H) == 5) {
    const bool f = iq::few(S, N, Nk, Hq, H);
    std::printf("%d %d %d %d\n", f, f ? iq::steps_of(Nk, H) : 0, iq::shares_of(S, N, Nk, Hq, H), 1 << iq::chunk_bits(S, N, Nk, Hq, H));
  }
  return 0;
}
