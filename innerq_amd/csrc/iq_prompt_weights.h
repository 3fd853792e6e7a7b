// How a call's keys are weighed (iq_prompt_weights.hip): the sizes of its workgroups' shares, chosen on the host.
#pragma once
#include "iq_common.h"

namespace iq {

constexpr int BK = 64;                                      // keys of a workgroup
constexpr int CHUNK_BITS = 11, SHARES = 16, GROUPS = 8192;  // rows (times heads) of a chunk at most; most workgroups of a key, in all

// Few rows over many keys: a workgroup holds up to FEW rows in LDS and walks over steps_of() times FEW_KEYS keys, as many as
// leave FEW_GROUPS workgroups (two per CU: their beginning, some 10 us, is then paid once).
constexpr int FEW = 256, FEW_GROUPS = 512, MOST_STEPS = 64, FEW_WAVES = 8, FEW_THREADS = 64 * FEW_WAVES, FEW_KEYS = 32 * FEW_WAVES;

// Whether a call has few rows over many keys: up to FEW rows (times heads) a sequence by the mean, and keys for seven eighths of
// FEW_GROUPS workgroups (a whole call, us, weigh_few_kernel / weigh_kernel; 32 heads over 8, D = 128, fp16; sequences x rows x keys:
// 1 x 64 x 4096 33.1 / 29.8, 1 x 64 x 16000 63 / 67, 4 x 64 x 4096 59 / 62, 4 x 64 x 16000 145 / 175, 16 x 1 x 4096 103 / 128,
// 16 x 16 x 16000 336 / 435).  How the rows are spread is not known on the host, and a workgroup takes all rows of its sequence:
// no more than FEW_TURNS times FEW in all, whosever they are (4 sequences of 16000 keys, one of 253 rows, the others of 1:
// 235 / 215; 64 of 8000, one of 4033: 11990 / 1450; even ones of more rows pay for that: 16 x 64 x 4000 147 / 176, 128 x 4 x 2000
// 336 / 441).
constexpr int FEW_TURNS = 4;
inline bool few(int S, int N, int Nk, int Hq, int H) {
  return int64_t(N) * (Hq / H) <= int64_t(FEW) * (S < FEW_TURNS ? S : FEW_TURNS) && int64_t(Nk) >= int64_t(1024) * S &&
         int64_t(Nk) * H >= int64_t(FEW_KEYS) * (FEW_GROUPS - FEW_GROUPS / 8);
}

inline int steps_of(int Nk, int H) {
  const int64_t n = ceil_div(int64_t(Nk) * H, int64_t(FEW_KEYS) * FEW_GROUPS);
  return n < 1 ? 1 : n < MOST_STEPS ? int(n) : MOST_STEPS;
}

// Rows of a chunk, as their logarithm: 2048, or as many fewer, 256 at least, as make 1024 workgroups of a call of long sequences
// (by their mean; bf16, 32 heads over 8, D = 128, a whole call, us, 2048 / this: a prompt of 300 tokens 28.4 / 21.8, of 500 39.0 /
// 27.0, of 1500 77.7 / 69.4; of 77, one chunk, 16.0).
inline int chunk_bits(int S, int N, int Nk, int Hq, int H) {
  const int64_t rows = int64_t(N) * (Hq / H) / S, groups = (int64_t(Nk) / BK + S) * H;
  int bits = CHUNK_BITS;
  while (rows >= 1024 && bits > 8 && groups * ceil_div(rows, 1 << bits) < 1024) --bits;
  return bits;
}

// workgroups that share a key
inline int shares_of(int S, int N, int Nk, int Hq, int H) {
  const int64_t chunks = ceil_div(int64_t(N) * (Hq / H), 1 << chunk_bits(S, N, Nk, Hq, H)), most = GROUPS / ((int64_t(Nk) / BK + S) * H);
  const int64_t n = chunks < most ? chunks : most;
  return few(S, N, Nk, Hq, H) || n < 1 ? 1 : n < SHARES ? int(n) : SHARES;
}

}  // namespace iq
