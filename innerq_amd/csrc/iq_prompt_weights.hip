// The attention weights that a packed prompt's keys gather (gfx950): the launches behind an attention's own.
//
// weights[s][h][j] += sum over the rows i that see key j, and the query heads g of KV head h, of 2^(c q_gi k_j - base_gi) /
// sum_gi, with each row's base and sum from the attention's own launch.  A workgroup takes BK keys of one KV head of one
// sequence and walks over the rows that see any of them (query rows times heads, as the attention's tiles), in tiles of 64
// staged through LDS.  Keys stay in registers: with S^T = K Q^T a key is a register of the result and a row a lane, so a
// tile's weights are added up register by register, and lanes meet only once, at the end.  Waves: two halves of the keys by
// two halves of a tile's rows.
//
// A key at the beginning of a long prompt is seen by all its rows, so a workgroup takes at most CHUNK of them; where a
// sequence may have more, partial sums go to the workspace and a second launch adds them.  Rows are added in a fixed order:
// no atomics.
#include "iq_prompt.h"

using namespace iq;

namespace {

constexpr int WAVES = 4, THREADS = 64 * WAVES, BR = 64;  // rows of a tile
constexpr int KB = 1, BK = 2 * 32 * KB;                  // blocks of 32 keys of a wave, keys of a workgroup
constexpr int CHUNK = 2048, MOST_CHUNKS = 16;            // rows (times heads) of a workgroup, at least; chunks of a sequence

// A slot's sequence and keys, and the rows, as rows times heads one behind the other, that see any of them.
struct Keys {
  int s, q0, k0, j0, j1, off;  // off: row i stands at key i + off
  int keys, v0, v1, rows;      // rows: [.., rows) of the sequence see any of them
};
__device__ __forceinline__ bool keys_of(const WeighArgs& a, int slot, Keys& x) {
  // sequence s has the slots from first_slot(s) to first_slot(s + 1), at least as many as it has tiles of keys
  auto first_slot = [&](int i) { return min(max(a.cu_k[i], 0), a.Nk) / BK + i; };
  const int lane = threadIdx.x & 63;
  int s = 0;
  for (int m = a.S; m > 1;) {  // it is among the m from s on
    const int step = (m + 63) / 64, i = min(s + lane * step, a.S);
    const int at = 63 - __builtin_clzll(__ballot(lane * step < m && first_slot(i) <= slot) | 1);
    m = min(step, m - at * step);
    s += at * step;
  }
  x.s = __builtin_amdgcn_readfirstlane(s);
  int q1, k1;
  rows_of(a.cu_q, x.s, a.N, x.q0, q1);
  rows_of(a.cu_k, x.s, a.Nk, x.k0, k1);
  x.q0 = __builtin_amdgcn_readfirstlane(x.q0);
  x.k0 = __builtin_amdgcn_readfirstlane(x.k0);
  const int lq = __builtin_amdgcn_readfirstlane(q1) - x.q0;
  x.keys = __builtin_amdgcn_readfirstlane(k1) - x.k0;
  x.off = x.keys - lq;
  x.j0 = (slot - __builtin_amdgcn_readfirstlane(first_slot(x.s))) * BK;
  if (x.j0 >= x.keys || x.j0 >= a.T) return false;
  x.j1 = min(x.j0 + BK, x.keys);
  const int first = a.causal ? max(x.j0 - x.off, 0) : 0;
  const int64_t seen = int64_t(x.j1) - 1 + a.window - x.off;  // rows below it see a key, in a window
  x.rows = a.window && seen < lq ? int(seen) : lq;
  x.v0 = first * a.nrep;
  x.v1 = x.rows * a.nrep;
  return first < x.rows;
}

template <int D, bool BF>
__global__ __launch_bounds__(THREADS, 4 / KB) void weigh_kernel(WeighArgs a) {
#pragma clang fp contract(off)  // logits times c less the base: one fma, as in the attention
  constexpr int CH = D / 8, KS = D / 16, LOADS = BR * CH / THREADS;
  __shared__ u4_t tile0[BR * CH], tile1[BR * CH];
  __shared__ float halves[BK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hi = lane >> 5;
  const int kw = wave & 1, rw = wave >> 1;
  const int H = gridDim.x / a.slots, kvh = blockIdx.x % H;
  const int head0 = kvh / a.maps * a.nrep * a.maps + kvh % a.maps;  // its query heads: head0 + i * maps
  Keys x;
  if (!keys_of(a, blockIdx.x / H, x)) return;
  const int v0 = max(x.v0, int(blockIdx.y) * a.chunk), v1 = min(x.v1, int(blockIdx.y + 1) * a.chunk);
  if (v0 >= v1) return;
  const int q0 = x.q0, j0 = x.j0, tiles = (v1 - v0 + BR - 1) / BR;
  // of the rows, [vf, vg) see all of the keys
  const int vf = a.causal ? max(x.j1 - 1 - x.off, 0) * a.nrep : 0;
  const int64_t whole = int64_t(j0) + a.window - x.off;  // rows below it, in a window
  const int vg = !a.window || whole >= x.rows ? v1 : whole <= 0 ? 0 : min(v1, int(whole) * a.nrep);

  u4_t kx[KB][KS];  // A operands: key 32 kb + n of the wave's (past the last: that one again, not stored)
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int j = min(j0 + (kw * KB + kb) * 32 + n, x.keys - 1);
    const uint16_t* p = a.k + int64_t(x.k0 + j) * a.sk_n + kvh * a.sk_h + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kx[kb][ks] = *reinterpret_cast<const u4_t*>(p + 16 * ks);
  }
  // a row of the tiles in their order, as query row and head (a step of BR without a division)
  struct Place {
    int row, head;
  };
  const int step_row = BR / a.nrep, step_head = BR - step_row * a.nrep;
  auto place_of = [&](int v) {
    const int row = v / a.nrep;
    return Place{row, v - row * a.nrep};
  };
  auto advance = [&](Place& p) {
    p.row += step_row;
    p.head += step_head;
    if (p.head >= a.nrep) {
      p.head -= a.nrep;
      ++p.row;
    }
  };
  // Tiles go from memory to LDS without registers, one ahead, from a descriptor that begins at the tile's first row and ends
  // with the sequence's last: rows past the chunk's hold anything (a later row, or zeros) and count for nothing.  Where the
  // heads divide BR a tile's rows are at the same distances from its first one in every tile.
  const int fr = threadIdx.x / CH, fc = (chunk_at<D>(fr, threadIdx.x % CH) % CH) * 16;
  Place load[LOADS], begin = place_of(v0);
  uint32_t at[LOADS];
  auto offset_of = [&](const Place& p) {
    return uint32_t(p.row - begin.row) * uint32_t(a.sq_n) * 2 + uint32_t(p.head * a.maps) * uint32_t(a.sq_h) * 2 + fc;
  };
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    load[i] = place_of(v0 + i * (THREADS / CH) + fr);
    at[i] = offset_of(load[i]);
  }
  const uint16_t* from = a.q + int64_t(q0) * a.sq_n + int64_t(head0) * a.sq_h;
  auto fetch = [&](u4_t* lds) {
    const int64_t bytes = 2 * (int64_t(x.rows - 1 - begin.row) * a.sq_n + int64_t((a.nrep - 1) * a.maps) * a.sq_h + D);
    const uint32_t bound = bytes >> 32 ? ~0u : uint32_t(bytes);
    const rsrc_t d = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(from + int64_t(begin.row) * a.sq_n), 0,
                                                       int(bound), 0x00020000);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      load_to_lds(d, lds + i * THREADS + wave * 64, at[i]);
    if (step_head) {
      advance(begin);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        advance(load[i]);
        at[i] = offset_of(load[i]);
      }
    } else {
      begin.row += step_row;
    }
  };
  int qa[KS];  // this lane's operands in a tile, in bytes
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qa[ks] = chunk_at<D>(rw * 32 + n, 2 * ks + hi) * 16;

  float acc[16 * KB];  // of value 16 kb + i: key 32 kb + 8 (i / 4) + 4 hi + i % 4
#pragma unroll
  for (int i = 0; i < 16 * KB; ++i) acc[i] = 0.f;
  // this lane's row of the next tile, and its {base, 1 / sum} (past the last: that one again, not counted)
  Place mine = place_of(v0 + rw * 32 + n);
  int mine_v = v0 + rw * 32 + n;
  const float2* stats = a.stats + int64_t(q0) * a.Hq + head0;
  auto stats_of = [&] {
    return stats[int64_t(min(mine.row, x.rows - 1)) * a.Hq + (mine.row < x.rows ? mine.head : a.nrep - 1) * a.maps];
  };
  auto scores = [&](const u4_t* lds, f16_t (&st)[KB]) {
    u4_t y[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) y[ks] = *reinterpret_cast<const u4_t*>(reinterpret_cast<const char*>(lds) + qa[ks]);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kb][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) st[kb] = mma32<BF>(kx[kb][ks], y[ks], st[kb]);
    }
  };
  auto add_tile = [&](int t, const u4_t* lds, int row, bool real, float2 w) {
    f16_t st[KB];
    const int va = v0 + t * BR;
    if (va >= vf && va + BR <= vg && !__any(fabsf(w.x) > 65536.f)) {  // all rows see all keys
      scores(lds, st);
#pragma unroll
      for (int i = 0; i < 16 * KB; ++i)
        acc[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(st[i / 16][i % 16], a.scale.c, -w.x)), w.y, acc[i]);
      return;
    }
    scores(lds, st);
    float c = a.scale.c;
    if (__any(fabsf(w.x) > 65536.f)) {  // logits rounded as the base is
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) st[kb] *= c;
      c = 1.f;
    }
    // key j is seen iff first <= j < last, counted from the lane's first key
    const int base = j0 + kw * 32 * KB + 4 * hi;
    const int last = (real ? a.causal ? min(row + x.off + 1, x.keys) : x.keys : 0) - base;
    const int first = (a.window ? max(row + x.off + 1 - a.window, 0) : 0) - base;
#pragma unroll
    for (int i = 0; i < 16 * KB; ++i) {
      const int j = 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4;
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i / 16][i % 16], c, -w.x)) * w.y;
      acc[i] += j < last && j >= first ? y : 0.f;
    }
  };
  fetch(tile0);
  float2 next = stats_of();
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kx[kb][ks] = (kx[kb][ks] & a.scale.keep) ^ a.scale.sign;
  // (a buffer by name in each half of the loop: reads of one would wait for the loads to the other)
  auto turn = [&](int t, u4_t* here, u4_t* other) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the tile is there, and no wave reads the other buffer any more
    const int row = mine.row;
    const bool real = mine_v < v1;
    const float2 w = next;
    if (t + 1 < tiles) {
      fetch(other);
      mine_v += BR;
      advance(mine);
      next = stats_of();
    }
    add_tile(t, here, row, real, w);
  };
  for (int t = 0; t < tiles; t += 2) {
    turn(t, tile0, tile1);
    if (t + 1 < tiles) turn(t + 1, tile1, tile0);
  }
  // Sums over the 32 lanes of rows: halves of the values change places step by step, until lane n holds value n's sum (with
  // 16 values: lanes n and n + 16 each a half of value n % 16's, then the sum).
#pragma unroll
  for (int b = 8 * KB; b > 0; b /= 2) {
    const bool up = n & b;
#pragma unroll
    for (int i = 0; i < b; ++i) acc[i] = (up ? acc[i + b] : acc[i]) + __shfl_xor(up ? acc[i] : acc[i + b], b, 64);
  }
  if constexpr (KB == 1) acc[0] += __shfl_xor(acc[0], 16, 64);
  const int j = kw * 32 * KB + 32 * (n / 16 % KB) + 8 * (n % 16 / 4) + 4 * hi + n % 4;
  if (rw == 1) halves[j] = acc[0];
  __syncthreads();
  if (rw == 1 || n >= 16 * KB || j0 + j >= x.j1 || j0 + j >= a.T) return;
  const float sum = acc[0] + halves[j];
  if (a.part) a.part[(int64_t(blockIdx.y) * H + kvh) * a.Nk + x.k0 + j0 + j] = sum;
  else a.weights[x.s * a.sw_s + kvh * a.sw_h + j0 + j] += sum;
}

// adds the chunks' sums of BK keys
__global__ __launch_bounds__(64) void add_kernel(WeighArgs a) {
  const int H = gridDim.x / a.slots, kvh = blockIdx.x % H;
  Keys x;
  if (!keys_of(a, blockIdx.x / H, x)) return;
  for (int j = x.j0 + threadIdx.x; j < x.j1 && j < a.T; j += 64) {
    float sum = 0.f;
    for (int z = x.v0 / a.chunk; z <= (x.v1 - 1) / a.chunk; ++z) sum += a.part[(int64_t(z) * H + kvh) * a.Nk + x.k0 + j];
    a.weights[x.s * a.sw_s + kvh * a.sw_h + j] += sum;
  }
}

// rows (times heads) of a chunk, of a call with `rows` in all
inline int64_t chunk_of(int64_t rows) {
  const int64_t even = ceil_div(ceil_div(rows, MOST_CHUNKS), BR) * BR;
  return even < CHUNK ? CHUNK : even;
}

template <int D, bool BF>
int launch(const WeighArgs& a, dim3 grid, hipStream_t stream) {
  weigh_kernel<D, BF><<<grid, THREADS, 0, stream>>>(a);
  if (const int st = launch_status()) return st;
  if (!a.part) return IQ_OK;
  add_kernel<<<grid.x, 64, 0, stream>>>(a);
  return launch_status();
}

}  // namespace

namespace iq {
size_t prompt_weights_bytes(int N, int Nk, int Hq, int H) {
  const int64_t rows = int64_t(N) * (Hq / H), chunks = ceil_div(rows, chunk_of(rows));
  const size_t stats = (size_t(N) * Hq * sizeof(float2) + 15) / 16 * 16;
  return chunks > 1 ? stats + (size_t(chunks) * H * Nk * sizeof(float) + 15) / 16 * 16 : stats;
}

bool prompt_weights_fit(int S, int N, int Nk, int Hq, int H) {
  const int64_t rows = int64_t(N) * (Hq / H), chunk = chunk_of(rows), chunks = ceil_div(rows, chunk);
  return (int64_t(Nk) / BK + S) * H <= UINT32_MAX / THREADS / chunks && chunk * chunks <= INT32_MAX;
}

int launch_prompt_weights(WeighArgs a, int D, bool bf, hipStream_t stream) {
  const int64_t slots = int64_t(a.Nk) / BK + a.S;  // first_slot(S) at most
  const int64_t rows = int64_t(a.N) * a.nrep, chunk = chunk_of(rows), chunks = ceil_div(rows, chunk);
  const int H = a.Hq / a.nrep;
  a.slots = int(slots);
  a.chunk = int(chunk);
  a.part = chunks > 1 ? (float*)((char*)a.stats + (size_t(a.N) * a.Hq * sizeof(float2) + 15) / 16 * 16) : nullptr;
  const dim3 grid(unsigned(slots * H), unsigned(chunks));
  if (D == 128) return bf ? launch<128, true>(a, grid, stream) : launch<128, false>(a, grid, stream);
  return bf ? launch<64, true>(a, grid, stream) : launch<64, false>(a, grid, stream);
}
}  // namespace iq
