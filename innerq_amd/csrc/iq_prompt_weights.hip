// The attention weights that a packed prompt's keys gather (gfx950): the launches behind an attention's own.
//
// weights[s][h][j] += sum over the rows i that see key j, and the query heads g of KV head h, of 2^(c q_gi k_j - base_gi) /
// sum_gi, with each row's base and sum from the attention's own launch.  A workgroup takes BK keys of one KV head of one
// sequence and walks over the rows that see any of them (query rows times heads, as the attention's tiles), in tiles of 64
// staged through LDS.  Keys stay in registers: with S^T = K Q^T a key is a register of the result and a row a lane, so a
// tile's weights are added up register by register, and lanes meet only once, at the end.  Waves: two halves of the keys by
// two halves of a tile's rows.
//
// A key at the beginning of a long prompt is seen by all its rows, so up to SHARES workgroups share a key: each takes every
// so-manieth chunk of the rows, and a second launch adds their sums (how many rows a sequence has is not known on the host:
// a share that finds none ends at once, and the shares are as many as leave GROUPS workgroups).  Rows are added in a fixed
// order: no atomics.  (One share / 16 at most, a whole call, bf16, 32 heads over 8, D = 128: a prompt of 2000 tokens 134 / 90 us,
// of 8192 947 / 846, 16 of 25 .. 2000 324 / 307, 64 of 100 59 / 63.)
//
// Bound: neither unit alone.  2048 rows by 2048 keys of 64 heads: vector unit busy 49 % of the clocks (16 exponentials and 32
// multiply-adds per 16 logits of a lane, and as much again around them), matrix unit 31 %; without the tiles' loads the launch
// took three quarters of its time, without the exponentials seven eighths.  16 packed prompts of 25 .. 2000 tokens: 110 us, 41
// GFLOP, behind 165 of the attention's; a prompt of 77 tokens 8 us, its loads one behind the other.
#include "iq_prompt.h"
#include "iq_prompt_weights.h"

using namespace iq;

namespace {

constexpr int WAVES = 4, THREADS = 64 * WAVES, BR = 64;  // rows of a tile
static_assert(BK == 32 * WAVES / 2);

// A slot's sequence and keys (of `bk` a slot), and the rows, as rows times heads one behind the other, that see any of them.
struct Keys {
  int s, q0, k0, j0, j1, off;  // off: row i stands at key i + off
  int keys, v0, v1, rows;      // rows: [.., rows) of the sequence see any of them
};
__device__ __forceinline__ bool keys_of(const WeighArgs& a, int slot, int bk, Keys& x) {
  // sequence s has the slots from first_slot(s) to first_slot(s + 1), at least as many as it has tiles of keys
  auto first_slot = [&](int i) { return min(max(a.cu_k[i], 0), a.Nk) / bk + i; };
  const int lane = threadIdx.x & 63;
  int s = 0;
  for (int m = a.S; m > 1;) {  // it is among the m from s on
    const int step = (m + 63) / 64, i = min(s + lane * step, a.S);
    const int at = 63 - __builtin_clzll(__ballot(lane * step < m && first_slot(i) <= slot) | 1);
    m = min(step, m - at * step);
    s += at * step;
  }
  x.s = __builtin_amdgcn_readfirstlane(s);
  typedef const __attribute__((address_space(4))) int32_t* consts_t;  // (by scalar loads)
  int q1, k1;
  rows_of((consts_t)a.cu_q, x.s, a.N, x.q0, q1);
  rows_of((consts_t)a.cu_k, x.s, a.Nk, x.k0, k1);
  const int lq = q1 - x.q0;
  x.keys = k1 - x.k0;
  x.off = x.keys - lq;
  x.j0 = (slot - (x.k0 / bk + x.s)) * bk;
  if (x.j0 < 0 || x.j0 >= x.keys || x.j0 >= a.T) return false;  // (negative: a slot before the first sequence's)
  x.j1 = min(x.j0 + bk, x.keys);
  const int first = a.causal ? max(x.j0 - x.off, 0) : 0;
  const int64_t seen = int64_t(x.j1) - 1 + a.window - x.off;  // rows below it see a key, in a window
  x.rows = a.window && seen < lq ? int(seen) : lq;
  x.v0 = first * a.nrep;
  x.v1 = x.rows * a.nrep;
  return first < x.rows;
}

// Sums of 16 values over the 32 lanes of rows: halves of the values change places step by step, until lanes n and n + 16 hold
// halves of value n's sum, then the sum.
__device__ __forceinline__ float sum_rows(float (&acc)[16]) {
  const int n = threadIdx.x & 31;
#pragma unroll
  for (int b = 8; b > 0; b /= 2) {
    const bool up = n & b;
#pragma unroll
    for (int i = 0; i < b; ++i) {
      const float x = acc[i], y = acc[i + b];
      acc[i] = (up ? y : x) + __shfl_xor(up ? x : y, b, 64);
    }
  }
  return acc[0] + __shfl_xor(acc[0], 16, 64);
}

// A block of 32 rows (in LDS, this lane's operands at qa bytes) against a wave's 32 keys: the logits, s[i] of key 8 (i / 4) +
// 4 hi + i % 4 and row n.  st: {base, 1 / sum} of this lane's row.
template <int D, bool BF>
struct Block {
  static constexpr int KS = D / 16;
  static __device__ __forceinline__ f16_t logits(const u4_t* lds, const int (&qa)[KS], const u4_t (&kx)[KS]) {
    u4_t y[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) y[ks] = *reinterpret_cast<const u4_t*>(reinterpret_cast<const char*>(lds) + qa[ks]);
    f16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mma32<BF>(kx[ks], y[ks], s);
    return s;
  }
  // all rows see all keys
  static __device__ __forceinline__ void add_whole(const u4_t* lds, const int (&qa)[KS], const u4_t (&kx)[KS], float c, float2 st,
                                                   float (&acc)[16]) {
    const f16_t s = logits(lds, qa, kx);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      acc[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -st.x)), st.y, acc[i]);
  }
  // any rows: a lane's row sees the keys [first, last), counted from the lane's first key
  static __device__ __forceinline__ void add_some(const u4_t* lds, const int (&qa)[KS], const u4_t (&kx)[KS], float c, bool big,
                                                  float2 st, int first, int last, float (&acc)[16]) {
    f16_t s = logits(lds, qa, kx);
    if (big) {  // logits rounded as the base is
      s *= c;
      c = 1.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int j = 8 * (i / 4) + i % 4;
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -st.x)) * st.y;
      acc[i] += j < last && j >= first ? w : 0.f;
    }
  }
};
__device__ __forceinline__ bool big_base(float2 st) { return __any(fabsf(st.x) > 65536.f); }

// the first chunk of a share that has rows which see the keys (or one behind them)
__device__ __forceinline__ int share_chunk(const WeighArgs& a, const Keys& x, int share) {
  const int shares = a.shares, c = x.v0 >> a.chunk_bits, ahead = share - c % shares;
  return c + (ahead < 0 ? ahead + shares : ahead);
}

template <int D, bool BF>
__global__ __launch_bounds__(THREADS, 4) void weigh_kernel(WeighArgs a) {
#pragma clang fp contract(off)  // logits times c less the base: one fma, as in the attention
  constexpr int CH = D / 8, KS = D / 16, LOADS = BR * CH / THREADS;
  __shared__ u4_t tile0[BR * CH], tile1[BR * CH];
  __shared__ float halves[BK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hi = lane >> 5;
  const int kw = wave % (WAVES / 2), rw = wave / (WAVES / 2);  // halves of the keys, of a tile's rows
  const int H = gridDim.x / a.slots, kvh = blockIdx.x % H;
  const int head0 = kvh / a.maps * a.nrep * a.maps + kvh % a.maps;  // its query heads: head0 + i * maps
  Keys x;
  if (!keys_of(a, blockIdx.x / H, BK, x)) return;
  const int first_chunk = share_chunk(a, x, blockIdx.y), chunk_rows = 1 << a.chunk_bits;
  if (first_chunk * chunk_rows >= x.v1) return;
  const int q0 = x.q0, j0 = x.j0;
  // of the rows, [vf, vg) see all of the keys
  const int vf = a.causal ? max(x.j1 - 1 - x.off, 0) * a.nrep : 0;
  const int64_t whole = int64_t(j0) + a.window - x.off;  // rows below it, in a window
  const int vg = !a.window || whole >= x.rows ? x.v1 : whole <= 0 ? 0 : int(whole) * a.nrep;

  u4_t kx[KS];  // A operands: key n of the wave's (past the last: that one again, not stored)
  {
    const uint16_t* p = a.k + int64_t(x.k0 + min(j0 + kw * 32 + n, x.keys - 1)) * a.sk_n + kvh * a.sk_h + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kx[ks] = *reinterpret_cast<const u4_t*>(p + 16 * ks);
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
  Place load[LOADS], begin, mine;
  uint32_t at[LOADS];
  int v0, v1, tiles;  // of the chunk
  auto offset_of = [&](const Place& p) {
    return uint32_t(p.row - begin.row) * uint32_t(a.sq_n) * 2 + uint32_t(p.head * a.maps) * uint32_t(a.sq_h) * 2 + fc;
  };
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

  float acc[16];  // of key 8 (i / 4) + 4 hi + i % 4
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  // this lane's row of the next tile, and its {base, 1 / sum} (past the last: that one again, not counted)
  const float2* stats = a.stats + int64_t(q0) * a.Hq + head0;
  auto stats_of = [&] {
    return stats[int64_t(min(mine.row, x.rows - 1)) * a.Hq + (mine.row < x.rows ? mine.head : a.nrep - 1) * a.maps];
  };
  float2 next;
  // (a buffer by name in each half of the loop: reads of one would wait for the loads to the other)
  auto turn = [&](int t, u4_t* here, u4_t* other) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // the tile is there, and no wave reads the other buffer any more
    const int row = mine.row;
    const float2 st = next;
    if (t + 1 < tiles) {
      fetch(other);
      advance(mine);
      next = stats_of();
    }
    const int va = v0 + t * BR;
    const bool big = big_base(st);
    if (va >= vf && va + BR <= min(vg, v1) && !big) {
      Block<D, BF>::add_whole(here, qa, kx, a.scale.c, st, acc);
      return;
    }
    const int base = j0 + kw * 32 + 4 * hi;
    const int last = (va + rw * 32 + n < v1 ? a.causal ? min(row + x.off + 1, x.keys) : x.keys : 0) - base;
    const int first = (a.window ? max(row + x.off + 1 - a.window, 0) : 0) - base;
    Block<D, BF>::add_some(here, qa, kx, a.scale.c, big, st, first, last, acc);
  };
  for (int chunk = first_chunk; chunk * chunk_rows < x.v1; chunk += a.shares) {
    v0 = max(x.v0, chunk * chunk_rows);
    v1 = min(x.v1, (chunk + 1) * chunk_rows);
    tiles = (v1 - v0 + BR - 1) / BR;
    begin = place_of(v0);
    mine = place_of(v0 + rw * 32 + n);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      load[i] = place_of(v0 + i * (THREADS / CH) + fr);
      at[i] = offset_of(load[i]);
    }
    if (chunk > first_chunk) __syncthreads();  // nobody reads the last tile any more
    fetch(tile0);
    next = stats_of();
    if (chunk == first_chunk)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kx[ks] = (kx[ks] & a.scale.keep) ^ a.scale.sign;
    for (int t = 0; t < tiles; t += 2) {
      turn(t, tile0, tile1);
      if (t + 1 < tiles) turn(t + 1, tile1, tile0);
    }
  }
  const float half = sum_rows(acc);
  const int j = kw * 32 + 8 * (n % 16 / 4) + 4 * hi + n % 4;
  if (rw == 1) halves[j] = half;
  __syncthreads();
  if (rw == 1 || n >= 16 || j0 + j >= x.j1 || j0 + j >= a.T) return;
  const float sum = half + halves[j];
  if (a.part) a.part[(int64_t(blockIdx.y) * H + kvh) * a.Nk + x.k0 + j0 + j] = sum;
  else a.weights[x.s * a.sw_s + kvh * a.sw_h + j0 + j] += sum;
}

// The same for few rows over many keys.  The rows (up to FEW; more in turns) stay in LDS with their statistics, and a wave
// takes 32 of each step's FEW_KEYS keys over all of them: no barriers, and each key's sum is one wave's.  (64 rows behind 16000
// keys on 4 sequences, 8 KV heads, D = 128: 85 us by weigh_kernel, 52 here, where reading the keys takes 28 at a copy's rate
// and the products 25 at a library product's.)
template <int D, bool BF>
__global__ __launch_bounds__(FEW_THREADS, 4) void weigh_few_kernel(WeighArgs a) {
#pragma clang fp contract(off)
  constexpr int CH = D / 8, KS = D / 16, LOADS = FEW * CH / FEW_THREADS;
  __shared__ u4_t rows[FEW * CH];
  __shared__ float2 stats[FEW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hi = lane >> 5;
  const int H = gridDim.x / a.slots, kvh = blockIdx.x % H;
  const int head0 = kvh / a.maps * a.nrep * a.maps + kvh % a.maps;  // its query heads: head0 + i * maps
  Keys x;
  if (!keys_of(a, blockIdx.x / H, FEW_KEYS * a.steps, x)) return;
  const uint16_t* kp = a.k + int64_t(x.k0) * a.sk_n + kvh * a.sk_h + 8 * hi;
  auto load_keys = [&](int j, u4_t (&y)[KS]) {  // (past the last: that one again, not stored)
    const uint16_t* p = kp + int64_t(min(j + n, x.keys - 1)) * a.sk_n;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) y[ks] = *reinterpret_cast<const u4_t*>(p + 16 * ks);
  };
  int qa[KS];  // this lane's operands in a block of 32 rows, in bytes
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qa[ks] = chunk_at<D>(n, 2 * ks + hi) * 16;
  float* const to = a.weights + x.s * a.sw_s + kvh * a.sw_h;
  for (int v0 = x.v0; v0 < x.v1; v0 += FEW) {
    const int v1 = min(v0 + FEW, x.v1), blocks = (v1 - v0 + 31) / 32;
    if (v0 > x.v0) __syncthreads();  // nobody reads the last rows any more
    // (past the last row: that one again, not counted)
    const int r0 = threadIdx.x / CH, step = FEW_THREADS / CH, step_row = step / a.nrep, step_head = step - step_row * a.nrep;
    int row = (v0 + r0) / a.nrep, head = v0 + r0 - row * a.nrep;
    constexpr int BATCH = LOADS < 8 ? LOADS : 8;  // loads under way together
#pragma clang loop unroll(disable)
    for (int i0 = 0; i0 < LOADS; i0 += BATCH) {
      u4_t y[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const bool real = v0 + (i0 + i) * step + r0 < v1;
        y[i] = *reinterpret_cast<const u4_t*>(a.q + int64_t(x.q0 + (real ? row : x.rows - 1)) * a.sq_n +
                                              int64_t(head0 + (real ? head : a.nrep - 1) * a.maps) * a.sq_h +
                                              8 * (threadIdx.x % CH));
        row += step_row;
        head += step_head;
        if (head >= a.nrep) {
          head -= a.nrep;
          ++row;
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) rows[chunk_at<D>((i0 + i) * step + r0, threadIdx.x % CH)] = y[i];
    }
    if (threadIdx.x < FEW) {
      const int v = min(v0 + int(threadIdx.x), v1 - 1), row = v / a.nrep;
      stats[threadIdx.x] = a.stats[int64_t(x.q0 + row) * a.Hq + head0 + (v - row * a.nrep) * a.maps];
    }
    __syncthreads();
    for (int j0 = x.j0 + 32 * wave; j0 < x.j1; j0 += FEW_KEYS) {
      u4_t kx[KS];
      load_keys(j0, kx);
      // this lane's key after the sums, and what it has gathered
      const int key = j0 + 8 * (n % 16 / 4) + 4 * hi + n % 4;
      const bool mine = n < 16 && key < x.j1 && key < a.T;
      const float old = mine ? to[key] : 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kx[ks] = (kx[ks] & a.scale.keep) ^ a.scale.sign;
      float acc[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[i] = 0.f;
      // of the rows, [vf, vg) see all of these keys
      const int vf = a.causal ? max(min(j0 + 32, x.j1) - 1 - x.off, 0) * a.nrep : 0;
      const int64_t whole = int64_t(j0) + a.window - x.off;  // rows below it, in a window
      const int vg = !a.window || whole >= x.rows ? v1 : whole <= 0 ? 0 : min(v1, int(whole) * a.nrep);
#pragma clang loop unroll(disable)
      for (int b = 0; b < blocks; ++b) {
        const float2 st = stats[32 * b + n];
        const int va = v0 + 32 * b;
        const bool big = big_base(st);
        if (va >= vf && va + 32 <= vg && !big) {
          Block<D, BF>::add_whole(rows + 32 * b * CH, qa, kx, a.scale.c, st, acc);
          continue;
        }
        const int base = j0 + 4 * hi, v = va + n, row = v / a.nrep;
        const int last = (v < v1 ? a.causal ? min(row + x.off + 1, x.keys) : x.keys : 0) - base;
        const int first = (a.window ? max(row + x.off + 1 - a.window, 0) : 0) - base;
        Block<D, BF>::add_some(rows + 32 * b * CH, qa, kx, a.scale.c, big, st, first, last, acc);
      }
      const float sum = sum_rows(acc);
      if (mine) to[key] = old + sum;
    }
  }
}

// adds the shares' sums of BK keys
__global__ __launch_bounds__(64) void add_kernel(WeighArgs a) {
  const int H = gridDim.x / a.slots, kvh = blockIdx.x % H;
  Keys x;
  if (!keys_of(a, blockIdx.x / H, BK, x)) return;
  for (int j = x.j0 + threadIdx.x; j < x.j1 && j < a.T; j += 64) {
    float sum = 0.f;
    for (int z = 0; z < a.shares; ++z)
      if (share_chunk(a, x, z) << a.chunk_bits < x.v1) sum += a.part[(int64_t(z) * H + kvh) * a.Nk + x.k0 + j];
    a.weights[x.s * a.sw_s + kvh * a.sw_h + j] += sum;
  }
}

inline size_t stats_bytes(int N, int Hq) { return (size_t(N) * Hq * sizeof(float2) + 15) / 16 * 16; }

template <int D, bool BF>
int launch(const WeighArgs& a, bool few, dim3 grid, hipStream_t stream) {
  if (few) {
    weigh_few_kernel<D, BF><<<grid, FEW_THREADS, 0, stream>>>(a);
    return launch_status();
  }
  weigh_kernel<D, BF><<<grid, THREADS, 0, stream>>>(a);
  if (const int st = launch_status()) return st;
  if (!a.part) return IQ_OK;
  add_kernel<<<grid.x, 64, 0, stream>>>(a);
  return launch_status();
}

}  // namespace

namespace iq {
size_t prompt_weights_bytes(int S, int N, int Nk, int Hq, int H) {
  const int shares = shares_of(S, N, Nk, Hq, H);
  return stats_bytes(N, Hq) + (shares > 1 ? (size_t(shares) * H * Nk * sizeof(float) + 15) / 16 * 16 : 0);
}

bool prompt_weights_fit(int S, int N, int Nk, int Hq, int H) {
  return int64_t(N) * (Hq / H) <= INT32_MAX - (SHARES << CHUNK_BITS) &&
         (int64_t(Nk) / BK + S) * H <= UINT32_MAX / FEW_THREADS / shares_of(S, N, Nk, Hq, H);
}

int launch_prompt_weights(WeighArgs a, int D, bool bf, hipStream_t stream) {
  const int H = a.Hq / a.nrep;
  const bool f = few(a.S, a.N, a.Nk, a.Hq, H);
  a.steps = f ? steps_of(a.Nk, H) : 1;
  a.slots = int(int64_t(a.Nk) / (f ? FEW_KEYS * a.steps : BK) + a.S);  // first_slot(S) at most
  a.shares = shares_of(a.S, a.N, a.Nk, a.Hq, H);
  a.chunk_bits = chunk_bits(a.S, a.N, a.Nk, a.Hq, H);
  a.part = a.shares > 1 ? (float*)((char*)a.stats + stats_bytes(a.N, a.Hq)) : nullptr;
  const dim3 grid(unsigned(int64_t(a.slots) * H), unsigned(a.shares));
  if (D == 128) return bf ? launch<128, true>(a, f, grid, stream) : launch<128, false>(a, f, grid, stream);
  return bf ? launch<64, true>(a, f, grid, stream) : launch<64, false>(a, f, grid, stream);
}
}  // namespace iq
