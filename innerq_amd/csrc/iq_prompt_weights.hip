// The attention weights that a packed prompt's keys gather (gfx950): the second launch of iq_prompt_attention_weights.
//
// weights[s][h][j] += sum over the rows i that see key j, and the query heads g of KV head h, of 2^(c q_gi k_j - base_gi) /
// sum_gi, with each row's base and sum from the attention's own launch.  A workgroup takes 128 keys of one KV head of one
// sequence and walks over the rows that see any of them (query rows times heads, as the attention's tiles), in tiles of 64
// staged through LDS.  Keys stay in registers: with S^T = K Q^T a key is a register of the result and a row a lane, so a
// tile's weights are added up register by register, and lanes meet only once, at the end.  Every key has one workgroup that
// adds its rows in a fixed order: no atomics.  Waves: two halves of the keys by two halves of a tile's rows, so that each
// operand that is read from LDS meets 64 keys.
#include "iq_prompt.h"

using namespace iq;

namespace {

constexpr int WAVES = 4, THREADS = 64 * WAVES, BK = 128, BR = 64;  // keys and rows of a tile

template <int D, bool BF>
__global__ __launch_bounds__(THREADS, 2) void weigh_kernel(WeighArgs a) {
#pragma clang fp contract(off)  // logits times c less the base: one fma, as in the attention
  constexpr int CH = D / 8, KS = D / 16, LOADS = BR * CH / THREADS;
  __shared__ u4_t tile0[BR * CH], tile1[BR * CH];
  __shared__ float halves[BK];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hi = lane >> 5;
  const int kw = wave & 1, rw = wave >> 1;
  const int H = gridDim.x / a.slots, kvh = blockIdx.x % H, slot = blockIdx.x / H;
  const int head0 = kvh / a.maps * a.nrep * a.maps + kvh % a.maps;  // its query heads: head0 + i * maps
  // sequence s has the slots from first_slot(s) to first_slot(s + 1), at least as many as it has tiles of keys
  auto first_slot = [&](int i) { return min(max(a.cu_k[i], 0), a.Nk) / BK + i; };
  int s = 0;
  for (int m = a.S; m > 1;) {  // it is among the m from s on
    const int step = (m + 63) / 64, i = min(s + lane * step, a.S);
    const int at = 63 - __builtin_clzll(__ballot(lane * step < m && first_slot(i) <= slot) | 1);
    m = min(step, m - at * step);
    s += at * step;
  }
  s = __builtin_amdgcn_readfirstlane(s);
  int q0, q1, k0, k1;
  rows_of(a.cu_q, s, a.N, q0, q1);
  rows_of(a.cu_k, s, a.Nk, k0, k1);
  q0 = __builtin_amdgcn_readfirstlane(q0);
  q1 = __builtin_amdgcn_readfirstlane(q1);
  k0 = __builtin_amdgcn_readfirstlane(k0);
  k1 = __builtin_amdgcn_readfirstlane(k1);
  const int lq = q1 - q0, keys = k1 - k0, off = keys - lq, j0 = (slot - __builtin_amdgcn_readfirstlane(first_slot(s))) * BK;
  if (j0 >= keys || j0 >= a.T) return;
  const int j1 = min(j0 + BK, keys);
  // rows [ra, rz) see any of the keys, as rows times heads one behind the other
  const int ra = a.causal ? max(j0 - off, 0) : 0;
  const int rz = a.window ? int(min(int64_t(lq), int64_t(j1) - 1 + a.window - off)) : lq;
  if (ra >= rz) return;
  const int v0 = ra * a.nrep, v1 = rz * a.nrep, tiles = (v1 - v0 + BR - 1) / BR;

  u4_t kx[2][KS];  // A operands: key 32 kb + n of the wave's 64 (past the last: that one again, not stored)
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
    const int j = min(j0 + kw * 64 + kb * 32 + n, keys - 1);
    const uint16_t* p = a.k + int64_t(k0 + j) * a.sk_n + kvh * a.sk_h + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kx[kb][ks] = *reinterpret_cast<const u4_t*>(p + 16 * ks);
  }
  // tiles go from memory to LDS without registers, one ahead; rows past the last repeat it
  const int fr = threadIdx.x / CH, fc = (chunk_at<D>(fr, threadIdx.x % CH) % CH) * 16;
  auto fetch = [&](int t, u4_t* lds) {
    const int first = (v0 + t * BR) / a.nrep;  // the descriptor begins at the tile's first row
    const rsrc_t d = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t*>(a.q + int64_t(q0 + first) * a.sq_n + head0 * a.sq_h), 0, -1, 0x00020000);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int v = min(v0 + t * BR + i * (THREADS / CH) + fr, v1 - 1), row = v / a.nrep, head = v - row * a.nrep;
      const uint32_t at = uint32_t(row - first) * uint32_t(a.sq_n) * 2 + uint32_t(head * a.maps) * uint32_t(a.sq_h) * 2 + fc;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(lds + i * THREADS + wave * 64), 16,
                                               at, 0, 0, 0);
    }
  };
  int qa[KS];  // this lane's operands in a tile, in bytes
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qa[ks] = chunk_at<D>(rw * 32 + n, 2 * ks + hi) * 16;

  float acc[32];  // of value 16 kb + i: key 32 kb + 8 (i / 4) + 4 hi + i % 4
#pragma unroll
  for (int i = 0; i < 32; ++i) acc[i] = 0.f;
  struct Row {
    int row;  // of the sequence
    bool real;
    float2 st;
  };
  auto row_of = [&](int t) {
    const int v = v0 + t * BR + rw * 32 + n, w = min(v, v1 - 1), row = w / a.nrep;
    return Row{row, v < v1, a.stats[int64_t(q0 + row) * a.Hq + head0 + (w - row * a.nrep) * a.maps]};
  };
  auto add_tile = [&](int t, const u4_t* lds, const Row& r) {
    u4_t x[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) x[ks] = *reinterpret_cast<const u4_t*>(reinterpret_cast<const char*>(lds) + qa[ks]);
    f16_t st[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kb][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) st[kb] = mma32<BF>(kx[kb][ks], x[ks], st[kb]);
    }
    float c = a.scale.c;
    if (__any(fabsf(r.st.x) > 65536.f)) {  // logits rounded as the base is
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) st[kb] *= c;
      c = 1.f;
    }
    // do all rows of the tile see all keys of the workgroup?
    const int va = v0 + t * BR, ia = va / a.nrep, iz = (min(va + BR, v1) - 1) / a.nrep;
    if (va + BR <= v1 && (!a.causal || ia + off >= j1 - 1) && (!a.window || iz + off + 1 - a.window <= j0)) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        acc[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(st[i / 16][i % 16], c, -r.st.x)), r.st.y, acc[i]);
    } else {
      // key j is seen iff first <= j < last, counted from the lane's first key
      const int base = j0 + kw * 64 + 4 * hi;
      const int last = (r.real ? a.causal ? min(r.row + off + 1, keys) : keys : 0) - base;
      const int first = (a.window ? max(r.row + off + 1 - a.window, 0) : 0) - base;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int j = 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4;
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i / 16][i % 16], c, -r.st.x)) * r.st.y;
        acc[i] += j < last && j >= first ? w : 0.f;
      }
    }
  };
  auto arrived = [&] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
  fetch(0, tile0);
  Row next = row_of(0);
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kx[kb][ks] = (kx[kb][ks] & a.scale.keep) ^ a.scale.sign;
  for (int t = 0; t < tiles; ++t) {
    arrived();
    __syncthreads();  // the tile is there, and no wave reads the other buffer any more
    const Row r = next;
    if (t + 1 < tiles) {
      fetch(t + 1, t & 1 ? tile0 : tile1);
      next = row_of(t + 1);
    }
    add_tile(t, t & 1 ? tile1 : tile0, r);
  }
  // Sums over the 32 lanes of rows: halves of the values change places step by step, until lane n holds value n's sum.
#pragma unroll
  for (int b = 16; b > 0; b /= 2) {
    const bool up = n & b;
#pragma unroll
    for (int i = 0; i < b; ++i) acc[i] = (up ? acc[i + b] : acc[i]) + __shfl_xor(up ? acc[i] : acc[i + b], b, 64);
  }
  const int j = kw * 64 + 32 * (n / 16) + 8 * (n % 16 / 4) + 4 * hi + n % 4;
  if (rw == 1) halves[j] = acc[0];
  __syncthreads();
  if (rw == 0 && j0 + j < j1 && j0 + j < a.T) a.weights[s * a.sw_s + kvh * a.sw_h + j0 + j] += acc[0] + halves[j];
}

}  // namespace

namespace iq {
int launch_prompt_weights(WeighArgs a, int D, bool bf, hipStream_t stream) {
  const int64_t slots = int64_t(a.Nk) / BK + a.S;  // first_slot(S) at most
  const int H = a.Hq / a.nrep;
  IQ_CHECK(slots * H <= UINT32_MAX / THREADS, IQ_ERR_SHAPE);
  a.slots = int(slots);
  auto launch = [&]<int D_, bool BF>() {
    weigh_kernel<D_, BF><<<unsigned(slots * H), THREADS, 0, stream>>>(a);
    return launch_status();
  };
  if (D == 128) return bf ? launch.operator()<128, true>() : launch.operator()<128, false>();
  return bf ? launch.operator()<64, true>() : launch.operator()<64, false>();
}
}  // namespace iq
