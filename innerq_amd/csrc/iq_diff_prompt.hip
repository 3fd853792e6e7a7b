// Differential attention over packed prompts (gfx950): iq_diff_prompt_attention.
//
// out_j = (softmax(c q_2j K_2g^T) - lam_j softmax(c q_2j+1 K_2g+1^T)) V_g: query heads 2j, 2j + 1 are the two maps of output
// head j, KV heads 2g, 2g + 1 their keys (g = j / nrep), V's heads are 2 D wide.  As iq_prompt.hip, with S^T = K Q^T and O^T
// += V^T P^T on v_mfma_f32_32x32x16 over tiles of keys staged through LDS; here half of a workgroup's waves take one map
// and half the other, of the same rows, so that V's tile is staged once for both and a wave holds the sums of one map.
// Each map has a softmax of its own (running maximum and sum), so the difference is taken at the end: the second map's
// waves hand their normalised sums, times lam, over LDS in fp32.
//
// A wave holds 32 rows of 2 D sums: at D = 128 the 128 accumulators leave room for two waves per SIMD, a workgroup of 8 with
// tiles of 32 keys; at D = 64 workgroups of 4 with tiles of 64.  (At D = 128 registers spill from the first masked tile on whose V
// holds an infinity or NaN; when they did in every masked one, four such tiles took 40 us, now 3.)  Bound: as iq_prompt.hip the
// matrix unit and the softmax beside it.  A prompt of 8192 tokens, 32 query heads over 8 KV heads, D = 128, fp16: 765 - 801 us,
// 1030 - 1078 TFLOP/s, where a 16384^3 library product reaches 1324; D = 64, bf16: 421 us, 980 TFLOP/s of 1380; 16 packed prompts of
// 25 .. 2000 tokens, D = 64, bf16: 129 - 137 us, 676 - 719 TFLOP/s, what is less than a long prompt's being first and last tiles and a
// chip that short prompts do not fill.  A workgroup walks over all keys of its rows, however few there are: 64 rows behind 16000 keys
// on 4 sequences, D = 128, fp16: 575 us on 32 workgroups.  Each map by a call of iq_prompt_attention over both halves of V would take 1.5 times
// the products (K Q^T twice).
#include "iq_prompt.h"

using namespace iq;

namespace {

struct DiffArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  int64_t sq_n, sq_h, sk_n, sk_h, sv_n, sv_h, so_n, so_h;
  const int32_t *cu_q, *cu_k;
  const float* lam;  // of each output head
  int64_t s_lam;
  float2* stats;  // [N][Hq] {base, 1 / sum of weights} of each row of each map, or null
  int S, N, Nk, Hq, nrep, slots;  // nrep: output heads per pair of KV heads
  Scale scale;
  float slack;  // 8 / c
  int causal, window;
};

// rows of a workgroup (of each map) and keys of a tile
template <int D>
struct Shape {
  static constexpr int MAP_WAVES = D == 64 ? 2 : 4, WAVES = 2 * MAP_WAVES, THREADS = 64 * WAVES, BM = 32 * MAP_WAVES;
  static constexpr int BN = D == 64 ? 64 : 32;
};

template <int D, bool BF>
__global__ __launch_bounds__(Shape<D>::THREADS, 2) void diff_kernel(DiffArgs a) {
#pragma clang fp contract(off)  // logits times c and the maximum times c round alike
  using X = Shape<D>;
  constexpr int THREADS = X::THREADS, BM = X::BM, BN = X::BN, WAVES = X::WAVES;
  constexpr int CH = D / 8, KS = D / 16;        // chunks per key row, k steps of S
  constexpr int NV = D / 64, VCH = 16;          // V's tile: parts of 128 dims, of 16 chunks a row
  constexpr int KB = BN / 32, KC = BN / 16;     // blocks of 32 keys of S, of 16 of O
  constexpr int LK = BN * CH, LV = BN * VCH;    // chunks of a key tile (one map), of a part of V's
  constexpr int TILE = 2 * LK + NV * LV, VLOADS = NV * LV / THREADS;
  __shared__ u4_t tile0[TILE], tile1[TILE];
  __shared__ int lodd[2][WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hi = lane >> 5;
  const int map = wave / X::MAP_WAVES, rb = wave % X::MAP_WAVES;
  const int G = gridDim.x / a.slots, g = blockIdx.x % G, slot = blockIdx.x / G;

  // Sequence s has the slots from first_slot(s) to first_slot(s + 1), at least as many as it has tiles, its last tiles (the
  // longest) first.
  auto first_slot = [&](int i) { return int(int64_t(min(max(a.cu_q[i], 0), a.N)) * a.nrep / BM) + i; };
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
  const int lq = q1 - q0, keys = k1 - k0, off = keys - lq, rows = lq * a.nrep, tiles = int((int64_t(rows) + BM - 1) / BM);
  const int tile = tiles - 1 - (slot - __builtin_amdgcn_readfirstlane(first_slot(s)));
  if (tile < 0 || tile >= tiles) return;
  // this lane's row, and the keys that it sees: [first, last) (worked out for the queries, and once more behind the whole tiles,
  // which have no registers to keep them)
  int vrow, row, head, last, first;
  auto row_of = [&](int lane_row) {
    vrow = tile * BM + rb * 32 + lane_row;
    row = min(vrow, rows - 1) / a.nrep;
    head = g * a.nrep + min(vrow, rows - 1) - row * a.nrep;
    last = a.causal ? min(row + off + 1, keys) : keys;
    first = a.window ? max(row + off + 1 - a.window, 0) : 0;
  };
  row_of(n);
  // the tiles of keys that any row of the workgroup sees
  const int row_a = tile * BM / a.nrep, row_z = (min(tile * BM + BM, rows) - 1) / a.nrep;
  const int j_end = a.causal ? min(row_z + off + 1, keys) : keys, j_begin = a.window ? max(row_a + off + 1 - a.window, 0) : 0;
  const int t_begin = j_begin / BN, t_end = j_end > j_begin ? (j_end + BN - 1) / BN : t_begin;

  u4_t q[KS];  // B operand: row n, dims 16 ks + 8 hi + e (rows past the end repeat the last one and are not stored)
  {
    const uint16_t* p = a.q + int64_t(q0 + row) * a.sq_n + int64_t(2 * head + map) * a.sq_h + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = *reinterpret_cast<const u4_t*>(p + 16 * ks);
  }
  f16_t o[NV][4];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[v][b][i] = 0.f;
  float m = NEG_INF, l = 0.f;

  // Tiles go from memory to LDS without registers, one tile ahead, chunks spread by chunk_at in the source address; rows past
  // the last key that the workgroup sees are past the descriptor's bound and read as zeros.
  const uint16_t *kp = a.k + int64_t(k0) * a.sk_n + int64_t(2 * g) * a.sk_h, *vp = a.v + int64_t(k0) * a.sv_n + g * a.sv_h;
  const int sk = int(a.sk_n) * 2, sv = int(a.sv_n) * 2;
  const int kr = threadIdx.x / CH, vr = threadIdx.x / VCH;
  const int vk = kr * sk + (chunk_at<D>(kr, threadIdx.x % CH) % CH) * 16;
  const int vv = vr * sv + (chunk_at<128>(vr, threadIdx.x % VCH) % VCH) * 16;
  auto fetch1 = [&]<int C, int LOADS>(const uint16_t* p, int64_t stride, int bytes, int at, int t, u4_t* lds) {
    const int there = min(j_end - t * BN, BN);
    const rsrc_t d = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p + int64_t(t) * BN * stride), 0,
                                                       (there - 1) * bytes + C * 16, 0x00020000);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(lds + i * THREADS + wave * 64), 16,
                                               at, i * (THREADS / C) * bytes, 0, 0);
  };
  auto fetch = [&](int t, u4_t* to) {
#pragma unroll
    for (int i = 0; i < 2; ++i) fetch1.template operator()<CH, LK / THREADS>(kp + i * a.sk_h, a.sk_n, sk, vk, t, to + i * LK);
#pragma unroll
    for (int v = 0; v < NV; ++v)
      fetch1.template operator()<VCH, LV / THREADS>(vp + 128 * v, a.sv_n, sv, vv, t, to + 2 * LK + v * LV);
  };
  // This lane's operands in a tile, in bytes (blocks of 32 keys (K), of 16 (V) are at fixed distances from them): K's step ks is
  // at k_own ^ 32 ks, V's block b of dims in half h of 16 keys at (v_own ^ 64 b ^ 32 h) + 8 h rows.  At D = 128 worked out where
  // they are used: there are no registers to keep all of them.
  const int k_own = (map * LK + chunk_at<D>(n, hi)) * 16;
  const int v_own = (2 * LK + chunk_at<128>(hi * 4 + (lane & 15) / 4, (lane >> 4 & 1) * 2 + lane % 4 / 2)) * 16 + lane % 2 * 8;
  auto not_kept = [&](int at) {
    if constexpr (D == 128) asm volatile("" : "+v"(at));
    return at;
  };
  // S^T of a tile: st[kb][i] is key 32 kb + 8 (i/4) + 4 hi + i%4
  auto scores = [&](const u4_t* lt, f16_t (&st)[KB]) {
    const int ka = not_kept(k_own);
    auto at = [&](int kb, int ks) { return *reinterpret_cast<const u4_t*>(reinterpret_cast<const char*>(lt) + (ka ^ 32 * ks) + kb * 32 * CH * 16); };
    u4_t x[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) x[ks] = at(0, ks);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kb][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        st[kb] = mma32<BF>(x[ks], q[ks], st[kb]);
        if (kb + 1 < KB) x[ks] = at(kb + 1, ks);
      }
    }
  };
  // V^T's operand: dim 128 v + 32 b + n, keys 16 kc + 8 (e/4) + 4 hi + e%4
  auto v_operand = [&](const u4_t* lt, int va, int kc, int v, int b) {
    u4_t y;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* at = reinterpret_cast<const char*>(lt) + (va ^ 64 * b ^ 32 * h) + (v * LV + (kc * 16 + h * 8) * VCH) * 16;
      const u2_t w = __builtin_bit_cast(
          u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)at));
      y[2 * h] = w.x;
      y[2 * h + 1] = w.y;
    }
    return y;
  };
  // the running maximum over a tile (in both halves of the wave)
  auto maximum = [&](const f16_t (&st)[KB]) {
    float x[4] = {m, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i % 4] = fmaxf(x[i % 4], st[kb][i]);
    const float y = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1]));
  };
  // Weights are relative to 2^base, base = RN(m c), m a maximum that is replaced when a row's has grown past it by 8 in the
  // exponent (as iq_prompt.hip).
  auto base_of = [&](float x) { return x == NEG_INF ? 0.f : x * a.scale.c; };
  auto softmax = [&](f16_t (&st)[KB], u4_t (&p)[KC]) {
    float mx = maximum(st);
    const bool grown = __any(mx > m + a.slack);
    mx = grown ? mx : m;
    const float base = base_of(mx);
    if (grown) {
      const float f = __builtin_amdgcn_exp2f(m == NEG_INF ? NEG_INF : base_of(m) - base);
      l *= f;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int b = 0; b < 4; ++b) o[v][b] *= f;
    }
    m = mx;
    float c = a.scale.c;
    if (__any(fabsf(base) > 65536.f)) {  // logits rounded as the base is
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) st[kb] *= c;
      c = 1.f;
    }
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[kb][i], c, -base));
        sum[i % 4] += st[kb][i];
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    // rounded to the activation dtype, as the matrix unit's two operands have one type, V's; their sum takes them unrounded
#pragma unroll
    for (int kc = 0; kc < KC; ++kc)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[kc][i] = pack2<BF>(st[kc / 2][8 * (kc % 2) + 2 * i], st[kc / 2][8 * (kc % 2) + 2 * i + 1]);
  };
  auto products = [&](const u4_t* lt, const u4_t (&p)[KC]) {
    const int va = not_kept(v_own);
#pragma unroll
    for (int kc = 0; kc < KC; ++kc)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int b = 0; b < 4; ++b) o[v][b] = mma32<BF>(v_operand(lt, va, kc, v, b), p[kc], o[v][b]);
  };
  // Any tile: keys that a row does not see have weight 0.  ODD: V may hold an infinity or NaN, which 0 * inf would carry into
  // rows that do not see its key.
  auto any_tile = [&]<bool ODD>(int t, const u4_t* lt, bool odd) {
    const int j0 = t * BN;
    // this wave's rows: does any see the tile, do all see all of it?
    const int ra = tile * BM + rb * 32, wa = ra / a.nrep, wz = min(ra + 31, rows - 1) / a.nrep;
    const int w_last = a.causal ? min(wz + off + 1, keys) : keys, w_first = a.window ? max(wa + off + 1 - a.window, 0) : 0;
    if (ra >= rows || w_last <= j0 || w_first >= j0 + BN) return;
    const bool mask = (a.causal ? min(wa + off + 1, keys) : keys) < j0 + BN || (a.window && wz + off + 1 - a.window > j0);
    f16_t st[KB];
    scores(lt, st);
    if (mask) {
      const int z = last - j0 - 4 * hi, f = first - j0 - 4 * hi;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int j = 32 * kb + 8 * (i / 4) + i % 4;
          st[kb][i] = j >= z || j < f ? NEG_INF : st[kb][i];
        }
    }
    u4_t p[KC];
    softmax(st, p);
    if (!ODD || !mask || !odd) {
      products(lt, p);
      return;
    }
    // key by key, into the rows that see it
#pragma clang loop unroll(disable)
    for (int key = 0; key < BN; ++key) {
      const int at = key / 16 * 4 + key % 16 / 8 * 2 + key % 4 / 2, of = key % 8 / 4;  // p's word, in the lanes hi == of
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4 * KC; ++i)
        if (i == at) w = p[i / 4][i % 4];
      const auto y = __builtin_amdgcn_permlane32_swap(w, w, false, false);
      w = of ? y[1] : y[0];
      const float pk = key & 1 ? hi_half<BF>(w) : lo_half<BF>(w);
      if (j0 + key < last && j0 + key >= first) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const u2_t x = reinterpret_cast<const u2_t*>(&lt[2 * LK + v * LV + chunk_at<128>(key, 4 * b + i)])[hi];
              const uint32_t x0 = x.x, x1 = x.y;
              o[v][b][4 * i] = __builtin_fmaf(pk, lo_half<BF>(x0), o[v][b][4 * i]);
              o[v][b][4 * i + 1] = __builtin_fmaf(pk, hi_half<BF>(x0), o[v][b][4 * i + 1]);
              o[v][b][4 * i + 2] = __builtin_fmaf(pk, lo_half<BF>(x1), o[v][b][4 * i + 2]);
              o[v][b][4 * i + 3] = __builtin_fmaf(pk, hi_half<BF>(x1), o[v][b][4 * i + 3]);
            }
      }
    }
  };

  // The tiles' order: [whole_a, whole_z), which every row sees whole, then the others; tile number i of it goes through
  // buffer i % 2, and every wave passes the same barriers.
  int whole_a = a.window ? (max(row_z + off + 1 - a.window, 0) + BN - 1) / BN : 0;
  int whole_z = (a.causal ? min(row_a + off + 1, keys) : keys) / BN;
  if (whole_a >= whole_z || t_begin >= t_end) whole_a = whole_z = t_begin;
  const int nw = whole_z - whole_a, tail = t_end - whole_z, count = t_end - t_begin;
  auto tile_at = [&](int i) { return i < nw ? whole_a + i : i < nw + tail ? whole_z + i - nw : t_begin + i - nw - tail; };
  auto whole_tile = [&](const u4_t* lt) {
    f16_t st[KB];
    u4_t p[KC];
    scores(lt, st);
    softmax(st, p);
    products(lt, p);
  };
  // This wave's loads to LDS are there.  Every barrier that hands a tile over is behind such a wait: the compiler's own does
  // not cover them on all paths.
  auto arrived = [&] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
  if (count > 0) fetch(tile_at(0), tile0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = (q[ks] & a.scale.keep) ^ a.scale.sign;  // (the queries arrive with the first tile)
  int i = 0;
  while (i < nw) {
    arrived();
    __syncthreads();  // the tile is there, and no wave reads the other buffer any more
    if (i + 1 < count) fetch(tile_at(i + 1), tile1);
    whole_tile(tile0);
    if (++i >= nw) break;
    arrived();
    __syncthreads();
    if (i + 1 < count) fetch(tile_at(i + 1), tile0);
    whole_tile(tile1);
    ++i;
  }
  row_of(not_kept(n));
  // tile i is there; does its V hold an infinity or NaN?  Each wave looks through the part that it has loaded itself.
  auto next_is_odd = [&] {
    const u4_t* lt = i & 1 ? tile1 : tile0;
    arrived();
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < VLOADS; ++c) {
      const u4_t w = lt[2 * LK + c * THREADS + threadIdx.x];
#pragma unroll
      for (int y = 0; y < 4; ++y) top = max_halves(top, w[y] & 0x7fff7fffu);
    }
    const uint32_t e = BF ? 0x7f80u : 0x7c00u;
    const bool mine = __any((top & 0xffffu) >= e || (top >> 16) >= e);
    if (lane == 0) lodd[i & 1][wave] = mine;
    __syncthreads();
    bool odd = false;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) odd |= lodd[i & 1][w] != 0;
    return __builtin_amdgcn_readfirstlane(odd) != 0;
  };
  auto tail_tile = [&]<bool ODD>(bool odd) {
    if (i + 1 < count) fetch(tile_at(i + 1), i & 1 ? tile0 : tile1);
    any_tile.template operator()<ODD>(tile_at(i), i & 1 ? tile1 : tile0, odd);
  };
  // (from the first odd tile on in a loop of its own, whose need of registers would make both spill: 40 us for four tiles)
  for (; i < count && !next_is_odd(); ++i) tail_tile.template operator()<false>(false);
  for (; i < count; ++i) tail_tile.template operator()<true>(next_is_odd());
  {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(y[0]) + __uint_as_float(y[1]);
  }
  // The difference, 128 dims at a time: the second map's waves hand theirs to the first map's (the same rows and dims are in
  // the same lanes and registers), which store them through LDS, whole rows at a time.
  float inv = l == 0.f ? 0.f : 1.f / l;
  if (l == 0.f)  // no key that counts: 0, whatever V holds
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[v][b][i] = 0.f;
  if (a.stats && hi == 0 && vrow < rows) a.stats[int64_t(q0 + row) * a.Hq + 2 * head + map] = float2{base_of(m), inv};
  if (map) inv *= a.lam[head * a.s_lam];
  static_assert(X::MAP_WAVES * 64 * 64 * 4 <= 2 * TILE * 16, "a part of the difference fits the two tiles");
  const int64_t at = int64_t(q0 + row) * a.so_n + head * a.so_h;
  const int at0 = int(at), at1 = int(at >> 32);
  // (16 KB of a wave: within one of the two tiles)
  constexpr int PER = TILE / 1024;
  u4_t* const area = rb < PER ? tile0 + rb * 1024 : tile1 + (rb - PER) * 1024;
  float* const mine = reinterpret_cast<float*>(area) + lane;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    __syncthreads();  // nobody reads tiles, or the last part's rows, any more
    if (map) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) mine[(b * 16 + i) * 64] = o[v][b][i] * inv;
    }
    __syncthreads();
    if (map) continue;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[v][b][i] = o[v][b][i] * inv - mine[(b * 16 + i) * 64];
    wave_lds_sync();
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        reinterpret_cast<u2_t*>(area + chunk_at<128>(n, 4 * b + i))[hi] =
            u2_t{pack2<BF>(o[v][b][4 * i], o[v][b][4 * i + 1]), pack2<BF>(o[v][b][4 * i + 2], o[v][b][4 * i + 3])};
    wave_lds_sync();
#pragma unroll
    for (int j = 0; j < VCH / 2; ++j) {
      const int r = j * (64 / VCH) + lane / VCH, c = lane % VCH;  // row and chunk
      const int64_t to = int64_t(uint32_t(__shfl(at0, r, 64))) | int64_t(__shfl(at1, r, 64)) << 32;
      if (tile * BM + rb * 32 + r < rows) *reinterpret_cast<u4_t*>(a.out + to + 128 * v + 8 * c) = area[chunk_at<128>(r, c)];
    }
  }
}

}  // namespace

extern "C" int iq_diff_prompt_attention(const void* q, int64_t sq_n, int64_t sq_h, const void* k, int64_t sk_n, int64_t sk_h,
                                        const void* v, int64_t sv_n, int64_t sv_h, const float* lam, int64_t s_lam,
                                        const int32_t* cu_q, const int32_t* cu_k, int S, int N, int Nk, int Hq, int H, int D,
                                        int mode, float scale, int causal, int window, void* out, int64_t so_n, int64_t so_h,
                                        float* weights, int64_t sw_s, int64_t sw_h, int64_t T, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  IQ_CHECK(cu_q && cu_k && lam && (N == 0 || (q && out)) && (Nk == 0 || (k && v)), IQ_ERR_NULL);
  IQ_CHECK(base_mode(mode) == 0, IQ_ERR_MODE);
  IQ_CHECK(d_ok(D) && H > 0 && H % 2 == 0 && Hq > 0 && Hq % H == 0 && Hq <= 4096 && S > 0 && N >= 0 && Nk >= 0 && window >= 0,
           IQ_ERR_SHAPE);
  IQ_CHECK(!window || causal, IQ_ERR_MODE);
  for (const int64_t s : {sk_n, sv_n}) IQ_CHECK(s >= 0 && s < (1 << 23), IQ_ERR_SHAPE);  // a tile of rows in 32 bits
  IQ_CHECK(s_lam >= 0 && (!N || out != q), IQ_ERR_SHAPE);
  for (const int64_t s : {sq_n, sq_h, sk_n, sk_h, sv_n, sv_h, so_n, so_h}) IQ_CHECK(s % 8 == 0, IQ_ERR_ALIGN);
  IQ_CHECK(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(cu_q, 4) && aligned(cu_k, 4) &&
               aligned(lam, 4), IQ_ERR_ALIGN);
  if (weights) {
    // a tile's rows of q in 32 bits
    IQ_CHECK(sq_n >= 0 && sq_n < (1 << 23) && sq_h >= 0 && sq_h < (1 << 29) && sq_h * (Hq / H) < (1 << 29), IQ_ERR_SHAPE);
    IQ_CHECK(T >= 0 && sw_s >= 0 && sw_h >= 0, IQ_ERR_SHAPE);
    IQ_CHECK(aligned(weights, 4), IQ_ERR_ALIGN);
  }
  if (N == 0) return IQ_OK;
  if (weights) {
    IQ_CHECK(iq::prompt_weights_fit(S, N, Nk, Hq, H), IQ_ERR_SHAPE);
    IQ_CHECK(workspace && workspace_bytes >= iq_prompt_weights_workspace_bytes(S, N, Nk, Hq, H, D), IQ_ERR_WORKSPACE);
    IQ_CHECK(aligned(workspace, 16), IQ_ERR_ALIGN);
  }
  float2* const stats = weights ? (float2*)workspace : nullptr;
  const int G = H / 2, nrep = Hq / H;
  if (window >= Nk) window = 0;  // hides nothing
  const Scale sc = scale_of(scale);
  auto launch = [&]<int D_, bool BF>() -> int {
    using X = Shape<D_>;
    const int64_t rows = int64_t(N) * nrep, slots = rows / X::BM + S;  // first_slot(S) at most
    IQ_CHECK(rows <= INT32_MAX - X::BM && int64_t(N) + Nk <= INT32_MAX && slots * G <= UINT32_MAX / X::THREADS, IQ_ERR_SHAPE);
    const DiffArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)out, sq_n, sq_h, sk_n, sk_h, sv_n,
                     sv_h, so_n, so_h, cu_q, cu_k, lam, s_lam, stats, S, N, Nk, Hq, nrep, int(slots), sc, 8.f / sc.c, causal ? 1 : 0,
                     window};
    diff_kernel<D_, BF><<<unsigned(slots * G), X::THREADS, 0, (hipStream_t)stream>>>(a);
    return launch_status();
  };
  const bool bf = act_bf16(mode);
  const int st = D == 128 ? (bf ? launch.operator()<128, true>() : launch.operator()<128, false>())
                          : (bf ? launch.operator()<64, true>() : launch.operator()<64, false>());
  if (st || !weights || !Nk) return st;
  return launch_prompt_weights({(const uint16_t*)q, (const uint16_t*)k, sq_n, sq_h, sk_n, sk_h, stats, weights, sw_s, sw_h, T,
                                cu_q, cu_k, S, N, Nk, Hq, nrep, 0, sc, causal ? 1 : 0, window, 2, 0, nullptr, 1, 0}, D, bf, (hipStream_t)stream);
}
