// Attention over packed prompts (gfx950): iq_prompt_attention.
//
// Sequences of different lengths lie one behind the other; a workgroup takes 128 rows of one KV head of one sequence
// (query rows times the heads that share the KV head; four waves of 32) and walks over the sequence's keys in tiles of
// 64, staged through LDS.  Both products run transposed on v_mfma_f32_32x32x16: S^T = K Q^T leaves a query row per lane
// and its keys in the lane's registers, where the running softmax needs one exchange (with the lane of the other
// half-wave) per tile, and the exponentials, rounded to the activation dtype, are the B operand of O^T += V^T P^T as
// they are: V^T's A operand reads LDS with ds_read_b64_tr_b16 in the same order of keys.  (Rounded, because the matrix
// unit's two operands have one type, V's; a weight moves by half a step at most, and its sum takes it unrounded: outputs'
// error 1.1 - 1.4 times that of fp32 weights, against 64 bits.)
//
// A tile holds the rows of all heads of a group, so short prompts fill tiles and stage their keys once (32 query heads
// over 8, a tile per query head before: 128 prompts of 16 tokens 58 us, now 18; one of 77 11.8, now 8.0).
// Bound: the matrix unit and the softmax's vector work, which two workgroups per CU overlap.  A prompt of 16384 tokens
// (32 query, 8 KV heads, D = 128, bf16): 1.94 ms, 1130 TFLOP/s, where a 16384^3 bf16 library product reaches 1370; the
// matrix unit is busy 60 % of the clocks, HBM moves 0.8 GB.  With D = 64 there are half the products per exponential: the
// vector unit is busy 79 % of the clocks, the matrix unit 50 % (1.11 - 1.18 ms, 930 - 990 TFLOP/s).  Short prompts wait for
// their first tile: 77 tokens 7.4 us.
#include "iq_paged.h"

using namespace iq;

namespace {

typedef float f16_t __attribute__((ext_vector_type(16)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;

constexpr int WAVES = 4, THREADS = 64 * WAVES, BM = 32 * WAVES, BN = 64;
constexpr float NEG_INF = -__builtin_inff();

struct PromptArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  int64_t sq_n, sq_h, sk_n, sk_h, sv_n, sv_h, so_n, so_h;
  const int32_t *cu_q, *cu_k;
  int S, N, Nk, Hq, nrep, slots;
  float c;              // |scale| log2(e); 1 for a scale of 0
  float slack;          // 8 / c
  uint32_t keep, sign;  // and-ed, xor-ed into the queries: a scale of 0 clears them, a negative one flips their signs
  int causal, window;
};

// rows [r0, r1) of sequence s in a packed tensor of n rows (whatever cu holds)
__device__ __forceinline__ void rows_of(const int32_t* cu, int s, int n, int& r0, int& r1) {
  r0 = min(max(cu[s], 0), n);
  r1 = min(max(cu[s + 1], r0), n);
}

// tiles of BM rows that a KV head's share of a sequence of lq query rows makes
__device__ __forceinline__ int tiles_of(int lq, int nrep) { return int((int64_t(lq) * nrep + BM - 1) / BM); }

template <bool BF>
__device__ __forceinline__ f16_t mma32(u4_t a, u4_t b, f16_t c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
  typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2_t, a), __builtin_bit_cast(us2_t, b)));
}

// 16-byte chunk c of row r in an LDS tile: spread so that neither K's reads (one chunk of 16 rows) nor V's transposed
// ones (four chunks of 4 rows) meet in a bank
template <int D>
__device__ __forceinline__ int chunk_at(int r, int c) {
  if constexpr (D == 128) return r * 16 + (c ^ ((r & 3) << 2 | (r >> 2 & 3)));
  else return r * 8 + (c ^ ((r >> 1 & 1) << 2 | (r >> 2 & 3)));
}

template <int D, bool BF>
__global__ __launch_bounds__(THREADS, 2) void prompt_kernel(PromptArgs a) {
#pragma clang fp contract(off)  // logits times c and the maximum times c round alike
  constexpr int CH = D / 8, KS = D / 16, DB = D / 32;  // chunks per row, k steps of S, blocks of 32 dims
  constexpr int LOADS = BN * CH / THREADS;             // chunks per thread and tile
  __shared__ u4_t lk0[BN * CH], lk1[BN * CH], lv0[BN * CH], lv1[BN * CH];
  __shared__ int lodd[2][WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hi = lane >> 5;

  // This workgroup's KV head and slot.  Blocks go round robin over the 8 XCDs: with the heads innermost, an XCD keeps to
  // one or a few heads' keys, and where XCDs share a head each has its share of long and short tiles (a run of slots per
  // XCD: a prompt of 8192 tokens, 8 query heads over one KV head 274 us, now 168; 32 over 4 652, now 497).
  const int H = gridDim.x / a.slots, kvh = blockIdx.x % H, slot = blockIdx.x / H;

  // The slot's sequence and tile of rows, a sequence's last tiles (the longest) first.
  int s = 0, q0, q1, k0, k1, tile;
  if (a.S == 1) {
    rows_of(a.cu_q, 0, a.N, q0, q1);
    rows_of(a.cu_k, 0, a.Nk, k0, k1);
    tile = tiles_of(q1 - q0, a.nrep) - 1 - slot;
    if (tile < 0) return;
    // (prompts of 16 tokens, us here / with the search below: 64 9.4 / 12.5, 128 17 / 20, 256 32 / 32, 512 65 / 57)
  } else if (a.S <= 256) {  // the sequences' tiles lie behind one another
    uint64_t past;
    for (int before = 0;; s += 64) {
      rows_of(a.cu_q, min(s + lane, a.S - 1), a.N, q0, q1);
      rows_of(a.cu_k, min(s + lane, a.S - 1), a.Nk, k0, k1);
      const int end = before + wave_scan(s + lane < a.S ? tiles_of(q1 - q0, a.nrep) : 0);
      past = __ballot(end > slot);
      if (past) {
        const int l = __builtin_ctzll(past);
        s += l;
        q0 = __builtin_amdgcn_readlane(q0, l);
        q1 = __builtin_amdgcn_readlane(q1, l);
        k0 = __builtin_amdgcn_readlane(k0, l);
        k1 = __builtin_amdgcn_readlane(k1, l);
        tile = __builtin_amdgcn_readlane(end, l) - 1 - slot;
        break;
      }
      if (s + 64 >= a.S) return;
      before = __builtin_amdgcn_readlane(end, 63);
    }
  } else {
    // Sequence s has the slots from first_slot(s) to first_slot(s + 1), at least as many as it has tiles: found among 64
    // starts at a time, without a sum over the sequences before it.
    auto first_slot = [&](int i) { return int(int64_t(min(max(a.cu_q[i], 0), a.N)) * a.nrep / BM) + i; };
    for (int n = a.S; n > 1;) {  // it is among the n from s on
      const int step = (n + 63) / 64, i = min(s + lane * step, a.S);
      const int at = 63 - __builtin_clzll(__ballot(lane * step < n && first_slot(i) <= slot) | 1);
      n = min(step, n - at * step);
      s += at * step;
    }
    rows_of(a.cu_q, s, a.N, q0, q1);
    rows_of(a.cu_k, s, a.Nk, k0, k1);
    tile = tiles_of(q1 - q0, a.nrep) - 1 - (slot - first_slot(s));
    if (tile < 0 || tile >= tiles_of(q1 - q0, a.nrep)) return;
  }
  s = __builtin_amdgcn_readfirstlane(s);  // (uniform, which the compiler does not see: it would loop over lanes at each load)
  q0 = __builtin_amdgcn_readfirstlane(q0);
  q1 = __builtin_amdgcn_readfirstlane(q1);
  tile = __builtin_amdgcn_readfirstlane(tile);
  k0 = __builtin_amdgcn_readfirstlane(k0);
  k1 = __builtin_amdgcn_readfirstlane(k1);
  const int lq = q1 - q0, keys = k1 - k0, off = keys - lq, rows = lq * a.nrep;
  // this lane's row of the KV head's rows, which are its query rows' heads one behind the other: row * nrep + head
  const int vrow = tile * BM + wave * 32 + n, row = min(vrow, rows - 1) / a.nrep, head = kvh * a.nrep + min(vrow, rows - 1) % a.nrep;
  // key j is seen iff first <= j < last
  const int last = a.causal ? min(row + off + 1, keys) : keys, first = a.window ? max(row + off + 1 - a.window, 0) : 0;
  // the tiles of keys that any row of the workgroup sees
  const int row_a = tile * BM / a.nrep, row_z = (min(tile * BM + BM, rows) - 1) / a.nrep;
  const int j_end = a.causal ? min(row_z + off + 1, keys) : keys, j_begin = a.window ? max(row_a + off + 1 - a.window, 0) : 0;
  const int t_begin = j_begin / BN, t_end = j_end > j_begin ? (j_end + BN - 1) / BN : t_begin;

  u4_t q[KS];  // B operand: row n, dims 16 ks + 8 hi + e (rows past the end repeat the last one and are not stored)
  {
    const uint16_t* p = a.q + int64_t(q0 + row) * a.sq_n + head * a.sq_h + 8 * hi;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = *reinterpret_cast<const u4_t*>(p + 16 * ks);
  }
  f16_t o[DB];
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[b][i] = 0.f;
  float m = NEG_INF, l = 0.f;

  // Tiles go from memory to LDS without registers, one tile ahead.  LDS is written in lane order, so the spreading of
  // chunk_at is in the source address: a thread's chunk of every pass of THREADS chunks has the same place in its row.
  // Rows past the last key that the workgroup sees are past the descriptor's bound and read as zeros (the bound counts the
  // scalar offset too, also where that alone is past it).
  const uint16_t *kp = a.k + int64_t(k0) * a.sk_n + kvh * a.sk_h, *vp = a.v + int64_t(k0) * a.sv_n + kvh * a.sv_h;
  const int sk = int(a.sk_n) * 2, sv = int(a.sv_n) * 2, fr = threadIdx.x / CH, fc = (chunk_at<D>(fr, threadIdx.x % CH) % CH) * 16;
  const int vk = fr * sk + fc, vv = fr * sv + fc;
  auto fetch1 = [&](const uint16_t* p, int64_t stride, int bytes, int at, int t, u4_t* lds) {
    const int rows = min(j_end - t * BN, BN);
    const rsrc_t d = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p + int64_t(t) * BN * stride), 0,
                                                       (rows - 1) * bytes + D * 2, 0x00020000);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)(lds + i * THREADS + wave * 64), 16,
                                               at, i * (THREADS / CH) * bytes, 0, 0);
  };
  auto fetch = [&](int t, u4_t* lk, u4_t* lv) {
    fetch1(kp, a.sk_n, sk, vk, t, lk);
    fetch1(vp, a.sv_n, sv, vv, t, lv);
  };
  // this lane's operands in a tile, in bytes; blocks of 32 keys (K), of 16 (V) are at fixed distances from them
  int ka[KS], va[DB][2];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) ka[ks] = chunk_at<D>(n, 2 * ks + hi) * 16;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = lane & 15, d = b * 32 + (lane >> 4 & 1) * 16 + j % 4 * 4;
      va[b][h] = chunk_at<D>(h * 8 + hi * 4 + j / 4, d / 8) * 16 + d % 8 * 2;
    }
  // S^T of a tile: st[kb][i] is key 32 kb + 8 (i/4) + 4 hi + i%4.  All of one block's operands are on their way before
  // its products begin, the next block's take their places.
  auto scores = [&](const u4_t* lk, f16_t (&st)[2]) {
    auto at = [&](int kb, int ks) { return *reinterpret_cast<const u4_t*>(reinterpret_cast<const char*>(lk) + ka[ks] + kb * 32 * CH * 16); };
    u4_t x[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) x[ks] = at(0, ks);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kb][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        st[kb] = mma32<BF>(x[ks], q[ks], st[kb]);
        if (kb == 0) x[ks] = at(1, ks);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x100, KS, 0);  // LDS reads
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, KS, 0);
  };
  // V^T's operand: dim 32 b + n, keys 16 kc + 8 (e/4) + 4 hi + e%4
  auto v_operand = [&](const u4_t* lv, int kc, int b) {
    u4_t y;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* at = reinterpret_cast<const char*>(lv) + va[b][h] + kc * 16 * CH * 16;
      const u2_t w = __builtin_bit_cast(
          u2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)at));
      y[2 * h] = w.x;
      y[2 * h + 1] = w.y;
    }
    return y;
  };
  // the running maximum over a tile (in both halves of the wave)
  auto maximum = [&](const f16_t (&st)[2]) {
    float x[4] = {m, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i % 4] = fmaxf(x[i % 4], st[kb][i]);
    const float y = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return fmaxf(__uint_as_float(z[0]), __uint_as_float(z[1]));
  };
  // Weights are relative to 2^base, base = RN(m c), m a maximum that is replaced when a row's has grown past it by 8 in
  // the exponent: weights stay below 2^8, and the accumulators are rescaled once or twice in a row's life.
  auto base_of = [&](float x) { return x == NEG_INF ? 0.f : x * a.c; };
  auto rescaled = [&](float mx) {  // base for a tile of maximum mx
    const bool grown = __any(mx > m + a.slack);
    mx = grown ? mx : m;
    const float base = base_of(mx);
    if (grown) {
      const float f = __builtin_amdgcn_exp2f(m == NEG_INF ? NEG_INF : base_of(m) - base);
      l *= f;
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] *= f;
    }
    m = mx;
    return base;
  };
  // exponents to weights: their sum into l, rounded and in pairs into p (keys as v_operand's)
  auto weigh = [&](f16_t (&st)[2], u4_t (&p)[4]) {
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[kb][i] = __builtin_amdgcn_exp2f(st[kb][i]);
        sum[i % 4] += st[kb][i];
      }
    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
    for (int kc = 0; kc < 4; ++kc)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[kc][i] = pack2<BF>(st[kc / 2][8 * (kc % 2) + 2 * i], st[kc / 2][8 * (kc % 2) + 2 * i + 1]);
  };
  auto products = [&](const u4_t* lv, const u4_t (&p)[4]) {
#pragma unroll
    for (int kc = 0; kc < 4; ++kc)
#pragma unroll
      for (int b = 0; b < DB; ++b) o[b] = mma32<BF>(v_operand(lv, kc, b), p[kc], o[b]);
  };

  // logits to weights.  One fma per logit leaves all weights of a row a common factor of 2^(the error of base), which the
  // sum shares; where base is so large that this shows in a rounded weight, logits are rounded as base is.
  auto softmax = [&](f16_t (&st)[2], u4_t (&p)[4]) {
    const float base = rescaled(maximum(st));
    float c = a.c;
    if (__any(fabsf(base) > 65536.f)) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) st[kb] *= a.c;
      c = 1.f;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[kb][i] = __builtin_fmaf(st[kb][i], c, -base);
    weigh(st, p);
  };

  // Any tile: keys that a row does not see have weight 0.
  // odd: V holds an infinity or NaN, which 0 * inf would carry into rows that do not see its key.
  auto any_tile = [&](int t, const u4_t* lk, const u4_t* lv, bool odd) {
    const int j0 = t * BN;
    // this wave's rows: does any see the tile, do all see all of it?
    const int va = tile * BM + wave * 32, wa = va / a.nrep, wz = min(va + 31, rows - 1) / a.nrep;
    const int w_last = a.causal ? min(wz + off + 1, keys) : keys, w_first = a.window ? max(wa + off + 1 - a.window, 0) : 0;
    if (va >= rows || w_last <= j0 || w_first >= j0 + BN) return;
    const bool mask = (a.causal ? min(wa + off + 1, keys) : keys) < j0 + BN || (a.window && wz + off + 1 - a.window > j0);
    f16_t st[2];
    scores(lk, st);
    if (mask) {
      const int z = last - j0 - 4 * hi, f = first - j0 - 4 * hi;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[kb][i] = 32 * kb + 8 * (i / 4) + i % 4 >= z ? NEG_INF : st[kb][i];
      if (a.window) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) st[kb][i] = 32 * kb + 8 * (i / 4) + i % 4 < f ? NEG_INF : st[kb][i];
      }
    }
    u4_t p[4];
    softmax(st, p);
    if (!mask || !odd) {
      products(lv, p);
      return;
    }
    // key by key, into the rows that see it
#pragma clang loop unroll(disable)
    for (int key = 0; key < BN; ++key) {
      const int at = key / 16 * 4 + key % 16 / 8 * 2 + key % 4 / 2, of = key % 8 / 4;  // p's word, in the lanes hi == of
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i == at) w = p[i / 4][i % 4];
      const auto y = __builtin_amdgcn_permlane32_swap(w, w, false, false);
      w = of ? y[1] : y[0];
      const float pk = key & 1 ? hi_half<BF>(w) : lo_half<BF>(w);
      if (j0 + key < last && j0 + key >= first) {
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const u2_t x = reinterpret_cast<const u2_t*>(&lv[chunk_at<D>(key, 4 * b + i)])[hi];
            const uint32_t x0 = x.x, x1 = x.y;
            o[b][4 * i] = __builtin_fmaf(pk, lo_half<BF>(x0), o[b][4 * i]);
            o[b][4 * i + 1] = __builtin_fmaf(pk, hi_half<BF>(x0), o[b][4 * i + 1]);
            o[b][4 * i + 2] = __builtin_fmaf(pk, lo_half<BF>(x1), o[b][4 * i + 2]);
            o[b][4 * i + 3] = __builtin_fmaf(pk, hi_half<BF>(x1), o[b][4 * i + 3]);
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
  int i = 0;
  auto whole_tile = [&](const u4_t* lk, const u4_t* lv) {
    f16_t st[2];
    u4_t p[4];
    scores(lk, st);
    softmax(st, p);
    products(lv, p);
  };
  // This wave's loads to LDS are there.  Every barrier that hands a tile over is behind such a wait: the compiler's own
  // does not cover them on all paths.
  auto arrived = [&] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
  if (count > 0) fetch(tile_at(0), lk0, lv0);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = (q[ks] & a.keep) ^ a.sign;  // (the queries arrive with the first tile)
  while (i < nw) {
    arrived();
    __syncthreads();  // the tile is there, and no wave reads the other buffer any more
    if (i + 1 < count) fetch(tile_at(i + 1), lk1, lv1);
    whole_tile(lk0, lv0);
    if (++i >= nw) break;
    arrived();
    __syncthreads();
    if (i + 1 < count) fetch(tile_at(i + 1), lk0, lv0);
    whole_tile(lk1, lv1);
    ++i;
  }
  for (; i < count; ++i) {
    u4_t *lk = i & 1 ? lk1 : lk0, *lv = i & 1 ? lv1 : lv0;
    // each wave looks through the part of V that it has loaded itself for infinities and NaN
    arrived();
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
      const u4_t w = lv[c * THREADS + threadIdx.x];
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
    odd = __builtin_amdgcn_readfirstlane(odd);
    if (i + 1 < count) fetch(tile_at(i + 1), i & 1 ? lk0 : lk1, i & 1 ? lv0 : lv1);
    any_tile(tile_at(i), lk, lv, odd);
  }
  {
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(y[0]) + __uint_as_float(y[1]);
  }
  // Rows leave through LDS: 16 lanes write a whole row of 128 dims, where a lane's own dims are 8 bytes here and there.
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __syncthreads();  // nobody reads tiles any more
  u4_t* const lo = (wave < 2 ? lk0 : lk1) + (wave & 1) * 32 * CH;
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<u2_t*>(lo + chunk_at<D>(n, 4 * b + i))[hi] =
          u2_t{pack2<BF>(o[b][4 * i] * inv, o[b][4 * i + 1] * inv), pack2<BF>(o[b][4 * i + 2] * inv, o[b][4 * i + 3] * inv)};
  wave_lds_sync();
  const int64_t at = int64_t(q0 + row) * a.so_n + head * a.so_h;
  const int at0 = int(at), at1 = int(at >> 32);
#pragma unroll
  for (int j = 0; j < CH / 2; ++j) {
    const int r = j * (64 / CH) + lane / CH, c = lane % CH;  // row and chunk
    const int64_t to = int64_t(uint32_t(__shfl(at0, r, 64))) | int64_t(__shfl(at1, r, 64)) << 32;
    if (tile * BM + wave * 32 + r < rows) *reinterpret_cast<u4_t*>(a.out + to + 8 * c) = lo[chunk_at<D>(r, c)];
  }
}

}  // namespace

extern "C" int iq_prompt_attention(const void* q, int64_t sq_n, int64_t sq_h, const void* k, int64_t sk_n, int64_t sk_h,
                                   const void* v, int64_t sv_n, int64_t sv_h, const int32_t* cu_q, const int32_t* cu_k,
                                   int S, int N, int Nk, int Hq, int H, int D, int mode, float scale, int causal, int window,
                                   void* out, int64_t so_n, int64_t so_h, void* stream) {
  IQ_CHECK(cu_q && cu_k && (N == 0 || (q && out)) && (Nk == 0 || (k && v)), IQ_ERR_NULL);
  IQ_CHECK(base_mode(mode) == 0, IQ_ERR_MODE);
  IQ_CHECK(d_ok(D) && H > 0 && Hq > 0 && Hq % H == 0 && Hq <= 4096 && S > 0 && N >= 0 && Nk >= 0 && window >= 0, IQ_ERR_SHAPE);
  IQ_CHECK(!window || causal, IQ_ERR_MODE);
  for (const int64_t s : {sk_n, sv_n}) IQ_CHECK(s >= 0 && s < (1 << 23), IQ_ERR_SHAPE);  // a tile of rows in 32 bits
  for (const int64_t s : {sq_n, sq_h, sk_n, sk_h, sv_n, sv_h, so_n, so_h}) IQ_CHECK(s % 8 == 0, IQ_ERR_ALIGN);
  IQ_CHECK(aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && aligned(out, 16) && aligned(cu_q, 4) && aligned(cu_k, 4),
           IQ_ERR_ALIGN);
  if (N == 0) return IQ_OK;
  const int64_t rows = int64_t(N) * (Hq / H);
  IQ_CHECK(rows <= INT32_MAX - BM && int64_t(N) + Nk <= INT32_MAX, IQ_ERR_SHAPE);
  const int64_t slots = rows / BM + S;  // first_slot(S) at most
  IQ_CHECK(slots * H <= UINT32_MAX / THREADS, IQ_ERR_SHAPE);
  if (window >= Nk) window = 0;  // hides nothing
  const float c = scale * 1.44269504088896340736f, abs_c = c == 0 ? 1.f : c < 0 ? -c : c;
  PromptArgs a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, (uint16_t*)out, sq_n, sq_h, sk_n, sk_h, sv_n,
               sv_h, so_n, so_h, cu_q, cu_k, S, N, Nk, Hq, Hq / H, int(slots), abs_c, 8.f / abs_c, c == 0 ? 0u : ~0u,
               c < 0 ? 0x80008000u : 0u, causal ? 1 : 0, window};
  auto launch = [&]<int D_, bool BF>() {
    prompt_kernel<D_, BF><<<unsigned(slots * H), THREADS, 0, (hipStream_t)stream>>>(a);
    return launch_status();
  };
  const bool bf = act_bf16(mode);
  if (D == 128) return bf ? launch.operator()<128, true>() : launch.operator()<128, false>();
  return bf ? launch.operator()<64, true>() : launch.operator()<64, false>();
}
