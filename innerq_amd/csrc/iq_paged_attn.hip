// Attention of one or a few new tokens per sequence over 4-bit pages (gfx950): iq_paged_attention.
//
// Flash decoding over a ragged batch: the pages of all (sequence, KV head, tile of query rows), each with PAD
// units before them, lie behind one another in one list, which the workgroups share out evenly (read from the
// sequences' lengths on the device, so a captured call follows them); a workgroup's four waves take its pages in
// turn, each with its own running maximum, sum and accumulators, merged over LDS at the end of each (sequence, head).
// Where a (sequence, head) spans several workgroups, their fp32 partials go to the workspace and a second launch
// merges them in a fixed order.
//
// One page, one wave: K's words become the A operands of v_mfma_f32_16x16x32 (16 tokens x 32 dims; the B operand is
// the query rows, held in registers), whose result has a query row per lane and 4 tokens per lane; its exponentials,
// rounded to the activation dtype, are the B operand of V^T P^T as they are (iq_paged.h's V blocks).  The codes go
// from memory to registers, one page ahead; LDS only merges the waves.
//
// Bound (8 KV heads, 32 query heads, D = 128): long sequences in fp16 by HBM and the vector unit alike (8 of 32768
// tokens: 336 MB in 63 us with the merge, 5.3 TB/s, where a large copy reaches 4.8; a wave spends about 1.3 us on a
// page); in bf16 by the conversion of the codes (48 of 130 .. 16001 tokens: 78 us, in fp16 62 us); short ones by the
// loads that wait for each other, lengths, table, page (one sequence of 1000 tokens: 10.4 us, 3.5 the merging launch).
//
// Keys' weights (iq_paged_attention_weights): a row's sum is known behind its last page, so the logits go to the workspace,
// 4 bytes per query head and token where the codes of a key that four heads share are 80, and the second launch reads them
// back beside its merging (weigh_pages).  The logits of 4 tokens and all heads lie side by side, so that lanes write whole
// lines.  8 sequences of 32768 tokens, fp16: 77 us (61 with stores that reach no memory) and 16 for merge and weights, 336 MB of
// pages and 34 MB of logits twice; 48 of 286 .. 16001, bf16: 86 - 91 and 17, the vector unit busy 47 % of the clocks.
//
// Differential attention (iq_diff_paged_attention, at the end): both maps of a pair of heads in one workgroup, so that V's
// codes are read and converted once.  8 sequences of 32768 tokens, 32 query heads over 8, D = 64, fp16: 168 MB in 40 us, the
// rate of a large copy (with the keys' weights 48 and 15); 3 new tokens on 24 of 93 .. 6001, D = 128, bf16: 39 and 6 for the
// merge, bound by no unit: a wave holds both maps' sums over 2 D dims, so that a SIMD has one wave, whose loads, conversions,
// products and exponentials follow one another with nothing beside them (vector unit busy 33 % of the clocks, matrix unit 5 %).
//
// The exponentials are rounded because the matrix unit's two operands have one type, that of V's values: each weight
// moves by half a step at most, and its sum takes it unrounded (outputs' error 1.1 - 1.4 times that of fp32 weights,
// against 64 bits).
#include "iq_paged.h"

using namespace iq;

namespace {

constexpr int WAVES = SHARE_LEAST, THREADS = 64 * WAVES, ROWS = 16;  // rows of an MFMA operand: a tile has T times as many
// What a (sequence, head, tile) costs beside its pages, in pages: its queries, its first page's latency and the
// merge of the waves.  Counted where the workgroups share out the list; without it a workgroup whose share was many
// short sequences came last (48 sequences of 130 .. 16001 tokens, bf16: 181 us against 82).
constexpr int PAD = 8;
constexpr float NEG_INF = -__builtin_inff();

struct AttnArgs {
  iq_paged p;
  const uint16_t* q;
  int64_t sq_s, sq_m, sq_h;
  uint16_t* out;
  int64_t so_s, so_m, so_h;
  int heads;           // KV heads, or pairs of them (MAPS = 2)
  int m, nrep, tiles;  // new tokens per sequence, (output) heads per KV head or pair, tiles of rows (row = token * nrep + head)
  float scale;         // times log2(e)
  int window;          // 0: none
  int grid;
  float* ws;
  int each;            // sequences per lane where a wave adds up their pages (Part)
  int split;           // 0: a workgroup takes a whole (sequence, head, tile)
  const float* lam;    // of each output head (MAPS = 2)
  int64_t s_lam;
  // where the keys' weights are wanted (m = 1): the logits [S][H][P][16][nrep][4 tokens], {maximum, 1 / sum} of each
  // row [S][H][nrep], and the weights to add to, fp32 [S][H][>= 64 P]
  float* logits;
  float2* stats;
  float* weights;
  int64_t sw_s, sw_h;
  int items, weigh_each;  // workgroups of the second launch that merge; pages of one that weighs
};

// pages that sequence s reads: [lo, lo + n)
__device__ __forceinline__ int pages_of(const AttnArgs& a, int s, int& lo) {
  const int len = min(a.p.lens[s], a.p.P * PAGE);
  lo = a.window ? max(0, len - a.m + 1 - a.window) / PAGE : 0;
  return len > 0 ? (len + PAGE - 1) / PAGE - lo : 0;
}

// Where a lane's `each` sequences from s0 + each * lane on end in the list of units (a unit: a page of one head and
// tile), `base` the units before s0; n: the sequences' units.  A lane takes one sequence where there are at most 64,
// four (their loads under way together) where there are more.  One / four, 2 KV heads: 64 sequences of 1000 tokens
// 16.4 / 17.2 us, 128 21.4 / 21.7, 512 of 600 38 / 36.
constexpr int EACH = 4;
struct Part {
  int n[EACH], end;
};
__device__ __forceinline__ Part part_at(const AttnArgs& a, int s0, int base) {
  Part p;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    p.n[i] = 0;
    if (i >= a.each) continue;
    int lo;
    const int s = s0 + int(threadIdx.x & 63) * a.each + i, pages = pages_of(a, min(s, a.p.S - 1), lo);
    p.n[i] = s < a.p.S && pages > 0 ? (pages + PAD) * a.heads * a.tiles : 0;
    sum += p.n[i];
  }
  p.end = base + wave_scan(sum);
  return p;
}
__device__ __forceinline__ int total_units(const AttnArgs& a, const Part& first) {
  int end = __builtin_amdgcn_readlane(first.end, 63);
  for (int s0 = 64 * a.each; s0 < a.p.S; s0 += 64 * a.each) end = __builtin_amdgcn_readlane(part_at(a, s0, end).end, 63);
  return end;
}
// of the lane that holds sequence s: its units, and the unit after them
__device__ __forceinline__ void units_of(const AttnArgs& a, const Part& p, int s, int& n, int& end) {
  const int l = s / a.each % 64, k = s % a.each;
  end = __builtin_amdgcn_readlane(p.end, l);
  n = 0;
#pragma unroll
  for (int i = EACH - 1; i >= 0; --i) {
    const int x = __builtin_amdgcn_readlane(p.n[i], l);
    if (i > k) end -= x;
    if (i == k) n = x;
  }
}
// the sequence that holds unit u < total, and its first unit
__device__ __forceinline__ void find_unit(const AttnArgs& a, Part p, int u, int& s, int& first) {
  for (int s0 = 0;;) {
    const uint64_t past = __ballot(p.end > u);
    if (past) {
      s = s0 + __builtin_ctzll(past) * a.each + a.each - 1;  // the lane's last one that begins at or before u
      for (int n, end;; --s) {
        units_of(a, p, s, n, end);
        first = end - n;
        if (first <= u && n > 0) return;
      }
    }
    s0 += 64 * a.each;
    if (s0 >= a.p.S) return;
    p = part_at(a, s0, __builtin_amdgcn_readlane(p.end, 63));
  }
}
// Rows.  A tile has R rows of MAPS maps: T groups of 16 columns of the matrix unit's operand, column c being row c % R of
// map c / R.  (Differential attention: up to 8 rows of both maps share a group, more have a group for each map.)
template <int T, int MAPS>
constexpr int tile_rows() { return ROWS * T / MAPS; }
// row r of tile t of sequence s: its query head offset (head in the group, token)
struct Row {
  int token, head;
  bool real;
};
template <int R>
__device__ __forceinline__ Row row_of(const AttnArgs& a, int tile, int r) {
  const int i = tile * R + r, token = i / a.nrep;
  return {token, i - token * a.nrep, token < a.m};
}

// one lane's part of a page: its K words and meta (4 tiles of 16 tokens), its V words and meta (2 blocks)
struct KRegs {
  u4_t c[4];  // D = 64: two words used
  uint32_t m[4];
};
struct VRegs {
  u4_t c[2][2], s[2], z[2];
};

// A page is read through a buffer descriptor of its own (one page's bytes; none for a page outside the pool): lane
// offsets stay in 32 bits and the offsets within a page in the instructions' immediates.  Each byte is read once: the
// loads leave the caches to others (8 sequences of 32768 tokens, caches full of other data before each call: 68 us
// against 73 when measured, 48 of 130 .. 16001 tokens 79 against 84; a small cache called again and again is 2 % slower).
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr int STREAM = 2;  // non-temporal

template <int D>
struct Lane {
  uint32_t kc, km, vc, vm;  // the lane's byte offsets into a page
  __device__ __forceinline__ Lane() {
    constexpr int U = D / 8, G = D / 32;
    const uint32_t lane = threadIdx.x & 63, l = lane & 15, quarter = lane >> 4;
    const uint32_t octet = D == 128 ? l : l / 2;
    kc = (l * U + quarter * (U / 4)) * 4;
    km = (page_km(D) + l * G + (D == 128 ? quarter : quarter / 2)) * 4;
    vc = (page_vc(D) + (quarter * U + octet) * 8) * 4;
    vm = (page_vm(D) + (quarter * G + octet / 4) * 8) * 4;
  }
};
__device__ __forceinline__ u4_t bload4(rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, STREAM));
}

template <int D>
__device__ __forceinline__ void load_k(rsrc_t pg, const Lane<D>& at, KRegs& r) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t c = at.kc + t * 16 * (D / 8) * 4;
    if constexpr (D == 128) {
      r.c[t] = bload4(pg, c);
    } else {
      const u2_t x = __builtin_bit_cast(u2_t, __builtin_amdgcn_raw_buffer_load_b64(pg, c, 0, STREAM));
      r.c[t] = u4_t{x.x, x.y, 0, 0};
    }
    r.m[t] = __builtin_amdgcn_raw_buffer_load_b32(pg, at.km + t * 16 * (D / 32) * 4, 0, STREAM);
  }
}
template <int D>
__device__ __forceinline__ void load_v(rsrc_t pg, const Lane<D>& at, VRegs& r) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t c = at.vc + h * 4 * (D / 8) * 32, m = at.vm + h * 4 * (D / 32) * 32;
    r.c[h][0] = bload4(pg, c);
    r.c[h][1] = bload4(pg, c + 16);
    r.s[h] = bload4(pg, m);
    r.z[h] = bload4(pg, m + 16);
  }
}

template <bool BF>
__device__ __forceinline__ f4_t mma(u4_t a, u4_t b, f4_t c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
}

// the A operands of V^T for 32 tokens: x[j] holds, for the lane's dim j, its 8 tokens (D/16 dims per lane)
template <int D, bool BF>
__device__ __forceinline__ void v_operands(const u4_t (&c)[2], u4_t s, u4_t z, u4_t (&x)[D / 16]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int pr = 0; pr < 4; ++pr) {  // tokens 2 pr, 2 pr + 1
    const uint32_t w0 = c[pr / 2][pr % 2 * 2], w1 = c[pr / 2][pr % 2 * 2 + 1];
    const uint32_t sp = s[pr], zp = z[pr];  // (a bit_cast of a vector's element would take its first one)
#pragma unroll
    for (int half = 0; half < D / 64; ++half) {
      uint32_t f;  // 4 dims of the two tokens, two dims of each token in turn in a byte
      if constexpr (D == 128) f = __builtin_amdgcn_perm(w1, w0, half ? 0x07030602u : 0x05010400u);
      else f = __builtin_amdgcn_perm(w1, w0, lane & 1 ? 0x07030602u : 0x05010400u);
      const u2_t e = values4<BF>(f & 0x0f0f0f0fu, sp, zp), o = values4<BF>((f >> 4) & 0x0f0f0f0fu, sp, zp);
      const uint32_t e0 = e.x, e1 = e.y, o0 = o.x, o1 = o.y;
      x[half * 4][pr] = e0;
      x[half * 4 + 1][pr] = o0;
      x[half * 4 + 2][pr] = e1;
      x[half * 4 + 3][pr] = o1;
    }
  }
}

template <int D, bool BF, int MAPS>
struct Acc {
  f4_t o[MAPS * D / 16];  // of V head h: o[h D/16 + j], dims row * D/16 + j of column lane % 16, row = lane/16 * 4 + i
  float m, l;
};

// the logits of a page's 64 tokens: s[g][t][i] of token 16 t + 4 (lane/16) + i for column 16 g + lane % 16
template <int D, bool BF, int T, int MAPS, int NQ>
__device__ __forceinline__ void logits(const KRegs (&r)[MAPS], const u4_t (&q)[NQ][D / 32], float scale, f4_t (&s)[T][4]) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    f4_t x[NQ];
#pragma unroll
    for (int g = 0; g < NQ; ++g) x[g] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < MAPS; ++h)
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const u4_t k = k_values<BF>(r[h].c[t][j], r[h].m[t]);
#pragma unroll
        for (int g = 0; g < NQ; ++g)
          if (MAPS == 1 || g == h) x[g] = mma<BF>(k, q[g][j], x[g]);
      }
    // (two maps in one group of columns: each had all columns, so that no value of one's keys meets the other's)
    if constexpr (MAPS == 2 && T == 1) s[0][t] = (threadIdx.x & 15) < 8 ? x[0] : x[1];
    else
#pragma unroll
      for (int g = 0; g < T; ++g) s[g][t] = x[g];
#pragma unroll
    for (int g = 0; g < T; ++g) s[g][t] *= scale;
    __builtin_amdgcn_sched_barrier(0);
  }
}

// the running softmax over 64 more logits; s becomes the weights
template <int D, bool BF, int MAPS>
__device__ __forceinline__ void weights(f4_t (&s)[4], Acc<D, BF, MAPS>& acc) {
  float mx = acc.m;
#pragma unroll
  for (int t = 0; t < 4; ++t) mx = fmaxf(mx, fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])));
  {
    auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    x = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    mx = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  }
  const float base = mx == NEG_INF ? 0.f : mx;  // a row that has seen nothing yet
  if (__any(mx != acc.m)) {
    const float f = __builtin_amdgcn_exp2f(acc.m - base);
    acc.l *= f;
#pragma unroll
    for (int j = 0; j < MAPS * D / 16; ++j) acc.o[j] *= f;
    acc.m = mx;
  }
  float sum = 0.f;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[t][i] = __builtin_amdgcn_exp2f(s[t][i] - base);
      sum += s[t][i];
    }
  acc.l += sum;
}

// is any value of the tokens with these scales and zeros (pairs) an infinity or NaN?  It is where z or 15 s + z is.
template <bool BF>
__device__ __forceinline__ bool odd_values(uint32_t s, uint32_t z) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float zz = i ? hi_half<BF>(z) : lo_half<BF>(z), ss = i ? hi_half<BF>(s) : lo_half<BF>(s);
    const float top = __builtin_fmaf(15.f, ss, zz);
    const uint32_t t = pack2<BF>(top, zz);  // rounded as the values are
    const uint32_t e = BF ? 0x7f80u : 0x7c00u;
    odd |= (t & e) == e || ((t >> 16) & e) == e;
  }
  return odd;
}

// Readies 32 tokens of a page that not every row sees all of (k0: the first token's number; a row sees [low, lim),
// no row sees tokens outside [lo, len)): tokens that no row sees, whose page rows may hold anything, get values 0.
// A token whose values hold an infinity or NaN is taken by itself, into the rows that see it (the product would carry
// it into every row, as 0 * inf), and then gets values 0 too.
template <int D, bool BF, int T, int MAPS>
__device__ __forceinline__ void unseen_values(const u4_t (&c)[2], u4_t& s, u4_t& z, const u4_t (&p)[T],
                                              Acc<D, BF, MAPS> (&acc)[T], int o0, int k0, const int (&lim)[T], const int (&low)[T], int lo, int len) {
  const int quarter = (threadIdx.x & 63) >> 4;
  bool odd = false;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t keep = 0;
#pragma unroll
    for (int e = 2 * w; e < 2 * w + 2; ++e) {
      const int k = k0 + e / 4 * 16 + quarter * 4 + e % 4;
      if (k < len && k >= lo) keep |= e & 1 ? 0xffff0000u : 0x0000ffffu;
    }
    s[w] &= keep;
    z[w] &= keep;
    odd |= odd_values<BF>(s[w], z[w]);
  }
  if (!__any(odd)) return;
#pragma clang loop unroll(disable)
  for (int t = 0; t < 32; ++t) {
    const int qd = t / 8, e = t % 8, k = k0 + e / 4 * 16 + qd * 4 + e % 4;
    const uint32_t half = quarter == qd ? (e & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
    u4_t st, zt;
    odd = false;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t at = w == e / 2 ? half : 0u;
      st[w] = s[w] & at;
      zt[w] = z[w] & at;
      odd |= odd_values<BF>(st[w], zt[w]);
    }
    if (!__any(odd)) continue;
    u4_t x[D / 16];
    v_operands<D, BF>(c, st, zt, x);
#pragma unroll
    for (int g = 0; g < T; ++g) {
      const bool sees = k < lim[g] && k >= low[g];
      u4_t pt;
#pragma unroll
      for (int w = 0; w < 4; ++w) pt[w] = p[g][w] & (w == e / 2 ? half : 0u);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const f4_t y = mma<BF>(x[j], pt, acc[g].o[o0 + j]);
        if (sees) acc[g].o[o0 + j] = y;
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t at = w == e / 2 ? half : 0u;
      s[w] &= ~at;
      z[w] &= ~at;
    }
  }
}

// o0: the V head's first accumulator
template <int D, bool BF, int T, int MAPS>
__device__ __forceinline__ void values(VRegs& r, const f4_t (&s)[T][4], Acc<D, BF, MAPS> (&acc)[T], int o0, bool mask, int tok0,
                                       const int (&lim)[T], const int (&low)[T], int lo, int len) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u4_t p[T];
#pragma unroll
    for (int g = 0; g < T; ++g)
      p[g] = u4_t{pack2<BF>(s[g][2 * h][0], s[g][2 * h][1]), pack2<BF>(s[g][2 * h][2], s[g][2 * h][3]),
                  pack2<BF>(s[g][2 * h + 1][0], s[g][2 * h + 1][1]), pack2<BF>(s[g][2 * h + 1][2], s[g][2 * h + 1][3])};
    if (mask) unseen_values<D, BF, T, MAPS>(r.c[h], r.s[h], r.z[h], p, acc, o0, tok0 + h * 32, lim, low, lo, len);
    u4_t x[D / 16];
    v_operands<D, BF>(r.c[h], r.s[h], r.z[h], x);
#pragma unroll
    for (int j = 0; j < D / 16; ++j)
#pragma unroll
      for (int g = 0; g < T; ++g) acc[g].o[o0 + j] = mma<BF>(x[j], p[g], acc[g].o[o0 + j]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// a slot of the workspace: C = 16 T columns of W = MAPS D sums, C maxima, C sums of weights
template <int W, int C>
__device__ __forceinline__ float* slot_of(float* ws, int i) { return ws + int64_t(i) * (C * W + 2 * C); }

// R: rows of a tile
template <int D, bool BF, int R>
__device__ __forceinline__ void store_row(const AttnArgs& a, int s, int head, int tile, int r, int d, const float (&v)[8],
                                          float inv) {
  const Row w = row_of<R>(a, tile, r);
  if (!w.real) return;
  u4_t x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = pack2<BF>(v[2 * i] * inv, v[2 * i + 1] * inv);
  *reinterpret_cast<u4_t*>(a.out + s * a.so_s + w.token * a.so_m + (int64_t(head) * a.nrep + w.head) * a.so_h + d) = x;
}

// workgroups per CU (registers: D = 128 with T = 2 would spill 209 of them at two.  Spilled as it is: D = 64 with T = 2 6
// registers, 31 in bf16, and D = 128 with T = 1 in bf16 22, in the masked path and where a (sequence, head) begins and
// ends; D = 64 is faster so: 48 of 1500 tokens, bf16, 26 us against 30)
// Two maps: one, so that none spills (8 sequences of 16384 tokens, D = 128, at two / one: fp16 85 / 49 us, bf16 117 / 55; 3 new
// tokens on 24 of 60 .. 6001, D = 64: 53 / 29; 8 of 32768, D = 64: 51 / 49).
constexpr int per_cu(int D, int T, int maps) { return maps == 1 && (T == 1 || D == 64) ? 2 : 1; }

// the second map's factor of row r of a tile, negated
template <int R>
__device__ __forceinline__ float minus_lam(const AttnArgs& a, int head, int tile, int r) {
  const Row w = row_of<R>(a, tile, r);
  return w.real ? -a.lam[(int64_t(head) * a.nrep + w.head) * a.s_lam] : 0.f;
}

// a row's softmax, for the keys' weights: {maximum, 1 / sum}; a row without a sum gives weights of 0
__device__ __forceinline__ float2 row_stats(float mx, float sum) {
  return {mx == NEG_INF ? 0.f : mx, sum == 0.f ? 0.f : 1.f / sum};
}
__device__ __forceinline__ void store_stats(const AttnArgs& a, int s, int head, int r, float mx, float sum) {
  if (r < a.nrep) a.stats[(int64_t(s) * a.p.H + head) * a.nrep + r] = row_stats(mx, sum);  // (head: of the store)
}

// W: the logits and the rows' sums are kept, for weigh_pages.  MAPS = 2: differential attention (see the end of the
// file): KV heads in pairs, whose keys are the two maps' and whose V heads are the halves of one of 2 D dims.
template <int D, bool BF, int T, bool W, int MAPS>
__global__ __launch_bounds__(THREADS, per_cu(D, T, MAPS)) void attn_kernel(AttnArgs a) {
  constexpr int J = D / 16, C = ROWS * T, R = tile_rows<T, MAPS>(), DV = MAPS * D, NQ = MAPS == 1 ? T : MAPS;
  __shared__ float so[WAVES][C][DV + 4];
  __shared__ float sm[WAVES][C], sl[WAVES][C];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 15,
            quarter = lane >> 4;
  const int H = a.heads;
  int u, u1, s = 0, first = 0;
  if (a.split) {
    const Part part = part_at(a, 0, 0);
    const int total = total_units(a, part), per = units_per_group(total, a.grid);
    u = share_begin(blockIdx.x, per, total);
    u1 = share_begin(blockIdx.x + 1, per, total);
    if (u < u1) find_unit(a, part, u, s, first);
  } else {
    s = blockIdx.x / (H * a.tiles);
    int lo;
    const int n = pages_of(a, s, lo);
    u = first = 0;
    const int hr = blockIdx.x - s * H * a.tiles;
    u = hr * (n + PAD);
    u1 = n > 0 ? u + n + PAD : u;
  }
  // sequences without tokens: rows of zeros
  for (int e = a.split ? blockIdx.x : s; e < (a.split ? a.p.S : s + 1); e += a.grid) {
    int lo;
    if (pages_of(a, e, lo) > 0) continue;
    if (a.p.lens[e] < 0 && threadIdx.x == 0) atomicOr(a.p.status, PAGED_BAD_TOKEN);
    const float zero[8] = {};
    const int rows = a.m * a.nrep, nh = a.split ? H : 1;
    for (int i = threadIdx.x; i < nh * rows * (DV / 8); i += THREADS) {
      const int d = i % (DV / 8) * 8, r = i / (DV / 8) % rows;
      const int h = a.split ? i / (DV / 8) / rows : blockIdx.x / a.tiles % H;
      store_row<D, BF, R>(a, e, h, r / R, r % R, d, zero, 0.f);
    }
  }
  while (u < u1) {
    int lo;
    int n = __builtin_amdgcn_readfirstlane(pages_of(a, s, lo));
    if (n <= 0) { ++s; continue; }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int hr = (u - first) / (n + PAD), x0 = (u - first) - hr * (n + PAD), x1 = min(n + PAD, x0 + u1 - u);
    const int p0 = max(x0 - PAD, 0), cnt = x1 - PAD - p0;  // this workgroup's pages of the head and tile
    u += x1 - x0;
    const bool over = a.split && u - first >= (n + PAD) * H * a.tiles;
    if (cnt <= 0) continue;
    const int head = hr / a.tiles, tile = hr - head * a.tiles;
    const int len = __builtin_amdgcn_readfirstlane(min(a.p.lens[s], a.p.P * PAGE));
    // the query rows of this lane's columns (16 g + l), their octets in the order of k_values' pairs
    u4_t q[NQ][D / 32];  // (rows past the last repeat it and are not stored)
    int lim[T], low[T];  // a column's row sees keys [low, lim)
    Acc<D, BF, MAPS> acc[T];
#pragma unroll
    for (int g = 0; g < NQ; ++g) {
      const Row row = row_of<R>(a, tile, MAPS == 1 ? ROWS * g + l : l % R);
      const int token = min(row.token, a.m - 1), h = row.real ? row.head : a.nrep - 1;
      const uint16_t* x = a.q + s * a.sq_s + token * a.sq_m +
                          ((int64_t(head) * a.nrep + h) * MAPS + (MAPS == 1 ? 0 : g)) * a.sq_h + quarter * (D / 4);
      u4_t w[D / 32];
#pragma unroll
      for (int j = 0; j < D / 32; ++j) w[j] = *reinterpret_cast<const u4_t*>(x + 8 * j);
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          q[g][j][e] = __builtin_amdgcn_perm(w[j][e % 2 * 2 + 1], w[j][e % 2 * 2], e / 2 ? 0x07060302u : 0x05040100u);
    }
#pragma unroll
    for (int g = 0; g < T; ++g) {
      const Row row = row_of<R>(a, tile, (ROWS * g + l) % R);
      lim[g] = len - (a.m - 1 - row.token);
      low[g] = a.window ? lim[g] - a.window : 0;
#pragma unroll
      for (int j = 0; j < MAPS * J; ++j) acc[g].o[j] = f4_t{0.f, 0.f, 0.f, 0.f};
      acc[g].m = NEG_INF;
      acc[g].l = 0.f;
    }
    // (read as constants, by scalar loads: a vector load here would wait for the pages under way)
    typedef const __attribute__((address_space(4))) int32_t* consts_t;
    const consts_t table = (consts_t)(a.p.table + s * a.p.s_table + lo + p0);
    const int mine = wave < cnt ? (cnt - wave + WAVES - 1) / WAVES : 0;  // this wave's pages: wave, wave + WAVES, ...
    const uint32_t* pages = a.p.pages + int64_t(head) * MAPS * page_words(D);
    const int64_t stride = int64_t(a.p.H) * page_words(D);
    // the page of the wave's turn i: one outside the pool is not read and counts as NaN
    bool bad = false;
    if (a.p.lens[s] > a.p.P * PAGE) {  // more tokens than the table has pages for: NaN too
      bad = true;
      if (threadIdx.x == 0) atomicOr(a.p.status, PAGED_BAD_TOKEN);
    }
    // past its last page a wave loads from a descriptor of no bytes: the loop has no branch that a load depends on,
    // which the wait counts would have to allow for
    auto id_of = [&](int i) { return i < mine ? table[wave + i * WAVES] : 0; };
    struct Page {
      rsrc_t head[MAPS];
    };
    auto page_of = [&](int id, bool there) {
      const bool b = id < 0 || id >= a.p.n_pages;
      if (b && there) {
        bad = true;
        if (lane == 0) atomicOr(a.p.status, PAGED_BAD_PAGE);
      }
      Page pg;
#pragma unroll
      for (int h = 0; h < MAPS; ++h)
        pg.head[h] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint32_t*>(pages + (b ? 0 : id) * stride + h * page_words(D)),
                                                       0, b || !there ? 0 : page_words(D) * 4, 0x00020000);
      return pg;
    };
    // K of the next page is on its way from the moment this page's logits are done, V from its product's end
    const Lane<D> at;
    KRegs kr[MAPS];
    VRegs vr[MAPS];
    {
      const Page pg = page_of(id_of(0), mine > 0);
#pragma unroll
      for (int h = 0; h < MAPS; ++h) load_k<D>(pg.head[h], at, kr[h]);
#pragma unroll
      for (int h = 0; h < MAPS; ++h) load_v<D>(pg.head[h], at, vr[h]);
    }
    uint32_t keep_at[T];  // where the columns' logits go, in bytes from the page's; past the descriptor's end: nowhere
    if constexpr (W)
#pragma unroll
      for (int g = 0; g < T; ++g) {
        const int c = ROWS * g + l, r = tile * R + c % R;
        keep_at[g] = r < a.nrep ? uint32_t(c / R) * uint32_t(a.p.P) * a.nrep * (PAGE * 4) + (quarter * a.nrep + r) * 16 : 1u << 31;
      }
    const int keep_bytes = ((C / R - 1) * a.p.P + 1) * a.nrep * (PAGE * 4);  // to the end of the last column's map's page
    const int see0 = a.window ? max(0, len - a.m + 1 - a.window) : 0;  // the first key that any row sees
    int id = id_of(1);
    for (int i = 0; i < mine; ++i) {
      const int tok0 = (lo + p0 + wave + i * WAVES) * PAGE;
      const bool mask = tok0 + PAGE > len - a.m + 1 || (a.window && tok0 < len - a.window);
      f4_t w[T][4];
      logits<D, BF, T, MAPS, NQ>(kr, q, a.scale, w);
      const Page next = page_of(id, i + 1 < mine);
      id = id_of(i + 2);
#pragma unroll
      for (int h = 0; h < MAPS; ++h) load_k<D>(next.head[h], at, kr[h]);
      if (mask) {
#pragma unroll
        for (int g = 0; g < T; ++g)
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int k = tok0 + t * 16 + quarter * 4 + e;
              if (k >= lim[g] || k < low[g]) w[g][t][e] = NEG_INF;
            }
      }
      if constexpr (W) {  // (whole lines: the rows of 4 tokens lie side by side; no branch, as with the loads)
        const int64_t first = ((int64_t(s) * a.p.H + head * MAPS) * a.p.P + tok0 / PAGE) * a.nrep * PAGE;
        const rsrc_t d = __builtin_amdgcn_make_buffer_rsrc(a.logits + first, 0, keep_bytes, 0x00020000);
#pragma unroll
        for (int g = 0; g < T; ++g)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4_t, w[g][t]), d, keep_at[g], t * 64 * a.nrep, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int g = 0; g < T; ++g) weights<D, BF, MAPS>(w[g], acc[g]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < MAPS; ++h) {
        values<D, BF, T, MAPS>(vr[h], w, acc, h * J, mask, tok0, lim, low, see0, len);
        load_v<D>(next.head[h], at, vr[h]);
      }
    }
    // the waves' sums
#pragma unroll
    for (int g = 0; g < T; ++g) {
      float sum = bad ? __builtin_nanf("") : acc[g].l;
      auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
      sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
      x = __builtin_amdgcn_permlane16_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
      sum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
      if (quarter == 0) {
        sm[wave][ROWS * g + l] = acc[g].m;
        sl[wave][ROWS * g + l] = sum;
      }
#pragma unroll
      for (int h = 0; h < MAPS; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < J; j += 4)
            *reinterpret_cast<f4_t*>(&so[wave][ROWS * g + l][h * D + (quarter * 4 + i) * J + j]) =
                f4_t{acc[g].o[h * J + j][i], acc[g].o[h * J + j + 1][i], acc[g].o[h * J + j + 2][i], acc[g].o[h * J + j + 3][i]};
    }
    __syncthreads();
    const bool whole = cnt == n;
    float* slot = whole ? nullptr : slot_of<DV, C>(a.ws, 2 * blockIdx.x + (p0 == 0 ? 1 : 0));
    // 8 dims of a column over the waves
    auto merge = [&](int c, int d, float& mx, float& sum, float (&v)[8]) {
      mx = NEG_INF;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) mx = fmaxf(mx, sm[w][c]);
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float f = sm[w][c] == NEG_INF ? 0.f : exp2f(sm[w][c] - mx);
        sum += sl[w][c] == 0.f ? 0.f : sl[w][c] * (sl[w][c] != sl[w][c] ? 1.f : f);
        if (f != 0.f)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += f * so[w][c][d + e];
      }
    };
    for (int i = threadIdx.x; i < (MAPS == 2 && whole ? R : C) * (DV / 8); i += THREADS) {
      const int rr = i / (DV / 8), d = i % (DV / 8) * 8;
      float mx, sum, v[8];
      merge(rr, d, mx, sum, v);
      if (whole) {
        if constexpr (W)
          if (d == 0) store_stats(a, s, head * MAPS, tile * R + rr, mx, sum);
        float inv = sum == 0.f ? 0.f : 1.f / sum;
        if constexpr (MAPS == 2) {
          float mx2, sum2, v2[8];
          merge(R + rr, d, mx2, sum2, v2);
          if constexpr (W)
            if (d == 0) store_stats(a, s, head * MAPS + 1, tile * R + rr, mx2, sum2);
          const float f = minus_lam<R>(a, head, tile, rr) * (sum2 == 0.f ? 0.f : 1.f / sum2);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = v[e] * inv + f * v2[e];
          inv = 1.f;
        }
        store_row<D, BF, R>(a, s, head, tile, rr, d, v, inv);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) slot[rr * DV + d + e] = v[e];
        if (d == 0) {
          slot[C * DV + rr] = mx;
          slot[C * DV + C + rr] = sum;
        }
      }
    }
    __syncthreads();
    if (over) {
      first += (n + PAD) * H * a.tiles;
      ++s;
    }
  }
}

// Adds each key's softmax weights, over a KV head's query rows, to what it has gathered: from the logits that attn_kernel
// has kept, a wave a page, a lane a key.  Rows are added in their order, WEIGH_ROWS of WEIGH_PAGES pages under way together.
// The rows' statistics are attn_kernel's, or, where several workgroups computed them, merged here as they are beside it.
constexpr int WEIGH_PAGES = 4, WEIGH_ROWS = 4;
template <int T, int MAPS, int DV>
__device__ __forceinline__ void weigh_pages(const AttnArgs& a, int block) {
  constexpr int C = ROWS * T, R = tile_rows<T, MAPS>();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x / 64;
  const int chunk = block / (a.p.S * a.p.H), sh = block - chunk * (a.p.S * a.p.H), s = sh / a.p.H, h = sh - s * a.p.H, head = h / MAPS, map = h - head * MAPS;
  int lo;
  const int n = pages_of(a, s, lo), first = lo + chunk * a.weigh_each, len = min(a.p.lens[s], a.p.P * PAGE);
  const int low = a.window ? len - a.window : 0;  // the row sees tokens [low, len); the others are left alone, a NaN row's too
  if (n <= 0 || first >= lo + n) return;
  int units = 0, end = 0, per = 1;
  if (a.split) {
    Part part = part_at(a, 0, 0);
    per = units_per_group(total_units(a, part), a.grid);
    for (int s0 = 64 * a.each; s0 <= s; s0 += 64 * a.each) part = part_at(a, s0, __builtin_amdgcn_readlane(part.end, 63));
    units_of(a, part, s, units, end);
  }
  for (int p0 = first + wave; p0 < min(first + a.weigh_each, lo + n); p0 += waves * WEIGH_PAGES) {
    const float* x[WEIGH_PAGES];
    float* to[WEIGH_PAGES];
    bool there[WEIGH_PAGES];
    float old[WEIGH_PAGES], sum[WEIGH_PAGES];
#pragma unroll
    for (int i = 0; i < WEIGH_PAGES; ++i) {
      const int page = min(p0 + i * waves, lo + n - 1), t = page * PAGE + lane;
      there[i] = p0 + i * waves < min(first + a.weigh_each, lo + n) && t < len && t >= low;
      x[i] = a.logits + ((int64_t(sh) * a.p.P + page) * PAGE + lane / 4 * 4) * a.nrep + lane % 4;
      to[i] = a.weights + s * a.sw_s + h * a.sw_h + min(t, len - 1);
      old[i] = *to[i];
      sum[i] = 0.f;
    }
    for (int r0 = 0; r0 < a.nrep; r0 += 64) {
      // a lane's row: its statistics
      const int r = min(r0 + lane, a.nrep - 1), tile = r / R, c = map * R + r - tile * R;
      float2 st = {NEG_INF, 0.f};
      int g0 = 0, g1 = 0;
      if (a.split) {
        const int each = units / (a.heads * a.tiles), u0 = end - units + (head * a.tiles + tile) * each;
        g0 = (u0 + PAD) / per;
        g1 = (u0 + each - 1) / per;
      }
      if (g0 == g1) {
        st = a.stats[int64_t(sh) * a.nrep + r];
      } else {
#pragma unroll 4
        for (int g = g0; g <= g1; ++g) {
          const float* p = slot_of<DV, C>(a.ws, 2 * g + (g == g0 ? 1 : 0)) + C * DV + c;
          const float m = p[0], l = p[C], mx = fmaxf(st.x, m);
          const float keep = st.x == NEG_INF ? 0.f : exp2f(st.x - mx), f = m == NEG_INF ? 0.f : exp2f(m - mx);
          st.y = (st.x == NEG_INF ? st.y : st.y * keep) + (l != l ? l : f * l);
          st.x = mx;
        }
        st = row_stats(st.x, st.y);
      }
      for (int rb = 0; rb < min(64, a.nrep - r0); rb += WEIGH_ROWS) {
        float y[WEIGH_ROWS][WEIGH_PAGES];
#pragma unroll
        for (int e = 0; e < WEIGH_ROWS; ++e)
#pragma unroll
          for (int i = 0; i < WEIGH_PAGES; ++i) y[e][i] = x[i][min(r0 + rb + e, a.nrep - 1) * 4];
#pragma unroll
        for (int e = 0; e < WEIGH_ROWS; ++e) {
          if (r0 + rb + e >= a.nrep) break;
          const float mx = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(st.x), rb + e));
          const float inv = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(st.y), rb + e));
#pragma unroll
          for (int i = 0; i < WEIGH_PAGES; ++i)
            sum[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(y[e][i] - mx), inv, sum[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < WEIGH_PAGES; ++i)
      if (there[i]) *to[i] = old[i] + sum[i];
  }
}

// One workgroup per (sequence, head, tile): merges the slots of those that several workgroups computed, in order.  W: behind
// these (where there are any), the workgroups that weigh the keys.
template <int D, bool BF, int T, bool W, int MAPS>
__global__ __launch_bounds__(ROWS * T * (MAPS * D / 8)) void combine_kernel(AttnArgs a) {
  constexpr int C = ROWS * T, R = tile_rows<T, MAPS>(), DV = MAPS * D;
  if constexpr (W)
    if (blockIdx.x >= unsigned(a.items)) return weigh_pages<T, MAPS, DV>(a, blockIdx.x - a.items);
  const int per_seq = a.heads * a.tiles, s = blockIdx.x / per_seq, hr = blockIdx.x - s * per_seq;
  Part part = part_at(a, 0, 0);
  const int total = total_units(a, part), per = units_per_group(total, a.grid);
  for (int s0 = 64 * a.each; s0 <= s; s0 += 64 * a.each) part = part_at(a, s0, __builtin_amdgcn_readlane(part.end, 63));
  int units, end;
  units_of(a, part, s, units, end);
  const int n = units / per_seq;
  if (n <= 0) return;
  const int u0 = end - units + hr * n, g0 = (u0 + PAD) / per, g1 = (u0 + n - 1) / per;
  if (g0 == g1) return;
  // lanes of DV/8 take a column's dims, `parts` of them its slots in runs
  const int tile = hr % a.tiles, per_map = min(R, a.m * a.nrep - tile * R), rows = MAPS * per_map;
  const int parts = g1 - g0 < 4 ? 1 : C / rows;
  const int grp = threadIdx.x / (DV / 8), part_i = grp / rows, ri = grp - part_i * rows, d = threadIdx.x % (DV / 8) * 8;
  const int map = MAPS == 1 ? 0 : ri / per_map, r = ri - map * per_map, rr = map * R + r;
  const int run = (g1 - g0 + parts) / parts, ga = g0 + part_i * run, gz = part_i < parts ? min(ga + run - 1, g1) : -1;
  constexpr int B = 4;  // slots whose loads are under way together
  float mx = NEG_INF, sum = 0.f, v[8] = {};
  for (int g = ga; g <= gz; g += B) {
    float m[B], l[B];
    f4_t x[B][2];
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const int gi = min(g + i, gz);
      const float* p = slot_of<DV, C>(a.ws, 2 * gi + (gi == g0 ? 1 : 0));
      m[i] = p[C * DV + rr];
      l[i] = p[C * DV + C + rr];
      x[i][0] = *reinterpret_cast<const f4_t*>(p + rr * DV + d);
      x[i][1] = *reinterpret_cast<const f4_t*>(p + rr * DV + d + 4);
    }
    const float was = mx;
#pragma unroll
    for (int i = 0; i < B; ++i) mx = fmaxf(mx, m[i]);
    const float keep = was == NEG_INF ? 0.f : exp2f(was - mx);
    sum *= keep;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= keep;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (g + i > gz) break;
      const float f = m[i] == NEG_INF ? 0.f : exp2f(m[i] - mx);
      sum += l[i] != l[i] ? l[i] : f * l[i];
      if (f != 0.f)  // (a slot that saw nothing, or nothing that counts)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += f * x[i][e / 4][e % 4];
    }
  }
  __shared__ float sv[C][DV], sm[C], sl[C];
  if (parts > 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sv[grp][d + e] = v[e];
    if (d == 0) {
      sm[grp] = mx;
      sl[grp] = sum;
    }
    __syncthreads();
    for (int i = 1; i < (part_i > 0 ? 1 : parts); ++i) {
      const int o = i * rows + ri;
      const float was = mx;
      mx = fmaxf(mx, sm[o]);
      const float keep = was == NEG_INF ? 0.f : exp2f(was - mx), f = sm[o] == NEG_INF ? 0.f : exp2f(sm[o] - mx);
      sum = (was == NEG_INF ? sum : sum * keep) + (sl[o] != sl[o] ? sl[o] : f * sl[o]);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = keep * v[e] + (f != 0.f ? f * sv[o][d + e] : 0.f);
    }
  }
  const int head = hr / a.tiles;
  float inv = sum == 0.f ? 0.f : 1.f / sum;
  if constexpr (MAPS == 2) {
    if (parts > 1) __syncthreads();  // nobody reads the parts any more
    if (part_i == 0 && map == 1) {
      const float f = minus_lam<R>(a, head, tile, r) * inv;
#pragma unroll
      for (int e = 0; e < 8; ++e) sv[r][d + e] = f * v[e];
    }
    __syncthreads();
    if (map == 0)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = v[e] * inv + sv[r][d + e];
    inv = 1.f;
  }
  if (part_i > 0 || map > 0) return;
  store_row<D, BF, R>(a, s, head, tile, r, d, v, inv);
}

constexpr int GRID = 512;  // two workgroups per CU

struct Launch {
  int T, tiles, split, grid;  // split: workgroups share out the pages, or each takes a whole (sequence, head, tile)
};
// T: a tile of more than 16 rows takes two groups of 16 to each page, which is loaded and converted once for both.  With
// D = 128 their accumulators leave room for one workgroup per CU, so the batch has to be large enough: 8192 pages of 16
// rows.  us with one / two groups (8 KV heads, 8 new tokens on 32 query heads, D = 128; fp16, bf16):
//   8 sequences of 16384 tokens  66 / 52, 79 / 56;  48 of 1500  39 / 42, 56 / 45;  64 of 500  24 / 23, 32 / 25
//   16 of 1000 (4096 pages)  13 / 17;  16 new tokens, 48 of 1500  78 / 63, 101 / 68
// Whole items, one launch and no list to go through, while tables are narrow: up to 8 pages per sequence, 16 with 64
// items, 32 with 256.  us whole / shared out (8 KV heads, D = 128, fp16):
//   sequences of 500 tokens (P = 8)  1: 8.7 / 10.4;  16: 9.0 / 13.4;  128: 24 / 28
//   of 1000 (P = 16)                 1: 12.1 / 10.6;  8: 12.3 / 12.4;  32: 13.7 / 20.3;  128: 36 / 40
//   of 1500 (P = 24)                 8: 15.8 / 14.7;  16: 16.1 / 17.0;  32: 17.6 / 23.9;  128: 46 / 52
//   of 4032 (P = 63)                64: 61 / 63, but of 50 .. 4096 tokens 48 / 36
// The lengths are on the device, so the table's width P stands for them: a caller whose tables are wider than any sequence
// passes the columns that are needed (16 sequences of 500 tokens: P = 8 8.2 us, P = 512 13.2; bf16 10.8, 16.7).
// Two maps: a group for each where there are more than 8 rows (a tile of 8 would read its pages again for the others).
// The same widths for two maps, whose items are half as many (P pages each, 8 KV heads, D = 128, fp16; us whole / shared out):
//   1 x 8 13.0 / 14.6;  1 x 12 15.8 / 14.8;  8 x 16 19.1 / 15.3;  16 x 16 19.2 / 19.9;  16 x 24 25.0 / 20.0;  32 x 16 20.0 / 22.6;
//   32 x 24 25.6 / 25.5;  64 x 32 34.3 / 40.6;  64 x 40 40.6 / 45.0;  4 new tokens, 1 x 8 17.7 / 19.8, 16 x 16 26.1 / 26.3, 64 x 32
//   45.5 / 49.2;  bf16, 16 x 16 23.8 / 22.1
// and with the keys' weights, where whole items take a second launch too:
//   1 x 8 11.9 / 11.4;  1 x 12 13.4 / 11.7;  16 x 8 12.6 / 15.0;  16 x 16 16.1 / 17.7;  16 x 24 19.2 / 18.7;  32 x 24 21.0 / 26.3;
//   64 x 32 44.1 / 47.1;  64 x 40 57.4 / 57.6;  two maps: 1 x 8 17.5 / 16.0;  16 x 8 18.4 / 18.0;  16 x 16 25.0 / 21.8;
//   16 x 24 31.4 / 22.4;  32 x 16 26.3 / 25.8;  64 x 32 48.6 / 49.6
inline Launch plan_of(int S, int P, int m, int nrep, int heads, int D, int maps) {
  const int64_t rows = int64_t(m) * nrep, pages = int64_t(S) * heads * P * ceil_div(rows, ROWS);
  Launch p;
  p.T = maps == 2 ? (rows > ROWS / 2 ? 2 : 1) : rows > ROWS && pages >= 8192 ? 2 : 1;
  p.tiles = int(ceil_div(rows, ROWS * p.T / maps));
  const int64_t items = int64_t(S) * heads * p.tiles;
  p.split = P > (items >= 256 ? 32 : items >= 64 ? 16 : 8);
  p.grid = p.split ? GRID / 2 * per_cu(D, p.T, maps) : int(items);
  return p;
}

inline size_t slots_bytes(const Launch& p, int D, int maps) {
  return p.split ? size_t(2 * GRID) * (ROWS * p.T) * (maps * D + 2) * sizeof(float) : 0;
}
inline size_t stats_bytes(int S, int Hq) { return (size_t(S) * Hq * sizeof(float2) + 15) / 16 * 16; }

}  // namespace

namespace iq {
int check_paged(const iq_paged* p);
}

namespace {
// slots, then for the keys' weights the rows' statistics and the logits
size_t workspace_bytes_of(int S, int P, int m, int Hq, int H, int D, int maps, bool weights) {
  if (S <= 0 || P <= 0 || m <= 0 || Hq <= 0 || H <= 0 || Hq % H || H % maps || !d_ok(D)) return 0;
  const size_t slots = slots_bytes(plan_of(S, P, m, Hq / H, H / maps, D, maps), D, maps);
  return weights ? slots + stats_bytes(S, Hq) + size_t(S) * Hq * P * PAGE * sizeof(float) : slots;
}

template <int MAPS>
int attention(const iq_paged* p, const void* q, int64_t sq_s, int64_t sq_m, int64_t sq_h, int m, int Hq, const float* lam,
              int64_t s_lam, float scale, int window, void* out, int64_t so_s, int64_t so_m, int64_t so_h, float* weights,
              int64_t sw_s, int64_t sw_h, int64_t Tw, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int st = iq::check_paged(p)) return st;
  IQ_CHECK(q && out && (MAPS == 1 || lam), IQ_ERR_NULL);
  IQ_CHECK(m > 0 && m <= 16 && Hq > 0 && Hq % p->H == 0 && p->H % MAPS == 0 && Hq <= 4096 && window >= 0 && s_lam >= 0,
           IQ_ERR_SHAPE);
  IQ_CHECK(MAPS == 1 || out != q, IQ_ERR_SHAPE);  // an output row lies over several heads' queries
  IQ_CHECK(aligned(q, 16) && aligned(out, 16) && sq_s % 8 == 0 && sq_m % 8 == 0 && sq_h % 8 == 0 && so_s % 8 == 0 &&
               so_m % 8 == 0 && so_h % 8 == 0 && aligned(lam, 4), IQ_ERR_ALIGN);
  const int nrep = Hq / p->H, heads = p->H / MAPS;
  const Launch pl = plan_of(p->S, p->P, m, nrep, heads, p->D, MAPS);
  IQ_CHECK(int64_t(p->S) * (p->P + PAD) * heads * pl.tiles <= INT32_MAX &&
               int64_t(p->S) * heads * pl.tiles <= UINT32_MAX / (ROWS * 2 * MAPS * 16), IQ_ERR_SHAPE);
  if (weights) {
    IQ_CHECK(m == 1 && Tw >= int64_t(p->P) * PAGE && sw_s >= 0 && sw_h >= 0, IQ_ERR_SHAPE);
    IQ_CHECK((int64_t(p->P) + 1) * nrep < INT32_MAX / (PAGE * 4), IQ_ERR_SHAPE);  // a map's logits in 32 bits
    IQ_CHECK(aligned(weights, 4), IQ_ERR_ALIGN);
  }
  const size_t need = workspace_bytes_of(p->S, p->P, m, Hq, p->H, p->D, MAPS, weights != nullptr);
  IQ_CHECK(!need || (workspace && workspace_bytes >= need), IQ_ERR_WORKSPACE);
  IQ_CHECK(aligned(workspace, 16), IQ_ERR_ALIGN);
  if (window >= p->P * PAGE) window = 0;  // hides nothing
  AttnArgs a{*p, (const uint16_t*)q, sq_s, sq_m, sq_h, (uint16_t*)out, so_s, so_m, so_h, heads, m, nrep, pl.tiles,
             scale * 1.44269504088896340736f, window, pl.grid, (float*)workspace, p->S > 64 ? EACH : 1, pl.split, lam, s_lam,
             nullptr, nullptr, weights, sw_s, sw_h, pl.split ? p->S * heads * pl.tiles : 0, 0};
  if (weights) {
    char* const ws = (char*)workspace + slots_bytes(pl, p->D, MAPS);
    a.stats = (float2*)ws;
    a.logits = (float*)(ws + stats_bytes(p->S, Hq));
  }
  auto launch = [&]<int D, bool BF, int T, bool W>() -> int {
    constexpr int threads = ROWS * T * (MAPS * D / 8);
    int64_t groups = a.items;  // of the second launch
    if constexpr (W) {
      a.weigh_each = threads / 64 * WEIGH_PAGES;
      groups += int64_t(p->S) * p->H * ceil_div(p->P, a.weigh_each);
      IQ_CHECK(groups <= INT32_MAX / threads, IQ_ERR_SHAPE);
    }
    attn_kernel<D, BF, T, W, MAPS><<<pl.grid, THREADS, 0, (hipStream_t)stream>>>(a);
    if (const int st = launch_status()) return st;
    if (groups) combine_kernel<D, BF, T, W, MAPS><<<unsigned(groups), threads, 0, (hipStream_t)stream>>>(a);
    return launch_status();
  };
  auto with = [&]<int D, bool BF>() {
    if (weights) return pl.T == 2 ? launch.template operator()<D, BF, 2, true>() : launch.template operator()<D, BF, 1, true>();
    return pl.T == 2 ? launch.template operator()<D, BF, 2, false>() : launch.template operator()<D, BF, 1, false>();
  };
  const bool bf = act_bf16(p->mode);
  if (p->D == 128) return bf ? with.template operator()<128, true>() : with.template operator()<128, false>();
  return bf ? with.template operator()<64, true>() : with.template operator()<64, false>();
}
}  // namespace

extern "C" size_t iq_paged_attention_workspace_bytes(int S, int P, int m, int Hq, int H, int D) {
  return workspace_bytes_of(S, P, m, Hq, H, D, 1, false);
}

extern "C" int iq_paged_attention(const iq_paged* p, const void* q, int64_t sq_s, int64_t sq_m, int64_t sq_h, int m, int Hq,
                                  float scale, int window, void* out, int64_t so_s, int64_t so_m, int64_t so_h,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  return attention<1>(p, q, sq_s, sq_m, sq_h, m, Hq, nullptr, 0, scale, window, out, so_s, so_m, so_h, nullptr, 0, 0, 0,
                      workspace, workspace_bytes, stream);
}

extern "C" size_t iq_paged_attention_weights_workspace_bytes(int S, int P, int Hq, int H, int D) {
  return workspace_bytes_of(S, P, 1, Hq, H, D, 1, true);
}

extern "C" int iq_paged_attention_weights(const iq_paged* p, const void* q, int64_t sq_s, int64_t sq_h, int Hq, float scale,
                                          int window, void* out, int64_t so_s, int64_t so_h, float* weights, int64_t sw_s,
                                          int64_t sw_h, int64_t T, void* workspace, size_t workspace_bytes, void* stream) {
  IQ_CHECK(weights, IQ_ERR_NULL);
  return attention<1>(p, q, sq_s, 0, sq_h, 1, Hq, nullptr, 0, scale, window, out, so_s, 0, so_h, weights, sw_s, sw_h, T,
                      workspace, workspace_bytes, stream);
}

// Differential attention (MAPS = 2).  KV heads 2g, 2g + 1 of a page are the keys of the two maps and the two halves of V; a
// workgroup takes a pair, so each page is read once for both maps.  Up to 8 rows of both maps share the 16 columns of a group
// (one softmax, one product with V for both), more take a group for each map.  Their sums stay apart until the waves, or the
// workgroups, are merged: then out = first / sum - lam second / sum in fp32.
extern "C" size_t iq_diff_paged_attention_workspace_bytes(int S, int P, int m, int Hq, int H, int D, int weights) {
  return workspace_bytes_of(S, P, m, Hq, H, D, 2, weights != 0);
}

extern "C" int iq_diff_paged_attention(const iq_paged* p, const void* q, int64_t sq_s, int64_t sq_m, int64_t sq_h, int m, int Hq,
                                       const float* lam, int64_t s_lam, float scale, int window, void* out, int64_t so_s,
                                       int64_t so_m, int64_t so_h, float* weights, int64_t sw_s, int64_t sw_h, int64_t T,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  return attention<2>(p, q, sq_s, sq_m, sq_h, m, Hq, lam, s_lam, scale, window, out, so_s, so_m, so_h, weights, sw_s, sw_h, T,
                      workspace, workspace_bytes, stream);
}
