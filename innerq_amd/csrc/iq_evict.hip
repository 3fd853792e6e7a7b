// Dropping tokens from 4-bit pages by the attention weight that they have gathered (gfx950): iq_paged_evict.
//
// Of a sequence of n > keep tokens each KV head (or run of `shared` heads) keeps its last `recent` tokens and, of the
// others, the `sinks` first ones and those of most weight.  Attention does not ask for the order of a cache's rows, so
// only the rows that have to move do: with B = keep - recent, a kept token below B stays; the places below B that a
// dropped token leaves are filled, in order, by the kept ones from B on; the last `recent` tokens move down to B .. keep.
// A step that drops a page of 64 tokens from 2048 moves some 60 rows and the recent ones, where keeping the order would
// move all of them.
//
// Three steps, one behind the other (each reads what the next one writes over), each a launch, or all of them in one by a
// workgroup per (sequence, run of heads):
//   select  one workgroup per (sequence, run of heads): the B-th largest weight by three passes over the bits of the
//           weights (11, 11, 10 from the top), then the lists of free places and of the rows that come.
//   fill    rows and their weights into the free places: sources from B on, destinations below B, in any order.
//   shift   the last `recent` rows: where they overlap their destinations one workgroup per (sequence, head), in order,
//           each batch read whole before it is written.  Weights from `keep` on become 0.
//
// Bound: latency: in each step loads wait for each other (length, weights or lists, table, page).  32 sequences of 2112 tokens to
// 2048, 256 of them recent (8 heads, D = 128): 24.5 us in one launch, 30 where other data passes between.  8 of 32768 to 2048,
// 512 recent: 26, 25 and 13 us in three.  There a third of select's time loads the weights and counts their first digits
// (weights of one size share bins, whose atomics take turns: with one copy of the counts, and words one by one, 30 us), and fill
// reads rows from all over: a token's V lies in D / 8 sectors of 32 bytes with 7 other tokens', so 8 bytes come for each used.
#include "iq_paged.h"

using namespace iq;

namespace {

constexpr int SELECT = 1024, FILL = 256, SHIFT = 1024;
constexpr int BATCH = 4;                        // rows of a lane that are under way together
constexpr int BITS[3] = {11, 11, 10}, BINS = 1 << 11;
constexpr int WAVES = SELECT / 64;
// One launch does it all where each (sequence, run of heads) has few rows to move, or there are as many of them as seven eighths of
// the CUs.  us in one launch / in three (8 heads, D = 128; sequences x tokens -> keep, recent):
//   1 x 80 -> 64, 8  14.9 / 17.9;  1 x 2112 -> 2048, 256  20.8 / 25.1;  32 of them  24.5 / 30.6;  128  86 / 91
//   32 x 8192 -> 2048, 512  84 / 98;  32 x 16384 -> 8192, 1024  246 / 256;  64 x 4096 -> 2048, 256  118 / 125
//   8 x 32768 -> 2048, 512  82 / 57;  2 x 16384 -> 8192, 4096  194 / 41;  32 x 2112 -> 2048, 256, heads in pairs  32.9 / 30.4
constexpr int FULL = 224, FEW_ROWS = 512;
constexpr int KEYS = 32, ROUND = KEYS * SELECT;  // weights of a thread, of a workgroup
constexpr int COPIES = 2;                       // of the digits' counts, by lane: equal digits of a wave take turns

typedef float f4_any_t __attribute__((ext_vector_type(4), aligned(4)));

struct EvictArgs {
  iq_paged p;
  const float* w;
  int64_t sw_s, sw_h;
  float* wo;
  int64_t so_s, so_h, T;
  int keep, recent, sinks, shared, most;  // most: rows that can come, at most
  int32_t* lens_out;
  int32_t* ws;
  int chunks;  // workgroups per (sequence, head)
};

// a (sequence, run of heads)'s part of the workspace: its tokens if it drops any (else 0), the rows that come, the free
// places, the rows
__device__ __forceinline__ int32_t* plan_of(const EvictArgs& a, int64_t run) { return a.ws + run * (2 + 2 * int64_t(a.most)); }

// inclusive sum over the workgroup; `total` the whole sum
__device__ __forceinline__ int group_scan(int v, int& total) {
  __shared__ int part[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  __syncthreads();  // (nobody reads the last call's sums any more)
  if (lane == 63) part[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const int y = part[i];
    if (i < wave) before += y;
    total += y;
  }
  return before + x;
}

// every thread of the workgroup has what it has read in registers: what it read may be written over
__device__ __forceinline__ void all_read() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// What a (sequence, run of heads) keeps: the tokens of a sequence that drops any (else 0), and how many rows come; the free
// places and the rows that come, in their order, to the plan.  By a workgroup of SELECT threads.
struct Plan {
  int n, count;
};
__device__ __forceinline__ Plan select(const EvictArgs& a, int run) {
  __shared__ int hist[COPIES][BINS];
  __shared__ int found[2];  // the digit, and how many of its keys are wanted
  __shared__ u4_t keys[ROUND / 4];
  const int runs = a.p.H / a.shared, s = run / runs, h0 = (run - s * runs) * a.shared, tid = threadIdx.x;
  const float* w = a.w + s * a.sw_s + h0 * a.sw_h;
  float* wo = a.wo + s * a.so_s + h0 * a.so_h;
  int32_t* plan = plan_of(a, run);
  const int n = a.p.lens[s];
  const bool there = n >= 0 && n <= int64_t(a.p.P) * PAGE;
  if (!there && tid == 0) atomicOr(a.p.status, PAGED_BAD_TOKEN);
  if (!there || n <= a.keep) return {0, 0};
  const int old = n - a.recent, B = a.keep - a.recent;  // B of the first `old` tokens stay
  if (a.wo != a.w)  // the weights below B (those of free places are written over by the next launch)
    for (int h = 0; h < a.shared; ++h)
      for (int i = tid; i < B; i += SELECT) wo[h * a.so_h + i] = w[h * a.sw_h + i];
  // Weights as whole numbers of the same order: NaN above all, -0 as 0.  The sinks are above all too, and come first.  A
  // round's keys lie in LDS, a thread's being those of `per` neighbouring tokens, 0 (less than any weight's) past the end.
  const bool one = old <= ROUND;
  const int groups = one ? (old + 4 * SELECT - 1) / (4 * SELECT) : KEYS / 4, per = 4 * groups;
  // four neighbouring keys lie together: a run of them, and the threads' own ones of one place, both meet no bank twice
  auto four_at = [&](int g) -> u4_t& { return keys[g ^ (g >> 4 & 7)]; };
  int* const counts = hist[tid % COPIES];
  auto load = [&](int round, bool count) {  // count: the first pass's digits too
    auto four = [&](const float* p, int i) {  // weights i .. i + 3, which may be the row's last
      if (i + 4 <= a.T) return f4_t(*reinterpret_cast<const f4_any_t*>(p + i));
      f4_t x = {0.f, 0.f, 0.f, 0.f};
      for (int e = 0; e < 4; ++e)
        if (i + e < a.T) x[e] = p[i + e];
      return x;
    };
    f4_t x[KEYS / 4];
#pragma unroll
    for (int v = 0; v < KEYS / 4; ++v) {
      const int i = round + (v * SELECT + tid) * 4;
      x[v] = i < old ? four(w, i) : f4_t{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();  // nobody reads the last round's keys any more
#pragma clang loop unroll(disable)
    for (int v = 0; v < groups; ++v) {  // (unrolled its code took 2 us more to fetch)
      const int i = round + (v * SELECT + tid) * 4;
      f4_t y;
#pragma unroll
      for (int u = 0; u < KEYS / 4; ++u)
        if (u == v) y = x[u];
      y += 0.f;
      if (i < old)
        for (int h = 1; h < a.shared; ++h) y += four(w + h * a.sw_h, i);
      u4_t k;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = y[e];
        const uint32_t b = __float_as_uint(z), q = i + e < a.sinks || z != z ? ~0u : b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
        k[e] = i + e < old ? q : 0u;
        if (count && i + e < old) atomicAdd(&counts[q >> (32 - BITS[0])], 1);
      }
      four_at(v * SELECT + tid) = k;
    }
    __syncthreads();
  };
  int* const all_counts = &hist[0][0];
  for (int i = tid; i < COPIES * BINS; i += SELECT) all_counts[i] = 0;
  if (one) load(0, B > 0);
  uint32_t least = 0;  // the B-th largest key
  int ties = 0;        // of the tokens whose key it is, the first `ties` stay
  if (B > 0) {
    uint32_t mask = 0;
    int want = B;
    for (int pass = 0, low = 32; pass < 3; ++pass) {
      const int bits = BITS[pass];
      low -= bits;
      if (pass > 0)
        for (int i = tid; i < COPIES * BINS; i += SELECT) all_counts[i] = 0;
      __syncthreads();
      for (int round = 0; round < old; round += ROUND) {
        if (!one) load(round, false);
        else if (pass == 0) break;
        for (int g = 0; g < groups; ++g) {
          const u4_t k = four_at(g * SELECT + tid);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k[e] && (k[e] & mask) == least) atomicAdd(&counts[k[e] >> low & ((1u << bits) - 1)], 1);
        }
      }
      __syncthreads();
      const int hi = BINS - 1 - 2 * tid;
      int c0 = 0, c1 = 0;
#pragma unroll
      for (int c = 0; c < COPIES; ++c) {
        c0 += hist[c][hi];
        c1 += hist[c][hi - 1];
      }
      int total;
      const int end = group_scan(c0 + c1, total), before = end - c0 - c1;
      if (before < want && want <= end) {
        const bool second = before + c0 < want;
        found[0] = second ? hi - 1 : hi;
        found[1] = second ? want - before - c0 : want - before;
      }
      __syncthreads();
      least |= uint32_t(found[0]) << low;
      mask |= ((1u << bits) - 1) << low;
      want = found[1];
    }
    ties = want;
  }
  // the places below B that become free, and the tokens from B on that stay (as many), each in order
  int count[2] = {0, 0}, tied = 0;
  for (int round = 0; round < old; round += ROUND) {
    if (!one) load(round, false);
    const int first = round + tid * per;
    uint32_t stay = 0, same = 0;  // a bit of each of the thread's tokens
    for (int g = 0; g < groups; ++g) {
      const u4_t k = four_at(tid * groups + g);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        stay |= uint32_t(k[e] > least) << (4 * g + e);
        same |= uint32_t(k[e] == least) << (4 * g + e);
      }
    }
    // (the thread's tokens below B, and below the end)
    auto up_to = [&](int end) { return end <= first ? 0u : end - first >= 32 ? ~0u : (1u << (end - first)) - 1; };
    const uint32_t all = per == 32 ? ~0u : (1u << per) - 1, low = up_to(B) & all, real = up_to(old) & all;
    same &= real;
    if (B > 0) {
      int total, rank = tied + group_scan(__builtin_popcount(same), total) - __builtin_popcount(same);
      tied += total;
      for (uint32_t left = same; left && rank < ties; left &= left - 1, ++rank) stay |= left & -left;
    } else {
      stay = 0;
    }
    const uint32_t in[2] = {real & low & ~stay, real & ~low & stay};
#pragma unroll
    for (int list = 0; list < 2; ++list) {
      int total, at = count[list] + group_scan(__builtin_popcount(in[list]), total) - __builtin_popcount(in[list]);
      count[list] += total;
      int32_t* to = plan + 2 + list * int64_t(a.most);
      for (uint32_t left = in[list]; left; left &= left - 1) to[at++] = first + __builtin_ctz(left);
    }
  }
  return {n, count[0]};
}

__global__ __launch_bounds__(SELECT) void select_kernel(EvictArgs a) {
  const Plan x = select(a, blockIdx.x);
  if (threadIdx.x == 0) {
    int32_t* plan = plan_of(a, blockIdx.x);
    plan[0] = x.n;
    plan[1] = x.count;
  }
}

// A lane's share of one token's row of one head: word o of K and V, and for o % 4 == 0 their group's scales and zeros.
struct Piece {
  uint32_t k, v, km;
  uint16_t vs, vz;
};
template <int D>
__device__ __forceinline__ Piece load_piece(const uint32_t* pg, int row, int o) {
  constexpr int U = D / 8, G = D / 32;
  const int b = v_block(row), e = v_place(row);
  Piece x{pg[row * U + o], pg[page_vc(D) + (b * U + o) * 8 + e], 0, 0, 0};
  if (o % 4 == 0) {
    const uint16_t* m = reinterpret_cast<const uint16_t*>(pg + page_vm(D)) + (b * G + o / 4) * 16 + e;
    x.km = pg[page_km(D) + row * G + o / 4];
    x.vs = m[0];
    x.vz = m[8];
  }
  return x;
}
template <int D>
__device__ __forceinline__ void store_piece(uint32_t* pg, int row, int o, const Piece& x) {
  constexpr int U = D / 8, G = D / 32;
  const int b = v_block(row), e = v_place(row);
  pg[row * U + o] = x.k;
  pg[page_vc(D) + (b * U + o) * 8 + e] = x.v;
  if (o % 4 == 0) {
    uint16_t* m = reinterpret_cast<uint16_t*>(pg + page_vm(D)) + (b * G + o / 4) * 16 + e;
    pg[page_km(D) + row * G + o / 4] = x.km;
    m[0] = x.vs;
    m[8] = x.vz;
  }
}

// token t's page of head h, null if the table names none of the pool
template <int D>
__device__ __forceinline__ uint32_t* page_of(const EvictArgs& a, int s, int h, int t) {
  const int id = a.p.table[s * a.p.s_table + t / PAGE];
  return id < 0 || id >= a.p.n_pages ? nullptr : a.p.pages + (int64_t(id) * a.p.H + h) * page_words(D);
}

// BATCH rows of a lane, and their tokens' weights, from tokens `from` to `to` (from < 0: none): reads all, calls `between`,
// writes all.  A row whose page is missing is not read and becomes NaN; one whose place has no page is not written.
template <int D, typename F>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int s, int h, int o, const int (&from)[BATCH],
                                          const int (&to)[BATCH], F&& between) {
  constexpr uint16_t nan = 0x7fff;  // of both activation dtypes
  const uint32_t* src[BATCH];
  uint32_t* dst[BATCH];
  Piece x[BATCH];
  float weight[BATCH];
  const float* w = a.w + s * a.sw_s + h * a.sw_h;
  float* wo = a.wo + s * a.so_s + h * a.so_h;
#pragma unroll
  for (int e = 0; e < BATCH; ++e) {
    src[e] = from[e] < 0 ? nullptr : page_of<D>(a, s, h, from[e]);
    dst[e] = from[e] < 0 ? nullptr : page_of<D>(a, s, h, to[e]);
    if (from[e] >= 0 && (!src[e] || !dst[e]) && o == 0) atomicOr(a.p.status, PAGED_BAD_PAGE);
  }
#pragma unroll
  for (int e = 0; e < BATCH; ++e)
    x[e] = src[e] ? load_piece<D>(src[e], from[e] % PAGE, o) : Piece{0, 0, nan | uint32_t(nan) << 16, nan, nan};
#pragma unroll
  for (int e = 0; e < BATCH; ++e) weight[e] = o == 1 && from[e] >= 0 ? w[from[e]] : 0.f;
  between();
#pragma unroll
  for (int e = 0; e < BATCH; ++e) {
    if (dst[e]) store_piece<D>(dst[e], to[e] % PAGE, o, x[e]);
    if (o == 1 && from[e] >= 0) wo[to[e]] = weight[e];
  }
}

// the rows that come to their places, by `chunks` workgroups of THREADS
template <int D, int THREADS>
__device__ __forceinline__ void fill(const EvictArgs& a, int s, int h, const int32_t* plan, int count, int chunk, int chunks) {
  constexpr int U = D / 8, ROWS = THREADS / U * BATCH;  // rows of a workgroup's turn
  const int o = threadIdx.x % U;
  for (int r0 = chunk * ROWS + threadIdx.x / U; r0 < count; r0 += chunks * ROWS) {
    int from[BATCH], to[BATCH];
#pragma unroll
    for (int e = 0; e < BATCH; ++e) {
      const int r = r0 + e * (THREADS / U);
      to[e] = plan[2 + min(r, count - 1)];
      from[e] = r < count ? plan[2 + int64_t(a.most) + r] : -1;
    }
    move_rows<D>(a, s, h, o, from, to, [] {});
  }
}

// the last rows to their places, and zeros for the weights behind, by `chunks` workgroups of SHIFT threads
template <int D>
__device__ __forceinline__ void shift(const EvictArgs& a, int s, int h, int n, int chunk, int chunks) {
  constexpr int U = D / 8, ROWS = SHIFT / U * BATCH;
  const int o = threadIdx.x % U;
  float* wo = a.wo + s * a.so_s + h * a.so_h;
  const int64_t first = chunk * int64_t(SHIFT) + threadIdx.x, step = int64_t(chunks) * SHIFT;
  if (!n) {  // a sequence that drops nothing
    if (a.wo != a.w)
      for (int64_t i = first; i < a.T; i += step) wo[i] = a.w[s * a.sw_s + h * a.sw_h + i];
    return;
  }
  const int src = n - a.recent;
  const bool apart = n - a.keep >= a.recent;  // the rows and their places: they move in any order
  if (apart || chunk == 0)
    for (int r0 = chunk * ROWS; r0 < a.recent; r0 += (apart ? chunks : 1) * ROWS) {
      int from[BATCH], to[BATCH];
#pragma unroll
      for (int e = 0; e < BATCH; ++e) {
        const int r = r0 + e * (SHIFT / U) + threadIdx.x / U;
        from[e] = r < a.recent ? src + r : -1;
        to[e] = a.keep - a.recent + min(r, a.recent - 1);
      }
      move_rows<D>(a, s, h, o, from, to, [] { all_read(); });
      // no weight is left where its token was: this batch's, or (they overlap) all from `keep` on, at the end
      if (apart)
        for (int i = threadIdx.x; i < min(ROWS, a.recent - r0); i += SHIFT) wo[src + r0 + i] = 0.f;
    }
  // nor behind, nor, of the others, before them
  for (int64_t i = a.keep + first; i < src; i += step) wo[i] = 0.f;
  for (int64_t i = n + first; i < a.T; i += step) wo[i] = 0.f;
  if (!apart && chunk == 0) {
    all_read();
    for (int i = max(a.keep, src) + threadIdx.x; i < n; i += SHIFT) wo[i] = 0.f;
  }
}

template <int D>
__global__ __launch_bounds__(FILL) void fill_kernel(EvictArgs a) {
  const int sh = blockIdx.x / a.chunks, chunk = blockIdx.x - sh * a.chunks, s = sh / a.p.H, h = sh - s * a.p.H;
  const int32_t* plan = plan_of(a, int64_t(s) * (a.p.H / a.shared) + h / a.shared);
  if (h == 0 && chunk == 0 && threadIdx.x == 0) a.lens_out[s] = plan[0] ? a.keep : a.p.lens[s];
  fill<D, FILL>(a, s, h, plan, plan[1], chunk, a.chunks);
}

template <int D>
__global__ __launch_bounds__(SHIFT) void shift_kernel(EvictArgs a) {
  const int sh = blockIdx.x / a.chunks, chunk = blockIdx.x - sh * a.chunks, s = sh / a.p.H, h = sh - s * a.p.H;
  shift<D>(a, s, h, plan_of(a, int64_t(s) * (a.p.H / a.shared) + h / a.shared)[0], chunk, a.chunks);
}

// All of it in one launch, a workgroup per (sequence, run of heads).
template <int D>
__global__ __launch_bounds__(SELECT) void evict_kernel(EvictArgs a) {
  static_assert(SELECT == SHIFT);
  const int runs = a.p.H / a.shared, s = blockIdx.x / runs, h0 = (blockIdx.x - s * runs) * a.shared;
  const Plan x = select(a, blockIdx.x);
  all_read();  // (and written: the lists, and the weights below B)
  for (int h = h0; h < h0 + a.shared; ++h) fill<D, SELECT>(a, s, h, plan_of(a, blockIdx.x), x.count, 0, 1);
  all_read();
  for (int h = h0; h < h0 + a.shared; ++h) shift<D>(a, s, h, x.n, 0, 1);
  if (a.lens_out != a.p.lens && h0 == 0 && threadIdx.x == 0) a.lens_out[s] = x.n ? a.keep : a.p.lens[s];
}
// its lengths in place: behind it, as its workgroups read them
__global__ __launch_bounds__(64) void lens_kernel(EvictArgs a) {
  const int s = blockIdx.x * 64 + threadIdx.x;
  if (s >= a.p.S) return;
  const int n = a.p.lens[s];
  if (n > a.keep && n <= int64_t(a.p.P) * PAGE) a.lens_out[s] = a.keep;
}

inline int64_t rows_that_come(int P, int keep, int recent) {
  const int64_t past = int64_t(P) * PAGE - keep;
  return past <= 0 ? 0 : past < keep - recent ? past : keep - recent;
}

}  // namespace

namespace iq {
int check_paged(const iq_paged* p);
}

extern "C" size_t iq_paged_evict_workspace_bytes(int S, int P, int H, int keep, int recent, int shared) {
  if (S <= 0 || P <= 0 || H <= 0 || keep <= 0 || recent < 0 || recent > keep || shared <= 0 || H % shared) return 0;
  return size_t(S) * (H / shared) * size_t(2 + 2 * rows_that_come(P, keep, recent)) * sizeof(int32_t);
}

extern "C" int iq_paged_evict(const iq_paged* p, const float* weights, int64_t sw_s, int64_t sw_h, float* weights_out,
                              int64_t so_s, int64_t so_h, int64_t T, int keep, int recent, int sinks, int shared,
                              int32_t* lens_out, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int st = iq::check_paged(p)) return st;
  IQ_CHECK(weights && weights_out && lens_out, IQ_ERR_NULL);
  IQ_CHECK(keep > 0 && recent >= 0 && sinks >= 0 && int64_t(recent) + sinks <= keep, IQ_ERR_SHAPE);
  IQ_CHECK(shared > 0 && p->H % shared == 0 && T >= int64_t(p->P) * PAGE, IQ_ERR_SHAPE);
  IQ_CHECK(sw_s >= 0 && sw_h >= 0 && so_s >= 0 && so_h >= 0, IQ_ERR_SHAPE);
  // (the strides of one sequence, or of one head, are of no account)
  IQ_CHECK(weights != weights_out || ((sw_s == so_s || p->S == 1) && (sw_h == so_h || p->H == 1)), IQ_ERR_SHAPE);
  IQ_CHECK(int64_t(p->S) * p->H <= INT32_MAX / SHIFT && p->P < INT32_MAX / PAGE - SELECT, IQ_ERR_SHAPE);
  IQ_CHECK(aligned(weights, 4) && aligned(weights_out, 4) && aligned(lens_out, 4), IQ_ERR_ALIGN);
  const size_t need = iq_paged_evict_workspace_bytes(p->S, p->P, p->H, keep, recent, shared);
  IQ_CHECK(workspace && workspace_bytes >= need, IQ_ERR_WORKSPACE);
  IQ_CHECK(aligned(workspace, 4), IQ_ERR_ALIGN);
  const int64_t most = rows_that_come(p->P, keep, recent), sh = int64_t(p->S) * p->H;
  // workgroups per (sequence, head) for `n` rows in turns of `rows`: at most 8192 in all, the longer lists in turns
  auto chunks_of = [&](int64_t n, int64_t rows) {
    const int64_t turns = sh < 8192 ? 8192 / sh : 1, c = ceil_div(n, rows);
    return int(c < 1 ? 1 : c < turns ? c : turns);
  };
  const int lanes = p->D / 8;
  EvictArgs a{*p, weights, sw_s, sw_h, weights_out, so_s, so_h, T, keep, recent, sinks, shared, int(most), lens_out,
              (int32_t*)workspace, chunks_of(most, FILL / lanes * BATCH)};
  const hipStream_t q = (hipStream_t)stream;
  const int64_t groups = int64_t(p->S) * (p->H / shared);
  if ((most + recent) * shared <= FEW_ROWS || groups >= FULL) {
    if (p->D == 128) evict_kernel<128><<<unsigned(groups), SELECT, 0, q>>>(a);
    else evict_kernel<64><<<unsigned(groups), SELECT, 0, q>>>(a);
    if (const int st = launch_status()) return st;
    if (lens_out != p->lens) return IQ_OK;
    lens_kernel<<<unsigned(ceil_div(p->S, 64)), 64, 0, q>>>(a);
    return launch_status();
  }
  select_kernel<<<p->S * (p->H / shared), SELECT, 0, q>>>(a);
  if (const int st = launch_status()) return st;
  auto rest = [&]<int D>() -> int {
    fill_kernel<D><<<unsigned(sh * a.chunks), FILL, 0, q>>>(a);
    if (const int st = launch_status()) return st;
    // a workgroup's turn: SHIFT / lanes * BATCH of the recent rows, and 8 weights per thread
    const int64_t rows = ceil_div(recent < p->P * int64_t(PAGE) ? recent : p->P * int64_t(PAGE), SHIFT / lanes * BATCH);
    const int64_t zeros = ceil_div(T, SHIFT * 8);
    a.chunks = chunks_of(rows > zeros ? rows : zeros, 1);
    shift_kernel<D><<<unsigned(sh * a.chunks), SHIFT, 0, q>>>(a);
    return launch_status();
  };
  return p->D == 128 ? rest.operator()<128>() : rest.operator()<64>();
}
