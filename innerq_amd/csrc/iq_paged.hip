// Appending to and reading 4-bit pages (gfx950): iq_paged_append, iq_paged_read; their status word: iq_paged_take_status.
//
// append: U = D/8 lanes hold one token of one head, 8 values each.  A lane that rotates reads its own 8 values and
// the 8 of its partner half (the second read hits L1), so neither the rotation nor a q rotated in place needs LDS;
// the group's minimum and maximum go over the 4 lanes of a group by DPP.  Each value is read once and each word
// written once: with many tokens both calls are bound by HBM (8 KV heads, 32 query heads, D = 128, bf16, 32760 tokens:
// append moves 713 MB in 150 us, 4.8 TB/s, what a large copy reaches; read 176 MB in 33 .. 40 us), with few by the
// loads that wait for each other: cu, the length, the table's entry, the angles (one token: 4 us).
#include "iq_paged.h"
#include "iq_quantize.h"

namespace {

constexpr int THREADS = 256;
constexpr int MOST_TOKENS = 1 << 27;  // of a call: a grid has less than 2^32 threads
constexpr int BATCH = 4;  // heads whose loads are under way together

struct AppendArgs {
  iq_paged p;
  const int32_t* cu;
  int N, Hq;
  const uint16_t *k, *v, *q;
  int64_t sk_n, sk_h, sv_n, sv_h, sq_n, sq_h;
  uint16_t* qo;
  int64_t so_n, so_h;
  const float *cos, *sin;
  int64_t n_pos;
  int R;
  const int32_t* evicted;  // tokens that each sequence has dropped (null: none): what its places are behind its positions
};

template <bool BF>
__device__ __forceinline__ void unpack8(u4_t w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = lo16(w[i], BF);
    f[2 * i + 1] = hi16(w[i], BF);
  }
}

// min / max over the 4 lanes of a quad, NaN propagating
template <int CTRL>
__device__ __forceinline__ float in_quad(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_min(float x) {
  x = __builtin_elementwise_minimum(x, in_quad<0xb1>(x));
  return __builtin_elementwise_minimum(x, in_quad<0x4e>(x));
}
__device__ __forceinline__ float quad_max(float x) {
  x = __builtin_elementwise_maximum(x, in_quad<0xb1>(x));
  return __builtin_elementwise_maximum(x, in_quad<0x4e>(x));
}

// 8 floats rounded to the activation dtype, in pairs (a conversion instruction per pair)
template <bool BF>
__device__ __forceinline__ u4_t pack8(const float (&f)[8]) {
  return u4_t{pack2<BF>(f[0], f[1]), pack2<BF>(f[2], f[3]), pack2<BF>(f[4], f[5]), pack2<BF>(f[6], f[7])};
}

// the 4-bit word of 8 values and its group's meta word (quant.py's asymmetric form, every op rounded to the type)
template <bool BF>
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], uint32_t& meta) {
  float mn = x[0], mx = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    mn = __builtin_elementwise_minimum(mn, x[i]);
    mx = __builtin_elementwise_maximum(mx, x[i]);
  }
  const GroupQ g = group_params<4, IQ_MODE_ASYM, BF>(quad_min(mn), quad_max(mx), 0.f);
  uint32_t w = 0;
  if (!g.slow) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = x[i] - g.z;
    unpack8<BF>(pack8<BF>(y), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(y[i], g.r);
    unpack8<BF>(pack8<BF>(y), y);
#pragma unroll
    for (int i = 0; i < 8; ++i)  // the code is in the low bits of clamp_rne's pattern
      w += __float_as_uint(clamp_rne<4>(y[i], false)) << (4 * i);
    w -= shifted_sum(RNE_BITS, 8, 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= asym_field_b(asym_code_b(x[i], g.z, g.s, 4, BF), 4) << (4 * i);
  }
  meta = meta_word(g.s, g.z, BF);
  return w;
}

// rotation of the 8 values f (dims 8o ..) with their partners p (s negated in the first half): fp32 products, each
// rounded, as separate torch ops
__device__ __forceinline__ void rotate8(float (&f)[8], const float (&p)[8], const float (&c)[8], const float (&s)[8]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = f[i] * c[i], b = p[i] * s[i];
    f[i] = a + b;
  }
}

// A lane's share of token n, which cannot be appended: its queries are NaN, and so is its row of its page, where it has
// one (a token past the rotation's rows), so that nothing computed from it passes for a result.
template <int D>
__device__ __forceinline__ void refuse(const AppendArgs& a, int n, int page, int row, int h0, int h1) {
  constexpr int U = D / 8;
  constexpr uint32_t nan2 = 0x7fff7fffu;  // of both activation dtypes
  const int o = threadIdx.x % U, H = a.p.H, b = v_block(row), e = v_place(row);
#pragma clang loop unroll(disable)
  for (int h = h0; h < h1; ++h) {
    if (h >= 2 * H) {
      *reinterpret_cast<u4_t*>(a.qo + n * a.so_n + (h - 2 * H) * a.so_h + 8 * o) = u4_t{nan2, nan2, nan2, nan2};
    } else if (page >= 0) {
      uint32_t* pg = a.p.pages + (int64_t(page) * H + (h < H ? h : h - H)) * page_words(D);
      if (h < H) {
        pg[row * U + o] = 0;
        if (o % 4 == 0) pg[page_km(D) + row * (D / 32) + o / 4] = nan2;
      } else {
        pg[page_vc(D) + (b * U + o) * 8 + e] = 0;
        if (o % 4 == 0) {
          uint16_t* m = reinterpret_cast<uint16_t*>(pg + page_vm(D)) + (b * (D / 32) + o / 4) * 16 + e;
          m[0] = m[8] = uint16_t(nan2);
        }
      }
    }
  }
}

template <int D, bool BF>
__global__ __launch_bounds__(THREADS) void append_kernel(AppendArgs a, int heads_per_block) {
  constexpr int U = D / 8, TOK = THREADS / U;
  const int o = threadIdx.x % U, n = blockIdx.x * TOK + threadIdx.x / U;
  int s, i;
  if (n >= a.N || !sequence_of(a.cu, a.p.S, n, s, i)) return;
  const int held = a.p.lens[s];
  const int64_t at = int64_t(held) + i;
  const int H = a.p.H, heads = 2 * H + (a.q ? a.Hq : 0);
  const int64_t pos = at + (a.evicted ? a.evicted[s] : 0);
  int32_t bad = 0, page = -1;
  if (held < 0 || at >= int64_t(a.p.P) * PAGE) bad = PAGED_BAD_TOKEN;
  else {
    page = a.p.table[s * a.p.s_table + at / PAGE];
    if (page < 0 || page >= a.p.n_pages) {
      bad = PAGED_BAD_PAGE;
      page = -1;
    }
    if (a.cos && (pos < 0 || pos >= a.n_pos)) bad |= PAGED_BAD_TOKEN;
  }
  const int row = int(at % PAGE);
  if (bad) {
    if (o == 0 && blockIdx.y == 0) atomicOr(a.p.status, bad);
    refuse<D>(a, n, page, row, blockIdx.y * heads_per_block, min(heads, int(blockIdx.y + 1) * heads_per_block));
    return;
  }
  const bool turn = a.cos && 8 * o < a.R, second = 16 * o >= a.R;
  float c[8], sn[8];
  if (turn) {
    const int64_t d = pos * (a.R / 2) + 8 * o - (second ? a.R / 2 : 0);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f4_t x = *reinterpret_cast<const f4_t*>(a.cos + d + 4 * j), y = *reinterpret_cast<const f4_t*>(a.sin + d + 4 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) { c[4 * j + e] = x[e]; sn[4 * j + e] = second ? y[e] : -y[e]; }
    }
  }
  const int partner = (second ? -a.R : a.R) / 2, h1 = min(heads, int(blockIdx.y + 1) * heads_per_block);
  for (int h0 = blockIdx.y * heads_per_block; h0 < h1; h0 += BATCH) {
    u4_t own[BATCH], other[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {  // (past the block's last head: that one again)
      const int h = min(h0 + i, h1 - 1);
      const uint16_t* x = h < H ? a.k + n * a.sk_n + h * a.sk_h : h < 2 * H ? a.v + n * a.sv_n + (h - H) * a.sv_h
                                                                           : a.q + n * a.sq_n + (h - 2 * H) * a.sq_h;
      own[i] = *reinterpret_cast<const u4_t*>(x + 8 * o);
      other[i] = turn ? *reinterpret_cast<const u4_t*>(x + 8 * o + partner) : u4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = h0 + i;
      if (h >= h1) break;
      const bool isv = h >= H && h < 2 * H;
      float f[8];
      u4_t x = own[i];
      if (turn && !isv) {
        float p[8];
        unpack8<BF>(x, f);
        unpack8<BF>(other[i], p);
        rotate8(f, p, c, sn);
        x = pack8<BF>(f);
      }
      if (h >= 2 * H) {
        // (non-temporal: 4 prompts of 8190 tokens 193 us against 197 with their read, a ragged batch 58 against 62; a
        // step's attention right behind it takes the same time)
        __builtin_nontemporal_store(x, reinterpret_cast<u4_t*>(a.qo + n * a.so_n + (h - 2 * H) * a.so_h + 8 * o));
        continue;
      }
      unpack8<BF>(x, f);
      uint32_t meta;
      const uint32_t w = quantize8<BF>(f, meta);
      uint32_t* pg = a.p.pages + (int64_t(page) * H + (isv ? h - H : h)) * page_words(D);
      if (!isv) {
        pg[row * U + o] = w;
        if (o % 4 == 0) pg[page_km(D) + row * (D / 32) + o / 4] = meta;
      } else {
        const int b = v_block(row), e = v_place(row);
        pg[page_vc(D) + (b * U + o) * 8 + e] = w;
        if (o % 4 == 0) {
          uint16_t* m = reinterpret_cast<uint16_t*>(pg + page_vm(D)) + (b * (D / 32) + o / 4) * 16 + e;
          m[0] = uint16_t(meta);
          m[8] = uint16_t(meta >> 16);
        }
      }
    }
  }
}

struct ReadArgs {
  iq_paged p;
  const int32_t* cu;
  int N;
  uint16_t *k, *v;
  int64_t sk_n, sk_h, sv_n, sv_h;
};

// a lane: 8 values of one token, for each of the block's heads of K and V
template <int D, bool BF>
__global__ __launch_bounds__(THREADS) void read_kernel(ReadArgs a, int heads_per_block) {
  constexpr int U = D / 8, TOK = THREADS / U;
  const int o = threadIdx.x % U, n = blockIdx.x * TOK + threadIdx.x / U;
  int s, i;
  if (n >= a.N || !sequence_of(a.cu, a.p.S, n, s, i)) return;
  const int held = a.p.lens[s];
  const int64_t at = int64_t(held) + i;
  const int H = a.p.H;
  int32_t bad = 0, page = 0;
  if (held < 0 || at >= int64_t(a.p.P) * PAGE) bad = PAGED_BAD_TOKEN;
  else {
    page = a.p.table[s * a.p.s_table + at / PAGE];
    if (page < 0 || page >= a.p.n_pages) bad = PAGED_BAD_PAGE;
  }
  if (bad && o == 0 && blockIdx.y == 0) atomicOr(a.p.status, bad);
  const int row = int(at % PAGE), b = v_block(row), e = v_place(row);
  const int h1 = min(2 * H, int(blockIdx.y + 1) * heads_per_block);
  for (int h0 = blockIdx.y * heads_per_block; h0 < h1; h0 += BATCH) {
    uint32_t w[BATCH], s16[BATCH], z16[BATCH];
    if (!bad) {
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {  // (past the block's last head: that one again)
        const int h = min(h0 + i, h1 - 1);
        const bool isv = h >= H;
        const uint32_t* pg = a.p.pages + (int64_t(page) * H + (isv ? h - H : h)) * page_words(D);
        const uint16_t* m = reinterpret_cast<const uint16_t*>(pg);
        w[i] = pg[isv ? page_vc(D) + (b * U + o) * 8 + e : row * U + o];
        const int at16 = isv ? 2 * page_vm(D) + (b * (D / 32) + o / 4) * 16 + e : 2 * (page_km(D) + row * (D / 32) + o / 4);
        s16[i] = m[at16];
        z16[i] = m[at16 + (isv ? 8 : 1)];
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = h0 + i;
      if (h >= h1) break;
      u4_t r = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};  // no such token: NaN
      if (!bad) {
        const u4_t x = k_values<BF>(w[i], s16[i] | z16[i] << 16);  // pairs (0,2) (4,6) (1,3) (5,7) -> (0,1) (2,3) (4,5) (6,7)
        r = u4_t{__builtin_amdgcn_perm(x[2], x[0], 0x05040100u), __builtin_amdgcn_perm(x[2], x[0], 0x07060302u),
                 __builtin_amdgcn_perm(x[3], x[1], 0x05040100u), __builtin_amdgcn_perm(x[3], x[1], 0x07060302u)};
      }
      uint16_t* out = h >= H ? a.v + n * a.sv_n + (h - H) * a.sv_h : a.k + n * a.sk_n + h * a.sk_h;
      *reinterpret_cast<u4_t*>(out + 8 * o) = r;
    }
  }
}

__global__ void take_status_kernel(int32_t* status, int32_t* taken) { *taken = atomicExch(status, 0); }

// Heads that a block does for its tokens: one while there are few blocks; then as many as leave `blocks` blocks, up to
// `most`, a power of two (finding a token, three or more loads that wait for each other, then serves all of them).
//   append, 768 blocks, 16 heads at most (8 KV, 32 query heads, D = 128, bf16; us with 1, 2, 4, 8, 16 heads per block):
//     256 tokens 4.9 5.1 6.1 8.5 13; 1024: 12 9.0 7.3 9.8 15; 2048: 24 17 13 12 17; 32768: 418 257 175 164 149
//     (2 KV, 8 query heads, 4096 tokens: 12 9.1 7.4 8.6 9.8; 32 and 32, 256 tokens: 7.2 5.7 6.3 8.6 13)
//   read, 256 blocks, 4 heads: 256 tokens 3.8 3.9 4.1 5.1 6.4; 1024: 5.2 4.7 4.6 5.5 6.8; 32768: 72 43 33 33 33
inline int heads_per_block(int tiles, int heads, int blocks, int most) {
  int n = 1;
  while (2 * n <= most && int64_t(tiles) * heads >= int64_t(blocks) * 2 * n) n *= 2;
  return n;
}

inline bool rows_ok(const void* p, int64_t s_n, int64_t s_h) { return aligned(p, 16) && s_n % 8 == 0 && s_h % 8 == 0; }

template <typename F>
int by_format(int D, int mode, F&& f) {
  if (D == 128) return mode & IQ_MODE_BF16 ? f.template operator()<128, true>() : f.template operator()<128, false>();
  return mode & IQ_MODE_BF16 ? f.template operator()<64, true>() : f.template operator()<64, false>();
}

}  // namespace

namespace iq {
int check_paged(const iq_paged* p) {
  IQ_CHECK(p && p->pages && p->table && p->lens && p->status, IQ_ERR_NULL);
  IQ_CHECK(base_mode(p->mode) == IQ_MODE_ASYM, IQ_ERR_MODE);
  IQ_CHECK(d_ok(p->D) && p->H > 0 && p->H <= 4096 && p->S > 0 && p->P > 0 && p->n_pages > 0, IQ_ERR_SHAPE);
  IQ_CHECK(p->P <= INT32_MAX / PAGE && p->n_pages <= INT32_MAX && p->s_table >= 0, IQ_ERR_SHAPE);
  IQ_CHECK(aligned(p->pages, 16) && aligned(p->table, 4) && aligned(p->lens, 4) && aligned(p->status, 4), IQ_ERR_ALIGN);
  return IQ_OK;
}
}  // namespace iq

extern "C" int iq_page_bytes(int H, int D, int64_t* bytes) {
  IQ_CHECK(bytes, IQ_ERR_NULL);
  IQ_CHECK(d_ok(D) && H > 0 && H <= 4096, IQ_ERR_SHAPE);
  *bytes = int64_t(H) * page_words(D) * 4;
  return IQ_OK;
}

extern "C" int iq_paged_take_status(int32_t* status, int32_t* taken, void* stream) {
  IQ_CHECK(status && taken, IQ_ERR_NULL);
  IQ_CHECK(aligned(status, 4) && aligned(taken, 4), IQ_ERR_ALIGN);
  take_status_kernel<<<1, 1, 0, (hipStream_t)stream>>>(status, taken);
  return launch_status();
}

extern "C" int iq_paged_append(const iq_paged* p, const int32_t* cu, int N, const void* k, int64_t sk_n, int64_t sk_h,
                               const void* v, int64_t sv_n, int64_t sv_h, const float* cos, const float* sin,
                               int64_t n_pos, int R, const void* q, int64_t sq_n, int64_t sq_h, int Hq, void* q_out,
                               int64_t so_n, int64_t so_h, void* stream) {
  return iq_paged_append_at(p, cu, N, k, sk_n, sk_h, v, sv_n, sv_h, cos, sin, n_pos, R, nullptr, q, sq_n, sq_h, Hq, q_out, so_n,
                            so_h, stream);
}

extern "C" int iq_paged_append_at(const iq_paged* p, const int32_t* cu, int N, const void* k, int64_t sk_n, int64_t sk_h,
                                  const void* v, int64_t sv_n, int64_t sv_h, const float* cos, const float* sin,
                                  int64_t n_pos, int R, const int32_t* evicted, const void* q, int64_t sq_n, int64_t sq_h,
                                  int Hq, void* q_out, int64_t so_n, int64_t so_h, void* stream) {
  if (const int st = iq::check_paged(p)) return st;
  IQ_CHECK((N == 0 || (k && v && (!q || q_out))) && (!cos == !sin), IQ_ERR_NULL);
  IQ_CHECK(N >= 0 && N <= MOST_TOKENS && (cu || N == p->S), IQ_ERR_SHAPE);
  IQ_CHECK(!q || (Hq > 0 && Hq <= 4096), IQ_ERR_SHAPE);
  IQ_CHECK(!cos || (R > 0 && R <= p->D && R % 16 == 0 && n_pos > 0), IQ_ERR_SHAPE);
  IQ_CHECK(rows_ok(k, sk_n, sk_h) && rows_ok(v, sv_n, sv_h) && aligned(cos, 16) && aligned(sin, 16), IQ_ERR_ALIGN);
  IQ_CHECK(!q || (rows_ok(q, sq_n, sq_h) && rows_ok(q_out, so_n, so_h)), IQ_ERR_ALIGN);
  IQ_CHECK(aligned(evicted, 4), IQ_ERR_ALIGN);
  if (N == 0) return IQ_OK;
  const AppendArgs a{*p, cu, N, Hq, (const uint16_t*)k, (const uint16_t*)v, (const uint16_t*)q, sk_n, sk_h, sv_n, sv_h,
                     sq_n, sq_h, (uint16_t*)q_out, so_n, so_h, cos, sin, n_pos, R, evicted};
  return by_format(p->D, p->mode, [&]<int D, bool BF>() {
    const int tiles = int(ceil_div(N, THREADS / (D / 8))), heads = 2 * p->H + (q ? Hq : 0);
    const int hpb = heads_per_block(tiles, heads, 768, 16);
    append_kernel<D, BF><<<dim3(tiles, unsigned(ceil_div(heads, hpb))), THREADS, 0, (hipStream_t)stream>>>(a, hpb);
    return launch_status();
  });
}

extern "C" int iq_paged_read(const iq_paged* p, const int32_t* cu, int N, void* k_out, int64_t sk_n, int64_t sk_h,
                             void* v_out, int64_t sv_n, int64_t sv_h, void* stream) {
  if (const int st = iq::check_paged(p)) return st;
  IQ_CHECK(N == 0 || (k_out && v_out), IQ_ERR_NULL);
  IQ_CHECK(N >= 0 && N <= MOST_TOKENS && (cu || N == p->S), IQ_ERR_SHAPE);
  IQ_CHECK(rows_ok(k_out, sk_n, sk_h) && rows_ok(v_out, sv_n, sv_h), IQ_ERR_ALIGN);
  if (N == 0) return IQ_OK;
  const ReadArgs a{*p, cu, N, (uint16_t*)k_out, (uint16_t*)v_out, sk_n, sk_h, sv_n, sv_h};
  return by_format(p->D, p->mode, [&]<int D, bool BF>() {
    const int tiles = int(ceil_div(N, THREADS / (D / 8))), hpb = heads_per_block(tiles, 2 * p->H, 256, 4);
    read_kernel<D, BF><<<dim3(tiles, unsigned(ceil_div(2 * p->H, hpb))), THREADS, 0, (hipStream_t)stream>>>(a, hpb);
    return launch_status();
  });
}
