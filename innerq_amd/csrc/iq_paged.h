// 4-bit pages (gfx950), shared by iq_paged.hip (append, read) and iq_paged_attn.hip.
//
// A page holds 64 tokens of every KV head, K and V both in 4-bit asym groups of 32 along head_dim, so a token is
// whole in its page as soon as it is appended: sequences of any lengths append one token or many without an fp16
// window, and no two tokens share a word of codes.  One (page, head) is one run of 32-bit words (U = D/8, G = D/32):
//
//   K codes  [64 tokens][U]            a token's row: one 16-byte load per lane is one group (D = 128)
//   K meta   [64 tokens][G]            {scale, zero} halves
//   V codes  [8 blocks][U][8 tokens]   one lane's two 16-byte loads are 8 dims of the 8 tokens of an MFMA operand
//   V meta   [8 blocks][G][8 scales | 8 zeros]
//
// A word is 8 codes of one token (dims 8o .. 8o+7, code i at bits 4i).  V block b = t/32*4 + t%16/4 holds the tokens
// whose logits one lane of the QK^T product's result holds (t%4 and t/16%2 give the place in it), so the softmax
// weights are the next product's operand where they are, with no exchange between lanes.
#pragma once
#include "iq_common.h"
#include "iq_device.h"

namespace iq {

constexpr int PAGE = 64;
__host__ __device__ constexpr int page_km(int D) { return PAGE * (D / 8); }                 // K meta's first word
__host__ __device__ constexpr int page_vc(int D) { return PAGE * (D / 8 + D / 32); }        // V codes'
__host__ __device__ constexpr int page_vm(int D) { return page_vc(D) + PAGE * (D / 8); }    // V meta's
__host__ __device__ constexpr int page_words(int D) { return 2 * PAGE * (D / 8 + D / 32); }
__host__ __device__ constexpr int v_block(int t) { return t / 32 * 4 + t % 16 / 4; }
__host__ __device__ constexpr int v_place(int t) { return t % 4 + t / 16 % 2 * 4; }

// bits of a store's status word (iq_paged.status)
constexpr int32_t PAGED_BAD_PAGE = IQ_PAGED_BAD_PAGE, PAGED_BAD_TOKEN = IQ_PAGED_BAD_TOKEN;

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
typedef float fl2_t __attribute__((ext_vector_type(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));

// two floats rounded to the activation dtype (nearest even), as one dword
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const fl2_t x = {a, b};
  if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf2_t));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, h2_t));
}

template <bool BF>
__device__ __forceinline__ float lo_half(uint32_t w) { return BF ? __uint_as_float(w << 16) : float(__builtin_bit_cast(h2_t, w).x); }
template <bool BF>
__device__ __forceinline__ float hi_half(uint32_t w) {
  return BF ? __uint_as_float(w & 0xffff0000u) : float(__builtin_bit_cast(h2_t, w).y);
}

// ---- values of packed codes: RN(c s + z) in the activation dtype ---------------------------------------------
// Codes leave their nibbles for bytes, and a byte 0 .. 15 is, as an OCP e4m3 number, exactly its code times 2^-9: one
// conversion per two codes.  fp16: one packed fma rounds c s + z once.  bf16 has no packed arithmetic on gfx950: fp32
// (c s is exact there, the sum rounds to 24 bits first, as the reference's fp32 dequantization followed by a cast).

// codes in bytes 0, 1 (HI: 2, 3) of x
template <bool HI>
__device__ __forceinline__ fl2_t codes2(uint32_t x) { return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, 512.f, HI); }
template <bool HI>
__device__ __forceinline__ h2_t codes2h(uint32_t x) {
  return __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 512.f, HI));
}

// the values of four codes in the bytes of x: of the pair in bytes 0, 1 with scales s and zeros z (a pair of halves
// each), of that in bytes 2, 3
template <bool BF>
__device__ __forceinline__ u2_t values4(uint32_t x, uint32_t s, uint32_t z) {
  if constexpr (!BF) {
    const h2_t sh = __builtin_bit_cast(h2_t, s), zh = __builtin_bit_cast(h2_t, z);
    return u2_t{__builtin_bit_cast(uint32_t, __builtin_elementwise_fma(codes2h<false>(x), sh, zh)),
                __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(codes2h<true>(x), sh, zh))};
  } else {
    const float s0 = lo_half<BF>(s), s1 = hi_half<BF>(s), z0 = lo_half<BF>(z), z1 = hi_half<BF>(z);
    const fl2_t a = codes2<false>(x), b = codes2<true>(x);
    return u2_t{pack2<true>(__builtin_fmaf(a.x, s0, z0), __builtin_fmaf(a.y, s1, z1)),
                pack2<true>(__builtin_fmaf(b.x, s0, z0), __builtin_fmaf(b.y, s1, z1))};
  }
}

// the values of one token's word w with meta {s, z}: dwords of the pairs (0,2), (4,6), (1,3), (5,7)
template <bool BF>
__device__ __forceinline__ u4_t k_values(uint32_t w, uint32_t meta) {
  const uint32_t s = __builtin_amdgcn_perm(meta, meta, 0x01000100u), z = __builtin_amdgcn_perm(meta, meta, 0x03020302u);
  const u2_t e = values4<BF>(w & 0x0f0f0f0fu, s, z), o = values4<BF>((w >> 4) & 0x0f0f0f0fu, s, z);
  return u4_t{e.x, e.y, o.x, o.y};
}

// inclusive sum over the wave's 64 lanes (of ints; every lane takes part): within rows of 16, then from row to row
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// ---- shares --------------------------------------------------------------------------------------------------
// A list of `total` units (up to 2^31 - 1) shared out evenly over `grid` workgroups: workgroup g's are the units from
// share_begin(g) to share_begin(g + 1), unit u's workgroup is u / per.  A page per wave (of four) at least.
constexpr int SHARE_LEAST = 4;
__host__ __device__ inline int units_per_group(int total, int grid) {
  const int n = total / grid + (total % grid ? 1 : 0);
  return n < SHARE_LEAST ? SHARE_LEAST : n;
}
__host__ __device__ inline int share_begin(int g, int per, int total) {
  const int64_t u = int64_t(g) * per;
  return int(u < total ? u : total);
}

// ---- sequences -----------------------------------------------------------------------------------------------
// token n of a flat list belongs to sequence s at place i (cu null: one token each); false: to none
__device__ __forceinline__ bool sequence_of(const int32_t* cu, int S, int n, int& s, int& i) {
  if (!cu) { s = n; i = 0; return n < S; }
  int lo = 0, hi = S;  // cu[lo] <= n < cu[hi], where there is such a sequence
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= n) lo = mid; else hi = mid;
  }
  s = lo;
  i = n - cu[lo];
  return i >= 0 && n < cu[lo + 1];
}

}  // namespace iq
