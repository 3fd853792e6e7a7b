// Attention over packed prompts (gfx950): what iq_prompt.hip (attention), iq_prompt_weights.hip (the weights that keys
// gather) and iq_diff_prompt.hip (differential attention) share.
#pragma once
#include "iq_paged.h"

namespace iq {

typedef float f16_t __attribute__((ext_vector_type(16)));
typedef short s4_t __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr float NEG_INF = -__builtin_inff();

// A scale as the kernels take it: |scale| log2(e) (1 for 0), and what is and-ed and xor-ed into the queries or keys: a
// scale of 0 clears them, a negative one flips their signs.
struct Scale {
  float c;
  uint32_t keep, sign;
};
inline Scale scale_of(float scale) {
  const float c = scale * 1.44269504088896340736f;
  return {c == 0 ? 1.f : c < 0 ? -c : c, c == 0 ? 0u : ~0u, c < 0 ? 0x80008000u : 0u};
}

// 16 bytes per lane from the descriptor's byte `at` (per lane) to LDS, lane by lane from `lds` on, without registers
__device__ __forceinline__ void load_to_lds(rsrc_t d, u4_t* lds, uint32_t at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (__attribute__((address_space(3))) void*)lds, 16, at, 0, 0, 0);
}

// rows [r0, r1) of sequence s in a packed tensor of n rows (whatever cu holds)
template <typename Cu>
__device__ __forceinline__ void rows_of(Cu cu, int s, int n, int& r0, int& r1) {
  r0 = min(max(cu[s], 0), n);
  r1 = min(max(cu[s + 1], r0), n);
}

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

// The weights of one attention call's keys (iq_prompt_weights.hip): q, k, lengths and masks as the call's, stats [N][Hq]
// {base, 1 / sum} of its rows: a weight is 2^(logit c - base) / sum.
struct WeighArgs {
  const uint16_t *q, *k;
  int64_t sq_n, sq_h, sk_n, sk_h;
  const float2* stats;
  float* weights;  // [S][H][T]
  int64_t sw_s, sw_h, T;
  const int32_t *cu_q, *cu_k;
  int S, N, Nk, Hq, nrep, slots;
  Scale scale;
  int causal, window;
  int maps;  // 2: differential attention, KV head 2g + i's rows are those of query heads 2j + i, j in its group
  // set by launch_prompt_weights: workgroups that share a key, and where several do, their sums [shares][H][Nk]
  int shares;
  float* part;
  int steps;  // tiles of keys of a workgroup
  int chunk_bits;  // rows of a chunk that a share takes in one go
};
// its workspace: the stats, then the sums
size_t prompt_weights_bytes(int S, int N, int Nk, int Hq, int H);  // (a multiple of 16)
bool prompt_weights_fit(int S, int N, int Nk, int Hq, int H);  // a launch's limits
int launch_prompt_weights(WeighArgs a, int D, bool bf, hipStream_t stream);

}  // namespace iq
