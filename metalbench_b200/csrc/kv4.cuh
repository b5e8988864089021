// The 4-bit paged KV cache: page layout shared by the storing kernels (kv4.cu)
// and the attention over it (attention_kv4.cu).
//
// cache = uint8 [num_pages][Hkv][KV4_BLOB]; the bytes of one page (64 tokens)
// and one kv head (128 dims) are
//   [0, 4096)     key codes: token t at byte 64 t, byte j = dim 2j (low four
//                 bits) and dim 2j + 1 (high four bits)
//   [4096, 8192)  value codes, the same, but the 16-byte piece c of token t
//                 stands at piece c ^ ((t >> 1) & 3), so that ldmatrix reads
//                 one piece of eight tokens from eight different bank groups
//   [8192, 8448)  per token: bf16 scale, bf16 minimum of the key
//   [8448, 8704)  per token: bf16 scale, bf16 minimum of the value
// A code u stands for minimum + scale * u. One page and head is one contiguous
// copy of 8704 bytes (a multiple of 512): keys, values and their scales travel
// together, and the page operations (kv_pages.cu) move pages without looking
// inside.
#pragma once
#include "common.cuh"

namespace kv4 {
constexpr int PAGE = 64;
constexpr int DH = 128;
constexpr int ROW = DH / 2;  // bytes of one token's codes
constexpr int V_CODES = PAGE * ROW;
constexpr int K_PARAMS = 2 * PAGE * ROW;
constexpr int V_PARAMS = K_PARAMS + PAGE * 4;
constexpr int BLOB = V_PARAMS + PAGE * 4;  // 8704

// Byte of word w (8 dims) of token t's value codes.
__host__ __device__ constexpr int v_word(int t, int w) {
  return V_CODES + t * ROW + (((w >> 2) ^ ((t >> 1) & 3)) << 4) + ((w & 3) << 2);
}
__device__ __forceinline__ float lo_bf(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// The exponent that takes a largest magnitude to [2^14, 2^15), within
// [-112, 113] (all of bf16 but its subnormals; 0 for a maximum of 0): x 2^-e is
// then an fp16 number to 2^-11 of itself down to 2^-29 of the largest, and to
// 2^-40 of the largest below.
__device__ __forceinline__ int fp16_exp(float most) {
  return most > 0.f ? max(-112, min(113, (__float_as_int(most) >> 23) - 127 - 14)) : 0;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((127 + e) << 23); }  // |e| <= 126
}  // namespace kv4
