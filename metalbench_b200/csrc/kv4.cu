// Storing tokens in the 4-bit paged KV cache and reading them back (layout in
// kv4.cuh). The 4-bit counterpart of the cache write that the decoder layer's
// QKV epilogue does in bf16.
//
// For the 128 dims x of one token and kv head (keys and values alike):
//   m = min x,  s = bf16((max x - m) / 15),  u = clamp(rint((x - m) / s), 0, 15)
// with u = 0 where s = 0; the stored value is m + s u. m is exact (x is bf16);
// s is rounded to bf16 (2^-9 relative: at most 3 % of one code step at u = 15)
// because its 2 bytes a token are read by every later step. The arithmetic is
// IEEE fp32 with one rounding per operation.
#include "kv4.cuh"
#include "kernels.h"

namespace {
using namespace kv4;

__device__ __forceinline__ float min_nan(float a, float b) {  // a NaN stays one
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Page of position `pos` of sequence b, or -1 (recorded in the status word).
__device__ __forceinline__ int page_of(const int* __restrict__ table, int max_pages, int num_pages,
                                       int b, int64_t pos, uint32_t* status) {
  int pg = -1;
  if (pos >= 0 && pos < (int64_t)max_pages * PAGE) pg = table[(int64_t)b * max_pages + pos / PAGE];
  if (pg >= 0 && pg < num_pages) return pg;
  atomicOr(status, MB_DEV_BAD_PAGE);
  return -1;
}

// One warp stores one (token, kv head): lanes 0-15 the key, lanes 16-31 the
// value, eight dims a lane, so that minimum and maximum take four shuffles and
// every lane packs one 32-bit word of codes.
__global__ void __launch_bounds__(256) kv4_append_kernel(
    const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int64_t stride_b,
    int64_t stride_s, int64_t stride_h, int64_t vstride_b, int64_t vstride_s, int64_t vstride_h,
    uint8_t* __restrict__ cache, int num_pages, int Hkv, const int* __restrict__ table,
    int max_pages, const int* __restrict__ start_pos, const int* __restrict__ new_len, int64_t total,
    int S, uint32_t* status) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= total) return;
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const int64_t tok = item / Hkv;
  const int h = (int)(item - tok * Hkv);
  const int b = (int)(tok / S), s = (int)(tok - (int64_t)b * S);
  if (new_len && s >= new_len[b]) return;
  const int64_t pos = (int64_t)start_pos[b] + s;
  const uint16_t* src = half ? v + b * vstride_b + s * vstride_s + h * vstride_h
                             : k + b * stride_b + s * stride_s + h * stride_h;
  const uint4 raw = *reinterpret_cast<const uint4*>(src + l * 8);
  const int pg = page_of(table, max_pages, num_pages, b, pos, status);
  if (pg < 0) return;
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = lo_bf(w[i]);
    x[2 * i + 1] = hi_bf(w[i]);
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, x[i]);
    hi = max_nan(hi, x[i]);
  }
#pragma unroll
  for (int off = 8; off; off >>= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, off));
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(hi - lo, 15.f));
  const float sc = __bfloat162float(sb);
  uint32_t code = 0;
  if (sc > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = fminf(fmaxf(rintf(__fdiv_rn(x[i] - lo, sc)), 0.f), 15.f);
      code |= (uint32_t)u << (4 * i);
    }
  }
  uint8_t* blob = cache + ((int64_t)pg * Hkv + h) * BLOB;
  const int t = (int)(pos & (PAGE - 1));
  *reinterpret_cast<uint32_t*>(blob + (half ? v_word(t, l) : t * ROW + l * 4)) = code;
  if (l == 0) {
    const uint32_t par = (uint32_t)__bfloat16_as_ushort(sb) | (__float_as_uint(lo) & 0xFFFF0000u);
    *reinterpret_cast<uint32_t*>(blob + (half ? V_PARAMS : K_PARAMS) + t * 4) = par;
  }
}

// Positions start_pos[b] .. start_pos[b] + S - 1 back as fp32 [B][S][Hkv][128]
// (zeros at and past kv_len[b]); lanes as in the storing kernel.
__global__ void __launch_bounds__(256) kv4_gather_kernel(
    const uint8_t* __restrict__ cache, int num_pages, int Hkv, const int* __restrict__ table,
    int max_pages, const int* __restrict__ start_pos, const int* __restrict__ kv_len, int64_t total,
    int S, float* __restrict__ ko, float* __restrict__ vo, uint32_t* status) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= total) return;
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const int64_t tok = item / Hkv;
  const int h = (int)(item - tok * Hkv);
  const int b = (int)(tok / S), s = (int)(tok - (int64_t)b * S);
  const int64_t pos = (int64_t)start_pos[b] + s;
  float o[8] = {};
  if (pos < kv_len[b]) {
    const int pg = page_of(table, max_pages, num_pages, b, pos, status);
    if (pg >= 0) {
      const uint8_t* blob = cache + ((int64_t)pg * Hkv + h) * BLOB;
      const int t = (int)(pos & (PAGE - 1));
      const uint32_t code =
          *reinterpret_cast<const uint32_t*>(blob + (half ? v_word(t, l) : t * ROW + l * 4));
      const uint32_t par =
          *reinterpret_cast<const uint32_t*>(blob + (half ? V_PARAMS : K_PARAMS) + t * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i)  // one rounding: scale * code is exact (8 + 4 bits)
        o[i] = fmaf(lo_bf(par), (float)((code >> (4 * i)) & 15u), hi_bf(par));
    }
  }
  float4* dst = reinterpret_cast<float4*>((half ? vo : ko) + item * DH + l * 8);
  dst[0] = make_float4(o[0], o[1], o[2], o[3]);
  dst[1] = make_float4(o[4], o[5], o[6], o[7]);
}

// Pages of B sequences as bf16 pages [B * max_pages][Hkv][64][128], with the
// block table, lengths and first positions that go with them: one CTA a page
// and kv head, lanes as in the storing kernel. A value is rounded to bf16 here
// (2^-9 relative), as a bf16 cache would hold it.
__global__ void __launch_bounds__(256) kv4_expand_kernel(
    const uint8_t* __restrict__ cache, int num_pages, int Hkv, const int* __restrict__ table,
    int max_pages, const int* __restrict__ kv_len, const int* __restrict__ start_pos,
    uint16_t* __restrict__ ko, uint16_t* __restrict__ vo, int* __restrict__ table_o,
    int* __restrict__ len_o, int* __restrict__ start_o, uint32_t* status) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int page = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int L = max(0, min(kv_len[b], max_pages * PAGE));
  if (threadIdx.x == 0 && h == 0 && page == 0) {
    len_o[b] = L;
    start_o[b] = start_pos ? min(start_pos[b], L) : L;
  }
  if (page * PAGE >= L) return;
  const int64_t to = (int64_t)b * max_pages + page;
  if (threadIdx.x == 0 && h == 0) table_o[to] = (int)to;
  const int pg = page_of(table, max_pages, num_pages, b, (int64_t)page * PAGE, status);
  const uint8_t* blob = cache + ((int64_t)max(pg, 0) * Hkv + h) * BLOB;
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  uint16_t* dst = (half ? vo : ko) + (to * Hkv + h) * (PAGE * DH) + l * 8;
  const int par_at = half ? V_PARAMS : K_PARAMS;
#pragma unroll
  for (int i = 0; i < PAGE / 8; ++i) {
    const int t = i * 8 + (threadIdx.x >> 5);
    uint32_t w[4] = {};
    if (pg >= 0 && page * PAGE + t < L) {  // the rest is read as zeros: what stands there may be anything
      const uint32_t code = *reinterpret_cast<const uint32_t*>(blob + (half ? v_word(t, l) : t * ROW + l * 4));
      const uint32_t par = *reinterpret_cast<const uint32_t*>(blob + par_at + t * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(
            fmaf(lo_bf(par), (float)((code >> (8 * j)) & 15u), hi_bf(par)),
            fmaf(lo_bf(par), (float)((code >> (8 * j + 4)) & 15u), hi_bf(par)));
        w[j] = *reinterpret_cast<const uint32_t*>(&x);
      }
    }
    *reinterpret_cast<uint4*>(dst + t * DH) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace

namespace mb {
int kv4_expand(const uint8_t* cache, int num_pages, int Hkv, const int* table, int max_pages,
               const int* kv_len, const int* start_pos, int B, uint16_t* ko, uint16_t* vo,
               int* table_o, int* len_o, int* start_o, uint32_t* status, cudaStream_t s) {
  MB_CUDA(launch_pdl(kv4_expand_kernel, dim3(max_pages, Hkv, B), dim3(256), 0, s, cache, num_pages,
                     Hkv, table, max_pages, kv_len, start_pos, ko, vo, table_o, len_o, start_o,
                     status));
  return MB_OK;
}
}  // namespace mb

extern "C" size_t mb_kv4_page_bytes(int Hkv) { return Hkv > 0 ? (size_t)Hkv * kv4::BLOB : 0; }

extern "C" int mb_kv4_append_bf16(const uint16_t* k, const uint16_t* v, int64_t k_batch,
                                  int64_t k_token, int64_t k_head, int64_t v_batch, int64_t v_token,
                                  int64_t v_head, uint8_t* cache, int num_pages, int Hkv,
                                  const int* block_table, int max_pages, const int* start_pos,
                                  const int* new_len, int B, int S, void* stream) {
  MB_REQUIRE(B >= 0 && S >= 0 && Hkv > 0 && num_pages >= 0 && max_pages >= 0,
             "kv4 append: bad sizes");
  if (B == 0 || S == 0) return MB_OK;
  MB_REQUIRE(k && v && cache && block_table && start_pos,
             "kv4 append: null pointer");
  MB_REQUIRE(((uintptr_t)k | (uintptr_t)v | (uintptr_t)cache) % 16 == 0,
             "kv4 append: k, v and the cache must be 16-byte aligned");
  MB_REQUIRE((k_batch | k_token | k_head | v_batch | v_token | v_head) % 8 == 0,
             "kv4 append: strides must be multiples of 8 elements");
  uint32_t* status = mb::device_status_ptr();
  MB_REQUIRE(status, "kv4 append: no status word");
  const int64_t total = (int64_t)B * S * Hkv;
  MB_REQUIRE((total + 7) / 8 <= 0x7fffffff, "kv4 append: too many tokens");
  MB_CUDA(mb::launch_pdl(kv4_append_kernel, dim3((unsigned)((total + 7) / 8)), dim3(256), 0,
                         static_cast<cudaStream_t>(stream), k, v, k_batch, k_token, k_head,
                         v_batch, v_token, v_head, cache, num_pages, Hkv, block_table, max_pages, start_pos, new_len, total, S, status));
  return MB_OK;
}

extern "C" int mb_kv4_gather_f32(const uint8_t* cache, int num_pages, int Hkv,
                                 const int* block_table, int max_pages, const int* start_pos,
                                 const int* kv_len, int B, int S, float* k_out, float* v_out,
                                 void* stream) {
  MB_REQUIRE(B >= 0 && S >= 0 && Hkv > 0 && num_pages >= 0 && max_pages >= 0,
             "kv4 gather: bad sizes");
  if (B == 0 || S == 0) return MB_OK;
  MB_REQUIRE(cache && block_table && start_pos && kv_len && k_out && v_out,
             "kv4 gather: null pointer");
  MB_REQUIRE(((uintptr_t)k_out | (uintptr_t)v_out | (uintptr_t)cache) % 16 == 0,
             "kv4 gather: the outputs and the cache must be 16-byte aligned");
  uint32_t* status = mb::device_status_ptr();
  MB_REQUIRE(status, "kv4 gather: no status word");
  const int64_t total = (int64_t)B * S * Hkv;
  MB_REQUIRE((total + 7) / 8 <= 0x7fffffff, "kv4 gather: too many tokens");
  MB_CUDA(mb::launch_pdl(kv4_gather_kernel, dim3((unsigned)((total + 7) / 8)), dim3(256), 0,
                         static_cast<cudaStream_t>(stream), cache, num_pages, Hkv, block_table,
                         max_pages, start_pos, kv_len, total, S, k_out, v_out, status));
  return MB_OK;
}
