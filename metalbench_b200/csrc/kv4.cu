// Storing tokens in the 4-bit paged KV cache and reading them back (layout in
// kv4.cuh). The 4-bit counterpart of the cache write that the decoder layer's
// QKV epilogue does in bf16.
//
// For the 128 dims x of one token and kv head (keys and values alike):
//   m = min x,  s = bf16((max x - m) / 15),  u = clamp(rint((x - m) / s), 0, 15)
// with u = 0 where s = 0; the stored value is m + s u. m is exact (x is bf16);
// s is rounded to bf16 (2^-8 relative: at most 6 % of one code step at u = 15)
// because its 2 bytes a token are read by every later step. Where max x - m is no
// fp32 number (NaN, infinities, a range of 2^128) s is none either, and the token
// reads as NaN; any other range gives finite values: 15 of half a step of s, 2^116 at
// most, are less than what fp32 has above the largest bf16 number (2^120 - 2^104).
#include "kv4.cuh"
#include "kernels.h"

namespace {
using namespace kv4;
static_assert(PAGE == 64, "positions are split by shifts");

// bf16 pairs; a NaN stays one.
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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

// W words (2 W dims) a lane of a row of 128, 64 / W lanes a row: W / 4 words of
// codes, and the row's scale and minimum (the same in all its lanes). A call,
// not inlined: copies in a loop over rows miss the instruction cache.
template <int W>
struct Row {
  uint32_t code[W / 4], par;
};
template <int W>
__device__ __noinline__ Row<W> quantise(uint4 ra, uint4 rb) {
  const uint32_t w[8] = {ra.x, ra.y, ra.z, ra.w, rb.x, rb.y, rb.z, rb.w};
  // minimum and maximum in packed bf16, then both at once as (min, -max)
  uint32_t mn = w[0], mx = w[0], tn = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < W; ++i) {
    mn = min2(mn, w[i]);
    mx = max2(mx, w[i]);
    tn = min2(tn, w[i] & 0x7FFF7FFFu);
  }
  uint32_t both = min2(__byte_perm(mn, mx ^ 0x80008000u, 0x5410), __byte_perm(mn, mx ^ 0x80008000u, 0x7632));
#pragma unroll
  for (int off = 32 / W; off; off >>= 1) both = min2(both, __shfl_xor_sync(0xffffffffu, both, off));
  const float lo = lo_bf(both), hi = -hi_bf(both);
  const float tiny = fminf(lo_bf(tn), hi_bf(tn));
  float x[2 * W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    x[2 * i] = lo_bf(w[i]);
    x[2 * i + 1] = hi_bf(w[i]);
  }
  // Quotients: y (1 / c) corrected once by its exact remainder is within half a
  // last place of y / c, and what is exactly halfway comes out exactly.
  const float range = hi - lo;
  const float q15 = range * (1.f / 15.f);
  const bool plain = range >= 0x1p-100f && range < INFINITY;  // no subnormals on the way
  const __nv_bfloat16 sb = __float2bfloat16_rn(plain ? fmaf(fmaf(-15.f, q15, range), 1.f / 15.f, q15)
                                                     : __fdiv_rn(range, 15.f));
  const float sc = __bfloat162float(sb);
  Row<W> r;
  r.par = (uint32_t)__bfloat16_as_ushort(sb) | (__float_as_uint(lo) & 0xFFFF0000u);
  // A remainder d - s q is exact (s has 8 bits), so with q' next to d / s adding
  // 1.5 * 2^23 rounds to the nearest whole number, ties to the even one: a d that
  // is no tie is off one by more than half a last place of q'. d = x - m is exact
  // too unless x is smaller than 2^-15 of the range (1 row in 60 of normal
  // numbers): there a quotient, off by 15 * 2^-24 at most, may round the wrong
  // way next to a tie, and only then the row goes the long way.
  bool slow = !plain;
  if (plain) {
    const float inv = __frcp_rn(sc);
    if (tiny < range * 0x1p-15f) {
      float far = 0.f;
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) {
        const float d = x[i] - lo, q = d * inv, y = fmaf(fmaf(-sc, q, d), inv, q);
        far = fmaxf(far, fabsf(y - rintf(y)));
      }
      slow = far > 0.5f - 0x1p-16f;
    }
#pragma unroll
    for (int k = 0; k < W / 4; ++k) {
      uint32_t sum = 0;  // of (bits of 1.5 * 2^23 + u) * 16^i: u <= 15, as s is within 2^-8 of range / 15
#pragma unroll
      for (int i = 7; i >= 0; --i) {
        const float d = x[8 * k + i] - lo, q = d * inv;
        sum = sum * 16u + __float_as_uint(fmaf(fmaf(-sc, q, d), inv, q) + 12582912.f);
      }
      r.code[k] = sum - 0x4B400000u * 0x11111111u;
    }
  }
  if (slow) {
    const float half = 0.5f * sc;
#pragma unroll
    for (int k = 0; k < W / 4; ++k) r.code[k] = 0;
    if (sc > 0.f) {
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) {
        const float d = x[i] - lo, b = d - x[i];
        const float lost = (x[i] - (d - b)) + (-lo - b);  // x - m = d + lost, exactly
        float u = fminf(fmaxf(rintf(__fdiv_rn(d, sc)), 0.f), 15.f);
        const float e = fmaf(-sc, u, d);
        const bool odd = (int)u & 1;
        if (e > half || (e == half && (lost > 0.f || (lost == 0.f && odd)))) u += 1.f;
        else if (e < -half || (e == -half && (lost < 0.f || (lost == 0.f && odd)))) u -= 1.f;
        r.code[i >> 3] |= (uint32_t)fminf(fmaxf(u, 0.f), 15.f) << (4 * (i & 7));
      }
    }
  }
  return r;
}

struct AppendArgs {
  const uint16_t *k, *v;
  int64_t kb, ks, kh, vb, vs, vh;  // element strides: batch, token, head
  uint8_t* cache;
  const int *table, *start_pos, *new_len, *kv_len;
  int num_pages, max_pages, Hkv, S;
  uint32_t* status;
};

__device__ __forceinline__ const uint16_t* row_at(const AppendArgs& a, int val, int b, int s, int h) {
  return val ? a.v + b * a.vb + s * a.vs + h * a.vh : a.k + b * a.kb + s * a.ks + h * a.kh;
}
template <int W>
__device__ __forceinline__ void put(uint8_t* blob, int val, int l, int t, const Row<W>& r) {
  uint8_t* at = blob + (val ? v_word(t, W / 4 * l) : t * ROW + l * W);
  if (W == 4) *reinterpret_cast<uint32_t*>(at) = r.code[0];
  else *reinterpret_cast<uint2*>(at) = make_uint2(r.code[0], r.code[W / 4 - 1]);
  if (l == 0) *reinterpret_cast<uint32_t*>(blob + (val ? V_PARAMS : K_PARAMS) + t * 4) = r.par;
}

// Few tokens a sequence (decode): a warp stores one (token, kv head), lanes
// 0-15 the key, lanes 16-31 the value. What bounds it is the chain of loads,
// length -> page -> store (64 tokens of 8 heads: 3.8 us, and 4.9 us with eight
// lanes a row, which stores prompts faster).
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a, int64_t total) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= total) return;
  const int lane = threadIdx.x & 31, val = lane >> 4, l = lane & 15;
  const int64_t tok = item / a.Hkv;
  const int h = (int)(item - tok * a.Hkv), b = (int)(tok / a.S), s = (int)(tok - (int64_t)b * a.S);
  const uint4 x = reinterpret_cast<const uint4*>(row_at(a, val, b, s, h))[l];
  if (a.new_len && s >= a.new_len[b]) return;
  const int64_t pos = (int64_t)a.start_pos[b] + s;
  if (a.kv_len && pos >= a.kv_len[b]) return;
  const int pg = page_of(a.table, a.max_pages, a.num_pages, b, pos, a.status);
  if (pg < 0) return;
  put(a.cache + ((int64_t)pg * a.Hkv + h) * BLOB, val, l, (int)(pos & (PAGE - 1)), quantise<4>(x, x));
}

// Many tokens a sequence (prompts): a CTA stores all heads of 2^lt tokens that
// lie in one page, 64 rows (token, head) at a time, heads first, so that it
// reads whole rows of a projection's output, looks one page up, and has four
// rows a quarter-warp in flight. (A CTA a page and head, 256-byte pieces 6 KB
// apart, took twice as long for 4 x 2048 tokens of 8 heads.)
__global__ void __launch_bounds__(256) kv4_append_tokens_kernel(const AppendArgs a, int lt) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 31, val = (lane >> 3) & 1, l = lane & 7;
  const int64_t start = a.start_pos[b];
  const int n = a.new_len ? min(a.new_len[b], a.S) : a.S;
  const int64_t p0 = ((start >> lt) + blockIdx.x) << lt;  // first position of this CTA
  const int64_t from = max(p0, start), end = a.kv_len ? min(start + n, (int64_t)a.kv_len[b]) : start + n;
  const int64_t to = min(p0 + (1 << lt), end);
  if (from >= to) return;
  const int rows = (int)(to - from) * a.Hkv;
  // a lane's rows are 16 apart: token and head step along without dividing
  const int first = (threadIdx.x >> 5) * 2 + (lane >> 4), ds = 16 / a.Hkv, dh = 16 - ds * a.Hkv;
  const int64_t ss = val ? a.vs : a.ks, sh = val ? a.vh : a.kh;
  const uint16_t* src = row_at(a, val, b, (int)(from - start), 0) + l * 16;
  int s0 = first / a.Hkv, h0 = first - s0 * a.Hkv, pg = -1;
  uint8_t* page = a.cache;
  for (int base = 0; base < rows; base += 64) {
    uint4 x[4], y[4];
    int s = s0, h = h0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = y[i] = make_uint4(0, 0, 0, 0);
      if (base + i * 16 + first < rows) {
        const uint4* p = reinterpret_cast<const uint4*>(src + s * ss + h * sh);
        x[i] = p[0], y[i] = p[1];
      }
      s += ds, h += dh;
      if (h >= a.Hkv) h -= a.Hkv, ++s;
    }
    if (base == 0) {
      pg = page_of(a.table, a.max_pages, a.num_pages, b, p0, a.status);
      if (pg < 0) return;
      page += (int64_t)pg * a.Hkv * BLOB;
    }
    const int t0 = (int)(from & (PAGE - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Row<8> r = quantise<8>(x[i], y[i]);  // all lanes: they shuffle
      if (base + i * 16 + first < rows) put(page + (int64_t)h0 * BLOB, val, l, t0 + s0, r);
      s0 += ds, h0 += dh;
      if (h0 >= a.Hkv) h0 -= a.Hkv, ++s0;
    }
  }
}

// Positions start_pos[b] .. start_pos[b] + S - 1 back as fp32 [B][S][Hkv][128]
// (zeros at and past kv_len[b]); rows, lanes and the two forms as for storing.
struct GatherArgs {
  const uint8_t* cache;
  const int *table, *start_pos, *kv_len;
  float *ko, *vo;
  int num_pages, max_pages, Hkv, S;
  uint32_t* status;
};

// Lane l of a half-warp: dims 4 l .. 4 l + 3 (low half of x) and 64 more, so
// that both 16-byte stores of a row are contiguous over the lanes.
__device__ __forceinline__ uint2 get(const uint8_t* blob, int half, int l, int t) {
  const uint8_t* p = half ? blob + v_word(t, l >> 1) : blob + t * ROW + (l >> 1) * 4;
  const uint8_t* p2 = half ? blob + v_word(t, 8 + (l >> 1)) : p + 32;
  const uint32_t c = *reinterpret_cast<const uint16_t*>(p + (l & 1) * 2), c2 = *reinterpret_cast<const uint16_t*>(p2 + (l & 1) * 2);
  return make_uint2(c | (c2 << 16), *reinterpret_cast<const uint32_t*>(blob + (half ? V_PARAMS : K_PARAMS) + t * 4));
}
__device__ __forceinline__ void write_row(float* row, int l, uint2 x) {
  float o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)  // one rounding: scale * code is exact (8 + 4 bits)
    o[j] = fmaf(lo_bf(x.y), (float)((x.x >> (4 * j)) & 15u), hi_bf(x.y));
  __stcs(reinterpret_cast<float4*>(row) + l, make_float4(o[0], o[1], o[2], o[3]));
  __stcs(reinterpret_cast<float4*>(row) + 16 + l, make_float4(o[4], o[5], o[6], o[7]));
}

__global__ void __launch_bounds__(256) kv4_gather_kernel(const GatherArgs a, int64_t total) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= total) return;
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const int64_t tok = item / a.Hkv;
  const int h = (int)(item - tok * a.Hkv), b = (int)(tok / a.S), s = (int)(tok - (int64_t)b * a.S);
  const int64_t pos = (int64_t)a.start_pos[b] + s;
  uint2 x = make_uint2(0, 0);  // reads as zeros
  if (pos < a.kv_len[b]) {
    const int pg = page_of(a.table, a.max_pages, a.num_pages, b, pos, a.status);
    if (pg >= 0) x = get(a.cache + ((int64_t)pg * a.Hkv + h) * BLOB, half, l, (int)(pos & (PAGE - 1)));
  }
  write_row((half ? a.vo : a.ko) + item * DH, l, x);
}

__global__ void __launch_bounds__(256) kv4_gather_tokens_kernel(const GatherArgs a, int lt) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15;
  const int64_t start = a.start_pos[b], end = a.kv_len[b];
  const int64_t p0 = ((start >> lt) + blockIdx.x) << lt;
  const int64_t from = max(p0, start), to = min(p0 + (1 << lt), start + a.S);
  if (from >= to) return;
  int pg = -1;
  if (from < end) pg = page_of(a.table, a.max_pages, a.num_pages, b, p0, a.status);
  const int rows = (int)(to - from) * a.Hkv;
  const int there = pg < 0 ? 0 : (int)(min(to, end) - from) * a.Hkv;  // the rest reads as zeros
  const int64_t out = (((int64_t)b * a.S + (from - start)) * a.Hkv) * DH;
  for (int base = 0; base < rows; base += 64) {
    uint2 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = base + i * 8 + (threadIdx.x >> 5), s = r / a.Hkv;
      x[i] = make_uint2(0, 0);
      if (r < there)
        x[i] = get(a.cache + ((int64_t)pg * a.Hkv + (r - s * a.Hkv)) * BLOB, half, l, (int)((from + s) & (PAGE - 1)));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = base + i * 8 + (threadIdx.x >> 5);
      if (r < rows) write_row((half ? a.vo : a.ko) + out + (int64_t)r * DH, l, x[i]);
    }
  }
}

// Tokens a CTA takes in the form for many: 64 rows, a power of two within a
// page; -1: few tokens a sequence, a warp each.
int log_tokens(int S, int Hkv) {
  int lt = 6;
  while (lt > 0 && (Hkv << lt) > 64) --lt;
  return S >= 32 && S >= (1 << lt) ? lt : -1;
}

__device__ __forceinline__ float max_of_16(float x) {  // over the 16 lanes of a half warp
#pragma unroll
  for (int d = 8; d; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
  return x;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The pages of B sequences in fp16 for the tcgen05 kernel (attention_kv4_tc.cu):
// one CTA a page and kv head, lanes as in the storing kernel. Tiles are two
// pages: what a sequence's last tile lacks is written as zeros.
__global__ void __launch_bounds__(256) kv4_expand_kernel(
    const uint8_t* __restrict__ cache, int num_pages, int Hkv, const int* __restrict__ table,
    int max_pages, int max_len, const int* __restrict__ kv_len, mb::Kv4Expanded o, uint32_t* status) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int page = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int L = max(0, min(kv_len[b], max_len));
  if (page / 2 * 2 * PAGE >= L) return;
  const int lane = threadIdx.x & 31, half = lane >> 4, l = lane & 15, warp = threadIdx.x >> 5;
  const int64_t to = ((int64_t)b * Hkv + h) * o.pages + page;
  const int pg = page * PAGE < L ? page_of(table, max_pages, num_pages, b, (int64_t)page * PAGE, status) : -1;
  const uint8_t* blob = cache + ((int64_t)max(pg, 0) * Hkv + h) * BLOB;
  uint16_t* dst = (half ? o.v : o.k) + to * (PAGE * DH) + l * 8;
  const int there = pg >= 0 ? min(PAGE, L - page * PAGE) : 0;  // the rest may be anything: it is taken as zeros
  __shared__ uint32_t pars[2][PAGE];  // keys', values'
  uint32_t code[PAGE / 8];            // (all loads on their way before the first is used)
#pragma unroll
  for (int i = 0; i < PAGE / 8; ++i) {
    const int t = i * 8 + warp;
    code[i] = t < there ? *reinterpret_cast<const uint32_t*>(blob + (half ? v_word(t, l) : t * ROW + l * 4)) : 0;
  }
  if (threadIdx.x < 2 * PAGE) {
    const int t = threadIdx.x % PAGE;
    pars[threadIdx.x / PAGE][t] = t < there ? *reinterpret_cast<const uint32_t*>(blob + K_PARAMS + threadIdx.x * 4) : 0;
  }
  static_assert(V_PARAMS == K_PARAMS + PAGE * 4, "the values' parameters follow the keys'");
  __syncthreads();
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < PAGE / 16; ++i) {
    const uint32_t par = pars[half][i * 16 + l];
    if (lo_bf(par) < INFINITY) most = fmaxf(most, fmaxf(fabsf(hi_bf(par)), fabsf(fmaf(lo_bf(par), 15.f, hi_bf(par)))));
  }
  // values that are all zero must not raise the rows' references above what other
  // pages need (any factor is right for them: a low one, far enough from fp32's end
  // that the terms' sum, which takes 2^60 in return, stays finite)
  constexpr int ZERO_VALUES = -60;
  most = max_of_16(most);
  const int e = half && most == 0.f ? ZERO_VALUES : fp16_exp(most);
  const float f = pow2i(-e);
  if (warp == 0 && l == 0) {
    int2* to_e = o.page_exp + to;
    (half ? to_e->y : to_e->x) = e;
  }
#pragma unroll
  for (int i = 0; i < PAGE / 8; ++i) {
    const int t = i * 8 + warp;
    const uint32_t kpar = pars[0][t], vpar = pars[1][t], par = half ? vpar : kpar;
    // stored of what was no number or infinite: the key's scores make the rows that see it
    // NaN, and its value is 0, since a weight of 0 times NaN would spread to all rows
    const bool good = lo_bf(kpar) < INFINITY && lo_bf(vpar) < INFINITY;
    const float scale = good ? lo_bf(par) * f : 0.f, least = good ? hi_bf(par) * f : half ? 0.f : NAN;
    // code n of a half word stands at bit 4 n: 2^23 + u 16^n - 2^23 is u 16^n (a conversion
    // of every code to a float would be bound by its unit)
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t c = code[i] >> (16 * j);
      float x[4];
#pragma unroll
      for (int n = 0; n < 4; ++n)
        x[n] = fmaf(__uint_as_float((c & (15u << (4 * n))) | 0x4B000000u) - 8388608.f, scale * (1.f / (1 << (4 * n))), least);
      w[2 * j] = half2_of(x[0], x[1]);
      w[2 * j + 1] = half2_of(x[2], x[3]);
    }
    *reinterpret_cast<uint4*>(dst + t * DH) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace

namespace mb {
int kv4_expand(const uint8_t* cache, int num_pages, int Hkv, const int* table, int max_pages,
               int max_len, const int* kv_len, int B, const Kv4Expanded& o, uint32_t* status, cudaStream_t s) {
  MB_CUDA(launch_pdl(kv4_expand_kernel, dim3(o.pages, Hkv, B), dim3(256), 0, s, cache, num_pages, Hkv, table,
                     max_pages, max_len, kv_len, o, status));
  return MB_OK;
}
}  // namespace mb

extern "C" size_t mb_kv4_page_bytes(int Hkv) { return Hkv > 0 ? (size_t)Hkv * kv4::BLOB : 0; }

extern "C" int mb_kv4_append_bf16(const uint16_t* k, const uint16_t* v, int64_t k_batch,
                                  int64_t k_token, int64_t k_head, int64_t v_batch, int64_t v_token,
                                  int64_t v_head, uint8_t* cache, int num_pages, int Hkv,
                                  const int* block_table, int max_pages, const int* start_pos,
                                  const int* new_len, const int* kv_len, int B, int S, void* stream) {
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
  const AppendArgs a = {k,     v,           k_batch,   k_token, k_head,    v_batch,   v_token, v_head, cache,
                        block_table, start_pos, new_len, kv_len, num_pages, max_pages, Hkv,     S,      status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int lt = log_tokens(S, Hkv);
  if (lt >= 0 && B <= 65535) {
    MB_CUDA(mb::launch_pdl(kv4_append_tokens_kernel, dim3((S >> lt) + 2, B), dim3(256), 0, s, a, lt));
    return MB_OK;
  }
  const int64_t total = (int64_t)B * S * Hkv;
  MB_REQUIRE((total + 7) / 8 <= 0x7fffffff, "kv4 append: too many tokens");
  MB_CUDA(mb::launch_pdl(kv4_append_kernel, dim3((unsigned)((total + 7) / 8)), dim3(256), 0, s, a, total));
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
  const GatherArgs a = {cache, block_table, start_pos, kv_len, k_out, v_out, num_pages, max_pages, Hkv, S, status};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int lt = log_tokens(S, Hkv);
  if (lt >= 0 && B <= 65535) {
    MB_CUDA(mb::launch_pdl(kv4_gather_tokens_kernel, dim3((S >> lt) + 2, B), dim3(256), 0, s, a, lt));
    return MB_OK;
  }
  const int64_t total = (int64_t)B * S * Hkv;
  MB_REQUIRE((total + 7) / 8 <= 0x7fffffff, "kv4 gather: too many tokens");
  MB_CUDA(mb::launch_pdl(kv4_gather_kernel, dim3((unsigned)((total + 7) / 8)), dim3(256), 0, s, a, total));
  return MB_OK;
}
