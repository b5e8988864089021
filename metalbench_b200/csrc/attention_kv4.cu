// GQA attention over the 4-bit paged KV cache (layout in kv4.cuh); the 4-bit
// counterpart of mb_attention_decode_bf16 (reference semantics:
// mlx/kernels/full/llama_decoder_layer.py:30-37).
//
// Mathematics. Key j of a page stands for mk_j + sk_j * u_j (u_j its 128 whole
// codes), value j for mv_j + sv_j * w_j. So
//   score_j = c * (sk_j * (q . u_j) + mk_j * sum(q)),      c = log2(e) * scale
//   out     = (sum_j p_j sv_j w_j + sum_j p_j mv_j) / sum_j p_j,  p_j = 2^score_j
// and the tensor cores multiply the codes themselves: a code's four bits, left
// where they stand in the low bits of a 16-bit half, ARE the fp16 number
// u * 2^-24 (u * 2^-20 for the odd code of a byte), a subnormal that mma.sync
// multiplies exactly. Eight codes become four operand registers in five
// logic operations; the powers of two are taken out of q (2^-4) and of the
// sums. Each row of q is scaled by its own power of two into fp16's range, which
// loses nothing of a bf16 number down to 2^-20 of the row's largest (one power
// for a tile would let a padding row that holds anything take the others' bits).
// The value scale goes into the exponent: P_j = 2^(score_j + log2(sv_j) - R)
// with a running reference R per query row, so that P_j sv-weighted is what is
// cut to fp16 (11 bits, and 2^-24 absolute at a range up to 2^15), and the
// denominator is sum_j P_j / sv_j in fp32, of the same P_j. R only moves when a weight would
// pass 2^15, so most pages rescale nothing.
//
// Orientation: keys are the 16 MMA rows, query rows the 8 columns (S^T = K
// Q^T, O^T = V^T P^T), so a decode step's 8 query heads of a kv head fill a
// column tile and no row is wasted; P^T moves from the accumulator layout to
// the operand layout by movmatrix. Query rows are the S * G pairs (position,
// head of the group); NT column tiles of 8 per pass over the cache.
//
// Schedule: one CTA an SM. The flat list of (sequence, kv head, row tile, page)
// is cut into equal shares, one a warp, planned on the device from kv_len, so
// that ragged batches balance; every (sequence, kv head, row tile), a unit,
// counts UNIT_COST pages more than it has, for its start and end. Each warp
// streams its share through its own ring of whole-page bulk copies (8704
// bytes, one mbarrier each) without waiting for another. A unit that lies
// within a share is written at once. At the end the warps that stopped in the
// same unit join their states in shared memory; what is then still in parts
// (at most two a warp) goes to the workspace, and attn_kv4_combine_kernel,
// which plans for itself while the last warps stream, joins it.
#include <cuda_fp16.h>

#include <cmath>

#include "kv4.cuh"
#include "kernels.h"

namespace {
using namespace kv4;

// Warps of a CTA and pages in a warp's ring, for NT column tiles of 8 rows: as
// many warps as the registers of an SM hold (168 and 255 a thread; two column tiles
// use all 255, of which the compiler spills 24 bytes), and as many pages in flight
// as its shared memory does.
template <int NT> struct Shape;
template <> struct Shape<1> { static constexpr int NW = 12, ST = 2; };
template <> struct Shape<2> { static constexpr int NW = 8, ST = 3; };
constexpr int MAX_B = 512;  // most sequences a launch: their page counts are planned in shared memory
constexpr int UNIT_COST = 2;  // pages that starting and ending a unit cost

struct Args {
  const uint16_t* q;
  const uint8_t* cache;
  const int* table;
  const int* kv_len;
  const int* start_pos;  // null: every key below kv_len is seen
  uint16_t* out;
  float* part_o;   // [warps][2][cols][DH]: unit began before this share, in it
  float* part_ml;  // [warps][2][cols][2]
  uint32_t* status;
  int64_t ldq, ldo;  // elements between two positions' rows
  int num_pages, max_pages, max_len, B, S, Hkv, G, RT;
  int warps;  // shares
  int active; // warps of a CTA that have one
  float scale_log2;
};

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// The codes of one 32-bit word as four fp16 pairs: codes 0|4, 1|5 (x16), 2|6, 3|7 (x16).
__device__ __forceinline__ void spread(uint32_t w, uint32_t (&e)[4]) {
  e[0] = w & 0x000F000Fu;
  e[1] = w & 0x00F000F0u;
  w >>= 8;
  e[2] = w & 0x000F000Fu;
  e[3] = w & 0x00F000F0u;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A weight cut to fp16's 11 bits before it goes into any sum: the terms of codes and
// minimum cancel in the output, and with the codes' weight alone rounded its error
// counts as often as the code is larger than the value (64 x 8193: error of the result
// 0.00179 then, 0.00172 so, of 0.00166 that the output's own rounding makes; no time).
// Cutting takes one operation, rounding two. Half a step, the mean of what is cut off,
// is a factor of every weight alike and drops out of the quotient; from there an error
// is at most half a step.
__device__ __forceinline__ float cut_to_h(float p) { return __uint_as_float(__float_as_uint(p) & 0xFFFFE000u); }

// unit / RT and row / G; one row tile and one position are the decode step's
__device__ __forceinline__ int head_of(const Args& a, int unit) { return a.RT == 1 ? unit : unit / a.RT; }
__device__ __forceinline__ int pos_of(const Args& a, int r) { return a.S == 1 ? 0 : r / a.G; }
__device__ __forceinline__ float fast_log2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Attended keys of sequence b (from L2: the combine kernel plans before it has
// waited for the main one).
__device__ __forceinline__ int seq_len(const Args& a, int b) {
  return max(0, min(__ldcg(a.kv_len + b), a.max_len));
}

// Flat page list of the batch, in shared memory.
struct Plan {
  int2 wsum[12];
  int pre[MAX_B + 1];   // index of the first page of sequence b; [B]: how many there are
  int vpre[MAX_B + 1];  // the same with UNIT_COST more pages a unit
};

template <int NW>
__device__ __forceinline__ void make_plan(const Args& a, Plan& p) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int MOST = (MAX_B + NW * 32 - 1) / (NW * 32);
  const int per = (a.B + NW * 32 - 1) / (NW * 32), b0 = min(a.B, tid * per);
  const int units = a.Hkv * a.RT;
  int pages[MOST];
  int2 sum = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    pages[i] = i < per && b0 + i < a.B ? (seq_len(a, b0 + i) + PAGE - 1) / PAGE : 0;
    sum.x += pages[i] * units;
    sum.y += pages[i] ? (pages[i] + UNIT_COST) * units : 0;
  }
  int2 inc = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc.x, off), y = __shfl_up_sync(0xffffffffu, inc.y, off);
    if (lane >= off) inc.x += x, inc.y += y;
  }
  if (lane == 31) p.wsum[warp] = inc;
  __syncthreads();
  int2 run = make_int2(inc.x - sum.x, inc.y - sum.y);
#pragma unroll
  for (int w = 0; w < NW; ++w)
    if (w < warp) run.x += p.wsum[w].x, run.y += p.wsum[w].y;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    if (i < per && b0 + i < a.B) {
      p.pre[b0 + i] = run.x;
      p.vpre[b0 + i] = run.y;
    }
    run.x += pages[i] * units;
    run.y += pages[i] ? (pages[i] + UNIT_COST) * units : 0;
  }
  if (tid == NW * 32 - 1) {
    p.pre[a.B] = run.x;  // the last thread's end is everybody's
    p.vpre[a.B] = run.y;
  }
  __syncthreads();
}

// The last i < n with list[i] <= v (list ascends, list[0] <= v): a warp together.
__device__ __forceinline__ int find_warp(const int* list, int n, int v) {
  int c = 0;
  for (int i = threadIdx.x & 31; i - (int)(threadIdx.x & 31) < n; i += 32)
    c += __popc(__ballot_sync(0xffffffffu, i < n && list[i] <= v));
  return c - 1;
}

// Pages whose place in the costed list lies before v.
__device__ __forceinline__ int pages_before(const Plan& p, int B, int units, int64_t v64) {
  if (v64 >= p.vpre[B]) return p.pre[B];
  const int v = (int)v64, b = find_warp(p.vpre, B, v);
  const int pages = (p.pre[b + 1] - p.pre[b]) / units;
  const int rem = v - p.vpre[b], unit = rem / (pages + UNIT_COST);
  return p.pre[b] + unit * pages + max(0, rem - unit * (pages + UNIT_COST) - UNIT_COST);
}

// Sequence of flat page f: pre[b] <= f < pre[b + 1].
__device__ __forceinline__ int find_seq(const int* pre, int B, int f) {
  int lo = 0, hi = B;  // pre[lo] <= f < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= f) lo = mid; else hi = mid;
  }
  return lo;
}

// A key's numbers as the scores use them, worked out once a page by the lane
// that owns the key and read by the four lanes that need it.
struct __align__(16) KeyParams {
  float sk, mk;  // key scale and minimum
  float lg, rv;  // log2 and reciprocal of the value scale
};

// Floats of a warp's state of one column tile, while warps join: 4 pieces of
// 8 x 32 accumulators, each one bank further, and R, l, om of the 8 columns.
constexpr int STATE = 1028 + 32;

// A warp's running state over the pages of one unit: NT column tiles of 8.
template <int NT>
struct State {
  float o[NT][4][2][4];  // [32-dim piece][dim pair][accumulator]
  float R[NT][2], l[NT][2], om[NT][2];
  uint32_t qf[NT][16];   // q as B fragments
  float qs[NT][2];       // sum of q's dims, scaled as the products are
  float qc[NT][2];       // what takes these to scores in log2 units
  int lim[NT][2];        // keys below lim are seen by column 2 tig + e

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][c][h][e] = 0.f;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        R[t][e] = -INFINITY;
        l[t][e] = om[t][e] = 0.f;
      }
    }
  }

  // q of row tile rt as B fragments, each row scaled by a power of two. L keys in
  // all, row s sees those at positions <= first + s.
  __device__ __forceinline__ void load_q(const Args& a, int b, int kvh, int rt, int L, int first) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
    float x[NT][32];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = rt * (NT * 8) + t * 8 + gid;
      const int s = pos_of(a, r);
      if (r < a.S * a.G) {
        const uint4* p = reinterpret_cast<const uint4*>(
            a.q + ((int64_t)b * a.S + s) * a.ldq + (kvh * a.G + (r - s * a.G)) * DH + 32 * tig);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w = p[i];
          x[t][8 * i] = lo_bf(w.x), x[t][8 * i + 1] = hi_bf(w.x), x[t][8 * i + 2] = lo_bf(w.y);
          x[t][8 * i + 3] = hi_bf(w.y), x[t][8 * i + 4] = lo_bf(w.z), x[t][8 * i + 5] = hi_bf(w.z);
          x[t][8 * i + 6] = lo_bf(w.w), x[t][8 * i + 7] = hi_bf(w.w);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) x[t][i] = 0.f;
      }
      float sum = 0.f, big = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        big = fmaxf(big, fabsf(x[t][i]));
        sum += x[t][i];
      }
#pragma unroll
      for (int off = 1; off <= 2; off <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, off);
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
      }
      // 2^e brings the row's largest to [2^11, 2^12)
      const int e = max(-100, min(100, 11 - ((int)(__float_as_uint(big) >> 23) - 127)));
      const float up = __uint_as_float((uint32_t)(127 + e) << 23), up16 = up * 0.0625f;
      const float back = a.scale_log2 * __uint_as_float((uint32_t)(127 + 24 - e) << 23);
      sum *= up * 0x1p-24f;
      const int mylim = min(L, first + s + 1);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = (2 * tig + c) * 4;  // a lane whose fragment row is column 2 tig + c
        qs[t][c] = __shfl_sync(0xffffffffu, sum, from);
        qc[t][c] = __shfl_sync(0xffffffffu, back, from);
        lim[t][c] = __shfl_sync(0xffffffffu, mylim, from);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        qf[t][4 * w] = pack_h2(x[t][8 * w] * up, x[t][8 * w + 4] * up);
        qf[t][4 * w + 1] = pack_h2(x[t][8 * w + 1] * up16, x[t][8 * w + 5] * up16);
        qf[t][4 * w + 2] = pack_h2(x[t][8 * w + 2] * up, x[t][8 * w + 6] * up);
        qf[t][4 * w + 3] = pack_h2(x[t][8 * w + 3] * up16, x[t][8 * w + 7] * up16);
      }
    }
  }

  // l and om are sums over a lane's keys until here.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
          l[t][c] += __shfl_xor_sync(0xffffffffu, l[t][c], off);
          om[t][c] += __shfl_xor_sync(0xffffffffu, om[t][c], off);
        }
  }

  // The state in shared memory (STATE floats a column tile), for warps to join.
  __device__ __forceinline__ void deposit(float* at) const {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float* to = at + t * STATE + lane;
#pragma unroll
      for (int i = 0; i < 32; ++i)  // a piece's 8 numbers a lane; pieces one bank apart for the readers
        to[i * 32 + (i >> 3)] = o[t][i >> 3][(i >> 2) & 1][i & 3] * ((i & 2) ? 0x1p20f : 0x1p24f);
      if (gid == 0) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<float4*>(at + t * STATE + 1028 + (2 * tig + c) * 4) =
              make_float4(R[t][c], l[t][c], om[t][c], 0.f);
      }
    }
  }

  // One page (pg, in shared memory) of keys key0 .. key0 + 63. MASKED: some of
  // them stand past the end (len) or are not seen by every column.
  template <bool MASKED>
  __device__ __forceinline__ void page(const uint8_t* pg, KeyParams* kp, float* vmin, int key0, int len) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = lane + 32 * i;
      uint32_t k = *reinterpret_cast<const uint32_t*>(pg + K_PARAMS + key * 4);
      uint32_t v = *reinterpret_cast<const uint32_t*>(pg + V_PARAMS + key * 4);
      if (MASKED && key0 + key >= len) k = v = 0;  // what stands past the end may be anything
      // A value scale of 0 (all dims alike, codes 0) must not enter the logarithm. Any
      // other number gives the right sums, but one far above the true scales beside it
      // would raise the reference and take the fp16 weights' bits: the minimum's own
      // size, for zeros 2^-60 (their terms are still fp32 numbers beside scales of 2^60).
      // (Scales below 2^-90 count as that: sums of 2^15 / s over 2^22 keys stay finite.)
      const float sv = lo_bf(v), flat = fmaxf(fabsf(hi_bf(v)) * 0.125f, 0x1p-60f);
      const float s = fminf(fmaxf(sv == 0.f ? flat : sv, 0x1p-90f), 0x1p126f);
      const float r = fast_rcp(s);
      // a key or value stored of what was no number or infinite has such a scale: it makes
      // the rows that see it NaN, by its score (a term of 0 * NaN would spread to all rows)
      const bool good = lo_bf(k) < INFINITY && sv < INFINITY;
      kp[key] = KeyParams{lo_bf(k), hi_bf(k), good ? fast_log2(s) : NAN, r};
      vmin[key] = good ? hi_bf(v) * r : 0.f;
    }
    __syncwarp();

    // ---- scores: log2 of the softmax terms times their value scales ----
    float sc[NT][4][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][mt][e] = 0.f;
    // KI key tiles side by side: their accumulators are independent, which
    // hides the latency of the eight products that follow one another in each
    constexpr int KI = 2;
#pragma unroll
    for (int m0 = 0; m0 < 4; m0 += KI) {
      uint32_t wd[KI][2][4];
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint4 k = *reinterpret_cast<const uint4*>(pg + ((m0 + i) * 16 + gid + 8 * r) * ROW + tig * 16);
          wd[i][r][0] = k.x, wd[i][r][1] = k.y, wd[i][r][2] = k.z, wd[i][r][3] = k.w;
        }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t ea[KI][4], eb[KI][4];
#pragma unroll
        for (int i = 0; i < KI; ++i) {
          spread(wd[i][0][w], ea[i]);
          spread(wd[i][1][w], eb[i]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < KI; ++i)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              mma_f16_16816(sc[t][m0 + i], ea[i][2 * h], eb[i][2 * h], ea[i][2 * h + 1], eb[i][2 * h + 1],
                            qf[t][4 * w + 2 * h], qf[t][4 * w + 2 * h + 1]);
      }
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = mt * 16 + gid + 8 * r;
        const KeyParams p = kp[key];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaf(qc[t][c], fmaf(p.mk, qs[t][c], p.sk * sc[t][mt][2 * r + c]), p.lg);
            if (MASKED && key0 + key >= lim[t][c]) x = -INFINITY;
            sc[t][mt][2 * r + c] = x;
          }
      }
    }

    // ---- reference ----
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float mx[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mx[c] = sc[t][0][c];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) mx[c] = fmaxf(mx[c], fmaxf(sc[t][mt][c], sc[t][mt][2 + c]));
      }
      // a lane whose own maximum passes the reference calls for all to raise it
      const bool raise = mx[0] > R[t][0] + 15.f || mx[1] > R[t][1] + 15.f;
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1)
            mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], off));
          const float Rn = mx[c] > R[t][c] + 15.f ? mx[c] - 8.f : R[t][c];
          const float f = R[t][c] == Rn ? 1.f : fast_exp2(R[t][c] - Rn);
          R[t][c] = Rn;
          l[t][c] *= f;
          om[t][c] *= f;
#pragma unroll
          for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              o[t][p][h][c] *= f;
              o[t][p][h][2 + c] *= f;
            }
        }
      }
    }

    // ---- weights, 16 keys at a time ----
    uint32_t pf[NT][4][2];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = mt * 16 + gid + 8 * r;
        const float rv = kp[key].rv, mv = vmin[key];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float p[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            // R is -inf while a column has seen nothing
            p[c] = cut_to_h(fast_exp2(sc[t][mt][2 * r + c] - (MASKED && R[t][c] == -INFINITY ? 0.f : R[t][c])));
            l[t][c] = fmaf(p[c], rv, l[t][c]);
            om[t][c] = fmaf(p[c], mv, om[t][c]);
          }
          pf[t][mt][r] = transpose8x8(pack_h2(p[0], p[1]));
        }
      }
    }

    // ---- O^T += V^T P^T ----
    // A page's products start from 0 and are added to the running sum with rounding:
    // the matrix unit cuts off what lies below its accumulator's last bits, and for one
    // that holds a long share's sum of codes, all of one sign, that is a bias which
    // grows with the share (30 x 131075 keys, 16 heads of 1: error of the result
    // 0.0028, here 0.0018, of 0.0016 that the output's own rounding makes; 64 x 8193
    // 118.7 -> 121.1 us).
    const uint32_t pg_s = mbd::smem_u32(pg);
#pragma unroll
    for (int p = 0; p < 4; p += 2) {
      float acc[NT][2][2][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i >> 3][(i >> 2) & 1][i & 3] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        const int key = mt * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
        const uint32_t rowp = pg_s + V_CODES + key * ROW;
        const int sw = (key >> 1) & 3;
        uint32_t v[4];  // octets 0, 1 of piece p, then of piece p + 1
        ldsm_x4_t(v, rowp + (((p + (lane >> 4)) ^ sw) << 4));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t e0[4], e1[4];
          spread(v[2 * j], e0);
          spread(v[2 * j + 1], e1);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16_16816(acc[t][j][0], e0[0], e0[1], e1[0], e1[1], pf[t][mt][0], pf[t][mt][1]);
            mma_f16_16816(acc[t][j][1], e0[2], e0[3], e1[2], e1[3], pf[t][mt][0], pf[t][mt][1]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][p + (i >> 3)][(i >> 2) & 1][i & 3] += acc[t][i >> 3][(i >> 2) & 1][i & 3];
    }
  }
};

// One column (query row) of the states that warps deposited STEP floats apart,
// `who` of them: reference, denominator, and four dims a lane. Every lane reads
// every state's numbers: that is shorter than reducing over lanes.
struct Joined {
  float R, l;
  float4 o;
};
template <int STEP, int MOST>
__device__ __forceinline__ Joined join_row(const float* states, int col, uint32_t who) {
  const int lane = threadIdx.x & 31;
  const float* ml = states + (col >> 3) * STATE + 1028 + (col & 7) * 4;
  const float* zp = states + (col >> 3) * STATE + (lane >> 3) * (8 * 32 + 1) + (lane & 7) * 4 + ((col & 7) >> 1) + (col & 1) * 32;
  // without branches, so that the loads of all states are in flight at once;
  // what stands in the place of a state that is not there is read and dropped
  float4 m[MOST];
  Joined j;
  j.R = -INFINITY;
#pragma unroll
  for (int w = 0; w < MOST; ++w) {
    m[w] = *reinterpret_cast<const float4*>(ml + w * STEP);
    if (!((who >> w) & 1)) m[w].x = -INFINITY;
    j.R = fmaxf(j.R, m[w].x);
  }
  j.l = 0.f;
  j.o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < MOST; ++w) {
    const float* z = zp + w * STEP;
    float4 v = make_float4(z[0] + m[w].z, z[64] + m[w].z, z[128] + m[w].z, z[192] + m[w].z);
    const bool in = (who >> w) & 1;
    const float f = m[w].x == -INFINITY ? 0.f : fast_exp2(m[w].x - j.R);
    j.l = in ? fmaf(m[w].y, f, j.l) : j.l;
    j.o.x = in ? fmaf(v.x, f, j.o.x) : j.o.x;
    j.o.y = in ? fmaf(v.y, f, j.o.y) : j.o.y;
    j.o.z = in ? fmaf(v.z, f, j.o.z) : j.o.z;
    j.o.w = in ? fmaf(v.w, f, j.o.w) : j.o.w;
  }
  return j;
}

// Where a row goes: finished to dst, or as a partial to o and ml, or (all null)
// nowhere.
struct To {
  uint16_t* dst;
  float *o, *ml;
};
__device__ __forceinline__ To row_to(const Args& a, int b, int kvh, int r, int slot, int col, int cols, bool whole) {
  To t = {nullptr, nullptr, nullptr};
  const int s = pos_of(a, r);
  if (whole) t.dst = a.out + ((int64_t)b * a.S + s) * a.ldo + (kvh * a.G + (r - s * a.G)) * DH;
  else t.o = a.part_o + ((int64_t)slot * cols + col) * DH, t.ml = a.part_ml + ((int64_t)slot * cols + col) * 2;
  return t;
}
__device__ __forceinline__ void store_row(To t, float R, float l, float4 o) {
  const int lane = threadIdx.x & 31;
  if (t.o) {
    *reinterpret_cast<float4*>(t.o + lane * 4) = o;
    if (lane == 0) *reinterpret_cast<float2*>(t.ml) = make_float2(R, l);
  }
  if (t.dst) {
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // 0: the row has seen no key
    const __nv_bfloat162 h0 = __floats2bfloat162_rn(o.x * inv, o.y * inv);
    const __nv_bfloat162 h1 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(t.dst + lane * 4) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
  }
}
// Not inlined: it runs once, at the end of a CTA's life, when every instruction
// of it would have to be fetched; a call without rows at the start, while the
// first pages are on their way, has it in the instruction cache by then.
template <int STEP, int MOST>
__device__ __noinline__ void join_store(const float* states, int col, uint32_t who, To t) {
  const Joined j = join_row<STEP, MOST>(states, col, who);
  store_row(t, j.R, j.l, j.o);
}

template <int NT>
struct Shared {
  static constexpr int NW = Shape<NT>::NW, ST = Shape<NT>::ST;
  static_assert(NT * STATE * 4 <= ST * BLOB && NW <= 16, "a warp's state takes the place of its pages");
  uint8_t ring[NW][ST][BLOB];
  KeyParams kp[NW][PAGE];
  float vmin[NW][PAGE];
  int4 seg[NW];       // last unit's first page, sequence, number, and whether it starts and ends here
  uint64_t bar[NW][ST];
  int page_ok[NW][ST];
  Plan plan;
};

template <int NT>
__global__ void __launch_bounds__(Shape<NT>::NW * 32) attn_kv4_kernel(const Args a) {
  constexpr int COLS = NT * 8, NW = Shape<NT>::NW, ST = Shape<NT>::ST;
  extern __shared__ __align__(128) uint8_t sm_raw[];
  Shared<NT>& sm = *reinterpret_cast<Shared<NT>*>(sm_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  uint8_t* ring = sm.ring[warp][0];
  uint64_t* bar = sm.bar[warp];
  int* ok_flag = sm.page_ok[warp];
  const int *pre = sm.plan.pre, *vpre = sm.plan.vpre;
  if (lane == 0)
    for (int i = 0; i < ST; ++i) mbd::mbar_init(bar + i, 1);
  mbd::fence_mbar_init();
  mbd::pdl_wait();
  mbd::pdl_trigger();  // after the wait: what the combine kernel plans from is complete
  make_plan<NW>(a, sm.plan);

  // sequences without keys: their rows are zeros
  const int row_elems = a.Hkv * a.G * DH;
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (pre[b] == pre[b + 1])
      for (int s = 0; s < a.S; ++s)
        for (int i = threadIdx.x * 8; i < row_elems; i += NW * 32 * 8)
          *reinterpret_cast<uint4*>(a.out + ((int64_t)b * a.S + s) * a.ldo + i) = make_uint4(0, 0, 0, 0);

  const int units = a.Hkv * a.RT;
  const int per = (vpre[a.B] + a.warps - 1) / a.warps;
  const int me = blockIdx.x * a.active + warp;  // share of this warp
  int begin = 0, end = 0;
  if (warp < a.active) {
    begin = pages_before(sm.plan, a.B, units, (int64_t)me * per);
    end = pages_before(sm.plan, a.B, units, (int64_t)(me + 1) * per);
  }
  const int mine = end - begin;

  // ---- this warp's loads, page after page ----
  int issued = 0;
  int win_pid = 0, win_ok = 0, win_kvh = 0;  // lane i: page (issued / 32) * 32 + i of this share
  auto issue = [&]() {
    if ((issued & 31) == 0) {
      const int f = begin + issued + lane;
      if (f < end) {
        const int b = find_seq(pre, a.B, f);
        const int rem = f - pre[b], pages = (pre[b + 1] - pre[b]) / units;
        const int unit = rem / pages;
        win_kvh = head_of(a, unit);
        const int pid = a.table[(int64_t)b * a.max_pages + (rem - unit * pages)];
        win_ok = pid >= 0 && pid < a.num_pages;
        win_pid = win_ok ? pid : 0;
        if (!win_ok) atomicOr(a.status, MB_DEV_BAD_PAGE);
      }
    }
    const int src = issued & 31;
    const int pid = __shfl_sync(0xffffffffu, win_pid, src);
    const int kvh = __shfl_sync(0xffffffffu, win_kvh, src);
    const int good = __shfl_sync(0xffffffffu, win_ok, src);
    const int st = issued % ST;
    if (lane == 0) {
      ok_flag[st] = good;
      mbd::mbar_expect_tx(bar + st, BLOB);
      mbd::bulk_load(ring + st * BLOB, a.cache + ((int64_t)pid * a.Hkv + kvh) * BLOB, BLOB, bar + st);
    }
    ++issued;
  };
  for (int i = 0; i < ST && i < mine; ++i) issue();
  if (warp == 0) join_store<ST * BLOB / 4, NW>(reinterpret_cast<const float*>(sm.ring), 0, 0, To{nullptr, nullptr, nullptr});
  int used = 0;       // pages consumed
  bool dead = false;  // a copy never arrived: consume and load nothing more
  int dead_at = 0;

  State<NT> z;
  // The state as finished rows (whole), or as the partial of a slot.
  auto emit = [&](int b, int unit, int slot, bool whole) {
    const int kvh = head_of(a, unit), rt = unit - kvh * a.RT;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = t * 8 + 2 * tig + c;
        const int r = rt * COLS + col;
        if (r >= a.S * a.G) continue;
        const float inv = z.l[t][c] > 0.f || z.l[t][c] != z.l[t][c] ? 1.f / z.l[t][c] : 0.f;
        const float om = z.om[t][c];
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)  // dim 32 (i / 4) + 4 gid + i % 4
          v[i] = fmaf(z.o[t][i >> 2][(i >> 1) & 1][2 * (i & 1) + c], (i & 1) ? 0x1p20f : 0x1p24f, om);
        if (whole) {
          const int s = pos_of(a, r);
          uint16_t* dst = a.out + ((int64_t)b * a.S + s) * a.ldo + (kvh * a.G + (r - s * a.G)) * DH;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const __nv_bfloat162 h0 = __floats2bfloat162_rn(v[4 * p] * inv, v[4 * p + 1] * inv);
            const __nv_bfloat162 h1 = __floats2bfloat162_rn(v[4 * p + 2] * inv, v[4 * p + 3] * inv);
            *reinterpret_cast<uint2*>(dst + 32 * p + 4 * gid) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
          }
        } else {
          float* po = a.part_o + ((int64_t)slot * COLS + col) * DH;
#pragma unroll
          for (int p = 0; p < 4; ++p)
            *reinterpret_cast<float4*>(po + 32 * p + 4 * gid) =
                make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
          if (gid == 0)
            *reinterpret_cast<float2*>(a.part_ml + ((int64_t)slot * COLS + col) * 2) =
                make_float2(z.R[t][c], z.l[t][c]);
        }
      }
  };
  int f0 = begin, ub = -1, b = 0, unit = 0, pages = 0;
  while (f0 < end) {
    // one segment: the pages of one unit (sequence, kv head, row tile) in this share
    b = find_warp(pre, a.B, f0);
    pages = (pre[b + 1] - pre[b]) / units;
    unit = (f0 - pre[b]) / pages;
    ub = pre[b] + unit * pages;  // flat index of the unit's first page
    const int f1 = min(end, ub + pages);
    const int kvh = head_of(a, unit), rt = unit - kvh * a.RT;
    const int L = seq_len(a, b);
    // row s sees the keys up to position first + s
    const int first = a.start_pos ? min(a.start_pos[b], L) : L;
    z.reset();
    {
      z.load_q(a, b, kvh, rt, L, first);
      const int all_seen = min(L, first + (rt * COLS) / a.G + 1);  // keys that every column sees

      for (int f = f0; f < f1; ++f) {
        const int st = used % ST;
        if (!dead) {
          dead = !mbd::mbar_wait(bar + st, (used / ST) & 1, a.status, MB_DEV_TIMEOUT_TMA);
          dead = __any_sync(0xffffffffu, dead);
          dead_at = used;
        }
        if (!dead && ok_flag[st]) {
          const int key0 = (f - ub) * PAGE;
          if (key0 + PAGE <= all_seen)
            z.template page<false>(ring + st * BLOB, sm.kp[warp], sm.vmin[warp], key0, L);
          else
            z.template page<true>(ring + st * BLOB, sm.kp[warp], sm.vmin[warp], key0, L);
        }
        __syncwarp();  // all lanes are done with this page
        ++used;
        if (issued < mine && !dead) issue();
      }
    }

    z.finish();
    if (f1 == end) break;  // the last one may go on in the next warp
    emit(b, unit, 2 * me, f0 == ub);
    f0 = f1;
  }
  // A warp that gave up leaves copies in flight: wait (bounded) for them.
  if (dead)
    for (int i = dead_at; i < issued; ++i) mbd::mbar_wait(bar + i % ST, (i / ST) & 1, nullptr, 0);

  // ---- neighbouring warps whose last unit is the same join their states ----
  if (lane == 0) {
    sm.seg[warp] = make_int4(ub, b, unit, (f0 == ub ? 1 : 0) | (end == ub + pages ? 2 : 0));
  }
  __syncthreads();  // every ring is free: a warp's state takes the place of its pages
  if (ub >= 0) z.deposit(reinterpret_cast<float*>(ring));
  __syncthreads();
  // lane w knows warp w's last unit; runs of warps with the same one, each a
  // row after the other, go round the warps
  const int4 sg = lane < NW ? sm.seg[lane] : make_int4(-1, 0, 0, 0);
  const int left = __shfl_up_sync(0xffffffffu, sg.x, 1);
  const bool leads = sg.x >= 0 && (lane == 0 || left != sg.x);
  const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
  const int nth = __popc(leaders & ((1u << lane) - 1)), items = __popc(leaders) * COLS;
  for (int i = warp; i < items; i += NW) {
    const int w0 = __ffs(__ballot_sync(0xffffffffu, leads && nth == i / COLS)) - 1, col = i % COLS;
    const int gub = __shfl_sync(0xffffffffu, sg.x, w0), gb = __shfl_sync(0xffffffffu, sg.y, w0);
    const int gunit = __shfl_sync(0xffffffffu, sg.z, w0), starts = __shfl_sync(0xffffffffu, sg.w, w0) & 1;
    const uint32_t who = __ballot_sync(0xffffffffu, sg.x == gub);
    const int ends = __shfl_sync(0xffffffffu, sg.w, 31 - __clz(who)) & 2;
    const int gkvh = head_of(a, gunit), r = (gunit - gkvh * a.RT) * COLS + col;
    if (r < a.S * a.G)
      join_store<ST * BLOB / 4, NW>(reinterpret_cast<const float*>(sm.ring), col, who,
                                    row_to(a, gb, gkvh, r, 2 * (blockIdx.x * a.active + w0) + starts, col, COLS,
                                           starts && ends));
  }
}

// One sequence (B = 1): every length is the same, so a cluster of CTAs takes a
// unit, its pages split evenly over the warps, and joins it over distributed
// shared memory: nothing to plan, no partials in memory and no second kernel.
// (8 kv heads: 517 keys 9.2 -> 6.6 us, 16000 keys 16.0 -> 12.5 us.)
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Address of the same shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(mbd::smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <int NT>
__global__ void __launch_bounds__(Shape<NT>::NW * 32) attn_kv4_one_kernel(const Args a) {
  constexpr int COLS = NT * 8, NW = Shape<NT>::NW, ST = Shape<NT>::ST;
  extern __shared__ __align__(128) uint8_t sm_raw[];
  Shared<NT>& sm = *reinterpret_cast<Shared<NT>*>(sm_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster_rank(), C = cluster_size();
  const int unit = blockIdx.x / C, kvh = head_of(a, unit), rt = unit - kvh * a.RT;
  uint8_t* ring = sm.ring[warp][0];
  uint64_t* bar = sm.bar[warp];
  int* ok_flag = sm.page_ok[warp];
  if (lane == 0)
    for (int i = 0; i < ST; ++i) mbd::mbar_init(bar + i, 1);
  mbd::fence_mbar_init();
  mbd::pdl_wait();
  mbd::pdl_trigger();
  const int L = seq_len(a, 0), pages = (L + PAGE - 1) / PAGE;
  // warps of different CTAs side by side: a short sequence is spread over them
  const int64_t share = warp * C + rank, shares = C * NW;
  const int begin = (int)(pages * share / shares), end = (int)(pages * (share + 1) / shares), mine = end - begin;
  int issued = 0, win_pid = 0, win_ok = 0;
  auto issue = [&]() {
    if ((issued & 31) == 0 && begin + issued + lane < end) {
      const int pid = a.table[begin + issued + lane];
      win_ok = pid >= 0 && pid < a.num_pages;
      win_pid = win_ok ? pid : 0;
      if (!win_ok) atomicOr(a.status, MB_DEV_BAD_PAGE);
    }
    const int pid = __shfl_sync(0xffffffffu, win_pid, issued & 31);
    const int good = __shfl_sync(0xffffffffu, win_ok, issued & 31);
    const int st = issued % ST;
    if (lane == 0) {
      ok_flag[st] = good;
      mbd::mbar_expect_tx(bar + st, BLOB);
      mbd::bulk_load(ring + st * BLOB, a.cache + ((int64_t)pid * a.Hkv + kvh) * BLOB, BLOB, bar + st);
    }
    ++issued;
  };
  for (int i = 0; i < ST && i < mine; ++i) issue();
  bool dead = false;  // a copy never arrived: consume and load nothing more
  int dead_at = 0;
  State<NT> z;
  z.reset();
  if (mine > 0) {
    const int first = a.start_pos ? min(a.start_pos[0], L) : L;
    z.load_q(a, 0, kvh, rt, L, first);
    const int all_seen = min(L, first + (rt * COLS) / a.G + 1);
    for (int used = 0; used < mine; ++used) {
      const int st = used % ST;
      if (!dead) {
        dead = !mbd::mbar_wait(bar + st, (used / ST) & 1, a.status, MB_DEV_TIMEOUT_TMA);
        dead = __any_sync(0xffffffffu, dead);
        dead_at = used;
      }
      if (!dead && ok_flag[st]) {
        const int key0 = (begin + used) * PAGE;
        if (key0 + PAGE <= all_seen)
          z.template page<false>(ring + st * BLOB, sm.kp[warp], sm.vmin[warp], key0, L);
        else
          z.template page<true>(ring + st * BLOB, sm.kp[warp], sm.vmin[warp], key0, L);
      }
      __syncwarp();
      if (issued < mine && !dead) issue();
    }
    if (dead)
      for (int i = dead_at; i < issued; ++i) mbd::mbar_wait(bar + i % ST, (i / ST) & 1, nullptr, 0);
    z.finish();
    z.deposit(reinterpret_cast<float*>(ring));
  }
  if (lane == 0) sm.seg[warp].x = mine;
  __syncthreads();
  // this CTA's part of every row, in place of the key numbers
  float* part = reinterpret_cast<float*>(sm.kp);  // [COLS][DH], then [COLS] (reference, denominator)
  static_assert(COLS * (DH + 2) * 4 <= NW * PAGE * 20, "a CTA's rows take the place of its key numbers");
  const uint32_t who = __ballot_sync(0xffffffffu, lane < NW && sm.seg[lane < NW ? lane : 0].x > 0);
  for (int col = warp; col < COLS; col += NW) {
    const Joined j = join_row<ST * BLOB / 4, NW>(reinterpret_cast<const float*>(sm.ring), col, who);
    *reinterpret_cast<float4*>(part + col * DH + lane * 4) = j.o;
    if (lane == 0) *reinterpret_cast<float2*>(part + COLS * DH + col * 2) = make_float2(j.R, j.l);
  }
  cluster_sync();
  for (int col = rank + warp * C; col < COLS; col += NW * C) {
    const int r = rt * COLS + col;
    if (r >= a.S * a.G) continue;
    float2 m = make_float2(-INFINITY, 0.f);
    if (lane < C) m = ld_cluster2(in_cta(part + COLS * DH + col * 2, lane));
    float R = m.x;
#pragma unroll
    for (int off = 8; off; off >>= 1) R = fmaxf(R, __shfl_xor_sync(0xffffffffu, R, off));
    R = __shfl_sync(0xffffffffu, R, 0);
    const float f = m.x == -INFINITY ? 0.f : fast_exp2(m.x - R);
    float l = m.y * f;
#pragma unroll
    for (int off = 8; off; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < C; ++c) {
      const float fc = __shfl_sync(0xffffffffu, f, c);
      const float4 v = ld_cluster4(in_cta(part + col * DH + lane * 4, c));
      o.x = fmaf(v.x, fc, o.x);
      o.y = fmaf(v.y, fc, o.y);
      o.z = fmaf(v.z, fc, o.z);
      o.w = fmaf(v.w, fc, o.w);
    }
    store_row(row_to(a, 0, kvh, r, 0, col, COLS, true), R, __shfl_sync(0xffffffffu, l, 0), o);
  }
  cluster_sync();  // nobody leaves while its rows are read
}

// Joins the partials of the units that more than one CTA worked on; before it
// waits for them it plans. A CTA takes a unit; its 8 warps take a query row
// each, or (SPLIT: few units, so many partials each) share one row's partials.
template <int NT, bool SPLIT>
__global__ void __launch_bounds__(256) attn_kv4_combine_kernel(const Args a) {
  __shared__ Plan plan;
  constexpr int COLS = NT * 8;
  mbd::pdl_trigger();
  make_plan<8>(a, plan);
  mbd::pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.Hkv * a.RT, act = a.active;
  const int per = (plan.vpre[a.B] + a.warps - 1) / a.warps;
  for (int u = blockIdx.x; u < a.B * units; u += gridDim.x) {
    const int b = u / units, unit = u - b * units;
    const int pages = (plan.pre[b + 1] - plan.pre[b]) / units;
    if (pages == 0) continue;
    const int v = plan.vpre[b] + unit * (pages + UNIT_COST) + UNIT_COST;  // place of the first page
    const int w0 = v / per, w1 = (v + pages - 1) / per, c0 = w0 / act, c1 = w1 / act;
    // w1's share ends with this unit: then it joined its CTA's other warps on it
    const bool ends = v + pages == plan.vpre[a.B] || v + pages + UNIT_COST >= (int64_t)(w1 + 1) * per;
    const int joined = c1 - c0 + (ends || w1 > max(w0, c1 * act) ? 1 : 0);
    const int n = joined + (ends ? 0 : 1);
    if (n < 2) continue;  // written by the main kernel
    const int kvh = head_of(a, unit), rt = unit - kvh * a.RT;
#pragma unroll
    for (int c8 = 0; c8 < (SPLIT ? 1 : NT); ++c8) {
      const int col = SPLIT ? blockIdx.y : c8 * 8 + warp;
      const int r = rt * COLS + col;
      if (r < a.S * a.G) {
        auto row = [&](int i) -> int64_t {
          const int w = i < joined ? max(w0, (c0 + i) * act) : w1;
          return (int64_t)(2 * w + (w == w0 ? 1 : 0)) * COLS + col;
        };
        // every lane keeps the same running reference
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = SPLIT ? warp : 0; i < n; i += SPLIT ? 32 : 4) {
          float2 ml[4];
          float4 o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int j = i + k * (SPLIT ? 8 : 1);
            ml[k] = make_float2(-INFINITY, 0.f);
            o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (j < n) {
              ml[k] = *reinterpret_cast<const float2*>(a.part_ml + row(j) * 2);
              o[k] = *reinterpret_cast<const float4*>(a.part_o + row(j) * DH + lane * 4);
            }
          }
          const float Mn = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M);
          const float f = M == -INFINITY ? 0.f : fast_exp2(M - Mn);
          M = Mn;
          L *= f;
          acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float w = ml[k].x == -INFINITY ? 0.f : fast_exp2(ml[k].x - Mn);
            L = fmaf(ml[k].y, w, L);
            acc.x = fmaf(o[k].x, w, acc.x);
            acc.y = fmaf(o[k].y, w, acc.y);
            acc.z = fmaf(o[k].z, w, acc.z);
            acc.w = fmaf(o[k].w, w, acc.w);
          }
        }
        if (SPLIT) {
          __shared__ float4 so[8][32];
          __shared__ float2 sl[8];
          so[warp][lane] = acc;
          if (lane == 0) sl[warp] = make_float2(M, L);
          __syncthreads();
          if (warp == 0) {
#pragma unroll
            for (int w = 1; w < 8; ++w) M = fmaxf(M, sl[w].x);
            L = 0.f;
            acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 8; ++w) {
              const float f = sl[w].x == -INFINITY ? 0.f : fast_exp2(sl[w].x - M);
              const float4 o = so[w][lane];
              L = fmaf(sl[w].y, f, L);
              acc.x = fmaf(o.x, f, acc.x);
              acc.y = fmaf(o.y, f, acc.y);
              acc.z = fmaf(o.z, f, acc.z);
              acc.w = fmaf(o.w, f, acc.w);
            }
          }
          __syncthreads();
          if (warp) continue;
        }
        store_row(row_to(a, b, kvh, r, 0, col, COLS, true), M, L, acc);
      }

    }
  }
}

struct Launch {
  int nt, rt, ctas, active;
  size_t bytes;
};

// Query rows of a kv head: S * G. Up to 8 take one column tile, more two (so
// that a page is unpacked once for 16 rows), in row tiles of 16.
Launch plan_launch(int B, int S, int Hq, int Hkv, int pages) {
  Launch p;
  const int64_t rows = (int64_t)S * (Hq / Hkv);
  p.nt = rows <= 8 ? 1 : 2;
  p.rt = (int)((rows + p.nt * 8 - 1) / (p.nt * 8));
  // shares of at least a page; as few warps a CTA as that leaves, over all SMs
  const int64_t most = (int64_t)(B < MAX_B ? B : MAX_B) * Hkv * p.rt * ((int64_t)pages + UNIT_COST);
  const int sms = mb::num_sms(), nw = p.nt == 1 ? Shape<1>::NW : Shape<2>::NW;
  p.ctas = (int)(most < sms ? most : sms);
  const int64_t act = (most + p.ctas - 1) / p.ctas;
  p.active = (int)(act < nw ? act : nw);
  p.bytes = (size_t)p.ctas * p.active * 2 * p.nt * 8 * (DH + 2) * sizeof(float);
  return p;
}

// Clusters of `size` CTAs of the one-sequence kernel that run at a time.
template <int NT>
int resident_clusters(int size) {
  static int known[64][5] = {};
  int dev = 0, slot = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 0;
  while ((1 << slot) < size) ++slot;
  if (!known[dev][slot]) {
    const void* fn = reinterpret_cast<const void*>(attn_kv4_one_kernel<NT>);
    int n = 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(size * 8);
    cfg.blockDim = dim3(Shape<NT>::NW * 32);
    cfg.dynamicSmemBytes = sizeof(Shared<NT>);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    if (mb::ensure_smem_attr(fn, (int)sizeof(Shared<NT>)) ||
        cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, attn_kv4_one_kernel<NT>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      n = 0;
    }
    known[dev][slot] = n + 1;
  }
  return known[dev][slot] - 1;
}

// Cluster size for one sequence, 0: the kernel for many. Expected times in us:
// 5.3, 0.3 more for a cluster of two and 0.6 for a larger one, and 0.2 for every
// page of a CTA's part of its unit; against 13, and 0.18 for every page of an SM's
// part of all units. Measured in graphs, the kernel for many / clusters of 1, 4, 8, 16:
//   8 kv heads,   517 keys    9.2 /   6.6   7.0   7.4  15.4
//                4000        10.4 /  17.5   9.0   7.4  15.4
//               16000        16.0 /  49.9  17.7  12.5  19.3
//               64000        24.2 / 182.0  50.9  29.9  37.5
//              131075        36.3 / 366.2  97.8  54.5  62.1
//   1 kv head,  16000        13.3 /  49.0  16.8  11.0   9.1
//               64000        14.8 / 180.7  50.1  28.3  18.4
// (Seven clusters of 16 run at a time: eight units take two rounds.)
template <int NT>
int one_cluster(int units, int pages) {
  const double flat = 13 + 0.18 * (double)units * pages / mb::num_sms();
  double best = flat;
  int at = 0;
  for (int c = 1; c <= 16; c <<= 1) {
    const double t = 5.3 + (c == 1 ? 0 : c == 2 ? 0.3 : 0.6) + 0.2 * pages / c;
    if (t < best && units <= resident_clusters<NT>(c)) best = t, at = c;
  }
  return at;
}

template <int NT>
int launch_one(const Args& a, int c, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(a.Hkv * a.RT * c);
  cfg.blockDim = dim3(Shape<NT>::NW * 32);
  cfg.dynamicSmemBytes = sizeof(Shared<NT>);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = mb::pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = c;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  MB_CUDA(cudaLaunchKernelEx(&cfg, attn_kv4_one_kernel<NT>, a));
  return MB_OK;
}

template <int NT>
int launch(const Args& a, int ctas, cudaStream_t s) {
  if (a.B == 1) {
    const int c = one_cluster<NT>(a.Hkv * a.RT, (a.max_len + PAGE - 1) / PAGE);
    if (c) return launch_one<NT>(a, c, s);
  }
  const int smem = (int)sizeof(Shared<NT>);
  int rc = mb::ensure_smem_attr(reinterpret_cast<const void*>(attn_kv4_kernel<NT>), smem);
  if (rc) return rc;
  MB_CUDA(mb::launch_pdl(attn_kv4_kernel<NT>, dim3(ctas), dim3(Shape<NT>::NW * 32), smem, s, a));
  if (a.warps == 1) return MB_OK;  // one share: nothing is in parts
  const int units = a.B * a.Hkv * a.RT, sms = mb::num_sms();
  // few units are many parts each (about sms / units): 8 warps to a row
  if (units * 8 <= sms)
    MB_CUDA(mb::launch_pdl(attn_kv4_combine_kernel<NT, true>, dim3(units, NT * 8), dim3(256), 0, s, a));
  else
    MB_CUDA(mb::launch_pdl(attn_kv4_combine_kernel<NT, false>, dim3(units < 4 * sms ? units : 4 * sms), dim3(256),
                           0, s, a));
  return MB_OK;
}

// Pieces of a prompt (64 rows a sequence or more): instead of unpacking every
// page once a row tile of 16, expand the cache once to fp16 pages in the
// workspace and run the tcgen05 prefill attention over those (the keys cut in
// parts when the row tiles are too few for the SMs), where the times (us) that
// expand_plan expects say so: 0.29 a page and row tile on one SM; or 1 a
// 128-key tile and 3 a wave of CTAs, and the bytes at 5.5 TB/s. Measured in us,
// expanded / unpacked:
//   2 sequences of 8192, 8 kv heads, 4 query heads each:  64 rows 58 / 83,
//     128 rows 62 / 151, 512 rows 151 / 549;
//   1 of 32768, 8, 4:  64 rows 118 / 145, 128 rows 107 / 276;
//   16 of 2048, 8, 4:  64 rows 114 / 167, 128 rows 125 / 307;
//   1 of 1024, 8, 1:  256 rows 18 / 13;  8 of 512, 8, 4:  64 rows 24 / 58;
//   1 of 8192, 1, 8:  64 rows 25 / 17.
constexpr int TC_ROWS = 64;
constexpr size_t MOST_EXPANDED = size_t(6) << 30;  // workspace: a sequence of 1.3 million tokens of 8 heads

struct Expand {
  int seqs;  // sequences expanded at a time: up to 512 MB of pages, at least one
  int splits;  // parts that a row tile's keys are cut into, to fill the SMs
  size_t half, part_at, bytes;  // keys or values; where the partials start; all
};

bool expand_plan(int B, int S, int Hq, int Hkv, int n_pages, Expand* e) {
  if (S < TC_ROWS || Hq > 65535 || Hkv > 65535 || (int64_t)(n_pages + 1) * Hkv * PAGE >= (1ll << 31)) return false;
  const int even = (n_pages + 1) / 2 * 2;
  const int64_t per_seq = (int64_t)even * Hkv * PAGE * DH * 2;
  int64_t n = (256ll << 20) / per_seq;
  n = n < 1 ? 1 : n > 65535 ? 65535 : n;
  e->seqs = (int)(n < B ? n : B);
  e->half = (size_t)per_seq * e->seqs;
  e->splits = mb::attention_split_plan(e->seqs, S, Hq, (int64_t)n_pages * PAGE);
  e->part_at = 2 * e->half + ((size_t)e->seqs * even * Hkv * sizeof(int2) + 15) / 16 * 16;
  e->bytes = e->part_at + (e->splits > 1 ? (size_t)e->seqs * S * Hq * e->splits * (DH + 2) * sizeof(float) : 0);
  if (e->bytes > MOST_EXPANDED) return false;
  const double sms = mb::num_sms(), pages = (double)B * Hkv * n_pages;
  const int rt = plan_launch(B, S, Hq, Hkv, n_pages).rt, sp = e->splits;
  const double unpack = 9 + (pages + 8.0 * B * Hkv) * rt * 0.29 / sms;  // a unit's start and end: 8 pages
  const double calls = std::ceil((double)B / e->seqs), ctas = (double)e->seqs * Hq * ((S + 127) / 128) * sp;
  const double tiles = ((n_pages + 1) / 2 + sp - 1) / sp;
  const double expand = 3 + calls * (3 + std::ceil(ctas / sms) * (3 + tiles) + (sp > 1 ? 6 : 0)) +
                        pages * (BLOB + 2 * PAGE * DH * 2) / 5.5e6;
  return expand < unpack;
}

}  // namespace

extern "C" size_t mb_attention_kv4_workspace_bytes(int B, int S, int Hq, int Hkv, int max_kv_len) {
  if (B <= 0 || S <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || max_kv_len <= 0) return 0;
  const int pages = (int)(((int64_t)max_kv_len + PAGE - 1) / PAGE);
  const size_t n = plan_launch(B, S, Hq, Hkv, pages).bytes;
  Expand e;
  return expand_plan(B, S, Hq, Hkv, pages, &e) && e.bytes > n ? e.bytes : n;
}

extern "C" int mb_attention_kv4_bf16(const uint16_t* q, int64_t ldq, const uint8_t* cache,
                                     int num_pages, const int* block_table, int max_pages,
                                     const int* kv_len, int max_kv_len, const int* start_pos, int B, int S,
                                     int Hq, int Hkv, int Dh, float scale, uint16_t* out, int64_t ldo,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  MB_REQUIRE(Dh == DH, "attention: head_dim must be 128 (got %d)", Dh);
  MB_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "attention: Hq must be a multiple of Hkv");
  MB_REQUIRE(B >= 0 && S >= 0 && num_pages > 0 && max_pages > 0, "attention kv4: bad sizes");
  if (B == 0 || S == 0) return MB_OK;
  MB_REQUIRE(q && cache && block_table && kv_len && out, "attention kv4: null pointer");
  MB_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache) % 16 == 0 && ldq % 8 == 0 && ldo % 8 == 0,
             "attention kv4: q, out and the cache must be 16-byte aligned");
  MB_REQUIRE((int64_t)S * Hq < (1ll << 30) && (int64_t)max_pages * PAGE < (1ll << 30),
             "attention kv4: too many rows or pages");
  MB_REQUIRE(max_kv_len > 0 && max_kv_len <= max_pages * PAGE, "attention kv4: max_kv_len must be in [1, max_pages*64]");
  const int pages = (max_kv_len + PAGE - 1) / PAGE;
  const Launch p = plan_launch(B, S, Hq, Hkv, pages);
  MB_REQUIRE(workspace && workspace_bytes >= p.bytes && (uintptr_t)workspace % 16 == 0,
             "attention kv4: workspace of %zu bytes required, 16-byte aligned", p.bytes);
  Expand e;
  const bool expand = expand_plan(B, S, Hq, Hkv, pages, &e) && scale > 0.f && ldq < (1 << 30) && ldo < (1 << 30) &&
                      mb::attention_prefill_tc_ok(q, (int)ldq, nullptr, nullptr, out, (int)ldo);
  // sequences a launch of the other form: its flat list of pages is counted in 32 bits
  const int64_t fit = ((1ll << 30) - 1) / ((int64_t)Hkv * p.rt * ((int64_t)pages + UNIT_COST));
  MB_REQUIRE(expand || fit > 0, "attention kv4: too many pages for the rows of one sequence");
  uint32_t* status = mb::device_status_ptr();
  MB_REQUIRE(status, "attention kv4: no status word");
  if (expand) {
    MB_REQUIRE(workspace_bytes >= e.bytes, "attention kv4: workspace of %zu bytes required", e.bytes);
    uint8_t* w = static_cast<uint8_t*>(workspace);
    mb::Kv4Rows r;
    r.x.k = reinterpret_cast<uint16_t*>(w);
    r.x.v = reinterpret_cast<uint16_t*>(w + e.half);
    r.x.page_exp = reinterpret_cast<int2*>(w + 2 * e.half);
    r.x.pages = (pages + 1) / 2 * 2;
    r.part = e.splits > 1 ? reinterpret_cast<float*>(w + e.part_at) : nullptr;
    r.splits = e.splits;
    r.ldq = ldq;
    r.ldo = ldo;
    r.max_len = max_kv_len;
    r.S = S;
    r.Hq = Hq;
    r.Hkv = Hkv;
    r.scale = scale;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    for (int b = 0; b < B; b += e.seqs) {
      r.B = B - b < e.seqs ? B - b : e.seqs;
      r.q = q + (int64_t)b * S * ldq;
      r.out = out + (int64_t)b * S * ldo;
      r.kv_len = kv_len + b;
      r.start_pos = start_pos ? start_pos + b : nullptr;
      int rc = mb::kv4_expand(cache, num_pages, Hkv, block_table + (int64_t)b * max_pages, max_pages, max_kv_len,
                              r.kv_len, r.B, r.x, status, s);
      if (!rc) rc = mb::attention_rows_kv4(r, s);
      if (rc) return rc;
    }
    return MB_OK;
  }
  const int step = (int)(fit < MAX_B ? fit : MAX_B);
  for (int b = 0; b < B; b += step) {
    Args a;
    a.q = q + (int64_t)b * S * ldq;
    a.cache = cache;
    a.table = block_table + (int64_t)b * max_pages;
    a.kv_len = kv_len + b;
    a.start_pos = start_pos ? start_pos + b : nullptr;
    a.out = out + (int64_t)b * S * ldo;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)p.ctas * p.active * 2 * p.nt * 8 * DH;
    a.status = status;
    a.ldq = ldq;
    a.ldo = ldo;
    a.num_pages = num_pages;
    a.max_pages = max_pages;
    a.max_len = max_kv_len;
    a.B = B - b < step ? B - b : step;
    a.S = S;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.RT = p.rt;
    a.warps = p.ctas * p.active;
    a.active = p.active;
    a.scale_log2 = scale * 1.4426950408889634f;
    const int rc = p.nt == 1 ? launch<1>(a, p.ctas, static_cast<cudaStream_t>(stream))
                             : launch<2>(a, p.ctas, static_cast<cudaStream_t>(stream));
    if (rc) return rc;
  }
  return MB_OK;
}
