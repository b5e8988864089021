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
// sums. q is scaled by a power of two into fp16's range, which loses nothing
// of a bf16 number down to 2^-20 of the tile's largest.
// The value scale goes into the exponent: P_j = 2^(score_j + log2(sv_j) - R)
// with a running reference R per query row, so that P_j sv-weighted is what is
// rounded to fp16 (11 bits, and 2^-24 absolute at a range up to 2^15), and the
// denominator is sum_j P_j / sv_j in fp32. R only moves when a weight would
// pass 2^15, so most pages rescale nothing.
//
// Orientation: keys are the 16 MMA rows, query rows the 8 columns (S^T = K
// Q^T, O^T = V^T P^T), so a decode step's 8 query heads of a kv head fill a
// column tile and no row is wasted; P^T moves from the accumulator layout to
// the operand layout by movmatrix. Query rows are the S * G pairs (position,
// head of the group); NT column tiles of 8 per pass over the cache.
//
// Schedule: the flat list of (sequence, kv head, row tile, page) is cut into
// equal shares, one a warp, planned on the device from kv_len, so that ragged
// batches balance; every (sequence, kv head, row tile), a unit, counts
// UNIT_COST pages more than it has, for its start and end. Each warp streams
// its share through its own ring of whole-page bulk copies (8704 bytes, one
// mbarrier each) without waiting for another. A unit that lies within a share
// is written at once. At the end the warps of a CTA that stopped in the same
// unit join their states in shared memory; what is then still in parts (at
// most two a warp) goes to the workspace, and attn_kv4_combine_kernel joins it.
#include <cuda_fp16.h>

#include "kv4.cuh"
#include "kernels.h"

namespace {
using namespace kv4;

constexpr int NW = 4;  // warps per CTA
constexpr int ST = 2;  // pages in a warp's ring
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
  int* plan;       // [2 (B + 1)]: pre, vpre for the combine kernel
  uint32_t* status;
  int64_t ldq, ldo;  // elements between two positions' rows
  int num_pages, max_pages, B, S, Hkv, G, RT;
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

// Attended keys of sequence b.
__device__ __forceinline__ int seq_len(const Args& a, int b) {
  return max(0, min(a.kv_len[b], a.max_pages * PAGE));
}

// pre[b] = flat index of the first page of sequence b, pre[B] = their number;
// vpre the same with UNIT_COST more pages a unit.
__device__ void plan(const Args& a, int* pre, int* vpre, int2* wsum) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + NW * 32 - 1) / (NW * 32);
  const int b0 = min(a.B, tid * per), b1 = min(a.B, b0 + per);
  const int units = a.Hkv * a.RT;
  int2 sum = make_int2(0, 0);
  for (int b = b0; b < b1; ++b) {
    const int pages = (seq_len(a, b) + PAGE - 1) / PAGE;
    sum.x += pages * units;
    sum.y += pages ? (pages + UNIT_COST) * units : 0;
  }
  int2 inc = sum;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc.x, off), y = __shfl_up_sync(0xffffffffu, inc.y, off);
    if (lane >= off) inc.x += x, inc.y += y;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  int2 run = make_int2(inc.x - sum.x, inc.y - sum.y);
  for (int w = 0; w < warp; ++w) run.x += wsum[w].x, run.y += wsum[w].y;
  for (int b = b0; b < b1; ++b) {
    pre[b] = run.x;
    vpre[b] = run.y;
    const int pages = (seq_len(a, b) + PAGE - 1) / PAGE;
    run.x += pages * units;
    run.y += pages ? (pages + UNIT_COST) * units : 0;
  }
  if (tid == NW * 32 - 1) {
    pre[a.B] = run.x;  // the last thread's end is everybody's
    vpre[a.B] = run.y;
  }
  __syncthreads();
}

// Pages whose place in the costed list lies before v.
__device__ __forceinline__ int pages_before(const int* pre, const int* vpre, int B, int units, int v) {
  if (v >= vpre[B]) return pre[B];
  int lo = 0, hi = B;  // vpre[lo] <= v < vpre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (vpre[mid] <= v) lo = mid; else hi = mid;
  }
  const int pages = (pre[lo + 1] - pre[lo]) / units;
  const int rem = v - vpre[lo], unit = rem / (pages + UNIT_COST);
  return pre[lo] + unit * pages + max(0, rem - unit * (pages + UNIT_COST) - UNIT_COST);
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
  float sk, mk;  // key scale and minimum, with the softmax scale and q's power of two
  float lg, rv;  // log2 and reciprocal of the value scale
};

// A warp's running state over the pages of one unit: NT column tiles of 8.
template <int NT>
struct State {
  float o[NT][4][2][4];  // [32-dim piece][dim pair][accumulator]
  float R[NT][2], l[NT][2], om[NT][2];
  uint32_t qf[NT][16];   // q as B fragments
  float qs[NT][2];       // sum of q's dims
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

  // One page (pg, in shared memory) of keys key0 .. key0 + 63. MASKED: some of
  // them stand past the end (len) or are not seen by every column.
  template <bool MASKED>
  __device__ __forceinline__ void page(const uint8_t* pg, KeyParams* kp, float* vmin, int key0, int len,
                                       float ck, float cm) {
    const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = lane + 32 * i;
      uint32_t k = *reinterpret_cast<const uint32_t*>(pg + K_PARAMS + key * 4);
      uint32_t v = *reinterpret_cast<const uint32_t*>(pg + V_PARAMS + key * 4);
      if (MASKED && key0 + key >= len) k = v = 0;  // what stands past the end may be anything
      // a value scale of 0 (all dims alike, codes 0) must not enter the logarithm
      const float sv = lo_bf(v), s = sv == 0.f ? 1.f : fminf(fmaxf(sv, 0x1p-90f), 0x1p90f);
      const float r = fast_rcp(s);
      kp[key] = KeyParams{lo_bf(k) * ck, hi_bf(k) * cm, fast_log2(s), r};
      // a scale that is no number makes the row none (clamping would hide it)
      vmin[key] = sv < INFINITY ? hi_bf(v) * r : NAN;
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
            float x = fmaf(p.mk, qs[t][c], fmaf(p.sk, sc[t][mt][2 * r + c], p.lg));
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

    // ---- weights and O^T += V^T P^T, 16 keys at a time ----
    const uint32_t pg_s = mbd::smem_u32(pg);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
      uint32_t pf[NT][2];
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
            p[c] = fast_exp2(sc[t][mt][2 * r + c] - (MASKED && R[t][c] == -INFINITY ? 0.f : R[t][c]));
            l[t][c] = fmaf(p[c], rv, l[t][c]);
            om[t][c] = fmaf(p[c], mv, om[t][c]);
          }
          pf[t][r] = transpose8x8(pack_h2(p[0], p[1]));
        }
      }
      const int key = mt * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
      const uint32_t rowp = pg_s + V_CODES + key * ROW;
      const int sw = (key >> 1) & 3;
#pragma unroll
      for (int p = 0; p < 4; p += 2) {
        uint32_t v[4];  // octets 0, 1 of piece p, then of piece p + 1
        ldsm_x4_t(v, rowp + (((p + (lane >> 4)) ^ sw) << 4));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t e0[4], e1[4];
          spread(v[2 * j], e0);
          spread(v[2 * j + 1], e1);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16_16816(o[t][p + j][0], e0[0], e0[1], e1[0], e1[1], pf[t][0], pf[t][1]);
            mma_f16_16816(o[t][p + j][1], e0[2], e0[3], e1[2], e1[3], pf[t][0], pf[t][1]);
          }
        }
      }
    }
  }
};

template <int NT>
__global__ void __launch_bounds__(NW * 32) attn_kv4_kernel(const Args a) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  constexpr int COLS = NT * 8;
  extern __shared__ __align__(128) uint8_t sm[];
  uint8_t* ring = sm + (threadIdx.x >> 5) * ST * BLOB;
  KeyParams* kp = reinterpret_cast<KeyParams*>(sm + NW * ST * BLOB) + (threadIdx.x >> 5) * PAGE;
  float* vmin = reinterpret_cast<float*>(sm + NW * (ST * BLOB + PAGE * 16)) + (threadIdx.x >> 5) * PAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + NW * (ST * BLOB + PAGE * 20));  // [NW][ST]
  int2* wsum = reinterpret_cast<int2*>(bars + NW * ST);               // [NW]
  int4* seg = reinterpret_cast<int4*>(wsum + NW);                     // [NW]
  int* page_ok = reinterpret_cast<int*>(seg + NW);                    // [NW][ST]
  int* pre = page_ok + NW * ST;                                       // [B + 1]
  int* vpre = pre + a.B + 1;                                          // [B + 1]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  uint64_t* bar = bars + warp * ST;
  int* ok_flag = page_ok + warp * ST;
  if (lane == 0)
    for (int i = 0; i < ST; ++i) mbd::mbar_init(bar + i, 1);
  mbd::fence_mbar_init();
  plan(a, pre, vpre, wsum);

  // sequences without keys: their rows are zeros
  const int row_elems = a.Hkv * a.G * DH;
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (pre[b] == pre[b + 1])
      for (int s = 0; s < a.S; ++s)
        for (int i = threadIdx.x * 8; i < row_elems; i += NW * 32 * 8)
          *reinterpret_cast<uint4*>(a.out + ((int64_t)b * a.S + s) * a.ldo + i) = make_uint4(0, 0, 0, 0);

  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < 2 * (a.B + 1); i += NW * 32) a.plan[i] = pre[i];

  const int units = a.Hkv * a.RT;
  const int me = blockIdx.x * NW + warp;
  const int per = (vpre[a.B] + gridDim.x * NW - 1) / (gridDim.x * NW);
  const int begin = pages_before(pre, vpre, a.B, units, min((int64_t)me * per, (int64_t)vpre[a.B]));
  const int end = pages_before(pre, vpre, a.B, units, min((int64_t)(me + 1) * per, (int64_t)vpre[a.B]));
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
        win_kvh = unit / a.RT;
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
  int used = 0;       // pages consumed
  bool dead = false;  // a copy never arrived: consume and load nothing more
  int dead_at = 0;

  State<NT> z;
  // The state as finished rows (whole), or as the partial of a slot.
  auto emit = [&](int b, int unit, int slot, bool whole) {
    const int kvh = unit / a.RT, rt = unit - kvh * a.RT;
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
          const int s = r / a.G;
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
    b = find_seq(pre, a.B, f0);
    pages = (pre[b + 1] - pre[b]) / units;
    unit = (f0 - pre[b]) / pages;
    ub = pre[b] + unit * pages;  // flat index of the unit's first page
    const int f1 = min(end, ub + pages);
    const int kvh = unit / a.RT, rt = unit - kvh * a.RT;
    const int L = seq_len(a, b);
    // row s sees the keys up to position first + s
    const int first = a.start_pos ? min(a.start_pos[b], L) : L;
    z.reset();
    {
      // ---- q of this unit as B fragments, scaled by a power of two ----
      float x[NT][32];
      float big = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int r = rt * COLS + t * 8 + gid;
        const int s = r / a.G;
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
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          big = fmaxf(big, fabsf(x[t][i]));
          sum += x[t][i];
        }
#pragma unroll
        for (int off = 1; off <= 2; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int mylim = min(L, first + s + 1);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int from = (2 * tig + c) * 4;  // a lane whose fragment row is column 2 tig + c
          z.qs[t][c] = __shfl_sync(0xffffffffu, sum, from);
          z.lim[t][c] = __shfl_sync(0xffffffffu, mylim, from);
        }
      }
#pragma unroll
      for (int off = 1; off <= 16; off <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
      // 2^e brings the tile's largest to [2^11, 2^12)
      const int e = max(-100, min(100, 11 - ((int)(__float_as_uint(big) >> 23) - 127)));
      const float up = __uint_as_float((uint32_t)(127 + e) << 23), up16 = up * 0.0625f;
      const float ck = a.scale_log2 * __uint_as_float((uint32_t)(127 + 24 - e) << 23);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          z.qf[t][4 * w] = pack_h2(x[t][8 * w] * up, x[t][8 * w + 4] * up);
          z.qf[t][4 * w + 1] = pack_h2(x[t][8 * w + 1] * up16, x[t][8 * w + 5] * up16);
          z.qf[t][4 * w + 2] = pack_h2(x[t][8 * w + 2] * up, x[t][8 * w + 6] * up);
          z.qf[t][4 * w + 3] = pack_h2(x[t][8 * w + 3] * up16, x[t][8 * w + 7] * up16);
        }
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
            z.template page<false>(ring + st * BLOB, kp, vmin, key0, L, ck, a.scale_log2);
          else
            z.template page<true>(ring + st * BLOB, kp, vmin, key0, L, ck, a.scale_log2);
        }
        __syncwarp();  // all lanes are done with this page
        ++used;
        if (issued < mine && !dead) issue();
      }
    }

#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
          z.l[t][c] += __shfl_xor_sync(0xffffffffu, z.l[t][c], off);
          z.om[t][c] += __shfl_xor_sync(0xffffffffu, z.om[t][c], off);
        }
    if (f1 == end) break;  // the last one may go on in the next warp
    emit(b, unit, 2 * me, f0 == ub);
    f0 = f1;
  }
  // A warp that gave up leaves copies in flight: wait (bounded) for them.
  if (dead)
    for (int i = dead_at; i < issued; ++i) mbd::mbar_wait(bar + i % ST, (i / ST) & 1, nullptr, 0);

  // ---- neighbouring warps whose last unit is the same join their states ----
  if (lane == 0) seg[warp] = make_int4(ub, f0, end, 0);
  __syncthreads();  // every ring is free: a warp's state takes the place of its pages
  const bool leads = ub >= 0 && (warp == 0 || seg[warp - 1].x != ub);
  if (ub >= 0 && !leads) {
    float* dst = reinterpret_cast<float*>(ring) + lane;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 32; ++i) dst[(t * 38 + i) * 32] = z.o[t][i >> 3][(i >> 2) & 1][i & 3];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        dst[(t * 38 + 32 + c) * 32] = z.R[t][c];
        dst[(t * 38 + 34 + c) * 32] = z.l[t][c];
        dst[(t * 38 + 36 + c) * 32] = z.om[t][c];
      }
    }
  }
  __syncthreads();
  if (!leads) return;
  int f1 = end;
  for (int w = warp + 1; w < NW && seg[w].x == ub; ++w) {
    f1 = seg[w].z;
    const float* src = reinterpret_cast<const float*>(ring + (w - warp) * ST * BLOB) + lane;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float fa[2], fb[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float Ro = src[(t * 38 + 32 + c) * 32];
        const float Rn = fmaxf(z.R[t][c], Ro);
        fa[c] = z.R[t][c] == -INFINITY ? 0.f : fast_exp2(z.R[t][c] - Rn);
        fb[c] = Ro == -INFINITY ? 0.f : fast_exp2(Ro - Rn);
        z.R[t][c] = Rn;
        z.l[t][c] = z.l[t][c] * fa[c] + src[(t * 38 + 34 + c) * 32] * fb[c];
        z.om[t][c] = z.om[t][c] * fa[c] + src[(t * 38 + 36 + c) * 32] * fb[c];
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        float& o = z.o[t][i >> 3][(i >> 2) & 1][i & 3];
        o = o * fa[i & 1] + src[(t * 38 + i) * 32] * fb[i & 1];
      }
    }
  }
  emit(b, unit, 2 * me + (f0 == ub ? 1 : 0), f0 == ub && f1 == ub + pages);
}

// Joins the partials of the units that more than one warp worked on. A CTA is
// one unit and COLS / gridDim.y of its query rows; its 8 warps take a row each
// (many units: few partials each), or share one row's partials (few units).
template <int NT, bool SPLIT>
__global__ void __launch_bounds__(256) attn_kv4_combine_kernel(const Args a, int warps) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  constexpr int COLS = NT * 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = a.Hkv * a.RT;
  const int b = blockIdx.x / units, unit = blockIdx.x - b * units;
  const int col = SPLIT ? blockIdx.y : blockIdx.y * 8 + warp;
  const int kvh = unit / a.RT, r = (unit - kvh * a.RT) * COLS + col;
  const int pages = (a.plan[b + 1] - a.plan[b]) / units;
  const int* vpre = a.plan + a.B + 1;
  const int per = (vpre[a.B] + warps - 1) / warps;
  const int v = vpre[b] + unit * (pages + UNIT_COST) + UNIT_COST;  // place of the first page
  if (pages == 0 || r >= a.S * a.G) return;
  const int w0 = v / per, w1 = (v + pages - 1) / per, c0 = w0 / NW, c1 = w1 / NW;
  // w1's share ends with this unit: then it joined its CTA's other warps on it
  const bool ends = v + pages == vpre[a.B] || v + pages + UNIT_COST >= (int64_t)(w1 + 1) * per;
  const int joined = c1 - c0 + (ends || w1 > max(w0, c1 * NW) ? 1 : 0);
  const int n = joined + (ends ? 0 : 1);
  if (n < 2) return;  // written by the main kernel
  auto row = [&](int i) -> int64_t {
    const int w = i < joined ? max(w0, (c0 + i) * NW) : w1;
    return (int64_t)(2 * w + (w == w0 ? 1 : 0)) * COLS + col;
  };
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, a.part_ml[row(i) * 2]);
#pragma unroll
  for (int off = 16; off; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  float L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = SPLIT ? warp : 0; i < n; i += SPLIT ? 8 : 1) {
    const int64_t at = row(i);
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
    const float4 o = *reinterpret_cast<const float4*>(a.part_o + at * DH + lane * 4);
    const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
    L = fmaf(ml.y, w, L);
    acc.x = fmaf(o.x, w, acc.x);
    acc.y = fmaf(o.y, w, acc.y);
    acc.z = fmaf(o.z, w, acc.z);
    acc.w = fmaf(o.w, w, acc.w);
  }
  if (SPLIT) {
    __shared__ float4 so[8][32];
    __shared__ float sl[8];
    so[warp][lane] = acc;
    if (lane == 0) sl[warp] = L;
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int w = 1; w < 8; ++w) {
      const float4 o = so[w][lane];
      acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
      L += sl[w];
    }
  }
  const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
  const __nv_bfloat162 h0 = __floats2bfloat162_rn(acc.x * inv, acc.y * inv);
  const __nv_bfloat162 h1 = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
  const int s = r / a.G;
  uint16_t* dst = a.out + ((int64_t)b * a.S + s) * a.ldo + (kvh * a.G + (r - s * a.G)) * DH;
  *reinterpret_cast<uint2*>(dst + lane * 4) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
}

constexpr int MAX_B = 4096;  // sequences a call: their page counts are planned in shared memory

constexpr int smem_bytes(int B) {
  return NW * (ST * BLOB + PAGE * 20) + NW * ST * 8 + NW * 24 + (NW * ST + 2 * (B + 1)) * 4;
}

// CTAs of one resident wave (with the shared memory of a batch of up to 64).
template <int NT>
int resident_ctas() {
  static int per_sm[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (!per_sm[dev]) {
    int nb = 0;
    if (mb::ensure_smem_attr(reinterpret_cast<const void*>(attn_kv4_kernel<NT>), smem_bytes(MAX_B)) ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&nb, attn_kv4_kernel<NT>, NW * 32,
                                                      smem_bytes(64)) != cudaSuccess || nb < 1)
      nb = 1;
    per_sm[dev] = nb;
  }
  return per_sm[dev] * mb::num_sms();
}

struct Plan {
  int nt, rt, grid;
  size_t bytes;
};

// Query rows of a kv head: S * G. Up to 8 take one column tile, more two (so
// that a page is unpacked once for 16 rows), in row tiles of 16.
Plan make_plan(int B, int S, int Hq, int Hkv, int max_pages) {
  Plan p;
  const int64_t rows = (int64_t)S * (Hq / Hkv);
  p.nt = rows <= 8 ? 1 : 2;
  p.rt = (int)((rows + p.nt * 8 - 1) / (p.nt * 8));
  const int64_t most = (int64_t)B * Hkv * p.rt * max_pages;
  const int res = p.nt == 1 ? resident_ctas<1>() : resident_ctas<2>();
  const int64_t ctas = (most * (1 + UNIT_COST) + NW - 1) / NW;
  p.grid = (int)(ctas < res ? ctas : res);
  p.bytes = ((size_t)2 * (B + 1) * sizeof(int) + 15) / 16 * 16 +
            (size_t)p.grid * NW * 2 * p.nt * 8 * (DH + 2) * sizeof(float);
  return p;
}

template <int NT>
int launch(const Args& a, int grid, cudaStream_t s) {
  const int smem = smem_bytes(a.B);
  int rc = mb::ensure_smem_attr(reinterpret_cast<const void*>(attn_kv4_kernel<NT>), smem_bytes(MAX_B));
  if (rc) return rc;
  MB_CUDA(mb::launch_pdl(attn_kv4_kernel<NT>, dim3(grid), dim3(NW * 32), smem, s, a));
  const int units = a.B * a.Hkv * a.RT;
  // few units are many partials each: 8 warps to a row
  if (units <= 2 * mb::num_sms())
    MB_CUDA(mb::launch_pdl(attn_kv4_combine_kernel<NT, true>, dim3(units, NT * 8), dim3(256), 0, s, a, grid * NW));
  else
    MB_CUDA(mb::launch_pdl(attn_kv4_combine_kernel<NT, false>, dim3(units, NT), dim3(256), 0, s, a, grid * NW));
  return MB_OK;
}

}  // namespace

extern "C" size_t mb_attention_kv4_workspace_bytes(int B, int S, int Hq, int Hkv, int max_pages) {
  if (B <= 0 || S <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv || max_pages <= 0) return 0;
  return make_plan(B, S, Hq, Hkv, max_pages).bytes;
}

extern "C" int mb_attention_kv4_bf16(const uint16_t* q, int64_t ldq, const uint8_t* cache,
                                     int num_pages, const int* block_table, int max_pages,
                                     const int* kv_len, const int* start_pos, int B, int S, int Hq,
                                     int Hkv, int Dh, float scale, uint16_t* out, int64_t ldo,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  MB_REQUIRE(Dh == DH, "attention: head_dim must be 128 (got %d)", Dh);
  MB_REQUIRE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0, "attention: Hq must be a multiple of Hkv");
  MB_REQUIRE(B >= 0 && S >= 0 && num_pages > 0 && max_pages > 0, "attention kv4: bad sizes");
  if (B == 0 || S == 0) return MB_OK;
  MB_REQUIRE(B <= MAX_B, "attention kv4: at most %d sequences a call", MAX_B);
  MB_REQUIRE(q && cache && block_table && kv_len && out, "attention kv4: null pointer");
  MB_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache) % 16 == 0 && ldq % 8 == 0 && ldo % 8 == 0,
             "attention kv4: q, out and the cache must be 16-byte aligned");
  const Plan p = make_plan(B, S, Hq, Hkv, max_pages);
  MB_REQUIRE((int64_t)B * Hkv * p.rt * ((int64_t)max_pages + UNIT_COST) < (1ll << 30) && (int64_t)max_pages * PAGE < (1ll << 30),
             "attention kv4: too many pages");
  MB_REQUIRE(workspace && workspace_bytes >= p.bytes && (uintptr_t)workspace % 16 == 0,
             "attention kv4: workspace of %zu bytes required, 16-byte aligned", p.bytes);
  uint32_t* status = mb::device_status_ptr();
  MB_REQUIRE(status, "attention kv4: no status word");
  Args a;
  a.q = q;
  a.cache = cache;
  a.table = block_table;
  a.kv_len = kv_len;
  a.start_pos = start_pos;
  a.out = out;
  a.plan = static_cast<int*>(workspace);
  a.part_o = reinterpret_cast<float*>(a.plan + (2 * (B + 1) + 3) / 4 * 4);
  a.part_ml = a.part_o + (size_t)p.grid * NW * 2 * p.nt * 8 * DH;
  a.status = status;
  a.ldq = ldq;
  a.ldo = ldo;
  a.num_pages = num_pages;
  a.max_pages = max_pages;
  a.B = B;
  a.S = S;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.RT = p.rt;
  a.scale_log2 = scale * 1.4426950408889634f;
  return p.nt == 1 ? launch<1>(a, p.grid, static_cast<cudaStream_t>(stream))
                   : launch<2>(a, p.grid, static_cast<cudaStream_t>(stream));
}
