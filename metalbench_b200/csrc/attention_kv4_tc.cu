// Attention of many query rows (pieces of prompts) over keys and values that
// were expanded from the 4-bit cache, on the 5th-generation tensor cores.
//
// The expanded pages (kv4_expand in kv4.cu) hold, in fp16, k 2^-x and v 2^-y
// with a power of two a page and kv head: [sequence][kv head][token][128].
// fp16 and not bf16, since a key rounded to bf16 (2^-8) costs more than the
// output's own rounding. With scores s in log2 units and a reference R of the
// row that is at least s + y of what it has seen, less 8,
//   p' = 2^(s + y - R + 6) <= 2^14,  out = sum p' v' / sum p' 2^-y
// (the 6 keeps terms down to 2^-30 of the largest out of fp16's underflow).
//
// One CTA = 128 query rows of one head (MMA M = 128), walking the keys in tiles
// of 128:
//   warp 0, 10  TMA producers of K and of V, so that neither waits for the
//               other's consumer.
//   warp 1      issues S_j = Q K_j^T into TMEM buffer j % 2 when S_{j-2} has
//               been read, warp 11 O += P_j V_j when P_j is there. (Eight MMAs
//               and their commits take a warp 750 cycles to issue; with one warp
//               for both that was the bottleneck.) P is an operand in TMEM, in
//               two buffers: in shared memory it would add 64 KB a tile to what
//               the port has to carry.
//   warps 2-9   softmax, a thread a row (TMEM lane): four warps take the even
//               tiles and four the odd ones, so that the exponentials of one
//               (900 cycles on the SFU) run while the other loads, masks and
//               stores; both halves of one tile at once took 2460 cycles a tile,
//               half of it with the SFU idle. First they take q, scale each row
//               by its own power of two and store it as fp16. A row's
//               reference goes from tile to tile through shared memory; it is
//               only raised when its maximum grows by more than 8, and only then
//               O is rescaled.
// TMEM: S0 | S1 | O (128 columns each) | P0 | P1 (64 each). Shared memory: rings
// of K and V, Q.
//
// Measured: 2 x 512 rows of 32 heads over 8192 keys of 8 in 151 us, 16 of them
// the expansion, 1850 cycles a tile (218 us and 2850 with two threads a row on
// one tile at a time and P in shared memory; 163 us with every exponential on the
// SFU, 1 in 4 or 1 in 16 on the FMA pipe 164 and 155). The MMAs take 1024 cycles
// of a tile, and the SFU 900; no unit is busy for more than 55 % of the time, loads
// are not waited for (leaving them out changes nothing): what is left is the chain
// S, softmax, P V of the two groups, which run in step since the one's reference
// waits for the other's maximum. (Taking turns on the SFU: 160 us; one warp for
// both products, or polling waits: more.)
//
// Few row tiles: `splits` CTAs share a row tile's keys and leave partials that
// a second kernel joins. Every wait is bounded and reports through the device
// status word; the teardown drains the MMA pipe and copies in flight. (All 168
// registers that 384 threads may have are used; the compiler spills 36 bytes.)
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace {

constexpr int TQ = 128, TK = 128, DHT = 128;
constexpr int CHUNK = 128 * 128;  // 64 elements of 128 rows, 128-byte swizzled
constexpr int TILE = 2 * CHUNK;
constexpr int KRING = 3, VRING = 3;
constexpr int OFF_V = KRING * TILE, OFF_Q = OFF_V + VRING * TILE, OFF_RED = OFF_Q + TILE;
constexpr int OFF_BAR = OFF_RED + 2 * TQ * 4;  // references [tile parity][row]
constexpr int NBAR = 2 * KRING + 2 * VRING + 21;
constexpr int SMEM_BYTES = 1024 + OFF_BAR + NBAR * 8 + 16;
constexpr int NSOFT = 256, THREADS = 128 + NSOFT;  // a group of TQ threads a tile
constexpr float RAISE = 8.f, BIAS = 6.f;

struct Args {
  CUtensorMap kmap, vmap;
  const uint16_t* q;
  int64_t ldq, ldo;
  uint16_t* out;
  const int* start_pos;  // null: not causal
  const int* kv_len;
  const int2* page_exp;  // [B][Hkv][pages]
  int max_len, pages, S, Hq, Hkv, G, n_qt, splits, tiles_per_split;
  float scale_log2;
  float* part_o;   // [B][Hq][S][splits][128]
  float* part_ml;  // [B][Hq][S][splits][2]
};

// D[tmem] (+)= A B[smem]^T, kind::f16, issued by the lane with `lead`. A predicate
// and no branch: descriptors stay warp-uniform, so that they are not moved from
// one lane's registers for every instruction.
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(mbd::smem_u32(bar)),
      "r"(lead)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 2^x for x < 64 on the FMA pipe (x below -126.5: 0, whose exponent field the last
// line makes of -127; a NaN stays one). Cody and
// Waite's reduction to f in [-1/2, 1/2], a polynomial of degree 4 there with the
// smallest largest relative error (2.6e-6, fitted by Lawson's reweighting).
__device__ __forceinline__ float ex2_fma(float x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(-127.f));
  const float whole = x + 12582912.f;  // 1.5 * 2^23: the nearest whole number in its low bits
  const float f = x - (whole - 12582912.f);
  const float y = fmaf(fmaf(fmaf(fmaf(0.009570101f, f, 0.05591786f), f, 0.24024744f), f, 0.6931218f), f, 0.9999993f);
  return y * __int_as_float((__float_as_int(whole) << 23) + 0x3F800000);
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bf2_of(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void pair_sync(int quad) {  // the two warps of a TMEM quadrant
  asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
}

__global__ void __launch_bounds__(THREADS, 1) attn_rows_kv4_kernel(const __grid_constant__ Args p, uint32_t* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(base + OFF_BAR);
  uint64_t *kfull = bars, *kempty = kfull + KRING, *vfull = kempty + KRING, *vempty = vfull + VRING;
  uint64_t *sfull = vempty + VRING, *sfree = sfull + 2, *qready = sfull + 4, *pfull = sfull + 5, *pfree = sfull + 7,
           *ofinal = sfull + 11, *sfinal = sfull + 12, *mready = sfull + 13;  // pfree [tile % 4], mready [quadrant][tile parity]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + NBAR);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* red = reinterpret_cast<float*>(base + OFF_RED);
  // (shuffles: what they return is known to be the same in a warp)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < KRING; ++i) {
      mbd::mbar_init(&kfull[i], 1);
      mbd::mbar_init(&kempty[i], 1);
    }
    for (int i = 0; i < VRING; ++i) {
      mbd::mbar_init(&vfull[i], 1);
      mbd::mbar_init(&vempty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbd::mbar_init(&sfull[i], 1);
      mbd::mbar_init(&sfree[i], TQ);
      mbd::mbar_init(&pfull[i], TQ);
    }
    mbd::mbar_init(qready, NSOFT);
    for (int i = 0; i < 4; ++i) mbd::mbar_init(&pfree[i], 1);
    for (int i = 0; i < 8; ++i) mbd::mbar_init(&mready[i], 32);
    mbd::mbar_init(ofinal, 1);
    mbd::mbar_init(sfinal, 1);
    *abort_flag = 0;
    mbd::fence_mbar_init();
    mbd::prefetch_tmap(&p.kmap);
    mbd::prefetch_tmap(&p.vmap);
  }
  if (warp == 1) mbd::tmem_alloc(tmem_slot, 512);
  __syncthreads();
  mbd::tc_fence_after();
  mbd::pdl_wait();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t tS = tmem, tO = tmem + 256, tP = tmem + 384;

  const int qt = p.n_qt - 1 - (int)blockIdx.x / p.splits;  // longest causal tiles first
  const int sp = (int)blockIdx.x % p.splits;
  const int h = blockIdx.y, b = blockIdx.z, kvh = h / p.G;
  const int L = max(0, min(p.kv_len[b], p.max_len));
  const bool causal = p.start_pos != nullptr;
  const int p0 = causal ? min(p.start_pos[b], L) : L;
  const int q_first = qt * TQ;
  const int kend = causal ? min(L, p0 + min(p.S - 1, q_first + TQ - 1) + 1) : L;
  const int jbase = sp * p.tiles_per_split;  // first key tile of this CTA
  const int n_tiles = __shfl_sync(
      0xffffffffu, max(0, min(kend > 0 ? (kend + TK - 1) / TK : 0, jbase + p.tiles_per_split) - jbase), 0);

  if (warp == 0 || warp == 10) {
    // ---------------- TMA producers ----------------
    if (lane == 0) {
      const CUtensorMap* map = warp ? &p.vmap : &p.kmap;
      uint64_t *full = warp ? vfull : kfull, *empty = warp ? vempty : kempty;
      uint8_t* ring = base + (warp ? OFF_V : 0);
      const int depth = warp ? VRING : KRING;
      const int row0 = ((b * p.Hkv + kvh) * p.pages) * kv4::PAGE + jbase * TK;
      int j = 0;
      for (; j < n_tiles; ++j) {
        const int st = j % depth;
        if (j >= depth && !mbd::mbar_wait(&empty[st], (j / depth - 1) & 1, status, MB_DEV_TIMEOUT_TMA, abort_flag)) break;
        mbd::mbar_expect_tx(&full[st], TILE);
        for (int c = 0; c < 2; ++c)
          mbd::tma_load_2d(ring + st * TILE + c * CHUNK, map, &full[st], c * 64, row0 + j * TK);
      }
      // no copy may still be landing in shared memory when the CTA exits
      for (int i = max(0, j - depth); i < j; ++i)
        mbd::mbar_wait(&full[i % depth], (i / depth) & 1, status, MB_DEV_TIMEOUT_TMA);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- S = Q K^T ----------------
    constexpr uint32_t idesc = mbd::make_idesc(0u, TQ, TK, 0, 0);
    const uint32_t lead = lane == 0;
    const uint64_t desc_q = mbd::sw128_desc(mbd::smem_u32(base + OFF_Q), 16, 1024);
    const uint64_t desc_k = mbd::sw128_desc(mbd::smem_u32(base), 16, 1024);
    bool ok = __all_sync(0xffffffffu, mbd::mbar_wait(qready, 0, status, MB_DEV_TIMEOUT_MMA, abort_flag));
    for (int j = 0; ok && j < n_tiles; ++j) {
      const int st = j % KRING, sb = j & 1;
      ok = __all_sync(0xffffffffu,
                      mbd::mbar_wait(&kfull[st], (j / KRING) & 1, status, MB_DEV_TIMEOUT_MMA, abort_flag) &&
                          mbd::mbar_wait(&sfree[sb], ((j >> 1) & 1) ^ 1, status, MB_DEV_TIMEOUT_MMA, abort_flag));
      if (!ok) break;
      mbd::tc_fence_after();
      const uint64_t dk = desc_k + (uint32_t)(st * (TILE >> 4));
#pragma unroll
      for (int kk = 0; kk < DHT / 16; ++kk) {  // K-major, two 64-element chunks; addresses count 16 bytes
        const uint32_t at = ((kk >> 2) * CHUNK + (kk & 3) * 32) >> 4;
        mma_ss(lead, tS + sb * TK, desc_q + at, dk + at, idesc, kk > 0);
      }
      commit(lead, &sfull[sb]);
      commit(lead, &kempty[st]);
    }
    commit(lead, sfinal);  // every MMA of this thread has completed: the drain before dealloc
    __syncwarp();
    mbd::mbar_wait(sfinal, 0, status, MB_DEV_TIMEOUT_MMA);
  } else if (warp == 11) {
    // ---------------- O += P V ----------------
    constexpr uint32_t idesc = mbd::make_idesc(0u, TQ, DHT, 0, 1);
    const uint32_t lead = lane == 0;
    const uint64_t desc_v = mbd::sw128_desc(mbd::smem_u32(base + OFF_V), CHUNK, 1024);
    bool ok = true;
    for (int j = 0; ok && j < n_tiles; ++j) {
      const int st = j % VRING;
      ok = __all_sync(0xffffffffu,
                      mbd::mbar_wait(&vfull[st], (j / VRING) & 1, status, MB_DEV_TIMEOUT_MMA, abort_flag) &&
                          mbd::mbar_wait(&pfull[j & 1], (j >> 1) & 1, status, MB_DEV_TIMEOUT_MMA, abort_flag));
      if (!ok) break;
      mbd::tc_fence_after();
      const uint64_t dv = desc_v + (uint32_t)(st * (TILE >> 4));
#pragma unroll
      for (int kk = 0; kk < TK / 16; ++kk)  // V tile [key][dim]: MN-major
        mma_ts(lead, tO, tP + (j & 1) * 64 + kk * 8, dv + kk * (2048 >> 4), idesc, j > 0 || kk > 0);
      commit(lead, &pfree[j & 3]);
      commit(lead, &vempty[st]);
    }
    commit(lead, ofinal);
    __syncwarp();
    mbd::mbar_wait(ofinal, 0, status, MB_DEV_TIMEOUT_MMA);
  } else {
    // ---------------- softmax + output (warps 2-9) ----------------
    const int quad = warp & 3;          // TMEM lane quadrant
    const int part = (warp - 2) >> 2;   // tiles part, part + 2, ...; dims [64 part, 64 part + 64)
    const int r = quad * 32 + lane;     // query row of the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const int row = q_first + r;
    const int c0 = part * 64;
    int4 pe_next = make_int4(0, 0, 0, 0);  // both pages' exponents
    const int4* pe = reinterpret_cast<const int4*>(p.page_exp + (int64_t)(b * p.Hkv + kvh) * p.pages) + jbase;
    if (part < n_tiles) pe_next = pe[part];
    // the row of q, scaled by a power of two, into TMEM
    float row_scale;
    {
      uint4 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = make_uint4(0, 0, 0, 0);
      if (row < p.S) {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + ((int64_t)b * p.S + row) * p.ldq + h * DHT + c0);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = src[i];
      }
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) most = fmaxf(most, fmaxf(fabsf(kv4::lo_bf(w[e])), fabsf(kv4::hi_bf(w[e]))));
      }
      red[part * TQ + r] = most;
      pair_sync(quad);
      const int e = kv4::fp16_exp(fmaxf(red[r], red[TQ + r]));
      const float f = kv4::pow2i(-e);
      row_scale = p.scale_log2 * kv4::pow2i(e);
      uint8_t* dst = base + OFF_Q + part * CHUNK + r * 128;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = half2_of(kv4::lo_bf(v[k]) * f, kv4::hi_bf(v[k]) * f);
        *reinterpret_cast<uint4*>(dst + ((i ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      mbd::fence_proxy_async();
      mbd::mbar_arrive(qready);
      pair_sync(quad);  // the maxima have been read
    }
    float m = -INFINITY, l = 0.f;  // reference of this thread's last tile, its terms' sum
    bool ok = true;
    for (int j = part; j < n_tiles; j += 2) {
      // clamped: 0 * inf and -inf * 0 must not meet
      const float scl[2] = {fminf(fmaxf(row_scale * kv4::pow2i(pe_next.x), 1e-37f), 3e38f),
                            fminf(fmaxf(row_scale * kv4::pow2i(pe_next.z), 1e-37f), 3e38f)};
      const float vexp[2] = {(float)pe_next.y, (float)pe_next.w};
      const float vinv[2] = {kv4::pow2i(-pe_next.y), kv4::pow2i(-pe_next.w)};
      if (j + 2 < n_tiles) pe_next = pe[j + 2];
      ok = __all_sync(0xffffffffu,
                      mbd::mbar_wait(&sfull[part], (j >> 1) & 1, status, MB_DEV_TIMEOUT_EPI, abort_flag));
      if (!ok) break;
      uint32_t s[8][16];
      mbd::tc_fence_after();
#pragma unroll
      for (int c = 0; c < 8; ++c) mbd::tmem_ld16(tS + part * TK + lane_off + c * 16, s[c]);
      mbd::tmem_ld_wait();
      mbd::tc_fence_before();
      mbd::mbar_arrive(&sfree[part]);
      // keys [0, lim] of this tile are seen
      const int lim = (causal ? min(L - 1, p0 + row) : L - 1) - (jbase + j) * TK;
      if (lim < TK - 1) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (c * 16 + e > lim) s[c][e] = __float_as_uint(-INFINITY);
      }
      float mt = -INFINITY;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(s[4 * g + c][e]));
        mt = fmaxf(mt, fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), scl[g], vexp[g]));
      }
      // the reference up to here, this tile's, and on to the next one
      float before = -INFINITY;
      if (j > 0) {
        ok = __all_sync(0xffffffffu, mbd::mbar_wait(&mready[quad * 2 + (part ^ 1)], ((j - 1) >> 1) & 1, status,
                                                    MB_DEV_TIMEOUT_EPI, abort_flag));
        if (!ok) break;
        before = red[(part ^ 1) * TQ + r];
      }
      red[part * TQ + r] = mt > before + RAISE ? mt : before;
      mbd::mbar_arrive(&mready[quad * 2 + part]);
      // read back, so that the exponentials are not scheduled before the arrival
      const float now = *const_cast<volatile float*>(red + part * TQ + r);
      const bool rescale = now != before && before != -INFINITY;
      const float mu = now == -INFINITY ? 0.f : now;
      float sum = 0.f;
      uint32_t w[64];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float off = vexp[g] + BIAS - mu;
        float sm[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float a = ex2(fmaf(__uint_as_float(s[4 * g + (i >> 3)][(2 * i) & 15]), scl[g], off));
          const float y = fmaf(__uint_as_float(s[4 * g + (i >> 3)][(2 * i + 1) & 15]), scl[g], off);
          const float c = (i & 3) == 1 ? ex2_fma(y) : ex2(y);  // 1 in 8 on the FMA pipe
          sm[(2 * i) & 3] += a;
          sm[(2 * i + 1) & 3] += c;
          w[32 * g + i] = half2_of(a, c);
        }
        sum = fmaf((sm[0] + sm[1]) + (sm[2] + sm[3]), vinv[g], sum);
      }
      l = m == now ? l + sum : fmaf(l, exp2f(m - now), sum);
      m = now;
      // this group's P is free once P_{j-2} V_{j-2} has completed; O may be
      // rescaled once P_{j-1} V_{j-1} has. (Four barriers, so that a parity is
      // not that of two phases ago: P_{j-5} V_{j-5} was waited for by the other
      // group before it passed on tile j - 1's reference, P_{j-6} V_{j-6} by this.)
      const bool any = __any_sync(0xffffffffu, rescale);
      if (j > 1)
        ok = __all_sync(0xffffffffu,
                        mbd::mbar_wait(&pfree[(j - 2) & 3], ((j - 2) >> 2) & 1, status, MB_DEV_TIMEOUT_EPI, abort_flag));
      if (any && ok)
        ok = __all_sync(0xffffffffu, mbd::mbar_wait(&pfree[(j - 1) & 3], ((j - 1) >> 2) & 1, status,
                                                    MB_DEV_TIMEOUT_EPI, abort_flag));
      if (!ok) break;
      mbd::tc_fence_after();
      if (any) {
        const float alpha = rescale ? exp2f(before - now) : 1.f;
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
          uint32_t o[16];
          mbd::tmem_ld16(tO + lane_off + c * 16, o);
          mbd::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
          tmem_st16(tO + lane_off + c * 16, o);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_st16(tP + part * 64 + lane_off + c * 16, w + c * 16);
      tmem_st_wait();
      mbd::tc_fence_before();
      mbd::mbar_arrive(&pfull[part]);
    }
    const bool fin =
        ok && __all_sync(0xffffffffu, mbd::mbar_wait(ofinal, 0, status, MB_DEV_TIMEOUT_EPI, abort_flag));
    // both groups' sums, under the last reference, which is O's
    // (in the quadrant's own rows of Q: every S has been made, and with no tile
    // the other quadrants may still be storing theirs)
    float2* ends = reinterpret_cast<float2*>(base + OFF_Q + quad * 4096) + lane;
    ends[part * 32] = make_float2(m, l);
    pair_sync(quad);
    const float2 other = ends[(part ^ 1) * 32];
    const float mine = m;
    m = fmaxf(mine, other.x);
    const float lt = (mine == -INFINITY ? l : l * exp2f(mine - m)) +
                     (other.x == -INFINITY ? other.y : other.y * exp2f(other.x - m));
    if (fin) mbd::tc_fence_after();
    if (fin && p.splits > 1) {
      // partial of this key split: unnormalised O, reference (log2 units), row sum
      const int64_t at = (((int64_t)b * p.Hq + h) * p.S + row) * p.splits + sp;
      float4* dst = reinterpret_cast<float4*>(p.part_o + at * DHT + c0);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[16];
        mbd::tmem_ld16(tO + lane_off + c0 + c * 16, o);
        mbd::tmem_ld_wait();
        if (row < p.S)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            dst[4 * c + e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                         __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
      }
      // a NaN that a row sees stays one; with no tile at all O was never written
      if (row < p.S && part == 0)
        *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(lt != lt ? 0.f : m, lt);
    } else if (fin) {
      const float inv = lt != 0.f ? 1.f / lt : 0.f;
      const uint32_t keep = lt != 0.f ? 0xFFFFFFFFu : 0u;  // no visible key: O may never have been written
      uint4* dst = reinterpret_cast<uint4*>(p.out + ((int64_t)b * p.S + row) * p.ldo + h * DHT + c0);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[16];
        mbd::tmem_ld16(tO + lane_off + c0 + c * 16, o);
        mbd::tmem_ld_wait();
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(o[e] & keep) * inv;
        if (row < p.S) {
          dst[2 * c] = make_uint4(bf2_of(v[0], v[1]), bf2_of(v[2], v[3]), bf2_of(v[4], v[5]), bf2_of(v[6], v[7]));
          dst[2 * c + 1] =
              make_uint4(bf2_of(v[8], v[9]), bf2_of(v[10], v[11]), bf2_of(v[12], v[13]), bf2_of(v[14], v[15]));
        }
      }
    }
  }
  mbd::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    mbd::tc_fence_after();
    mbd::tmem_dealloc(tmem, 512);
  }
}

// out = sum_s O_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), M = max m_s: a warp a row
__global__ void __launch_bounds__(256) attn_rows_kv4_join_kernel(const Args p, int64_t rows) {
  mbd::pdl_wait();
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);  // (b Hq + h) S + row
  const int lane = threadIdx.x & 31;
  if (id >= rows) return;
  const int64_t bh = id / p.S, b = bh / p.Hq;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + id * p.splits;
  const float4* po = reinterpret_cast<const float4*>(p.part_o + id * p.splits * DHT) + lane;
  float M = -INFINITY, l = 0.f;
  for (int s = 0; s < p.splits; ++s) M = fmaxf(M, ml[s].x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < p.splits; ++s) {
    if (ml[s].x == -INFINITY) continue;  // no visible key: O may never have been written
    const float w = exp2f(ml[s].x - M);
    const float4 v = po[s * (DHT / 4)];
    l = fmaf(ml[s].y, w, l);
    o.x = fmaf(v.x, w, o.x), o.y = fmaf(v.y, w, o.y), o.z = fmaf(v.z, w, o.z), o.w = fmaf(v.w, w, o.w);
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  uint16_t* dst = p.out + (b * p.S + id % p.S) * p.ldo + (bh % p.Hq) * DHT + lane * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(bf2_of(o.x * inv, o.y * inv), bf2_of(o.z * inv, o.w * inv));
}

}  // namespace

namespace mb {

int attention_rows_kv4(const Kv4Rows& a, cudaStream_t stream) {
  Args p;
  const auto half = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const auto sw = CU_TENSOR_MAP_SWIZZLE_128B;
  const uint64_t rows = (uint64_t)a.B * a.Hkv * a.x.pages * kv4::PAGE;
  int rc = make_tmap_2d(&p.kmap, a.x.k, half, 2, DHT, rows, DHT * 2, 64, TK, sw);
  if (!rc) rc = make_tmap_2d(&p.vmap, a.x.v, half, 2, DHT, rows, DHT * 2, 64, TK, sw);
  if (!rc) rc = ensure_smem_attr(reinterpret_cast<const void*>(attn_rows_kv4_kernel), SMEM_BYTES);
  if (rc) return rc;
  p.q = a.q;
  p.ldq = a.ldq;
  p.out = a.out;
  p.ldo = a.ldo;
  p.start_pos = a.start_pos;
  p.kv_len = a.kv_len;
  p.page_exp = a.x.page_exp;
  p.max_len = a.max_len;
  p.pages = a.x.pages;
  p.S = a.S;
  p.Hq = a.Hq;
  p.Hkv = a.Hkv;
  p.G = a.Hq / a.Hkv;
  p.n_qt = (a.S + TQ - 1) / TQ;
  p.splits = a.splits;
  p.tiles_per_split = (a.x.pages / 2 + a.splits - 1) / a.splits;
  p.scale_log2 = 1.4426950408889634f * a.scale;
  p.part_o = a.part;
  p.part_ml = a.part ? a.part + (size_t)a.B * a.S * a.Hq * a.splits * DHT : nullptr;
  uint32_t* status = device_status_ptr();
  MB_REQUIRE(status, "attention kv4: no status word");
  MB_CUDA(launch_pdl(attn_rows_kv4_kernel, dim3(p.n_qt * p.splits, a.Hq, a.B), dim3(THREADS), SMEM_BYTES, stream, p,
                     status));
  if (p.splits > 1) {
    const int64_t n = (int64_t)a.B * a.Hq * a.S;
    MB_CUDA(launch_pdl(attn_rows_kv4_join_kernel, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, stream, p, n));
  }
  return MB_OK;
}

}  // namespace mb
