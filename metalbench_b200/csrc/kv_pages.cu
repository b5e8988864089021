// Page operations of a paged KV cache: growing sequences, forking and freeing
// them, and compacting the pool. They work on the block table, the sequence
// lengths and a use count per page, all in device memory, and on any number of
// page pools (the keys and values of every layer, in 4 bits or bf16), whose
// pages are moved as bytes. Nothing returns to the host, so a decode loop that
// calls them can be captured in a CUDA graph.
//
// Rules. A sequence of `len` tokens owns the first ceil(len / 64) entries of
// its table row; what stands behind them is left alone. A page may be shared
// by sequences only while it is full; refs[p] counts the rows that name it, and
// 0 means free. New pages are the lowest-numbered free ones, given out in row
// order, so that results do not depend on timing. A call that cannot be served
// (too few free pages, an entry or a parent out of range) changes nothing.
//
// The bookkeeping of a call is one launch of one CTA or, for larger tables, one
// 8-CTA cluster: its 32 or 128 warps count (ballots over contiguous segments),
// meet at a barrier, read all counts and place what they counted. The pages' bytes move in a
// second launch over all SMs, bound by HBM.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace {

constexpr int PAGE = 64;
// CTAs of the bookkeeping's cluster and threads of each
template <int CTAS> constexpr int THREADS = CTAS == 1 ? 1024 : 512;
template <int CTAS> constexpr int WARPS = CTAS * THREADS<CTAS> / 32;
constexpr int MOST_WARPS = WARPS<8>;  // 128
constexpr int MAX_POOLS = 64;

struct Pools {
  uint8_t* base[MAX_POOLS];
  int64_t bytes[MAX_POOLS];  // one page
  int32_t piece[MAX_POOLS];  // bytes moved at once: a page in equal parts
  int n;
};

// Caller's workspace, as the kernels see it.
struct Work {
  int* cnt;     // [4][warps]
  int* head;    // [1] moves to make
  int2* moves;  // [max moves] from, to
  int* ids;     // free pages found / holes
  int* ids2;    // moved pages
  int* row;     // [B] per-row number
  int* row2;    // [B]
  int* stage;   // [B][max_pages] a fork's new rows
};

struct Meta {
  int* table;
  int* len;
  int* refs;
  int B, max_pages, num_pages;
  int* status;
  Work w;
};

template <int CTAS>
__device__ __forceinline__ void sync_all() {
  if (CTAS == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
template <int CTAS>
__device__ __forceinline__ int warp_id() { return (blockIdx.x * THREADS<CTAS> + threadIdx.x) >> 5; }

// This warp's contiguous part of n things: a multiple of 32.
template <int CTAS>
__device__ __forceinline__ void segment(int n, int& from, int& to) {
  const int size = ((n + WARPS<CTAS> - 1) / WARPS<CTAS> + 31) / 32 * 32;
  const int64_t f = (int64_t)warp_id<CTAS>() * size;
  from = (int)(f < n ? f : n);
  to = (int)(f + size < n ? f + size : n);
}

// Sum of one row of counts over the warps before this one, and over all.
template <int CTAS>
__device__ __forceinline__ int2 before_and_all(const int* cnt) {
  const int lane = threadIdx.x & 31, me = warp_id<CTAS>();
  int b = 0, a = 0;
#pragma unroll
  for (int i = 0; i < WARPS<CTAS> / 32; ++i) {
    const int v = __ldcg(cnt + i * 32 + lane);
    a += v;
    if (i * 32 + lane < me) b += v;
  }
  return make_int2(__reduce_add_sync(0xffffffffu, b), __reduce_add_sync(0xffffffffu, a));
}

__device__ __forceinline__ int pages_of(int len) { return (len + PAGE - 1) / PAGE; }

// How many pages of this warp's part of the pool are free / in use.
template <bool FREE>
__device__ int count_pages(const int* refs, int from, int to) {
  const int lane = threadIdx.x & 31;
  int n = 0;
#pragma unroll 4
  for (int i = from; i < to; i += 32) {
    const int p = i + lane;
    n += __popc(__ballot_sync(0xffffffffu, p < to && (FREE ? refs[p] == 0 : refs[p] > 0)));
  }
  return n;
}

// The first `want` free pages of the pool, in order, into ids.
__device__ void list_free(const int* refs, int from, int to, int rank, int want, int* ids) {
  const int lane = threadIdx.x & 31;
  for (int i = from; i < to && rank < want; i += 32) {
    const int p = i + lane;
    const bool is_free = p < to && refs[p] == 0;
    const uint32_t m = __ballot_sync(0xffffffffu, is_free);
    const int r = rank + __popc(m & ((1u << lane) - 1));
    if (is_free && r < want) ids[r] = p;
    rank += __popc(m);
  }
}

// ---------------------------------------------------------------------------
template <int CTAS>
__global__ void __cluster_dims__(CTAS) __launch_bounds__(THREADS<CTAS>)
    kv_extend_kernel(const Meta m, const int* add, int* __restrict__ start) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int lane = threadIdx.x & 31, me = warp_id<CTAS>();
  int r0, r1, p0, p1;
  segment<CTAS>(m.B, r0, r1);
  segment<CTAS>(m.num_pages, p0, p1);
  const int most = m.max_pages * PAGE;
  int need = 0, bad = 0;
  for (int i = r0; i < r1; i += 32) {
    const int b = i + lane;
    if (b < r1) {
      const int l = m.len[b], n = add[b];
      if (l < 0 || n < 0 || l > most || n > most - l) bad = 1;
      else need += pages_of(l + n) - pages_of(l);
    }
  }
  need = __reduce_add_sync(0xffffffffu, need);
  bad = __any_sync(0xffffffffu, bad);
  const int nfree = count_pages<true>(m.refs, p0, p1);
  if (lane == 0) {
    m.w.cnt[me] = need;
    m.w.cnt[WARPS<CTAS> + me] = nfree;
    m.w.cnt[2 * WARPS<CTAS> + me] = bad;
  }
  sync_all<CTAS>();
  const int2 nd = before_and_all<CTAS>(m.w.cnt), fr = before_and_all<CTAS>(m.w.cnt + WARPS<CTAS>);
  const bool any_bad = before_and_all<CTAS>(m.w.cnt + 2 * WARPS<CTAS>).y != 0;
  const int lack = nd.y > fr.y ? nd.y - fr.y : 0;
  const bool go = !any_bad && !lack;
  if (me == 0 && lane == 0) *m.status = any_bad ? -1 : lack;
  if (go) {
    list_free(m.refs, p0, p1, fr.x, nd.y, m.w.ids);
    int run = nd.x;  // pages given to rows before this one
    for (int i = r0; i < r1; i += 32) {
      const int b = i + lane;
      int n = 0;
      if (b < r1) n = pages_of(m.len[b] + add[b]) - pages_of(m.len[b]);
      int inc = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += y;
      }
      if (b < r1) m.w.row[b] = run + inc - n;
      run += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  sync_all<CTAS>();
  for (int b = me; b < m.B; b += WARPS<CTAS>) {  // one warp a row
    const int l = m.len[b], n = add[b];
    __syncwarp();  // every lane has read the lengths before they change (add may be len)
    if (lane == 0) start[b] = l;
    if (!go) continue;
    const int old = pages_of(l), k = pages_of(l + n) - old;
    const int off = __ldcg(m.w.row + b);
    for (int i = lane; i < k; i += 32) {
      const int p = __ldcg(m.w.ids + off + i);
      m.table[(int64_t)b * m.max_pages + old + i] = p;
      m.refs[p] = 1;
    }
    if (lane == 0) m.len[b] = l + n;
  }
}

// ---------------------------------------------------------------------------
template <int CTAS>
__global__ void __cluster_dims__(CTAS) __launch_bounds__(THREADS<CTAS>)
    kv_fork_kernel(const Meta m, const int* __restrict__ parent) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int lane = threadIdx.x & 31, me = warp_id<CTAS>();
  int r0, r1, p0, p1;
  segment<CTAS>(m.B, r0, r1);
  segment<CTAS>(m.num_pages, p0, p1);
  const int most = m.max_pages * PAGE;
  auto bad_len = [&](int l) { return l < 0 || l > most; };
  // ---- count: tail pages to copy, free pages; stage the parents' rows ----
  int tails = 0, bad = 0;
  for (int i = r0; i < r1; i += 32) {
    const int b = i + lane;
    int tail = 0;
    if (b < r1) {
      const int p = parent[b];
      if (p < -1 || p >= m.B || bad_len(m.len[b])) {
        bad = 1;
      } else {
        const int l = p < 0 ? 0 : m.len[p];
        if (bad_len(l)) bad = 1;
        else tail = p != b && l % PAGE != 0;
        m.w.row2[b] = l;
      }
    }
    tails += __popc(__ballot_sync(0xffffffffu, tail));
  }
  const int nfree = count_pages<true>(m.refs, p0, p1);
  for (int b = me; b < m.B; b += WARPS<CTAS>) {
    const int p = parent[b];
    if (p == b || p < -1 || p >= m.B) continue;
    const int old = pages_of(m.len[b]), now = p < 0 ? 0 : pages_of(m.len[p]);
    if (old < 0 || old > m.max_pages || now < 0 || now > m.max_pages) continue;  // bad, seen above
    for (int c = lane; c < old; c += 32)
      if ((unsigned)m.table[(int64_t)b * m.max_pages + c] >= (unsigned)m.num_pages) bad = 1;
    for (int c = lane; c < now; c += 32) {
      const int e = m.table[(int64_t)p * m.max_pages + c];
      if ((unsigned)e >= (unsigned)m.num_pages) bad = 1;
      m.w.stage[(int64_t)b * m.max_pages + c] = e;
    }
  }
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    m.w.cnt[me] = tails;
    m.w.cnt[WARPS<CTAS> + me] = nfree;
    m.w.cnt[2 * WARPS<CTAS> + me] = bad;
  }
  sync_all<CTAS>();
  const int2 tl = before_and_all<CTAS>(m.w.cnt), fr = before_and_all<CTAS>(m.w.cnt + WARPS<CTAS>);
  const bool any_bad = before_and_all<CTAS>(m.w.cnt + 2 * WARPS<CTAS>).y != 0;
  const int lack = tl.y > fr.y ? tl.y - fr.y : 0;
  const bool go = !any_bad && !lack;
  if (me == 0 && lane == 0) {
    *m.status = any_bad ? -1 : lack;
    *m.w.head = go ? tl.y : 0;
  }
  if (go) {
    list_free(m.refs, p0, p1, fr.x, tl.y, m.w.ids);
    int rank = tl.x;
    for (int i = r0; i < r1; i += 32) {
      const int b = i + lane;
      const bool tail = b < r1 && parent[b] >= 0 && parent[b] != b && m.len[parent[b]] % PAGE != 0;
      const uint32_t mask = __ballot_sync(0xffffffffu, tail);
      if (b < r1) m.w.row[b] = tail ? rank + __popc(mask & ((1u << lane) - 1)) : -1;
      rank += __popc(mask);
    }
  }
  sync_all<CTAS>();
  if (!go) return;
  // ---- place: uses, rows, lengths, and the list of pages to copy ----
  for (int b = me; b < m.B; b += WARPS<CTAS>) {
    if (parent[b] == b) continue;
    const int l = __ldcg(m.w.row2 + b), tail = __ldcg(m.w.row + b);
    const int old = pages_of(m.len[b]), now = pages_of(l);
    __syncwarp();
    int* row = m.table + (int64_t)b * m.max_pages;
    for (int c = lane; c < max(old, now); c += 32) {
      if (c < old) atomicSub(m.refs + row[c], 1);
      if (c < now) {
        int e = __ldcg(m.w.stage + (int64_t)b * m.max_pages + c);
        if (tail >= 0 && c == now - 1) {
          const int to = __ldcg(m.w.ids + tail);
          m.w.moves[tail] = make_int2(e, to);
          e = to;
        }
        atomicAdd(m.refs + e, 1);
        row[c] = e;
      }
    }
    if (lane == 0) m.len[b] = l;
  }
}

// ---------------------------------------------------------------------------
template <int CTAS>
__global__ void __cluster_dims__(CTAS) __launch_bounds__(THREADS<CTAS>)
    kv_compact_kernel(const Meta m, int* __restrict__ remap) {
  mbd::pdl_trigger();
  mbd::pdl_wait();
  const int lane = threadIdx.x & 31, me = warp_id<CTAS>();
  int p0, p1;
  segment<CTAS>(m.num_pages, p0, p1);
  const int live_here = count_pages<false>(m.refs, p0, p1);
  int bad = 0;
  for (int b = me; b < m.B; b += WARPS<CTAS>) {
    const int l = m.len[b];
    if (l < 0 || l > m.max_pages * PAGE) {
      bad = 1;
      continue;
    }
    for (int c = lane; c < pages_of(l); c += 32) {
      const int e = m.table[(int64_t)b * m.max_pages + c];
      if ((unsigned)e >= (unsigned)m.num_pages || m.refs[e] <= 0) bad = 1;
    }
  }
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) {
    m.w.cnt[me] = live_here;
    m.w.cnt[WARPS<CTAS> + me] = bad;
  }
  sync_all<CTAS>();
  const int2 lv = before_and_all<CTAS>(m.w.cnt);
  const bool go = before_and_all<CTAS>(m.w.cnt + WARPS<CTAS>).y == 0;
  const int live = lv.y;
  if (me == 0 && lane == 0) *m.status = go ? live : -1;
  // free pages below `live` are holes, pages in use from `live` on are moved
  // into them, in order; as many of the one as of the other
  int rank = lv.x, below = 0;
  for (int i = p0; i < p1; i += 32) {
    const int p = i + lane;
    const bool use = p < p1 && m.refs[p] > 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, use);
    const int lb = rank + __popc(mask & ((1u << lane) - 1));  // pages in use before p
    if (p < p1) {
      if (!go) remap[p] = p;
      else if (!use) remap[p] = -1;
      else if (p < live) remap[p] = p;
      if (go && !use && p < live) m.w.ids[p - lb] = p;
      if (go && use && p >= live) m.w.ids2[live - 1 - lb] = p;  // counted from the last one
    }
    below += __popc(__ballot_sync(0xffffffffu, use && p < live));
    rank += __popc(mask);
  }
  if (lane == 0) m.w.cnt[2 * WARPS<CTAS> + me] = below;
  sync_all<CTAS>();
  const int n = live - before_and_all<CTAS>(m.w.cnt + 2 * WARPS<CTAS>).y;
  if (me == 0 && lane == 0) *m.w.head = go ? n : 0;
  if (go)
    for (int i = me * 32 + lane; i < n; i += WARPS<CTAS> * 32) {
      const int from = __ldcg(m.w.ids2 + n - 1 - i), to = __ldcg(m.w.ids + i);
      m.w.moves[i] = make_int2(from, to);
      remap[from] = to;
      m.refs[to] = m.refs[from];
      m.refs[from] = 0;
    }
  sync_all<CTAS>();
  if (!go) return;
  for (int b = me; b < m.B; b += WARPS<CTAS>)
    for (int c = lane; c < pages_of(m.len[b]); c += 32) {
      int* e = m.table + (int64_t)b * m.max_pages + c;
      *e = __ldcg(remap + *e);
    }
}

// ---------------------------------------------------------------------------
// The listed pages of every pool: no page is both read and written (a fork
// writes free pages, a compaction moves pages above `live` below it). A CTA is
// one warp, whose first lane moves pieces of up to 16 KB through a ring in
// shared memory with bulk copies in both directions: no registers and no
// instructions a byte, and pieces on their way in while others go out. (2036
// pages of 4 pools of 68 KiB, 1.13 GB read and written: 193 us with 16-byte loads
// and stores by 256 threads and 8 CTAs an SM, 177 us here, 6.4 TB/s. Smaller pages
// cost as much a piece and have not been measured.)
constexpr int PIECE = 16384;
constexpr int RING = 6, LAG = 2;  // pieces; a piece's place is filled again LAG pieces after it went out
constexpr int COPY_SMEM = RING * PIECE + RING * 8;

__global__ void __launch_bounds__(32)
    kv_copy_kernel(const __grid_constant__ Pools pools, const int* __restrict__ head,
                   const int2* __restrict__ moves, int chunks, uint32_t* status) {
  extern __shared__ __align__(128) uint8_t ring[];
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + RING * PIECE);
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) mbd::mbar_init(full + i, 1);
    mbd::fence_mbar_init();
  }
  mbd::pdl_trigger();
  mbd::pdl_wait();
  if (threadIdx.x) return;
  const int64_t total = (int64_t)*head * chunks * pools.n;
  const int64_t mine = total > blockIdx.x ? (total - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  uint8_t* to[RING];
  uint32_t size[RING];
  auto load = [&](int64_t k, int st) {  // the k-th piece of this CTA
    const int64_t i = blockIdx.x + k * gridDim.x;
    int64_t rest, move;  // (piece within rest, then pool within move); short divisions where they do
    if (total <= 0xFFFFFFFFll) rest = (uint32_t)i / (uint32_t)chunks, move = (uint32_t)rest / (uint32_t)pools.n;
    else rest = i / chunks, move = rest / pools.n;
    const int pool = (int)(rest - move * pools.n);
    const int64_t bytes = pools.bytes[pool], piece = pools.piece[pool], at = (i - rest * chunks) * piece;
    const int2 mv = moves[move];
    size[st] = at < bytes ? (uint32_t)(bytes - at < piece ? bytes - at : piece) : 0;
    to[st] = pools.base[pool] + mv.y * bytes + at;
    if (size[st]) {
      mbd::mbar_expect_tx(full + st, size[st]);
      mbd::bulk_load(ring + st * PIECE, pools.base[pool] + mv.x * bytes + at, size[st], full + st);
    } else {
      mbd::mbar_arrive(full + st);
    }
  };
#pragma unroll
  for (int st = 0; st < RING; ++st)
    if (st < mine) load(st, st);
  bool ok = true;
  int64_t k = 0;
  for (uint32_t phase = 0; k < mine && ok; phase ^= 1) {
#pragma unroll
    for (int st = 0; st < RING; ++st, ++k) {
      if (k >= mine || !ok) break;
      ok = mbd::mbar_wait(full + st, phase, status, MB_DEV_TIMEOUT_TMA);
      if (!ok) break;
      if (size[st])
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to[st]),
                     "r"(mbd::smem_u32(ring + st * PIECE)), "r"(size[st])
                     : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      // the piece that went out LAG ago has been read: its place is free
      if (k >= LAG && k - LAG + RING < mine) {
        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LAG) : "memory");
        load(k - LAG + RING, (st + RING - LAG) % RING);
      }
    }
  }
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  if (!ok)  // a copy never came: wait (bounded) for the others before the memory goes
    for (int st = 0; st < RING; ++st) mbd::mbar_wait(full + st, 0, nullptr, 0, nullptr, 1000000);
}

size_t align16(size_t x) { return (x + 15) / 16 * 16; }

// Workspace of any of the page calls: counts, move list, page lists, rows.
size_t work_layout(int B, int max_pages, int num_pages, bool stage, Work* w, uint8_t* p) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    uint8_t* r = p + at;
    at += align16(bytes);
    return r;
  };
  int* cnt = reinterpret_cast<int*>(take(4 * MOST_WARPS * sizeof(int)));
  int* head = reinterpret_cast<int*>(take(sizeof(int)));
  int2* moves = reinterpret_cast<int2*>(take((size_t)num_pages * sizeof(int2)));
  int* ids = reinterpret_cast<int*>(take((size_t)num_pages * sizeof(int)));
  int* ids2 = reinterpret_cast<int*>(take((size_t)num_pages * sizeof(int)));
  int* row = reinterpret_cast<int*>(take((size_t)B * sizeof(int)));
  int* row2 = reinterpret_cast<int*>(take((size_t)B * sizeof(int)));
  int* st = reinterpret_cast<int*>(take(stage ? (size_t)B * max_pages * sizeof(int) : 0));
  if (w) *w = Work{cnt, head, moves, ids, ids2, row, row2, st};
  return at;
}

int fill_meta(const char* what, Meta* m, int* table, int* len, int* refs, int B, int max_pages,
              int num_pages, int* status, bool stage, void* ws, size_t ws_bytes) {
  MB_REQUIRE(B >= 0 && max_pages > 0 && num_pages >= 0 && max_pages < (1 << 24), "%s: bad sizes", what);
  MB_REQUIRE((table && len) || B == 0, "%s: null pointer", what);
  MB_REQUIRE(refs && status, "%s: null pointer", what);
  MB_REQUIRE((int64_t)B * max_pages < (1ll << 31), "%s: block table too large", what);
  const size_t need = work_layout(B, max_pages, num_pages, stage, nullptr, nullptr);
  MB_REQUIRE(ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0,
             "%s: workspace of %zu bytes required, 16-byte aligned", what, need);
  *m = Meta{table, len, refs, B, max_pages, num_pages, status, {}};
  work_layout(B, max_pages, num_pages, stage, &m->w, static_cast<uint8_t*>(ws));
  return MB_OK;
}

int copy_pages(const char* what, void* const* pools, const int64_t* bytes, int npools, const Work& w,
               int64_t most_moves, cudaStream_t s) {
  for (int at = 0; at < npools; at += MAX_POOLS) {
    Pools p = {};
    p.n = npools - at < MAX_POOLS ? npools - at : MAX_POOLS;
    int64_t big = 0;
    for (int i = 0; i < p.n; ++i) {
      p.base[i] = static_cast<uint8_t*>(pools[at + i]);
      p.bytes[i] = bytes[at + i];
      big = bytes[at + i] > big ? bytes[at + i] : big;
    }
    const int chunks = (int)((big + PIECE - 1) / PIECE);
    for (int i = 0; i < p.n; ++i) p.piece[i] = (int32_t)(((p.bytes[i] + chunks - 1) / chunks + 15) / 16 * 16);
    const int64_t all = most_moves * chunks * p.n, wave = (int64_t)mb::num_sms() * 2;
    if (all == 0) continue;
    uint32_t* status = mb::device_status_ptr();
    MB_REQUIRE(status, "%s: no status word", what);
    const int rc = mb::ensure_smem_attr(reinterpret_cast<const void*>(kv_copy_kernel), COPY_SMEM);
    if (rc) return rc;
    MB_CUDA(mb::launch_pdl(kv_copy_kernel, dim3((unsigned)(all < wave ? all : wave)), dim3(32), COPY_SMEM, s,
                           p, w.head, w.moves, chunks, status));
  }
  return MB_OK;
}

int check_pools(const char* what, void* const* pools, const int64_t* bytes, int npools) {
  MB_REQUIRE(npools >= 0 && (npools == 0 || (pools && bytes)), "%s: bad pools", what);
  for (int i = 0; i < npools; ++i)
    MB_REQUIRE(pools[i] && (uintptr_t)pools[i] % 16 == 0 && bytes[i] > 0 && bytes[i] % 16 == 0 &&
                   bytes[i] < (1ll << 40),
               "%s: pools must be 16-byte aligned and their pages a multiple of 16 bytes", what);
  return MB_OK;
}

}  // namespace

namespace {
// One CTA does the bookkeeping of a small table and pool sooner: a block's
// barrier is cheaper than a cluster's. Measured in us, 1 / 8 CTAs, in graphs:
//   pages, rows x columns    extend      fork (a quarter of the rows)   compact
//     256,   8 x 32        2.5 / 3.7        3.7 / 5.3        3.2 / 4.7
//    2048,  64 x 32        3.1 / 3.9        5.1 / 5.9        5.3 / 5.7
//    2048,  96 x 33        3.4 / 3.8        6.4 / 6.0        6.3 / 5.8
//    4096,  32 x 128       2.8 / 3.9        5.6 / 7.4        6.3 / 7.0
//    4096,  64 x 64        3.1 / 4.0        5.7 / 6.6        7.3 / 6.5
//    4096, 128 x 32        3.9 / 4.0        6.9 / 6.0        8.1 / 5.8
//    8192,  16 x 512       3.1 / 3.9       11.8 / 14.1      10.3 / 11.7
//    8192,  64 x 128       3.4 / 4.2        7.4 / 8.2       10.5 / 7.6
//    8192, 128 x 64        4.2 / 4.2        8.9 / 7.3       12.3 / 7.0
//   16384,  64 x 128       4.2 / 4.0        9.0 / 9.0       13.9 / 8.2
//   32768,  64 x 512       5.7 / 4.4       17.5 / 16.2      36.3 / 14.5
// A fork's time goes by its rows (32 warps take one each); a row of a compaction
// costs about as much as 64 entries.
template <typename F>
int launch_book(bool small, F launch) {
  return small ? launch(std::integral_constant<int, 1>()) : launch(std::integral_constant<int, 8>());
}
int64_t book_work(const Meta& m) { return (int64_t)m.B * (m.max_pages + 64); }
}  // namespace

extern "C" size_t mb_kv_pages_workspace_bytes(int B, int max_pages, int num_pages) {
  if (B < 0 || max_pages <= 0 || num_pages < 0) return 0;
  return work_layout(B, max_pages, num_pages, true, nullptr, nullptr);
}

extern "C" int mb_kv_pages_extend(int* block_table, int* seq_len, int* page_refs, int B,
                                  int max_pages, int num_pages, const int* new_len, int* start_pos,
                                  int* status, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  Meta m;
  int rc = fill_meta("kv_pages_extend", &m, block_table, seq_len, page_refs, B, max_pages, num_pages,
                     status, false, workspace, workspace_bytes);
  if (rc) return rc;
  MB_REQUIRE(B == 0 || (new_len && start_pos), "kv_pages_extend: null pointer");
  return launch_book(num_pages <= 8192 && book_work(m) <= 16384, [&](auto c) {
    MB_CUDA(mb::launch_pdl(kv_extend_kernel<c()>, dim3(c()), dim3(THREADS<c()>), 0, static_cast<cudaStream_t>(stream), m,
                           new_len, start_pos));
    return MB_OK;
  });
}

extern "C" int mb_kv_pages_fork(void* const* pools, const int64_t* page_bytes, int npools,
                                int* block_table, int* seq_len, int* page_refs, int B, int max_pages,
                                int num_pages, const int* parent, int* status, void* workspace,
                                size_t workspace_bytes, void* stream) {
  Meta m;
  int rc = fill_meta("kv_pages_fork", &m, block_table, seq_len, page_refs, B, max_pages, num_pages,
                     status, true, workspace, workspace_bytes);
  if (!rc) rc = check_pools("kv_pages_fork", pools, page_bytes, npools);
  if (rc) return rc;
  MB_REQUIRE(B == 0 || parent, "kv_pages_fork: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = launch_book(num_pages <= 8192 && B <= 64, [&](auto c) {
    MB_CUDA(mb::launch_pdl(kv_fork_kernel<c()>, dim3(c()), dim3(THREADS<c()>), 0, s, m, parent));
    return MB_OK;
  });
  if (rc) return rc;
  return copy_pages("kv_pages_fork", pools, page_bytes, npools, m.w, B < num_pages ? B : num_pages, s);
}

extern "C" int mb_kv_pages_compact(void* const* pools, const int64_t* page_bytes, int npools,
                                   int* block_table, const int* seq_len, int* page_refs, int B,
                                   int max_pages, int num_pages, int* remap, int* live,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  Meta m;
  int rc = fill_meta("kv_pages_compact", &m, block_table, const_cast<int*>(seq_len), page_refs, B,
                     max_pages, num_pages, live, false, workspace, workspace_bytes);
  if (!rc) rc = check_pools("kv_pages_compact", pools, page_bytes, npools);
  if (rc) return rc;
  MB_REQUIRE(num_pages == 0 || remap, "kv_pages_compact: null pointer");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = launch_book(num_pages <= 4096 && book_work(m) <= 6144, [&](auto c) {
    MB_CUDA(mb::launch_pdl(kv_compact_kernel<c()>, dim3(c()), dim3(THREADS<c()>), 0, s, m, remap));
    return MB_OK;
  });
  if (rc) return rc;
  return copy_pages("kv_pages_compact", pools, page_bytes, npools, m.w, num_pages / 2, s);
}
