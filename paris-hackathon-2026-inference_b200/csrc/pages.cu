// Page bookkeeping of the paged cache, all on the device and in stream order: grow, fork,
// free and compact.  The state is refs[page] (sequences that hold the page; 0 = free), the
// tables and the lengths; the free pages are those with refs 0, handed out lowest number
// first, so the same calls give the same pages on every run.
//
// What a call grants depends on what the entries before it took, so one CTA plans (1024 threads,
// marks and sums in shared memory, four refs a thread at a time): a chain of latencies, 7 to 8 us
// from cold caches, that neither bytes nor arithmetic bound.  The copies run on the whole GPU behind it and are
// bound by HBM: 32 prompts of up to 2000 tokens forked into 8 branches each, freed and grown
// (74 MB) 24 us with the host's part, 11.4 at the copy rate; packing a pool of ten layers (1.36 GB
// read and written) 243 us, of which the copies 223, 6.1 TB/s, 94 % of the copy rate.
#include "paged.cuh"
#include "pmoe_tma.cuh"

namespace pmoe {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPerThread = 4;

// Inclusive scan of x >= 0 over the block; *total gets the sum.  Sums stop at kMost, above any
// number of pages.
constexpr int kMost = 0x3fffffff;
__device__ __forceinline__ int block_scan(int x, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x = min(x + y, kMost);
  }
  __syncthreads();  // s_warp of the scan before has been read
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int w = s_warp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w = min(w + y, kMost);
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = __shfl_sync(0xffffffffu, w, warp == 0 ? 0 : warp - 1);
  return min(x + (warp == 0 ? 0 : before), kMost);
}

// The free pages among 4 * kPlanThreads refs, a thread's four loaded beforehand.
struct Refs4 {
  int r[kPerThread];
};
__device__ __forceinline__ Refs4 load_refs(const int32_t* refs, int n_pages, int p0) {
  Refs4 x;
  const int p = p0 + threadIdx.x * kPerThread;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) x.r[k] = p + k < n_pages ? refs[p + k] : 1;
  return x;
}

// The first `want` free pages in ascending order into pick; returns how many there were.
// `first`: the refs of the pages 0 .. 4095, which the caller loads while it does other things.
__device__ __forceinline__ int pick_free(const int32_t* refs, int n_pages, int want, Refs4 first,
                                         int32_t* pick, int* s_warp) {
  int found = 0;
  for (int p0 = 0; p0 < n_pages && found < want; p0 += kPlanThreads * kPerThread) {
    const Refs4 x = p0 == 0 ? first : load_refs(refs, n_pages, p0);
    const int p = p0 + threadIdx.x * kPerThread;
    int mine = 0, total;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) mine += x.r[k] == 0;
    int at = found + block_scan(mine, s_warp, &total) - mine;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (x.r[k] == 0) {
        if (at < want) pick[at] = p + k;
        ++at;
      }
    found += total;
  }
  return min(found, want);
}

// Room in shared memory for the marks of so many sequences and for the requests of one round;
// more go through the workspace.
constexpr int kMarks = 4096, kRequests = kPlanThreads;

// What a request asks for: pages (-1: refused), and the number asked for up to and with it.
struct Requests {
  int32_t *need, *end, *pick;
};
struct PlanSmem {
  int warp[32], mark[kMarks], need[kRequests], end[kRequests];
};
__device__ __forceinline__ Requests requests_of(PlanSmem& s, int32_t* ws, int n) {
  Requests q;
  q.need = n <= kRequests ? s.need : ws;
  q.end = n <= kRequests ? s.end : ws + n;
  q.pick = ws + 2 * size_t(n);
  return q;
}

// mark[slot] = the first request that names the slot.
__device__ __forceinline__ void mark_first(int32_t* mark, int S, const int32_t* slots, int n) {
  for (int s = threadIdx.x; s < S; s += kPlanThreads) mark[s] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads)
    if (slots[i] >= 0 && slots[i] < S) atomicMin(&mark[slots[i]], i);
  __syncthreads();
}

// Requests in order: need[i] = ask(i) pages, end[i] their running sum; returns how many pages
// there are for them.  A request is granted if need >= 0 and end <= that.
template <typename Ask>
__device__ __forceinline__ int serve(const Pool& p, int n, Refs4 first, PlanSmem& sm, Requests q, Ask ask) {
  int64_t carry = 0;
  for (int i0 = 0; i0 < n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    const int want = i < n ? ask(i) : -1;
    int total;
    const int64_t e = carry + block_scan(max(want, 0), sm.warp, &total);
    if (i < n) {
      q.need[i] = want;
      q.end[i] = int(min(e, int64_t(p.n_pages) + 1));  // beyond the pool: granted to nobody
    }
    carry += total;
  }
  const int found = pick_free(p.refs, p.n_pages, int(min(carry, int64_t(p.n_pages))), first, q.pick, sm.warp);
  __syncthreads();
  return found;
}

// ws: mark[S], need[n], end[n], pick[n_pages]
__global__ void __launch_bounds__(kPlanThreads) pages_grow_kernel(
    const Pool p, const int32_t* slots, const int32_t* add, int n, int32_t* ok, int32_t* ws) {
  __shared__ PlanSmem sm;
  const int tid = threadIdx.x, ps = 1 << p.page_shift;
  pdl_wait();
  const Refs4 first = load_refs(p.refs, p.n_pages, 0);
  int32_t* mark = p.S <= kMarks ? sm.mark : ws;
  const Requests q = requests_of(sm, ws + p.S, n);
  mark_first(mark, p.S, slots, n);
  const int found = serve(p, n, first, sm, q, [&](int i) {
    const int s = slots[i], a = add[i];
    if (s < 0 || s >= p.S || mark[s] != i || a < 0) return -1;
    const int64_t old = p.lens[s], len = old + a;
    if (old < 0 || len > int64_t(p.max_pages) << p.page_shift || len > 0x7fffffff) return -1;
    return int(((len + ps - 1) >> p.page_shift) - ((old + ps - 1) >> p.page_shift));
  });
  // the granted pages, a thread each: page k belongs to the first request with end > k
  for (int k = tid; k < found; k += kPlanThreads) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (q.end[mid] > k) hi = mid; else lo = mid + 1;
    }
    if (q.end[lo] > found) continue;  // the first that did not fit
    const int s = slots[lo], page = q.pick[k];
    const int have = int((int64_t(p.lens[s]) + ps - 1) >> p.page_shift);
    p.tables[s * p.table_stride + have + k - (q.end[lo] - q.need[lo])] = page;
    p.refs[page] = 1;
  }
  __syncthreads();  // the lengths have been read
  for (int i = tid; i < n; i += kPlanThreads) {
    const bool yes = q.need[i] >= 0 && q.end[i] <= found;
    if (yes) p.lens[slots[i]] += add[i];
    ok[i] = yes;
  }
}

// ws: plan[n] (fresh page, -1: none needed, -2: refused), mark[S], need[n], end[n], pick[n_pages]
__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(
    const Pool p, const int32_t* src, const int32_t* dst, const int32_t* keep, int n,
    int32_t* ok, int32_t* ws) {
  __shared__ PlanSmem sm;
  const int tid = threadIdx.x, ps = 1 << p.page_shift;
  pdl_wait();
  pdl_trigger();
  const Refs4 first = load_refs(p.refs, p.n_pages, 0);
  int32_t *plan = ws, *mark = p.S <= kMarks ? sm.mark : ws + n;
  const Requests q = requests_of(sm, ws + n + p.S, n);
  mark_first(mark, p.S, dst, n);
  const int found = serve(p, n, first, sm, q, [&](int i) {
    const int s = src[i], d = dst[i], k = keep[i];
    // a target is empty, named once and nobody's source
    if (s < 0 || s >= p.S || d < 0 || d >= p.S || mark[d] != i || mark[s] != 0x7fffffff || k < 0 ||
        k > int64_t(p.max_pages) << p.page_shift)
      return -1;
    const bool part = k & (ps - 1);  // the last page is partly filled: it is copied, so it must be there
    const int tail = part ? p.tables[s * p.table_stride + (k >> p.page_shift)] : 0;
    if (p.lens[d] != 0 || k > p.lens[s] || (part && (tail < 0 || tail >= p.n_pages))) return -1;
    return int(part);
  });
  for (int i = tid; i < n; i += kPlanThreads) {
    const bool yes = q.need[i] >= 0 && q.end[i] <= found;
    ok[i] = yes;
    plan[i] = !yes ? -2 : q.need[i] ? q.pick[q.end[i] - 1] : -1;
  }
}

// gridDim = (n, parts): part 0 copies the table row, all parts copy the tail page.
__global__ void __launch_bounds__(256) fork_copy_kernel(const Pool p, const int32_t* src,
                                                        const int32_t* dst, const int32_t* keep,
                                                        const int32_t* plan) {
  pdl_wait();
  const int i = blockIdx.x, fresh = plan[i];
  if (fresh == -2) return;
  const int k = keep[i], full = k >> p.page_shift, used = k & ((1 << p.page_shift) - 1);
  const int32_t* from = p.tables + src[i] * p.table_stride;
  if (blockIdx.y == 0) {
    int32_t* to = p.tables + dst[i] * p.table_stride;
    for (int j = threadIdx.x; j < full; j += blockDim.x) {
      const int page = from[j];
      to[j] = page;
      if (page >= 0 && page < p.n_pages) atomicAdd(&p.refs[page], 1);
    }
    if (threadIdx.x == 0) {
      if (fresh >= 0) {
        to[full] = fresh;
        p.refs[fresh] = 1;
      }
      p.lens[dst[i]] = k;
    }
  }
  if (fresh < 0) return;
  const size_t chunk = size_t(p.D) << p.page_shift;  // elements of one head's rows
  const __nv_bfloat16* s0 = p.pages + size_t(from[full]) * p.chunks * chunk;
  __nv_bfloat16* d0 = p.pages + size_t(fresh) * p.chunks * chunk;
  const int vec = used * p.D / 8;  // 16-byte pieces of a chunk's used rows
  // four chunks' pieces on their way at a time
  constexpr int kOnce = 4;
  for (int j = threadIdx.x; j < vec; j += blockDim.x)
    for (int c = blockIdx.y; c < p.chunks; c += kOnce * gridDim.y) {
      uint4 x[kOnce];
#pragma unroll
      for (int k = 0; k < kOnce; ++k)
        if (c + k * int(gridDim.y) < p.chunks)
          x[k] = reinterpret_cast<const uint4*>(s0 + (c + k * gridDim.y) * chunk)[j];
#pragma unroll
      for (int k = 0; k < kOnce; ++k)
        if (c + k * int(gridDim.y) < p.chunks) reinterpret_cast<uint4*>(d0 + (c + k * gridDim.y) * chunk)[j] = x[k];
    }
}

__global__ void __launch_bounds__(256) pages_free_kernel(const Pool p, const int32_t* slots,
                                                         int window, int sinks) {
  pdl_wait();
  const int s = slots[blockIdx.x];
  if (s < 0 || s >= p.S) return;
  int lo = 0, hi = p.max_pages;
  if (window > 0) {
    const int ps = 1 << p.page_shift, len = p.lens[s];
    lo = int((int64_t(sinks) + ps - 1) >> p.page_shift);
    hi = min(hi, len > window ? (len - window) >> p.page_shift : 0);
  }
  int32_t* row = p.tables + s * p.table_stride;
  for (int j = lo + threadIdx.x; j < hi; j += blockDim.x) {
    if (row[j] < 0) continue;
    // taken by one block alone where a slot is listed twice
    const int page = atomicExch(&row[j], -1);
    if (page >= 0 && page < p.n_pages) atomicSub(&p.refs[page], 1);
  }
  if (window == 0 && threadIdx.x == 0) p.lens[s] = 0;
}

// With n live pages, the k-th free page below n takes the k-th live page at or above it: a
// packed pool after the fewest moves.  ws[0]: moves; ws[16 + k]: the k-th page that moves,
// to remap[ws[16 + k]].
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const Pool p, int32_t* live,
                                                                    int32_t* remap, int32_t* ws) {
  __shared__ int s_warp[32];
  const int tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  int32_t* movers = ws + 16;
  int mine = 0, n_live;
  for (int q = tid; q < p.n_pages; q += kPlanThreads) mine += p.refs[q] > 0;
  block_scan(mine, s_warp, &n_live);
  int moves = 0;
  for (int q0 = 0; q0 < p.n_pages; q0 += kPlanThreads) {
    const int q = q0 + tid;
    const bool used = q < p.n_pages && p.refs[q] > 0;
    const bool move = used && q >= n_live;
    int total;
    const int at = moves + block_scan(move, s_warp, &total) - move;
    if (move) movers[at] = q;
    if (q < p.n_pages) remap[q] = used ? q : -1;
    moves += total;
  }
  __syncthreads();
  int holes = 0;
  for (int q0 = 0; q0 < n_live; q0 += kPlanThreads) {
    const int q = q0 + tid;
    const bool hole = q < n_live && p.refs[q] <= 0;
    int total;
    const int at = holes + block_scan(hole, s_warp, &total) - hole;
    if (hole) remap[movers[at]] = q;
    holes += total;
  }
  __syncthreads();
  for (int k = tid; k < moves; k += kPlanThreads) {
    const int from = movers[k], to = remap[from];
    p.refs[to] = p.refs[from];
    p.refs[from] = 0;
  }
  if (tid == 0) {
    live[0] = n_live;
    ws[0] = moves;
  }
}

__global__ void __launch_bounds__(256) compact_move_kernel(const Pool p, const int32_t* remap,
                                                           const int32_t* ws) {
  pdl_wait();
  const int moves = ws[0];
  const int64_t entries = int64_t(p.S) * p.max_pages;
  for (int64_t e = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; e < entries;
       e += int64_t(gridDim.x) * blockDim.x) {
    int32_t* at = p.tables + (e / p.max_pages) * p.table_stride + e % p.max_pages;
    const int page = *at;
    if (page >= 0 && page < p.n_pages) {
      const int to = remap[page];
      if (to >= 0 && to != page) *at = to;
    }
  }
  const size_t page_vec = (size_t(p.chunks) * p.D << p.page_shift) / 8;
  const size_t part = 2048;  // 16-byte pieces a block copies at a time
  const size_t parts = (page_vec + part - 1) / part;
  for (size_t w = blockIdx.x; w < parts * moves; w += gridDim.x) {
    const int from = ws[16 + w / parts], to = remap[from];
    const uint4* s = reinterpret_cast<const uint4*>(p.pages) + from * page_vec;
    uint4* d = reinterpret_cast<uint4*>(p.pages) + to * page_vec;
    const size_t j0 = (w % parts) * part, j1 = min(j0 + part, page_vec);
    uint4 x[8];  // all of the thread's pieces on their way at once
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const size_t j = j0 + threadIdx.x + k * 256;
      if (j < j1) x[k] = __ldcs(s + j);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const size_t j = j0 + threadIdx.x + k * 256;
      if (j < j1) __stcs(d + j, x[k]);
    }
  }
}

}  // namespace

cudaError_t launch_pages_grow(const Pool& p, const int32_t* slots, const int32_t* add, int n,
                              int32_t* ok, int32_t* ws, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  return launch_dependent(pages_grow_kernel, dim3(1), kPlanThreads, 0, 1, st, p, slots, add, n, ok, ws);
}

cudaError_t launch_pages_fork(const Pool& p, const int32_t* src, const int32_t* dst,
                              const int32_t* keep, int n, int32_t* ok, int32_t* ws,
                              cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  const cudaError_t e = launch_dependent(fork_plan_kernel, dim3(1), kPlanThreads, 0, 1, st, p, src, dst,
                                         keep, n, ok, ws);
  if (e != cudaSuccess) return e;
  return launch_dependent(fork_copy_kernel, dim3(n, p.chunks < 8 ? p.chunks : 8), 256, 0, 1, st, p, src,
                          dst, keep, static_cast<const int32_t*>(ws));
}

cudaError_t launch_pages_free(const Pool& p, const int32_t* slots, int n, int window, int sinks,
                              cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  return launch_dependent(pages_free_kernel, dim3(n), 256, 0, 1, st, p, slots, window, sinks);
}

cudaError_t launch_pages_compact(const Pool& p, int32_t* live, int32_t* remap, int32_t* ws,
                                 cudaStream_t st) {
  const cudaError_t e = launch_dependent(compact_plan_kernel, dim3(1), kPlanThreads, 0, 1, st, p, live,
                                         remap, ws);
  if (e != cudaSuccess) return e;
  return launch_dependent(compact_move_kernel, dim3(148 * 4), 256, 0, 1, st, p,
                          static_cast<const int32_t*>(remap), static_cast<const int32_t*>(ws));
}

}  // namespace pmoe
