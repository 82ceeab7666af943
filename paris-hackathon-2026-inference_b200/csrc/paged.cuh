// The paged key/value cache as the attention-half kernels see it.
//
// Keys and values of one layer are two views [n_pages, Hkv, page_size, D] of the
// cache's pool (inner three dimensions contiguous, any page stride that keeps
// 16-byte alignment).  Sequence b's key j lies in page table[b][j / page_size],
// row j % page_size.  An entry outside [0, n_pages) names no page: nothing is read or
// written through it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace pmoe {

struct PagedKV {
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  int64_t k_page_stride, v_page_stride;  // elements
  int n_pages, page_shift;               // page size = 1 << page_shift
  int Hkv, D;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;                         // entries of a table row
  const int32_t* kv_lens;                // [B], the call's new tokens included
  int B;
};

// Keys a sequence's tables can hold, and whether its length is beyond that.
__host__ __device__ __forceinline__ int kv_len_of(int len, int max_pages, int page_shift,
                                                  bool* over) {
  const int64_t cap = int64_t(max_pages) << page_shift;
  *over = len > cap;
  return len < 0 ? 0 : (len > cap ? int(cap) : len);
}

// Page that holds key j, or -1 where the table names none.
__host__ __device__ __forceinline__ int page_of(const PagedKV& kv, int b, int j) {
  const int i = j >> kv.page_shift;
  if (i < 0 || i >= kv.max_pages) return -1;
  const int p = kv.table[b * kv.table_stride + i];
  return (p < 0 || p >= kv.n_pages) ? -1 : p;
}

// The keys that the token at index p sees: [0, sink) and [lo, p].
__host__ __device__ __forceinline__ void visible_keys(int p, int window, int sinks, int* lo,
                                                      int* sink) {
  *lo = (window > 0 && p + 1 > window) ? p + 1 - window : 0;
  *sink = sinks < *lo ? sinks : *lo;
}

// The last b in [0, B) with key(b) <= x, or -1; key ascends.  32 places at a time by a whole
// warp: one step for 32 sequences, two for 1024.
template <typename Key>
__device__ __forceinline__ int last_at_or_before(int B, int x, Key key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B;
  while (n > 0) {
    const int step = (n + 31) / 32, at = lane * step;
    const bool before = at < n && key(lo + at) <= x;
    const int k = __popc(__ballot_sync(0xffffffffu, before));
    if (k == 0) return -1;
    lo += (k - 1) * step;
    n = step < n - (k - 1) * step ? step : n - (k - 1) * step;
    if (step == 1) break;
  }
  return B > 0 ? lo : -1;
}

struct AttnArgs {
  PagedKV kv;
  const __nv_bfloat16* q;
  int64_t q_stride_t, q_stride_h;  // elements
  int T, Hq;
  const int32_t* cu_q;             // [B+1], or null: row t is sequence t's one new token
  float scale;
  int window, sinks;               // window 0: none
  __nv_bfloat16* out;              // [T, Hq, D] contiguous
};

struct RopeArgs {
  PagedKV kv;
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // elements, token and head strides
  int T, Hq;
  const int64_t* positions;                    // [axes][pos_stride]
  int64_t pos_stride;
  int axes, half, interleaved;                 // half = rotary dims / 2
  int sections[4];
  const float* inv_freq;                       // [half]
  const __nv_bfloat16 *w_q, *w_k;              // [D] or null
  float eps, mscale;
  const int32_t* cu_q;
  __nv_bfloat16* q_out;                        // [T, Hq, D] contiguous
};

struct Pool {
  __nv_bfloat16* pages;    // [n_pages][chunks][page_size][D]
  int n_pages, chunks, page_shift, D;
  int32_t* refs;           // [n_pages]
  int32_t* tables;         // [S][table_stride], max_pages entries used
  int64_t table_stride;
  int max_pages, S;
  int32_t* lens;           // [S]
};

// CTAs of the decode kernel: one per SM of a B200.
constexpr int kDecodeCtas = 148;

// Launch with programmatic stream serialisation: the kernel's set-up may run while its
// predecessor in the stream ends.  Every kernel launched this way waits (griddepcontrol.wait)
// before it reads or writes anything that the predecessor might still use, on all its paths, so
// that a kernel behind it may rely on everything before it.
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem,
                             unsigned cluster, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {cluster, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

cudaError_t launch_rope_append(const RopeArgs& a, cudaStream_t st);
cudaError_t attn_decode_init();
cudaError_t attn_prefill_init();
cudaError_t launch_attn_prefill(const AttnArgs& a, void* ws, cudaStream_t st);
size_t attn_prefill_ws_bytes(int T, int B, int Hq, int Hkv, int D, int64_t keys);
cudaError_t launch_attn_decode(const AttnArgs& a, void* ws, cudaStream_t st);
size_t attn_decode_ws_bytes(int B, int Hq, int Hkv, int D);
cudaError_t launch_pages_grow(const Pool& p, const int32_t* slots, const int32_t* add, int n,
                              int32_t* ok, int32_t* ws, cudaStream_t st);
cudaError_t launch_pages_fork(const Pool& p, const int32_t* src, const int32_t* dst,
                              const int32_t* keep, int n, int32_t* ok, int32_t* ws,
                              cudaStream_t st);
cudaError_t launch_pages_free(const Pool& p, const int32_t* slots, int n, int window, int sinks,
                              cudaStream_t st);
cudaError_t launch_pages_compact(const Pool& p, int32_t* live, int32_t* remap, int32_t* ws,
                                 cudaStream_t st);
// 32-bit words of workspace of the page operations.
inline size_t pages_grow_words(int S, int n, int n_pages) { return size_t(S) + 2 * size_t(n) + n_pages; }
inline size_t pages_fork_words(int S, int n, int n_pages) { return size_t(S) + 3 * size_t(n) + n_pages; }
inline size_t pages_compact_words(int n_pages) { return size_t(n_pages) + 16; }

}  // namespace pmoe
