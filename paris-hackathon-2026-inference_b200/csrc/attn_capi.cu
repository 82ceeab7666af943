// extern "C" entry points of the paged-attention operators (declared in
// include/paris_moe.h): argument checks, then one launcher each.
#include <atomic>

#include "paged.cuh"
#include "pmoe_common.cuh"

using namespace pmoe;

namespace {

constexpr int kMaxDevices = 64;
std::atomic<int> g_ready[kMaxDevices];  // 0 unknown, 1 ready

int ensure_device() {
  int dev = 0, major = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return PMOE_ERR_CUDA;
  if (g_ready[dev].load(std::memory_order_acquire)) return PMOE_OK;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess)
    return PMOE_ERR_CUDA;
  if (major != 10) return PMOE_ERR_DEVICE;
  if (attn_decode_init() != cudaSuccess || attn_prefill_init() != cudaSuccess) return PMOE_ERR_CUDA;
  g_ready[dev].store(1, std::memory_order_release);
  return PMOE_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int page_shift_of(int page_size) {
  switch (page_size) {
    case 16: return 4;
    case 32: return 5;
    case 64: return 6;
    case 128: return 7;
    default: return -1;
  }
}

bool head_dim_ok(int D) { return D == 64 || D == 128 || D == 256; }
// A stride of a dimension of n entries, in elements: 16-byte steps.
bool stride_ok(int64_t s, int64_t n) { return n <= 1 || (s > 0 && s % 8 == 0); }

__nv_bfloat16* bfm(uint16_t* p) { return reinterpret_cast<__nv_bfloat16*>(p); }
const __nv_bfloat16* bf(const uint16_t* p) { return reinterpret_cast<const __nv_bfloat16*>(p); }

// The cache arguments that all attention entry points share.
int check_cache(int Hq, int Hkv, int D, int64_t kps, int64_t vps, int n_pages, int page_size,
                int64_t table_stride, int max_pages, int B) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || n_pages < 0 || max_pages < 0 || B < 0 ||
      (B > 1 && table_stride < max_pages))
    return PMOE_ERR_ARG;
  if (!head_dim_ok(D) || page_shift_of(page_size) < 0 || Hq / Hkv > 128 || Hkv > 65535)
    return PMOE_ERR_UNSUPPORTED;
  const int64_t page = int64_t(Hkv) * page_size * D;
  if (n_pages > 1 && (kps < page || vps < page)) return PMOE_ERR_ARG;
  if (kps % 8 != 0 || vps % 8 != 0) return PMOE_ERR_ALIGN;
  // key indexes and padded lengths are 32-bit
  if (int64_t(max_pages) * page_size > 0x7fff0000LL) return PMOE_ERR_UNSUPPORTED;
  return PMOE_OK;
}

PagedKV make_kv(const uint16_t* k, const uint16_t* v, int64_t kps, int64_t vps, int n_pages,
                int page_size, int Hkv, int D, const int32_t* table, int64_t table_stride,
                int max_pages, const int32_t* kv_lens, int B) {
  if (n_pages <= 1) kps = vps = int64_t(Hkv) * page_size * D;  // never stepped over
  return PagedKV{const_cast<__nv_bfloat16*>(bf(k)), const_cast<__nv_bfloat16*>(bf(v)), kps, vps,
                 n_pages, page_shift_of(page_size), Hkv, D, table, table_stride, max_pages,
                 kv_lens, B};
}

int attn_args(AttnArgs* a, const uint16_t* q, int T, int Hq, int64_t q_st, int64_t q_sh,
              const uint16_t* k, const uint16_t* v, int64_t kps, int64_t vps, int n_pages,
              int page_size, int Hkv, int D, const int32_t* table, int64_t table_stride,
              int max_pages, const int32_t* kv_lens, int B, const int32_t* cu_q, float scale,
              int window, int sinks, uint16_t* out) {
  if (T < 0 || window < 0 || sinks < 0) return PMOE_ERR_ARG;
  int s = check_cache(Hq, Hkv, D, kps, vps, n_pages, page_size, table_stride, max_pages, B);
  if (s != PMOE_OK) return s;
  if (int64_t(T) * Hq > 0x3fffffffLL) return PMOE_ERR_UNSUPPORTED;
  if (!stride_ok(q_st, T) || !stride_ok(q_sh, Hq)) return PMOE_ERR_ALIGN;
  if (T == 0) return PMOE_OK;
  if (!q || !out || !kv_lens || (n_pages > 0 && (!k || !v)) || (max_pages > 0 && !table))
    return PMOE_ERR_ARG;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned4(table) ||
      !aligned4(kv_lens) || !aligned4(cu_q))
    return PMOE_ERR_ALIGN;
  a->kv = make_kv(k, v, kps, vps, n_pages, page_size, Hkv, D, table, table_stride, max_pages,
                  kv_lens, B);
  a->q = bf(q);
  a->q_stride_t = q_st;
  a->q_stride_h = q_sh;
  a->T = T;
  a->Hq = Hq;
  a->cu_q = cu_q;
  a->scale = scale;
  a->window = window;
  a->sinks = sinks;
  a->out = bfm(out);
  return PMOE_OK;
}

int make_pool(Pool* p, uint16_t* pages, int n_pages, int chunks, int page_size, int D,
              int32_t* refs, int32_t* tables, int64_t table_stride, int max_pages, int S,
              int32_t* lens, bool need_lens) {
  if (n_pages < 0 || max_pages < 0 || S < 0 || (S > 1 && table_stride < max_pages))
    return PMOE_ERR_ARG;
  if (page_shift_of(page_size) < 0 || n_pages > 1 << 29) return PMOE_ERR_UNSUPPORTED;
  if (int64_t(max_pages) * page_size > 0x7fff0000LL) return PMOE_ERR_UNSUPPORTED;
  if ((n_pages > 0 && !refs) || (S > 0 && need_lens && !lens) ||
      (S > 0 && max_pages > 0 && !tables))
    return PMOE_ERR_ARG;
  if (!aligned4(refs) || !aligned4(tables) || !aligned4(lens) || !aligned16(pages))
    return PMOE_ERR_ALIGN;
  *p = Pool{bfm(pages), n_pages, chunks, page_shift_of(page_size), D, refs, tables,
            table_stride, max_pages, S, lens};
  return PMOE_OK;
}

}  // namespace

extern "C" {

int pmoe_rope_append(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h,
                     const uint16_t* k, int64_t k_stride_t, int64_t k_stride_h,
                     const uint16_t* v, int64_t v_stride_t, int64_t v_stride_h, int T, int Hq,
                     int Hkv, int D, const int64_t* positions, int64_t pos_stride, int axes,
                     const int* sections, int interleaved, const float* inv_freq, int rot,
                     const uint16_t* w_qnorm, const uint16_t* w_knorm, float eps, float mscale,
                     uint16_t* k_pages, uint16_t* v_pages, int64_t k_page_stride,
                     int64_t v_page_stride, int n_pages, int page_size, const int32_t* page_table,
                     int64_t table_stride, int max_pages, const int32_t* kv_lens,
                     const int32_t* cu_q, int B, uint16_t* q_out, void* stream) {
  if (T < 0 || axes < 1 || axes > 4 || !sections) return PMOE_ERR_ARG;
  int s = check_cache(Hq, Hkv, D, k_page_stride, v_page_stride, n_pages, page_size, table_stride,
                      max_pages, B);
  if (s != PMOE_OK) return s;
  if (rot < 0 || rot > D) return PMOE_ERR_ARG;
  if (rot % 16 != 0) return PMOE_ERR_UNSUPPORTED;
  int64_t sum = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0) return PMOE_ERR_ARG;
    sum += sections[i];
  }
  if (sum != rot / 2) return PMOE_ERR_ARG;
  if (!cu_q && T != B) return PMOE_ERR_ARG;
  if (!stride_ok(q_stride_t, T) || !stride_ok(q_stride_h, Hq) || !stride_ok(k_stride_t, T) ||
      !stride_ok(k_stride_h, Hkv) || !stride_ok(v_stride_t, T) || !stride_ok(v_stride_h, Hkv))
    return PMOE_ERR_ALIGN;
  if (T == 0) return PMOE_OK;
  if (!q || !k || !v || !q_out || !kv_lens || (rot > 0 && (!positions || !inv_freq)) ||
      (n_pages > 0 && (!k_pages || !v_pages)) || (max_pages > 0 && !page_table) ||
      (axes > 1 && pos_stride < T))
    return PMOE_ERR_ARG;
  const void* wide[8] = {q, k, v, q_out, w_qnorm, w_knorm, k_pages, v_pages};
  for (const void* p : wide)
    if (!aligned16(p)) return PMOE_ERR_ALIGN;
  if (!aligned4(page_table) || !aligned4(kv_lens) || !aligned4(cu_q) || !aligned4(inv_freq) ||
      (reinterpret_cast<uintptr_t>(positions) & 7u) != 0)
    return PMOE_ERR_ALIGN;
  if ((s = ensure_device()) != PMOE_OK) return s;
  RopeArgs a{};
  a.kv = make_kv(k_pages, v_pages, k_page_stride, v_page_stride, n_pages, page_size, Hkv, D,
                 page_table, table_stride, max_pages, kv_lens, B);
  a.q = bf(q);
  a.k = bf(k);
  a.v = bf(v);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k_st = k_stride_t;
  a.k_sh = k_stride_h;
  a.v_st = v_stride_t;
  a.v_sh = v_stride_h;
  a.T = T;
  a.Hq = Hq;
  a.positions = positions;
  a.pos_stride = pos_stride;
  a.axes = axes;
  a.half = rot / 2;
  a.interleaved = interleaved;
  for (int i = 0; i < axes; ++i) a.sections[i] = sections[i];
  a.inv_freq = inv_freq;
  a.w_q = bf(w_qnorm);
  a.w_k = bf(w_knorm);
  a.eps = eps;
  a.mscale = mscale;
  a.cu_q = cu_q;
  a.q_out = bfm(q_out);
  return launch_rope_append(a, static_cast<cudaStream_t>(stream)) == cudaSuccess ? PMOE_OK
                                                                                 : PMOE_ERR_CUDA;
}

int pmoe_attn_decode(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, int B, int Hq,
                     int Hkv, int D, const uint16_t* k_pages, const uint16_t* v_pages,
                     int64_t k_page_stride, int64_t v_page_stride, int n_pages, int page_size,
                     const int32_t* page_table, int64_t table_stride, int max_pages,
                     const int32_t* kv_lens, float scale, int window, int sinks, uint16_t* out,
                     void* workspace, size_t workspace_bytes, void* stream) {
  AttnArgs a{};
  int s = attn_args(&a, q, B, Hq, q_stride_t, q_stride_h, k_pages, v_pages, k_page_stride,
                    v_page_stride, n_pages, page_size, Hkv, D, page_table, table_stride,
                    max_pages, kv_lens, B, nullptr, scale, window, sinks, out);
  if (s != PMOE_OK || B == 0) return s;
  size_t need = 0;
  if ((s = pmoe_attn_decode_workspace(B, Hq, Hkv, D, &need)) != PMOE_OK) return s;
  if (need > 0 && (!workspace || workspace_bytes < need)) return PMOE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return PMOE_ERR_ALIGN;
  // the line of work units is counted in 32 bits per sequence
  if (int64_t(max_pages) * page_size / 16 * Hq > 0x7fffffffLL) return PMOE_ERR_UNSUPPORTED;
  if ((s = ensure_device()) != PMOE_OK) return s;
  return launch_attn_decode(a, workspace, static_cast<cudaStream_t>(stream)) == cudaSuccess
             ? PMOE_OK : PMOE_ERR_CUDA;
}

int pmoe_attn_decode_workspace(int B, int Hq, int Hkv, int D, size_t* bytes) {
  if (!bytes || B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0) return PMOE_ERR_ARG;
  if (!head_dim_ok(D)) return PMOE_ERR_UNSUPPORTED;
  *bytes = attn_decode_ws_bytes(B, Hq, Hkv, D);
  return PMOE_OK;
}

int pmoe_attn_prefill_workspace(int T, int B, int Hq, int Hkv, int D, int page_size, int max_pages,
                                size_t* bytes) {
  if (!bytes || T < 0 || B < 0 || max_pages < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0)
    return PMOE_ERR_ARG;
  if (!head_dim_ok(D) || page_shift_of(page_size) < 0 || Hq / Hkv > 128) return PMOE_ERR_UNSUPPORTED;
  *bytes = T == 0 || B == 0 ? 0 : attn_prefill_ws_bytes(T, B, Hq, Hkv, D, int64_t(max_pages) * page_size);
  return PMOE_OK;
}

int pmoe_attn_prefill(const uint16_t* q, int64_t q_stride_t, int64_t q_stride_h, int T, int Hq,
                      int Hkv, int D, const uint16_t* k_pages, const uint16_t* v_pages,
                      int64_t k_page_stride, int64_t v_page_stride, int n_pages, int page_size,
                      const int32_t* page_table, int64_t table_stride, int max_pages,
                      const int32_t* kv_lens, const int32_t* cu_q, int B, float scale, int window,
                      int sinks, uint16_t* out, void* workspace, size_t workspace_bytes,
                      void* stream) {
  if (B < 1 && T > 0) return PMOE_ERR_ARG;
  if (!cu_q && T > 0) return PMOE_ERR_ARG;
  AttnArgs a{};
  int s = attn_args(&a, q, T, Hq, q_stride_t, q_stride_h, k_pages, v_pages, k_page_stride,
                    v_page_stride, n_pages, page_size, Hkv, D, page_table, table_stride,
                    max_pages, kv_lens, B, cu_q, scale, window, sinks, out);
  if (s != PMOE_OK || T == 0) return s;
  const size_t need = attn_prefill_ws_bytes(T, B, Hq, Hkv, D, int64_t(max_pages) * page_size);
  if (need > 0 && (!workspace || workspace_bytes < need)) return PMOE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return PMOE_ERR_ALIGN;
  if ((s = ensure_device()) != PMOE_OK) return s;
  return launch_attn_prefill(a, workspace, static_cast<cudaStream_t>(stream)) == cudaSuccess ? PMOE_OK
                                                                                  : PMOE_ERR_CUDA;
}

int pmoe_pages_workspace(int S, int n, int n_pages, size_t* bytes) {
  if (!bytes || S < 0 || n < 0 || n_pages < 0) return PMOE_ERR_ARG;
  *bytes = sizeof(int32_t) * (pages_fork_words(S, n, n_pages) + pages_compact_words(n_pages));
  return PMOE_OK;
}

int pmoe_pages_grow(int32_t* refs, int n_pages, int page_size, int32_t* tables,
                    int64_t table_stride, int max_pages, int S, int32_t* lens,
                    const int32_t* slots, const int32_t* add, int n, int32_t* ok, void* workspace,
                    size_t workspace_bytes, void* stream) {
  Pool p;
  int s = make_pool(&p, nullptr, n_pages, 0, page_size, 0, refs, tables, table_stride, max_pages,
                    S, lens, true);
  if (s != PMOE_OK) return s;
  if (n < 0 || (n > 0 && (!slots || !add || !ok))) return PMOE_ERR_ARG;
  if (n == 0) return PMOE_OK;
  if (!workspace || workspace_bytes < sizeof(int32_t) * pages_grow_words(S, n, n_pages))
    return PMOE_ERR_WORKSPACE;
  if (!aligned16(workspace) || !aligned4(slots) || !aligned4(add) || !aligned4(ok))
    return PMOE_ERR_ALIGN;
  if ((s = ensure_device()) != PMOE_OK) return s;
  return launch_pages_grow(p, slots, add, n, ok, static_cast<int32_t*>(workspace),
                           static_cast<cudaStream_t>(stream)) == cudaSuccess ? PMOE_OK
                                                                             : PMOE_ERR_CUDA;
}

int pmoe_pages_fork(uint16_t* pages, int n_pages, int chunks, int page_size, int D, int32_t* refs,
                    int32_t* tables, int64_t table_stride, int max_pages, int S, int32_t* lens,
                    const int32_t* src, const int32_t* dst, const int32_t* keep, int n,
                    int32_t* ok, void* workspace, size_t workspace_bytes, void* stream) {
  Pool p;
  int s = make_pool(&p, pages, n_pages, chunks, page_size, D, refs, tables, table_stride,
                    max_pages, S, lens, true);
  if (s != PMOE_OK) return s;
  if (n < 0 || chunks < 1 || D < 1 || (n > 0 && (!src || !dst || !keep || !ok)) ||
      (n > 0 && n_pages > 0 && !pages))
    return PMOE_ERR_ARG;
  if (D % 8 != 0) return PMOE_ERR_UNSUPPORTED;
  if (n == 0) return PMOE_OK;
  if (!workspace || workspace_bytes < sizeof(int32_t) * pages_fork_words(S, n, n_pages))
    return PMOE_ERR_WORKSPACE;
  if (!aligned16(workspace) || !aligned4(src) || !aligned4(dst) || !aligned4(keep) || !aligned4(ok))
    return PMOE_ERR_ALIGN;
  if ((s = ensure_device()) != PMOE_OK) return s;
  return launch_pages_fork(p, src, dst, keep, n, ok, static_cast<int32_t*>(workspace),
                           static_cast<cudaStream_t>(stream)) == cudaSuccess ? PMOE_OK
                                                                             : PMOE_ERR_CUDA;
}

int pmoe_pages_free(int32_t* refs, int n_pages, int page_size, int32_t* tables,
                    int64_t table_stride, int max_pages, int S, int32_t* lens,
                    const int32_t* slots, int n, int window, int sinks, void* stream) {
  Pool p;
  int s = make_pool(&p, nullptr, n_pages, 0, page_size, 0, refs, tables, table_stride, max_pages,
                    S, lens, true);
  if (s != PMOE_OK) return s;
  if (n < 0 || window < 0 || sinks < 0 || (n > 0 && !slots)) return PMOE_ERR_ARG;
  if (!aligned4(slots)) return PMOE_ERR_ALIGN;
  if (n == 0) return PMOE_OK;
  if ((s = ensure_device()) != PMOE_OK) return s;
  return launch_pages_free(p, slots, n, window, sinks, static_cast<cudaStream_t>(stream)) ==
                 cudaSuccess ? PMOE_OK : PMOE_ERR_CUDA;
}

int pmoe_pages_compact(uint16_t* pages, int n_pages, int chunks, int page_size, int D,
                       int32_t* refs, int32_t* tables, int64_t table_stride, int max_pages, int S,
                       int32_t* live, int32_t* remap, void* workspace, size_t workspace_bytes,
                       void* stream) {
  Pool p;
  int s = make_pool(&p, pages, n_pages, chunks, page_size, D, refs, tables, table_stride,
                    max_pages, S, nullptr, false);
  if (s != PMOE_OK) return s;
  if (chunks < 1 || D < 1 || !live || (n_pages > 0 && (!remap || !pages))) return PMOE_ERR_ARG;
  if (D % 8 != 0) return PMOE_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < sizeof(int32_t) * pages_compact_words(n_pages))
    return PMOE_ERR_WORKSPACE;
  if (!aligned16(workspace) || !aligned4(live) || !aligned4(remap)) return PMOE_ERR_ALIGN;
  if ((s = ensure_device()) != PMOE_OK) return s;
  return launch_pages_compact(p, live, remap, static_cast<int32_t*>(workspace),
                              static_cast<cudaStream_t>(stream)) == cudaSuccess ? PMOE_OK
                                                                                : PMOE_ERR_CUDA;
}

}  // extern "C"
