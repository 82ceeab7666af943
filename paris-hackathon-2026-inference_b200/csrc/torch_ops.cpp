// torch.ops.paris_moe.*: the PyTorch operators over the C ABI of paris_moe.h.
//
// The drop-in surface for the reference's patched MoE forward
// (engine/kernels/moe_grouped_mlp.py:166-186, installed by
// engine/kernels/patch.py:43-84): moe_block takes the HF module's own bf16
// tensors, allocates its output and workspace with PyTorch's caching
// allocator, launches on the current CUDA stream and never synchronises the
// host, so it can be captured in a CUDA graph at the engine's decode buckets
// (engine/runtime/cuda_graphs.py:142).  A non-zero status from the library
// becomes a c10::Error (RuntimeError in Python) carrying the status code and
// its name; the CPU kernels only raise (no CPU fallback).  Meta
// kernels give the output shapes for tracing.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cstdint>
#include <optional>
#include <tuple>

#include "paris_moe.h"

namespace {

using at::Tensor;

#define PMOE_CALL(fn, ...)                                                             \
  do {                                                                                 \
    const int st_ = fn(__VA_ARGS__);                                                   \
    TORCH_CHECK(st_ == PMOE_OK, #fn " failed: status ", st_, " (",                      \
                pmoe_status_string(st_), ")");                                         \
  } while (0)

const uint16_t* bf(const Tensor& t) {
  return reinterpret_cast<const uint16_t*>(t.data_ptr());
}
uint16_t* bf_mut(Tensor& t) { return reinterpret_cast<uint16_t*>(t.data_ptr()); }

void check_bf16(const char* op, const char* name, const Tensor& t, const Tensor& x, int dim) {
  TORCH_CHECK(t.is_cuda(), "paris_moe.", op, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == x.device(), "paris_moe.", op, ": ", name, " is on ", t.device(),
              ", x on ", x.device());
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, "paris_moe.", op, ": ", name,
              " must be bf16, got ", t.scalar_type());
  TORCH_CHECK(t.is_contiguous(), "paris_moe.", op, ": ", name, " must be contiguous");
  TORCH_CHECK(t.dim() == dim, "paris_moe.", op, ": ", name, " must have ", dim,
              " dimensions, got ", t.dim());
}

struct Shapes {
  int T, H, E, I, Is;
};

// The HF module's layouts (modeling_qwen3_5_moe.py:713-792): gate.weight
// [E,H], experts.gate_up_proj [E,2I,H], experts.down_proj [E,H,I],
// shared_expert.{gate,up}_proj.weight [Is,H], down_proj.weight [H,Is],
// shared_expert_gate.weight [1,H].
Shapes check_block(const char* op, const Tensor& x, const Tensor& w_router,
                   const Tensor& w_gate_up, const Tensor& w_down, const Tensor& w_sh_gate,
                   const Tensor& w_sh_up, const Tensor& w_sh_down, const Tensor& w_sh_gvec) {
  check_bf16(op, "x", x, x, 2);
  check_bf16(op, "w_router", w_router, x, 2);
  check_bf16(op, "w_gate_up", w_gate_up, x, 3);
  check_bf16(op, "w_down", w_down, x, 3);
  check_bf16(op, "w_sh_gate", w_sh_gate, x, 2);
  check_bf16(op, "w_sh_up", w_sh_up, x, 2);
  check_bf16(op, "w_sh_down", w_sh_down, x, 2);
  check_bf16(op, "w_sh_gvec", w_sh_gvec, x, 2);
  Shapes s{int(x.size(0)), int(x.size(1)), int(w_router.size(0)), int(w_gate_up.size(1) / 2),
           int(w_sh_gate.size(0))};
  TORCH_CHECK(w_router.size(1) == s.H && w_gate_up.size(0) == s.E &&
                  w_gate_up.size(1) == 2 * s.I && w_gate_up.size(2) == s.H &&
                  w_down.size(0) == s.E && w_down.size(1) == s.H && w_down.size(2) == s.I &&
                  w_sh_up.size(0) == s.Is && w_sh_gate.size(1) == s.H &&
                  w_sh_up.size(1) == s.H && w_sh_down.size(0) == s.H &&
                  w_sh_down.size(1) == s.Is && w_sh_gvec.numel() == s.H,
              "paris_moe.", op, ": weight shapes do not match x [", s.T, ",", s.H,
              "] (E=", s.E, ", I=", s.I, ", Is=", s.Is, ")");
  return s;
}

void* stream_of(const Tensor& x) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
}

Tensor workspace(const Tensor& x, int T, int H, int E, int K, int I, int Is) {
  size_t nbytes = 0;
  PMOE_CALL(pmoe_workspace_size, T, H, E, K, I, Is, &nbytes);
  return at::empty({int64_t(nbytes)}, x.options().dtype(at::kByte));
}

// y[T,H] of the block.
//   top_k, flags             as pmoe_block_forward (flags: bit 0 shared expert,
//                            bit 1 routed experts)
//   expert_lo/hi             routed experts computed (hi < 0: E); ep_size 1 only
//   comm_handle != 0         a pmoe_comm_create handle: the full output on every
//                            rank via the NVLink exchanges (pmoe_block_forward_comm);
//                            ep_rank / ep_size must match the communicator
//   comm_handle 0, ep_size>1 this rank's partial: experts
//                            [ep_rank*E/ep_size, (ep_rank+1)*E/ep_size) and the
//                            shared expert of its token slice, for the caller to
//                            sum over ranks (the all_reduce of ep.py:140)
Tensor moe_block_cuda(const Tensor& x, const Tensor& w_router, const Tensor& w_gate_up,
                      const Tensor& w_down, const Tensor& w_sh_gate, const Tensor& w_sh_up,
                      const Tensor& w_sh_down, const Tensor& w_sh_gvec, int64_t top_k,
                      int64_t expert_lo, int64_t expert_hi, int64_t flags, int64_t ep_rank,
                      int64_t ep_size, int64_t comm_handle) {
  const Shapes s = check_block("moe_block", x, w_router, w_gate_up, w_down, w_sh_gate, w_sh_up,
                               w_sh_down, w_sh_gvec);
  TORCH_CHECK(ep_size >= 1 && ep_rank >= 0 && ep_rank < ep_size,
              "paris_moe.moe_block: bad ep_rank ", ep_rank, " / ep_size ", ep_size);
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({s.T, s.H}, x.options());
  if (s.T == 0) return y;
  const int K = int(top_k);
  Tensor ws = workspace(x, s.T, s.H, s.E, K, s.I, s.Is);
  void* st = stream_of(x);
  if (comm_handle != 0) {
    void* comm = reinterpret_cast<void*>(comm_handle);
    int rank = -1, world = 0;
    PMOE_CALL(pmoe_comm_info, comm, &rank, &world, nullptr, nullptr);
    TORCH_CHECK(rank == ep_rank && world == ep_size, "paris_moe.moe_block: ep_rank/ep_size ",
                ep_rank, "/", ep_size, " differ from the communicator's ", rank, "/", world);
    TORCH_CHECK(expert_lo == 0 && (expert_hi < 0 || expert_hi == s.E),
                "paris_moe.moe_block: an expert range cannot be combined with comm_handle");
    PMOE_CALL(pmoe_block_forward_comm, comm, bf(x), s.T, s.H, s.E, K, s.I, s.Is, bf(w_router),
              bf(w_gate_up), bf(w_down), bf(w_sh_gate), bf(w_sh_up), bf(w_sh_down),
              bf(w_sh_gvec), int(flags), bf_mut(y), ws.data_ptr(), size_t(ws.numel()), st,
              nullptr, 0);
    return y;
  }
  if (ep_size > 1) {
    TORCH_CHECK(expert_lo == 0 && (expert_hi < 0 || expert_hi == s.E),
                "paris_moe.moe_block: an expert range cannot be combined with ep_size > 1");
    const int r = int(ep_rank), n = int(ep_size);
    PMOE_CALL(pmoe_block_forward_ep, bf(x), s.T, s.H, s.E, K, s.I, s.Is, bf(w_router),
              bf(w_gate_up), bf(w_down), bf(w_sh_gate), bf(w_sh_up), bf(w_sh_down),
              bf(w_sh_gvec), int(int64_t(r) * s.E / n), int(int64_t(r + 1) * s.E / n),
              int(int64_t(r) * s.T / n), int(int64_t(r + 1) * s.T / n), int(flags), nullptr, 0,
              r, n, 0, bf_mut(y), ws.data_ptr(), size_t(ws.numel()), st);
    return y;
  }
  const int hi = expert_hi < 0 ? s.E : int(expert_hi);
  PMOE_CALL(pmoe_block_forward, bf(x), s.T, s.H, s.E, K, s.I, s.Is, bf(w_router), bf(w_gate_up),
            bf(w_down), bf(w_sh_gate), bf(w_sh_up), bf(w_sh_down), bf(w_sh_gvec),
            int(expert_lo), hi, int(flags), bf_mut(y), ws.data_ptr(), size_t(ws.numel()), st);
  return y;
}

Tensor moe_block_meta(const Tensor& x, const Tensor&, const Tensor&, const Tensor&,
                      const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t,
                      int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) {
  return at::empty_like(x);
}

// One MoE-only decoder layer x + block(RMSNorm(x)) (pmoe_layer_forward), on one
// GPU.
Tensor moe_layer_cuda(const Tensor& x, const Tensor& w_norm, double eps, const Tensor& w_router,
                      const Tensor& w_gate_up, const Tensor& w_down, const Tensor& w_sh_gate,
                      const Tensor& w_sh_up, const Tensor& w_sh_down, const Tensor& w_sh_gvec,
                      int64_t top_k, int64_t flags) {
  const Shapes s = check_block("moe_layer", x, w_router, w_gate_up, w_down, w_sh_gate, w_sh_up,
                               w_sh_down, w_sh_gvec);
  check_bf16("moe_layer", "w_norm", w_norm, x, 1);
  TORCH_CHECK(w_norm.size(0) == s.H, "paris_moe.moe_layer: w_norm must be [", s.H, "]");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({s.T, s.H}, x.options());
  if (s.T == 0) return y;
  const int K = int(top_k);
  Tensor ws = workspace(x, s.T, s.H, s.E, K, s.I, s.Is);
  PMOE_CALL(pmoe_layer_forward, bf(x), s.T, s.H, s.E, K, s.I, s.Is, bf(w_norm), float(eps),
            bf(w_router), bf(w_gate_up), bf(w_down), bf(w_sh_gate), bf(w_sh_up), bf(w_sh_down),
            bf(w_sh_gvec), 0, s.E, 0, s.T, int(flags), nullptr, 0, 0, 1, 0, bf_mut(y),
            ws.data_ptr(), size_t(ws.numel()), stream_of(x));
  return y;
}

Tensor moe_layer_meta(const Tensor& x, const Tensor&, double, const Tensor&, const Tensor&,
                      const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                      int64_t, int64_t) {
  return at::empty_like(x);
}

// Qwen3_5MoeRMSNorm (modeling_qwen3_5_moe.py:795-812).
Tensor rmsnorm_cuda(const Tensor& x, const Tensor& w_norm, double eps) {
  check_bf16("rmsnorm", "x", x, x, 2);
  check_bf16("rmsnorm", "w_norm", w_norm, x, 1);
  TORCH_CHECK(w_norm.size(0) == x.size(1), "paris_moe.rmsnorm: w_norm must be [H]");
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty_like(x);
  PMOE_CALL(pmoe_rmsnorm, bf(x), int(x.size(0)), int(x.size(1)), bf(w_norm), float(eps),
            bf_mut(y), stream_of(x));
  return y;
}

Tensor rmsnorm_meta(const Tensor& x, const Tensor&, double) { return at::empty_like(x); }

using RouteOut = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

// Router + top-k + CSR dispatch (pmoe_route): (topk_idx i32 [T,k], topk_w f32
// [T,k], offsets i32 [E+1], sorted_tok i32 [T*k], sorted_slot i32 [T*k],
// shared_gate f32 [T]).
RouteOut moe_route_cuda(const Tensor& x, const Tensor& w_router, const Tensor& w_sh_gvec,
                        int64_t k) {
  check_bf16("moe_route", "x", x, x, 2);
  check_bf16("moe_route", "w_router", w_router, x, 2);
  check_bf16("moe_route", "w_sh_gvec", w_sh_gvec, x, 2);
  const int T = int(x.size(0)), H = int(x.size(1)), E = int(w_router.size(0)), K = int(k);
  TORCH_CHECK(w_router.size(1) == H && w_sh_gvec.numel() == H,
              "paris_moe.moe_route: weight shapes do not match x");
  const c10::cuda::CUDAGuard guard(x.device());
  const auto i32 = x.options().dtype(at::kInt), f32 = x.options().dtype(at::kFloat);
  Tensor idx = at::empty({T, K}, i32), w = at::empty({T, K}, f32);
  Tensor offs = at::zeros({E + 1}, i32), stok = at::empty({int64_t(T) * K}, i32);
  Tensor sslot = at::empty({int64_t(T) * K}, i32), sg = at::empty({T}, f32);
  if (T == 0) return {idx, w, offs, stok, sslot, sg};
  Tensor ws = workspace(x, T, H, E, K, 64, 64);
  PMOE_CALL(pmoe_route, bf(x), T, H, E, K, bf(w_router), bf(w_sh_gvec), idx.data_ptr<int32_t>(),
            w.data_ptr<float>(), offs.data_ptr<int32_t>(), stok.data_ptr<int32_t>(),
            sslot.data_ptr<int32_t>(), sg.data_ptr<float>(), ws.data_ptr(), size_t(ws.numel()),
            stream_of(x));
  return {idx, w, offs, stok, sslot, sg};
}

RouteOut moe_route_meta(const Tensor& x, const Tensor& w_router, const Tensor&, int64_t k) {
  const int64_t T = x.size(0), E = w_router.size(0);
  const auto i32 = x.options().dtype(at::kInt), f32 = x.options().dtype(at::kFloat);
  return {at::empty({T, k}, i32),     at::empty({T, k}, f32),     at::empty({E + 1}, i32),
          at::empty({T * k}, i32), at::empty({T * k}, i32), at::empty({T}, f32)};
}

// ---- the attention half ------------------------------------------------------
using OptTensor = std::optional<Tensor>;

void check_int(const char* op, const char* name, const Tensor& t, at::ScalarType type, int dim,
               const Tensor& x) {
  TORCH_CHECK(t.is_cuda(), "paris_moe.", op, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == x.device(), "paris_moe.", op, ": ", name, " is on ", t.device(),
              ", expected ", x.device());
  TORCH_CHECK(t.scalar_type() == type, "paris_moe.", op, ": ", name, " must be ", type, ", got ",
              t.scalar_type());
  TORCH_CHECK(t.dim() == dim, "paris_moe.", op, ": ", name, " must have ", dim,
              " dimensions, got ", t.dim());
  TORCH_CHECK(t.numel() == 0 || t.size(dim - 1) <= 1 || t.stride(dim - 1) == 1, "paris_moe.", op,
              ": ", name, "'s last dimension must be contiguous");
}

int to_int(const char* op, const char* name, int64_t v) {
  TORCH_CHECK(v >= INT32_MIN && v <= INT32_MAX, "paris_moe.", op, ": ", name, " ", v,
              " is beyond 32 bits");
  return int(v);
}

// Element stride of a dimension; one of at most one entry is never stepped over.
int64_t stride_of(const Tensor& t, int dim) { return t.size(dim) <= 1 ? 0 : t.stride(dim); }

void check_no_grad(const char* op, const char* name, const Tensor& t) {
  TORCH_CHECK(!(t.requires_grad() && at::GradMode::is_enabled()), "paris_moe.", op, ": ", name,
              " requires grad, and the operator has no backward pass (call it under no_grad)");
}

// Rows [T, heads, D]: any token and head stride, contiguous heads.
void check_rows(const char* op, const char* name, const Tensor& t, const Tensor& x) {
  check_no_grad(op, name, t);
  TORCH_CHECK(t.is_cuda(), "paris_moe.", op, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == x.device(), "paris_moe.", op, ": ", name, " is on ", t.device(),
              ", expected ", x.device());
  TORCH_CHECK(t.scalar_type() == at::kBFloat16, "paris_moe.", op, ": ", name,
              " must be bf16, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == 3, "paris_moe.", op, ": ", name, " must be [tokens, heads, D]");
  TORCH_CHECK(t.size(2) <= 1 || t.stride(2) == 1, "paris_moe.", op, ": ", name,
              "'s last dimension must be contiguous");
}

// A cache view [n_pages, Hkv, page_size, D]: any page stride, contiguous pages.
struct CacheView {
  int n_pages, Hkv, page_size, D, B, max_pages;
  int64_t k_stride, v_stride, table_stride;
};
CacheView check_cache(const char* op, const Tensor& q, const Tensor& k, const Tensor& v,
                      const Tensor& table, const Tensor& lens) {
  for (const Tensor* t : {&k, &v}) {
    const char* name = t == &k ? "k_pages" : "v_pages";
    check_no_grad(op, name, *t);
    TORCH_CHECK(t->is_cuda() && t->device() == q.device(), "paris_moe.", op, ": ", name,
                " must be a CUDA tensor on ", q.device());
    TORCH_CHECK(t->scalar_type() == at::kBFloat16, "paris_moe.", op, ": ", name,
                " must be bf16, got ", t->scalar_type());
    TORCH_CHECK(t->dim() == 4, "paris_moe.", op, ": ", name,
                " must be [n_pages, kv_heads, page_size, D]");
    const int64_t d = t->size(3), ps = t->size(2);
    TORCH_CHECK(t->numel() == 0 || ((d <= 1 || t->stride(3) == 1) && (ps <= 1 || t->stride(2) == d) &&
                                    (t->size(1) <= 1 || t->stride(1) == ps * d)),
                "paris_moe.", op, ": ", name, "'s last three dimensions must be contiguous");
  }
  TORCH_CHECK(k.sizes() == v.sizes(), "paris_moe.", op, ": k_pages and v_pages differ in shape");
  check_int(op, "page_table", table, at::kInt, 2, q);
  check_int(op, "kv_lens", lens, at::kInt, 1, q);
  TORCH_CHECK(table.size(0) == lens.size(0), "paris_moe.", op, ": page_table has ", table.size(0),
              " rows, kv_lens ", lens.size(0));
  const int64_t page = k.size(1) * k.size(2) * k.size(3);
  return {to_int(op, "n_pages", k.size(0)), to_int(op, "kv_heads", k.size(1)),
          to_int(op, "page_size", k.size(2)), to_int(op, "D", k.size(3)),
          to_int(op, "batch", lens.size(0)), to_int(op, "max_pages", table.size(1)),
          k.size(0) <= 1 ? page : k.stride(0), v.size(0) <= 1 ? page : v.stride(0),
          table.size(0) <= 1 ? table.size(1) : table.stride(0)};
}

const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }
int32_t* i32_mut(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }
uint16_t* pages_mut(const Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }

const int32_t* check_cu(const char* op, const Tensor& cu, const CacheView& c, const Tensor& q) {
  check_int(op, "cu_q", cu, at::kInt, 1, q);
  TORCH_CHECK(cu.size(0) == c.B + 1, "paris_moe.", op, ": cu_q has ", cu.size(0),
              " entries, expected ", c.B + 1);
  return i32(cu);
}

Tensor rope_append_cuda(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions,
                        const Tensor& inv_freq, at::IntArrayRef sections, bool interleaved,
                        const Tensor& k_pages, const Tensor& v_pages, const Tensor& page_table,
                        const Tensor& kv_lens, const OptTensor& cu_q, const OptTensor& w_qnorm,
                        const OptTensor& w_knorm, double eps, double mscale) {
  const char* op = "rope_append";
  check_rows(op, "q", q, q);
  check_rows(op, "k", k, q);
  check_rows(op, "v", v, q);
  const CacheView c = check_cache(op, q, k_pages, v_pages, page_table, kv_lens);
  const int T = to_int(op, "tokens", q.size(0)), Hq = to_int(op, "heads", q.size(1));
  TORCH_CHECK(q.size(2) == c.D, "paris_moe.rope_append: q has D ", q.size(2), ", the cache ", c.D);
  TORCH_CHECK(k.size(0) == T && k.size(1) == c.Hkv && k.size(2) == c.D && v.sizes() == k.sizes(),
              "paris_moe.rope_append: k and v must be [", T, ", ", c.Hkv, ", ", c.D, "]");
  check_int(op, "positions", positions, at::kLong, 2, q);
  check_int(op, "inv_freq", inv_freq, at::kFloat, 1, q);
  TORCH_CHECK(positions.size(1) == T, "paris_moe.rope_append: positions must be [axes, ", T, "]");
  TORCH_CHECK(positions.size(0) >= 1 && positions.size(0) <= 4 &&
                  int64_t(sections.size()) == positions.size(0),
              "paris_moe.rope_append: one section for each of positions' 1 to 4 axes");
  int sec[4] = {0, 0, 0, 0};
  int64_t half = 0;
  for (size_t i = 0; i < sections.size(); ++i) {
    sec[i] = to_int(op, "section", sections[i]);
    TORCH_CHECK(sec[i] >= 0, "paris_moe.rope_append: sections must not be negative");
    half += sec[i];
  }
  TORCH_CHECK(half == inv_freq.size(0) && 2 * half <= c.D, "paris_moe.rope_append: sections add up to ",
              half, ", inv_freq has ", inv_freq.size(0), " entries, D/2 is ", c.D / 2);
  for (const OptTensor* w : {&w_qnorm, &w_knorm})
    if (w->has_value()) {
      check_no_grad(op, "norm weight", **w);
      check_bf16(op, "norm weight", **w, q, 1);
      TORCH_CHECK((*w)->size(0) == c.D, "paris_moe.rope_append: norm weights must be [", c.D, "]");
    }
  TORCH_CHECK(cu_q.has_value() || T == c.B, "paris_moe.rope_append: ", T, " tokens for ", c.B,
              " sequences need cu_q");
  const int32_t* cu = cu_q.has_value() ? check_cu(op, *cu_q, c, q) : nullptr;
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({T, Hq, c.D}, q.options());
  PMOE_CALL(pmoe_rope_append, bf(q), stride_of(q, 0), stride_of(q, 1), bf(k), stride_of(k, 0),
            stride_of(k, 1), bf(v), stride_of(v, 0), stride_of(v, 1), T, Hq, c.Hkv, c.D,
            static_cast<const int64_t*>(positions.data_ptr()),
            positions.size(0) <= 1 ? int64_t(T) : positions.stride(0), int(positions.size(0)), sec,
            interleaved ? 1 : 0, static_cast<const float*>(inv_freq.data_ptr()), int(2 * half),
            w_qnorm.has_value() ? bf(*w_qnorm) : nullptr,
            w_knorm.has_value() ? bf(*w_knorm) : nullptr, float(eps), float(mscale),
            pages_mut(k_pages), pages_mut(v_pages), c.k_stride, c.v_stride, c.n_pages, c.page_size,
            i32(page_table), c.table_stride, c.max_pages, i32(kv_lens), cu, c.B, bf_mut(out),
            stream_of(q));
  return out;
}
Tensor rope_append_meta(const Tensor& q, const Tensor&, const Tensor&, const Tensor&,
                        const Tensor&, at::IntArrayRef, bool, const Tensor&, const Tensor&,
                        const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                        const OptTensor&, double, double) {
  return at::empty(q.sizes(), q.options());
}

Tensor attn_decode_cuda(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                        const Tensor& page_table, const Tensor& kv_lens, double scale,
                        int64_t window, int64_t sinks) {
  const char* op = "attn_decode";
  check_rows(op, "q", q, q);
  const CacheView c = check_cache(op, q, k_pages, v_pages, page_table, kv_lens);
  const int Hq = to_int(op, "heads", q.size(1));
  TORCH_CHECK(q.size(0) == c.B && q.size(2) == c.D, "paris_moe.attn_decode: q must be [", c.B,
              ", heads, ", c.D, "]");
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({c.B, Hq, c.D}, q.options());
  size_t nbytes = 0;
  PMOE_CALL(pmoe_attn_decode_workspace, c.B, Hq, c.Hkv, c.D, &nbytes);
  Tensor ws = at::empty({int64_t(nbytes)}, q.options().dtype(at::kByte));
  PMOE_CALL(pmoe_attn_decode, bf(q), stride_of(q, 0), stride_of(q, 1), c.B, Hq, c.Hkv, c.D,
            bf(k_pages), bf(v_pages), c.k_stride, c.v_stride, c.n_pages, c.page_size,
            i32(page_table), c.table_stride, c.max_pages, i32(kv_lens), float(scale),
            to_int(op, "window", window), to_int(op, "sinks", sinks), bf_mut(out), ws.data_ptr(),
            nbytes, stream_of(q));
  return out;
}
Tensor attn_decode_meta(const Tensor& q, const Tensor&, const Tensor&, const Tensor&,
                        const Tensor&, double, int64_t, int64_t) {
  return at::empty(q.sizes(), q.options());
}

Tensor attn_prefill_cuda(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                         const Tensor& page_table, const Tensor& kv_lens, const Tensor& cu_q,
                         double scale, int64_t window, int64_t sinks) {
  const char* op = "attn_prefill";
  check_rows(op, "q", q, q);
  const CacheView c = check_cache(op, q, k_pages, v_pages, page_table, kv_lens);
  const int T = to_int(op, "tokens", q.size(0)), Hq = to_int(op, "heads", q.size(1));
  TORCH_CHECK(q.size(2) == c.D, "paris_moe.attn_prefill: q has D ", q.size(2), ", the cache ", c.D);
  const int32_t* cu = check_cu(op, cu_q, c, q);
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor out = at::empty({T, Hq, c.D}, q.options());
  size_t nbytes = 0;
  PMOE_CALL(pmoe_attn_prefill_workspace, T, c.B, Hq, c.Hkv, c.D, c.page_size, c.max_pages, &nbytes);
  Tensor ws;
  if (nbytes > 0) ws = at::empty({int64_t(nbytes)}, q.options().dtype(at::kByte));
  PMOE_CALL(pmoe_attn_prefill, bf(q), stride_of(q, 0), stride_of(q, 1), T, Hq, c.Hkv, c.D,
            bf(k_pages), bf(v_pages), c.k_stride, c.v_stride, c.n_pages, c.page_size,
            i32(page_table), c.table_stride, c.max_pages, i32(kv_lens), cu, c.B, float(scale),
            to_int(op, "window", window), to_int(op, "sinks", sinks), bf_mut(out),
            nbytes > 0 ? ws.data_ptr() : nullptr, nbytes, stream_of(q));
  return out;
}
Tensor attn_prefill_meta(const Tensor& q, const Tensor&, const Tensor&, const Tensor&,
                         const Tensor&, const Tensor&, double, int64_t, int64_t) {
  return at::empty(q.sizes(), q.options());
}

// The bookkeeping tensors of a page pool.
struct PoolView {
  int n_pages, max_pages, S;
  int64_t table_stride;
};
PoolView check_pool(const char* op, const Tensor& refs, const Tensor& tables) {
  check_int(op, "refs", refs, at::kInt, 1, refs);
  check_int(op, "tables", tables, at::kInt, 2, refs);
  return {to_int(op, "n_pages", refs.size(0)), to_int(op, "max_pages", tables.size(1)),
          to_int(op, "sequences", tables.size(0)),
          tables.size(0) <= 1 ? tables.size(1) : tables.stride(0)};
}
void check_lens(const char* op, const Tensor& lens, const PoolView& p, const Tensor& refs) {
  check_int(op, "lens", lens, at::kInt, 1, refs);
  TORCH_CHECK(lens.size(0) == p.S, "paris_moe.", op, ": lens has ", lens.size(0),
              " entries, tables ", p.S, " rows");
}
int check_list(const char* op, const char* name, const Tensor& t, int64_t n, const Tensor& refs) {
  check_int(op, name, t, at::kInt, 1, refs);
  TORCH_CHECK(t.size(0) == n, "paris_moe.", op, ": ", name, " has ", t.size(0),
              " entries, expected ", n);
  return to_int(op, name, n);
}
// The pool [n_pages, ..., page_size, D], contiguous.
struct PageShape {
  int chunks, page_size, D;
};
PageShape check_pages(const char* op, const Tensor& pages, const Tensor& refs) {
  TORCH_CHECK(pages.is_cuda() && pages.device() == refs.device(), "paris_moe.", op,
              ": pages must be a CUDA tensor on ", refs.device());
  TORCH_CHECK(pages.scalar_type() == at::kBFloat16, "paris_moe.", op, ": pages must be bf16, got ",
              pages.scalar_type());
  TORCH_CHECK(pages.dim() >= 3 && pages.is_contiguous(), "paris_moe.", op,
              ": pages must be contiguous [n_pages, ..., page_size, D]");
  TORCH_CHECK(pages.size(0) == refs.size(0), "paris_moe.", op, ": pages holds ", pages.size(0),
              " pages, refs ", refs.size(0));
  int64_t chunks = 1;
  for (int64_t i = 1; i + 2 < pages.dim(); ++i) chunks *= pages.size(i);
  return {to_int(op, "chunks", chunks), to_int(op, "page_size", pages.size(pages.dim() - 2)),
          to_int(op, "D", pages.size(pages.dim() - 1))};
}
Tensor pages_workspace(const Tensor& refs, int S, int n, int n_pages, size_t* nbytes) {
  PMOE_CALL(pmoe_pages_workspace, S, n, n_pages, nbytes);
  return at::empty({int64_t(*nbytes)}, refs.options().dtype(at::kByte));
}

Tensor pages_grow_cuda(const Tensor& refs, const Tensor& tables, const Tensor& lens,
                       const Tensor& slots, const Tensor& add, int64_t page_size) {
  const char* op = "pages_grow";
  const PoolView p = check_pool(op, refs, tables);
  check_lens(op, lens, p, refs);
  const int n = check_list(op, "slots", slots, slots.numel(), refs);
  check_list(op, "add", add, n, refs);
  const c10::cuda::CUDAGuard guard(refs.device());
  Tensor ok = at::empty({n}, refs.options());
  size_t nbytes = 0;
  Tensor ws = pages_workspace(refs, p.S, n, p.n_pages, &nbytes);
  PMOE_CALL(pmoe_pages_grow, i32_mut(refs), p.n_pages, to_int(op, "page_size", page_size),
            i32_mut(tables), p.table_stride, p.max_pages, p.S, i32_mut(lens), i32(slots), i32(add),
            n, i32_mut(ok), ws.data_ptr(), nbytes, stream_of(refs));
  return ok;
}
Tensor pages_grow_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor& slots,
                       const Tensor&, int64_t) {
  return at::empty(slots.sizes(), slots.options().dtype(at::kInt));
}

Tensor pages_fork_cuda(const Tensor& pages, const Tensor& refs, const Tensor& tables,
                       const Tensor& lens, const Tensor& src, const Tensor& dst,
                       const Tensor& keep) {
  const char* op = "pages_fork";
  const PoolView p = check_pool(op, refs, tables);
  check_lens(op, lens, p, refs);
  const PageShape g = check_pages(op, pages, refs);
  const int n = check_list(op, "src", src, src.numel(), refs);
  check_list(op, "dst", dst, n, refs);
  check_list(op, "keep", keep, n, refs);
  const c10::cuda::CUDAGuard guard(refs.device());
  Tensor ok = at::empty({n}, refs.options());
  size_t nbytes = 0;
  Tensor ws = pages_workspace(refs, p.S, n, p.n_pages, &nbytes);
  PMOE_CALL(pmoe_pages_fork, pages_mut(pages), p.n_pages, g.chunks, g.page_size, g.D,
            i32_mut(refs), i32_mut(tables), p.table_stride, p.max_pages, p.S, i32_mut(lens),
            i32(src), i32(dst), i32(keep), n, i32_mut(ok), ws.data_ptr(), nbytes, stream_of(refs));
  return ok;
}
Tensor pages_fork_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                       const Tensor& src, const Tensor&, const Tensor&) {
  return at::empty(src.sizes(), src.options().dtype(at::kInt));
}

void pages_free_cuda(const Tensor& refs, const Tensor& tables, const Tensor& lens,
                     const Tensor& slots, int64_t page_size, int64_t window, int64_t sinks) {
  const char* op = "pages_free";
  const PoolView p = check_pool(op, refs, tables);
  check_lens(op, lens, p, refs);
  const int n = check_list(op, "slots", slots, slots.numel(), refs);
  const c10::cuda::CUDAGuard guard(refs.device());
  PMOE_CALL(pmoe_pages_free, i32_mut(refs), p.n_pages, to_int(op, "page_size", page_size),
            i32_mut(tables), p.table_stride, p.max_pages, p.S, i32_mut(lens), i32(slots), n,
            to_int(op, "window", window), to_int(op, "sinks", sinks), stream_of(refs));
}
void pages_free_meta(const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t, int64_t,
                     int64_t) {}

std::tuple<Tensor, Tensor> pages_compact_cuda(const Tensor& pages, const Tensor& refs,
                                              const Tensor& tables) {
  const char* op = "pages_compact";
  const PoolView p = check_pool(op, refs, tables);
  const PageShape g = check_pages(op, pages, refs);
  const c10::cuda::CUDAGuard guard(refs.device());
  Tensor live = at::empty({1}, refs.options()), remap = at::empty({p.n_pages}, refs.options());
  size_t nbytes = 0;
  Tensor ws = pages_workspace(refs, p.S, 0, p.n_pages, &nbytes);
  PMOE_CALL(pmoe_pages_compact, pages_mut(pages), p.n_pages, g.chunks, g.page_size, g.D,
            i32_mut(refs), i32_mut(tables), p.table_stride, p.max_pages, p.S, i32_mut(live),
            i32_mut(remap), ws.data_ptr(), nbytes, stream_of(refs));
  return {live, remap};
}
std::tuple<Tensor, Tensor> pages_compact_meta(const Tensor&, const Tensor& refs, const Tensor&) {
  return {at::empty({1}, refs.options()), at::empty(refs.sizes(), refs.options())};
}

// CPU tensors: a clear error instead of a computation (there is no CPU path).
[[noreturn]] void no_cpu(const char* op) {
  TORCH_CHECK(false, "paris_moe.", op, ": tensors must be CUDA (no CPU fallback)");
}
Tensor moe_block_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                     const Tensor&, const Tensor&, const Tensor&, int64_t, int64_t, int64_t,
                     int64_t, int64_t, int64_t, int64_t) {
  no_cpu("moe_block");
}
Tensor moe_layer_cpu(const Tensor&, const Tensor&, double, const Tensor&, const Tensor&,
                     const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                     int64_t, int64_t) {
  no_cpu("moe_layer");
}
Tensor rmsnorm_cpu(const Tensor&, const Tensor&, double) { no_cpu("rmsnorm"); }
RouteOut moe_route_cpu(const Tensor&, const Tensor&, const Tensor&, int64_t) {
  no_cpu("moe_route");
}
Tensor rope_append_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                       at::IntArrayRef, bool, const Tensor&, const Tensor&, const Tensor&,
                       const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, double,
                       double) {
  no_cpu("rope_append");
}
Tensor attn_decode_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                       double, int64_t, int64_t) {
  no_cpu("attn_decode");
}
Tensor attn_prefill_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                        const Tensor&, double, int64_t, int64_t) {
  no_cpu("attn_prefill");
}
Tensor pages_grow_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                      int64_t) {
  no_cpu("pages_grow");
}
Tensor pages_fork_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                      const Tensor&, const Tensor&) {
  no_cpu("pages_fork");
}
void pages_free_cpu(const Tensor&, const Tensor&, const Tensor&, const Tensor&, int64_t, int64_t,
                    int64_t) {
  no_cpu("pages_free");
}
std::tuple<Tensor, Tensor> pages_compact_cpu(const Tensor&, const Tensor&, const Tensor&) {
  no_cpu("pages_compact");
}

}  // namespace

TORCH_LIBRARY(paris_moe, m) {
  m.def(
      "moe_block(Tensor x, Tensor w_router, Tensor w_gate_up, Tensor w_down, Tensor w_sh_gate, "
      "Tensor w_sh_up, Tensor w_sh_down, Tensor w_sh_gvec, int top_k=8, int expert_lo=0, "
      "int expert_hi=-1, int flags=3, *, int ep_rank=0, int ep_size=1, int comm_handle=0) "
      "-> Tensor");
  m.def(
      "moe_layer(Tensor x, Tensor w_norm, float eps, Tensor w_router, Tensor w_gate_up, "
      "Tensor w_down, Tensor w_sh_gate, Tensor w_sh_up, Tensor w_sh_down, Tensor w_sh_gvec, "
      "int top_k=8, int flags=3) -> Tensor");
  m.def("rmsnorm(Tensor x, Tensor w_norm, float eps) -> Tensor");
  m.def(
      "moe_route(Tensor x, Tensor w_router, Tensor w_sh_gvec, int k) -> "
      "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "rope_append(Tensor q, Tensor k, Tensor v, Tensor positions, Tensor inv_freq, "
      "int[] sections, bool interleaved, Tensor(a!) k_pages, Tensor(b!) v_pages, "
      "Tensor page_table, Tensor kv_lens, *, Tensor? cu_q=None, Tensor? w_qnorm=None, "
      "Tensor? w_knorm=None, float eps=1e-6, float mscale=1.0) -> Tensor");
  m.def(
      "attn_decode(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor kv_lens, "
      "float scale, int window=0, int sinks=0) -> Tensor");
  m.def(
      "attn_prefill(Tensor q, Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor kv_lens, "
      "Tensor cu_q, float scale, int window=0, int sinks=0) -> Tensor");
  m.def(
      "pages_grow(Tensor(a!) refs, Tensor(b!) tables, Tensor(c!) lens, Tensor slots, Tensor add, "
      "int page_size) -> Tensor");
  m.def(
      "pages_fork(Tensor(a!) pages, Tensor(b!) refs, Tensor(c!) tables, Tensor(d!) lens, "
      "Tensor src, Tensor dst, Tensor keep) -> Tensor");
  m.def(
      "pages_free(Tensor(a!) refs, Tensor(b!) tables, Tensor(c!) lens, Tensor slots, "
      "int page_size, int window=0, int sinks=0) -> ()");
  m.def(
      "pages_compact(Tensor(a!) pages, Tensor(b!) refs, Tensor(c!) tables) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(paris_moe, CUDA, m) {
  m.impl("moe_block", &moe_block_cuda);
  m.impl("moe_layer", &moe_layer_cuda);
  m.impl("rmsnorm", &rmsnorm_cuda);
  m.impl("moe_route", &moe_route_cuda);
  m.impl("rope_append", &rope_append_cuda);
  m.impl("attn_decode", &attn_decode_cuda);
  m.impl("attn_prefill", &attn_prefill_cuda);
  m.impl("pages_grow", &pages_grow_cuda);
  m.impl("pages_fork", &pages_fork_cuda);
  m.impl("pages_free", &pages_free_cuda);
  m.impl("pages_compact", &pages_compact_cuda);
}

TORCH_LIBRARY_IMPL(paris_moe, CPU, m) {
  m.impl("moe_block", &moe_block_cpu);
  m.impl("moe_layer", &moe_layer_cpu);
  m.impl("rmsnorm", &rmsnorm_cpu);
  m.impl("moe_route", &moe_route_cpu);
  m.impl("rope_append", &rope_append_cpu);
  m.impl("attn_decode", &attn_decode_cpu);
  m.impl("attn_prefill", &attn_prefill_cpu);
  m.impl("pages_grow", &pages_grow_cpu);
  m.impl("pages_fork", &pages_fork_cpu);
  m.impl("pages_free", &pages_free_cpu);
  m.impl("pages_compact", &pages_compact_cpu);
}

TORCH_LIBRARY_IMPL(paris_moe, Meta, m) {
  m.impl("moe_block", &moe_block_meta);
  m.impl("moe_layer", &moe_layer_meta);
  m.impl("rmsnorm", &rmsnorm_meta);
  m.impl("moe_route", &moe_route_meta);
  m.impl("rope_append", &rope_append_meta);
  m.impl("attn_decode", &attn_decode_meta);
  m.impl("attn_prefill", &attn_prefill_meta);
  m.impl("pages_grow", &pages_grow_meta);
  m.impl("pages_fork", &pages_fork_meta);
  m.impl("pages_free", &pages_free_meta);
  m.impl("pages_compact", &pages_compact_meta);
}

// The attention half serves only; its operators have no backward pass (and raise where their
// inputs ask for one), so calls go past autograd's boxed fallback, which costs several
// microseconds for a dozen tensors.
TORCH_LIBRARY_IMPL(paris_moe, Autograd, m) {
  m.impl("rope_append", torch::CppFunction::makeFallthrough());
  m.impl("attn_decode", torch::CppFunction::makeFallthrough());
  m.impl("attn_prefill", torch::CppFunction::makeFallthrough());
  m.impl("pages_grow", torch::CppFunction::makeFallthrough());
  m.impl("pages_fork", torch::CppFunction::makeFallthrough());
  m.impl("pages_free", torch::CppFunction::makeFallthrough());
  m.impl("pages_compact", torch::CppFunction::makeFallthrough());
}
