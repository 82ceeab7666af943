// Attention over the paged cache, one CTA per (packed query row, key/value head).
//   o = sum_j softmax_j(scale q.k_j) v_j over the keys that the row sees.
// One pass with a running maximum and sum per warp; the warps' parts are joined at the
// end.  No matrix instructions.
#include "paged.cuh"

namespace pmoe {

constexpr int kRowWarps = 8;

template <int D>
__global__ void __launch_bounds__(kRowWarps * 32) attn_rows_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float s_o[kRowWarps][D], s_m[kRowWarps], s_l[kRowWarps];
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.Hq / a.kv.Hkv;
  const int b = a.cu_q ? seq_of(a.cu_q, a.kv.B, t) : t;
  bool over = false;
  int p = -1, lo = 0, sink = 0;
  if (b >= 0) {
    const int len = kv_len_of(a.kv.kv_lens[b], a.kv.max_pages, a.kv.page_shift, &over);
    p = len - (a.cu_q ? a.cu_q[b + 1] - t : 1);
    if (p >= 0) visible_keys(p, a.window, a.sinks, &lo, &sink);
  }
  const int n = p >= 0 ? p + 1 - lo + sink : 0;  // visible keys: sinks first
  for (int g = 0; g < G; ++g) {
    const __nv_bfloat16* qr = a.q + t * a.q_stride_t + (h * G + g) * a.q_stride_h;
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      q[e] = __bfloat162float(qr[lane + 32 * e]);
      o[e] = 0.f;
    }
    for (int i = warp; i < n; i += kRowWarps) {
      const int j = i < sink ? i : lo + i - sink;
      const int page = page_of(a.kv, b, j);
      const int64_t row = ((int64_t(h) << a.kv.page_shift) + (j & ((1 << a.kv.page_shift) - 1))) * D;
      float s = 0.f;
      if (page >= 0) {
        const __nv_bfloat16* kr = a.kv.k + page * a.kv.k_page_stride + row;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], __bfloat162float(kr[lane + 32 * e]), s);
      }
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s = page >= 0 ? s * a.scale : NAN;
      const float m2 = fmaxf(m, s), base = m2 == -INFINITY ? 0.f : m2;
      const float keep = __expf(m - base), w = __expf(s - base);
      l = l * keep + w;
      m = m2;
      const __nv_bfloat16* vr = a.kv.v + (page >= 0 ? page : 0) * a.kv.v_page_stride + row;
#pragma unroll
      for (int e = 0; e < E; ++e)
        o[e] = o[e] * keep + (page >= 0 ? w * __bfloat162float(vr[lane + 32 * e]) : 0.f);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kRowWarps * 32) {
      float top = -INFINITY, sum = 0.f, acc = 0.f;
      for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, s_m[w]);
      const float base = top == -INFINITY ? 0.f : top;
      for (int w = 0; w < kRowWarps; ++w) {
        const float f = __expf(s_m[w] - base);
        sum += s_l[w] * f;
        acc += s_o[w][d] * f;
      }
      const float y = over ? NAN : n == 0 ? 0.f : acc / sum;
      a.out[(int64_t(t) * a.Hq + h * G + g) * D + d] = __float2bfloat16_rn(y);
    }
    __syncthreads();
  }
}

cudaError_t launch_attn_rows(const AttnArgs& a, cudaStream_t st) {
  if (a.T == 0) return cudaSuccess;
  const dim3 grid(a.T, a.kv.Hkv);
  switch (a.kv.D) {
    case 64: attn_rows_kernel<64><<<grid, kRowWarps * 32, 0, st>>>(a); break;
    case 128: attn_rows_kernel<128><<<grid, kRowWarps * 32, 0, st>>>(a); break;
    default: attn_rows_kernel<256><<<grid, kRowWarps * 32, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace pmoe
