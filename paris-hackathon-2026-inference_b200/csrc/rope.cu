// Rotary positions with several axes, the optional per-head RMSNorm, and the write of
// keys and values into the cache's pages.
//
// Pair (i, i + half) of a query or key row turns by angle = pos[axis(i)] * inv_freq[i]:
//   y_i = x_i c - x_{i+half} s,   y_{i+half} = x_{i+half} c + x_i s.
// The angle is formed and reduced to (-pi, pi] in 64 bits: at position 1e6 a 32-bit
// product is already off by 0.03 rad.  One rounding to bf16, at the store.
#include "paged.cuh"

namespace pmoe {

constexpr int kRopeThreads = 256;

__device__ __forceinline__ int rope_axis(const RopeArgs& a, int i) {
  if (a.interleaved) {
    const int x = i % a.axes;
    return i < a.axes * a.sections[x] ? x : 0;
  }
  int x = 0, end = a.sections[0];
  while (x + 1 < a.axes && i >= end) end += a.sections[++x];
  return x;
}

// One CTA per token: the token's cos/sin once in shared memory, then a warp per row
// (D/8 lanes of 16 bytes; the pair's other half comes from lane +- half/8).
template <int D>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const RopeArgs a) {
  __shared__ float s_cos[128], s_sin[128];
  __shared__ int64_t s_dst[2];  // element offsets of the token's key / value row, or -1
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < a.half; i += kRopeThreads) {
    const double turns = double(a.positions[rope_axis(a, i) * a.pos_stride + t]) *
                         double(a.inv_freq[i]) * 0.15915494309189533577;
    float s, c;
    sincospif(float(2.0 * (turns - rint(turns))), &s, &c);
    s_cos[i] = c * a.mscale;
    s_sin[i] = s * a.mscale;
  }
  if (tid == 0) {
    const int b = a.cu_q ? seq_of(a.cu_q, a.kv.B, t) : t;
    int64_t kd = -1, vd = -1;
    if (b >= 0 && b < a.kv.B) {
      const int after = a.cu_q ? a.cu_q[b + 1] - t : 1;  // tokens from t to the sequence's end
      const int j = a.kv.kv_lens[b] - after;
      const int p = j >= 0 ? page_of(a.kv, b, j) : -1;
      if (p >= 0) {
        const int64_t row = int64_t(j & ((1 << a.kv.page_shift) - 1)) * D;
        kd = p * a.kv.k_page_stride + row;
        vd = p * a.kv.v_page_stride + row;
      }
    }
    s_dst[0] = kd;
    s_dst[1] = vd;
  }
  __syncthreads();
  constexpr int kLanes = D / 8;            // lanes of a row
  constexpr int kRowsPerWarp = 32 / kLanes;
  const int rl = lane % kLanes;            // this lane's 8 elements: 8*rl ..
  const int rows = a.Hq + 2 * a.kv.Hkv;
  const int64_t head_stride = int64_t(D) << a.kv.page_shift;
  for (int r0 = warp * kRowsPerWarp; r0 < rows; r0 += kRopeThreads / 32 * kRowsPerWarp) {
    const int r = r0 + lane / kLanes;
    const bool live = r < rows;
    const bool is_q = r < a.Hq, is_k = !is_q && r < a.Hq + a.kv.Hkv;
    const __nv_bfloat16* src = nullptr;
    __nv_bfloat16* dst = nullptr;
    if (live) {
      if (is_q) {
        src = a.q + t * a.q_st + r * a.q_sh;
        dst = a.q_out + (int64_t(t) * a.Hq + r) * D;
      } else if (is_k) {
        const int h = r - a.Hq;
        src = a.k + t * a.k_st + h * a.k_sh;
        dst = s_dst[0] < 0 ? nullptr : a.kv.k + s_dst[0] + h * head_stride;
      } else {
        const int h = r - a.Hq - a.kv.Hkv;
        src = a.v + t * a.v_st + h * a.v_sh;
        dst = s_dst[1] < 0 ? nullptr : a.kv.v + s_dst[1] + h * head_stride;
      }
    }
    uint4 raw = live ? *reinterpret_cast<const uint4*>(src + 8 * rl) : uint4{0, 0, 0, 0};
    float x[8];
    const __nv_bfloat162* b2 = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __bfloat1622float2(b2[j]);
      x[2 * j] = f.x;
      x[2 * j + 1] = f.y;
    }
    const __nv_bfloat16* w = is_q ? a.w_q : is_k ? a.w_k : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w) {
      const float rs = rsqrtf(ss / float(D) + a.eps);
      const uint4 wraw = *reinterpret_cast<const uint4*>(w + 8 * rl);
      const __nv_bfloat162* w2 = reinterpret_cast<const __nv_bfloat162*>(&wraw);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(w2[j]);
        x[2 * j] *= rs * (1.f + f.x);
        x[2 * j + 1] *= rs * (1.f + f.y);
      }
    }
    const int hl = a.half >> 3;  // lanes of half the rotary dims
    const bool lo = rl < hl, hi = !lo && rl < 2 * hl;
    const int from = (lane - rl) + (lo ? rl + hl : hi ? rl - hl : rl);
    const bool turn = (is_q || is_k) && (lo || hi);
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = __shfl_sync(0xffffffffu, x[j], from);
      const int i = 8 * (lo ? rl : hi ? rl - hl : 0) + j;
      const float c = turn ? s_cos[i] : 1.f, s = turn ? s_sin[i] : 0.f;
      o[j] = turn ? (lo ? x[j] * c - y * s : x[j] * c + y * s) : x[j];
    }
    if (dst) {
      uint4 res;
      __nv_bfloat162* r2 = reinterpret_cast<__nv_bfloat162*>(&res);
#pragma unroll
      for (int j = 0; j < 4; ++j) r2[j] = __floats2bfloat162_rn(o[2 * j], o[2 * j + 1]);
      // a row that nothing changes keeps its bits (a NaN's payload among them)
      *reinterpret_cast<uint4*>(dst + 8 * rl) = (turn || w) ? res : raw;
    }
  }
}

cudaError_t launch_rope_append(const RopeArgs& a, cudaStream_t st) {
  if (a.T == 0) return cudaSuccess;
  switch (a.kv.D) {
    case 64: rope_append_kernel<64><<<a.T, kRopeThreads, 0, st>>>(a); break;
    case 128: rope_append_kernel<128><<<a.T, kRopeThreads, 0, st>>>(a); break;
    default: rope_append_kernel<256><<<a.T, kRopeThreads, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace pmoe
