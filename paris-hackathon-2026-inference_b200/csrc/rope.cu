// Rotary positions with several axes, the optional per-head RMSNorm, and the write of
// keys and values into the cache's pages.
//
// Pair (i, i + half) of a query or key row turns by angle = pos[axis(i)] * inv_freq[i]:
//   y_i = x_i c - x_{i+half} s,   y_{i+half} = x_{i+half} c + x_i s.
// The angle is formed and reduced to (-pi, pi] in 64 bits: at position 1e6 a 32-bit
// product is already off by 0.03 rad.  One rounding to bf16, at the store.
#include "paged.cuh"
#include "pmoe_tma.cuh"

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

// S warps share a token, and need nobody else.  A lane has the same 8 dims of every row (D/8
// lanes a row, 32/(D/8) rows at once), so the factors of its dims, with the norm's gains in
// them, stay in registers: y = (x own + partner other) r with own = g c, other = -+ g' s, and
// own = g, other = 0 behind the rotary dims.  The partner's 8 dims come from lane +- half/8 as they
// were loaded.  A batch of rows is on its way while the angles are worked out.
//
// 8192 tokens of 16 + 2 heads of 256 (168 MB): 34.5 us, 4.9 TB/s, 75 % of the copy rate.  Bound by
// instructions (128 a row, 63 % of the issue slots): the first version took 320 a row and
// 76 us, one with the factors in shared memory 51, this one with batches of 4 rows (110
// registers, half the warps) 44.  64 tokens, eight warps each: 4.5 us, a chain of latencies.
constexpr int kBatch = 2;  // row slots a warp holds at a time, and as many on their way

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 unpack(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ uint32_t word(const uint4& v, int j) {
  return j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
}

template <int D, int S>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_append_kernel(const RopeArgs a) {
  constexpr int kLanes = D / 8, kRows = 32 / kLanes, kWarps = kRopeThreads / 32;
  __shared__ float s_cos[kWarps][128], s_sin[kWarps][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = (blockIdx.x * kWarps + warp) / S, part = warp % S;
  if (t >= a.T) return;  // (a whole warp)
  pdl_wait();
  const int rl = lane % kLanes, sub = lane / kLanes;  // this lane's 8 dims 8*rl .., row of a slot
  // Rows r0, r0 + step, .. of q, then of k, then of v are this lane's.
  const int r0 = part * kRows + sub, step = S * kRows;
  const uint4* src;
  int64_t src_step;  // of `step` rows, in 16-byte pieces
  int n;
  auto open = [&](int kind) {
    const __nv_bfloat16* base = kind == 0 ? a.q + t * a.q_st : kind == 1 ? a.k + t * a.k_st : a.v + t * a.v_st;
    const int64_t sh = kind == 0 ? a.q_sh : kind == 1 ? a.k_sh : a.v_sh;
    src = reinterpret_cast<const uint4*>(base + r0 * sh) + rl;
    src_step = step * sh / 8;
    n = kind == 0 ? a.Hq : a.kv.Hkv;
  };
  uint4 next[kBatch];
  auto load = [&](int r) {  // rows r, r + step, ..; src advances
#pragma unroll
    for (int k = 0; k < kBatch; ++k, src += src_step)
      next[k] = r + k * step < n ? *src : uint4{0, 0, 0, 0};
  };
  open(0);
  load(r0);

  for (int x = lane; x < a.half; x += 32) {
    const double turns = double(a.positions[rope_axis(a, x) * a.pos_stride + t]) *
                         double(a.inv_freq[x]) * 0.15915494309189533577;
    float s, c;
    sincospif(float(2.0 * (turns - rint(turns))), &s, &c);
    s_cos[warp][x] = c * a.mscale;
    s_sin[warp][x] = s * a.mscale;
  }
  // where the token's keys and values go
  int64_t kd = -1, vd = -1;
  {
    const int32_t* cu = a.cu_q;
    int b = t;
    if (cu) b = last_at_or_before(a.kv.B, t, [=](int i) { return cu[i]; });
    if (b >= 0 && b < a.kv.B) {
      const int after = cu ? cu[b + 1] - t : 1;  // tokens from t to the sequence's end
      const int j = after > 0 ? a.kv.kv_lens[b] - after : -1;
      const int p = j >= 0 ? page_of(a.kv, b, j) : -1;
      if (p >= 0) {
        const int64_t row = int64_t(j & ((1 << a.kv.page_shift) - 1)) * D;
        kd = p * a.kv.k_page_stride + row;
        vd = p * a.kv.v_page_stride + row;
      }
    }
  }
  __syncwarp();

  const int hl = a.half >> 3;  // lanes of half the rotary dims
  const bool turn = rl < 2 * hl, low = rl < hl;
  const int partner = turn ? (low ? lane + hl : lane - hl) : lane;
  float2 own[4], other[4];
  bool norm = false;
  auto factors = [&](const __nv_bfloat16* w) {  // of q or of k
    norm = w != nullptr;
    float2 g[4], g2[4];  // this lane's gains and its partner's
    const uint4 v = w ? reinterpret_cast<const uint4*>(w)[rl] : uint4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack(word(v, j)), f2 = unpack(__shfl_sync(0xffffffffu, word(v, j), partner));
      g[j] = make_float2(1.f + f.x, 1.f + f.y);
      g2[j] = make_float2(1.f + f2.x, 1.f + f2.y);
    }
    const int at = 8 * (low ? rl : rl - hl);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      own[j] = g[j];
      other[j] = make_float2(0.f, 0.f);
      if (turn) {
        const float2 c = *reinterpret_cast<const float2*>(&s_cos[warp][at + 2 * j]);
        float2 s = *reinterpret_cast<const float2*>(&s_sin[warp][at + 2 * j]);
        if (low) s = make_float2(-s.x, -s.y);
        own[j] = mul2(g[j], c);
        other[j] = mul2(g2[j], s);
      }
    }
  };
  auto turned = [&](const uint4& x) {
    float2 v[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = unpack(word(x, j));
      const uint32_t m = __shfl_sync(0xffffffffu, word(x, j), partner);
      y[j] = unpack(turn ? m : 0u);
    }
    float2 rs = make_float2(1.f, 1.f);
    if (norm) {
      float2 ss = mul2(v[0], v[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) ss = fma2(v[j], v[j], ss);
      float sum = ss.x + ss.y;
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      rs.x = rs.y = rsqrtf(sum * (1.f / D) + a.eps);
    }
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = mul2(fma2(v[j], own[j], mul2(y[j], other[j])), rs);
      const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
      o[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
    // (a row that nothing changes keeps its bits, a NaN's payload among them)
    return turn || norm ? uint4{o[0], o[1], o[2], o[3]} : x;
  };
  const int64_t head = (int64_t(D) << a.kv.page_shift) / 8;  // 16-byte pieces between cache heads
#pragma unroll 1
  for (int kind = 0; kind < 3; ++kind) {
    if (kind < 2) factors(kind ? a.w_k : a.w_q);
    uint4* dst = kind == 0 ? reinterpret_cast<uint4*>(a.q_out + int64_t(t) * a.Hq * D)
                           : reinterpret_cast<uint4*>(kind == 1 ? a.kv.k + kd : a.kv.v + vd);
    const int64_t dst_row = kind == 0 ? D / 8 : head;
    const bool write = kind == 0 || (kind == 1 ? kd : vd) >= 0;
    dst += r0 * dst_row + rl;
    // all lanes take the turns that the first rows of the warp need
    for (int r = r0, w = part * kRows; w < n; r += kBatch * step, w += kBatch * step) {
      uint4 now[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) now[k] = next[k];
      if (w + kBatch * step < n) load(r + kBatch * step);
#pragma unroll
      for (int k = 0; k < kBatch; ++k, dst += step * dst_row) {
        if (w + k * step >= n) break;
        const uint4 y = kind < 2 ? turned(now[k]) : now[k];
        if (write && r + k * step < n) *dst = y;
      }
    }
    if (kind < 2) {
      open(kind + 1);
      load(r0);
    }
  }
}

template <int D, int S>
cudaError_t launch_split(const RopeArgs& a, cudaStream_t st) {
  const int64_t warps = int64_t(a.T) * S, per = kRopeThreads / 32;
  return launch_dependent(rope_append_kernel<D, S>, dim3(unsigned((warps + per - 1) / per)),
                          kRopeThreads, 0, 1, st, a);
}

template <int D>
cudaError_t launch_one(const RopeArgs& a, cudaStream_t st) {
  // Warps for every SM, and no more: a token's factors are worked out by each of its warps.  64
  // tokens: 4.5 us with 8 warps a token, 7.5 with one; 592: 7.0 with 2, 7.2 with 8; 1024: 8.2 with
  // 2, 11.6 with 8; 2368: 11.0 with one, 13.0 with 2.
  if (a.T >= 148 * 16) return launch_split<D, 1>(a, st);
  return a.T >= 148 * 4 ? launch_split<D, 2>(a, st) : launch_split<D, 8>(a, st);
}

cudaError_t launch_rope_append(const RopeArgs& a, cudaStream_t st) {
  if (a.T == 0) return cudaSuccess;
  switch (a.kv.D) {
    case 64: return launch_one<64>(a, st);
    case 128: return launch_one<128>(a, st);
    default: return launch_one<256>(a, st);
  }
}

}  // namespace pmoe
