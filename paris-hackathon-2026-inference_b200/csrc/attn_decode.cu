// Attention of one new token per sequence over the paged cache, split over the cache's
// length and joined.
//   o = sum_j softmax_j(scale q.k_j) v_j over the keys that the token sees.
//
// Work unit: 16 keys of one (sequence, key/value head, group of up to 8 NT query heads), an
// "item" of units(b) units.  All items' units lie in one line, and CTA c of n takes the piece
// [c U/n, (c+1) U/n): equal work whatever the lengths are, planned on the device from
// kv_lens (so a captured call follows new lengths).  Within a piece, unit i belongs to warp
// i % W.  Each warp runs alone: it fetches its own units with TMA into its own ring of slots
// (one box per operand: 16 rows x D of one page and head), and holds a running
// maximum and sum and its own O.  At the end of an item's part in the CTA the warps join
// through shared memory; an item that lies in one CTA is written out there, the parts of
// the others are joined by combine_kernel in CTA order.
//
// Keys are the M side of the products, so that G <= 8 query heads fill an instruction:
// S^T[16 keys][8 heads] = K Q^T, and O^T[16 dims][8 heads] += V^T P^T, with V^T read
// through the transposing ldmatrix and P^T turned in registers (movmatrix).
//
// The weights p are rounded to bf16 for the product with V (2^-8 relative at most,
// as bf16 V itself is); sums, maxima, O and the join stay in 32 bits.
//
// Bound by HBM: each visible key and value is read once.  64 sequences of up to 16384 keys
// (1.107 GB): 175 us, 6.3 TB/s, 98 % of the copy rate; three of up to 100001 in 16-token pages
// under a window of 30000: 62 us, 86 %; one of 333: 12.6 us, two launches and a chain of
// latencies.  192 KiB of slots per SM keep about 160 KiB in flight; one box per operand and
// unit, as a unit never leaves its page.
#include <algorithm>

#include "paged.cuh"
#include "pmoe_tma.cuh"

namespace pmoe {

namespace {

constexpr int kUnit = 16;     // keys of a unit
constexpr int kJoinDims = 32; // dims that the warps join at a time
constexpr int kJoinPitch = kJoinDims + 4;
constexpr float kLog2e = 1.4426950408889634f;

// The keys of a sequence that its new token sees, in units of 16: the sinks' units, then
// those from w0 on.
struct Seq {
  int len, lo, sink, ns, w0, units;
};

__device__ __forceinline__ Seq seq_geo(const AttnArgs& a, int b) {
  Seq s;
  bool over;
  s.len = kv_len_of(a.kv.kv_lens[b], a.kv.max_pages, a.kv.page_shift, &over);
  if (s.len == 0 || over) {  // nothing to read: combine_kernel writes the zeros (or NaN)
    s.lo = s.sink = s.ns = s.w0 = s.units = 0;
    return s;
  }
  visible_keys(s.len - 1, a.window, a.sinks, &s.lo, &s.sink);
  s.ns = (s.sink + kUnit - 1) / kUnit;
  s.w0 = max(s.lo / kUnit, s.ns);
  s.units = s.ns + (s.len + kUnit - 1) / kUnit - s.w0;
  return s;
}

__device__ __forceinline__ int unit_key(const Seq& s, int k) {
  return (k < s.ns ? k : s.w0 + k - s.ns) * kUnit;
}

// CTAs that share U units of `items` items: a warp's worth of units each at least, but not
// fewer than items, so that short sequences run side by side.
__device__ __forceinline__ int active_ctas(int64_t U, int64_t items, int warps) {
  int64_t n = max((U + warps - 1) / warps, items);
  n = min(n, U);
  return int(min(n, int64_t(kDecodeCtas)));
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int c1, int c3,
                                            int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %2, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(c1), "r"(c3), "r"(c4),
      "r"(smem_u32(bar))
      : "memory");
}

// Warps and slots per warp: 192 KiB of slots in all.  A D = 256 slot is 16 KiB.
template <int D> struct Ring {
  static constexpr int kWarps = D == 256 ? 6 : 8;
  static constexpr int kOperand = kUnit * D * 2;  // bytes of a slot's K (or V) part
  static constexpr int kSlots = 196608 / (kWarps * 2 * kOperand);
};
template <int D, int NT> constexpr int decode_smem() {
  using R = Ring<D>;
  return 1024 + R::kWarps * R::kSlots * 2 * R::kOperand +
         R::kWarps * 8 * NT * kJoinPitch * 4 + R::kWarps * R::kSlots * 8 +
         R::kWarps * 8 * NT * 2 * 4;
}

// Workspace: two partial results per CTA, O [8 NT][D], then (m, l) [8 NT][2], in 32 bits; then
// the first and the last CTA of every item.
struct DecodeWs {
  float* o;
  float* ml;
  int* ctas;  // [items][2]
};
__host__ __device__ inline DecodeWs decode_ws(void* ws, int heads, int D) {
  DecodeWs w;
  w.o = static_cast<float*>(ws);
  w.ml = w.o + size_t(2) * kDecodeCtas * heads * D;
  w.ctas = reinterpret_cast<int*>(w.ml + size_t(2) * kDecodeCtas * heads * 2);
  return w;
}

// Where a warp stands in the line of units.
struct Walk {
  int b, hc, k;
  Seq s;
};
// n units on; past the last sequence b = B.
__device__ __forceinline__ void walk(const AttnArgs& a, int Hc, Walk& w, int n) {
  w.k += n;
  while (w.b < a.kv.B && w.k >= w.s.units) {
    w.k -= w.s.units;
    if (w.s.units == 0 || ++w.hc == Hc) {
      w.hc = 0;
      if (++w.b < a.kv.B) w.s = seq_geo(a, w.b);
    }
  }
}

template <int D, int NT>
__global__ void __launch_bounds__(Ring<D>::kWarps * 32, 1) attn_decode_kernel(
    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
    const AttnArgs a, void* ws_raw) {
  using R = Ring<D>;
  constexpr int W = R::kWarps, S = R::kSlots, kThreads = W * 32, GH = 8 * NT;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* s_join = reinterpret_cast<float*>(smem + W * S * 2 * R::kOperand);  // [W][GH][pitch]
  uint64_t* s_bar = reinterpret_cast<uint64_t*>(s_join + W * GH * kJoinPitch);  // [W][S]
  float* s_m = reinterpret_cast<float*>(s_bar + W * S);                      // [W][GH]
  float* s_l = s_m + W * GH;
  __shared__ int64_t s_scan[W + 1], s_start[3];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.Hq / a.kv.Hkv, chunks = (G + GH - 1) / GH, Hc = a.kv.Hkv * chunks;
  const DecodeWs ws = decode_ws(ws_raw, GH, D);

  if (lane == 0)
    for (int s = 0; s < S; ++s) mbar_init(&s_bar[warp * S + s], 1);
  mbar_fence_init();
  pdl_wait();
  // combine_kernel's CTAs may take their places, read kv_lens (so not before the wait) and wait
  pdl_trigger();

  // ---- the plan: units per sequence, summed over the block --------------------
  const int per = (a.kv.B + kThreads - 1) / kThreads;
  const int b_lo = min(a.kv.B, tid * per), b_hi = min(a.kv.B, b_lo + per);
  int64_t mine = 0, items = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int u = seq_geo(a, b).units;
    mine += u;
    items += u > 0;
  }
  int64_t incl = mine, it = items;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o), z = __shfl_xor_sync(0xffffffffu, it, o);
    if (lane >= o) incl += y;
    it += z;
  }
  __shared__ int64_t s_items[W];
  __shared__ float s_inv[GH];
  if (lane == 31) s_scan[warp] = incl, s_items[warp] = it;
  __syncthreads();
  int64_t before = incl - mine, total = 0, n_items = 0;
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
    n_items += s_items[w];
  }
  const int64_t U = total * Hc;
  const int n = active_ctas(U, n_items * Hc, W);
  if (int(blockIdx.x) >= n) return;
  // equal pieces, the first U % n of them one longer
  const int64_t whole = U <= 0x7fffffff ? int64_t(int(U) / n) : U / n;
  const int more = int(U - whole * n), c = blockIdx.x;
  const int64_t u0 = c * whole + min(c, more), u1 = u0 + whole + (c < more);
  if (before * Hc <= u0 && u0 < (before + mine) * Hc) {
    int64_t at = before;
    int b = b_lo;
    for (;; ++b) {
      const int u = seq_geo(a, b).units;
      if (u0 < (at + u) * Hc) break;
      at += u;
    }
    s_start[0] = b;
    s_start[1] = at * Hc;
  }
  __syncthreads();

  // ---- per warp: fetch and consume ---------------------------------------------
  Walk seg;  // the CTA's current item
  seg.b = int(s_start[0]);
  seg.s = seq_geo(a, seg.b);
  {
    const int off = int(u0 - s_start[1]);  // (a sequence's units in all heads fit 32 bits)
    seg.hc = off / seg.s.units;
    seg.k = off - seg.hc * seg.s.units;
  }
  char* ring = smem + warp * S * 2 * R::kOperand;
  uint64_t* bars = s_bar + warp * S;
  int64_t u_fetch = u0 + warp, u = u0 + warp;  // next unit to fetch, to consume
  // Where the warp's next 32 units to fetch lie, a lane each: one page lookup's latency for
  // all of them.
  Walk ahead = seg;  // at the first of the 32
  walk(a, Hc, ahead, warp);
  int my_page = -1, my_row = 0, my_head = 0, nth = 0;
  auto look = [&]() {
    Walk w = ahead;
    my_page = -1;
    if (u_fetch + int64_t(lane) * W < u1) {
      walk(a, Hc, w, lane * W);
      const int key = unit_key(w.s, w.k);
      my_page = page_of(a.kv, w.b, key);
      my_row = key & ((1 << a.kv.page_shift) - 1);
      my_head = w.hc / chunks;
    }
  };
  look();
  uint32_t bad = 0;  // slots whose unit lies in no page
  int slot_f = 0, slot_c = 0, phase_c = 0, in_flight = 0;
  bool dead = false;
  auto fetch_one = [&]() {
    if (u_fetch >= u1 || dead) return;
    if (nth == 32) {
      walk(a, Hc, ahead, 32 * W);
      look();
      nth = 0;
    }
    const int page = __shfl_sync(0xffffffffu, my_page, nth), row = __shfl_sync(0xffffffffu, my_row, nth);
    const int h = __shfl_sync(0xffffffffu, my_head, nth);
    bad = page < 0 ? bad | 1u << slot_f : bad & ~(1u << slot_f);
    if (lane == 0) {
      const uint32_t dst = smem_u32(ring + slot_f * 2 * R::kOperand);
      const int at = page < 0 ? a.kv.n_pages : page;  // no page: zeros
      mbar_arrive_expect_tx(&bars[slot_f], 2 * R::kOperand);
      tma_load_5d(dst, &map_k, row, h, at, &bars[slot_f]);
      tma_load_5d(dst + R::kOperand, &map_v, row, h, at, &bars[slot_f]);
    }
    slot_f = slot_f + 1 == S ? 0 : slot_f + 1;
    ++in_flight;
    ++nth;
    u_fetch += W;
  };
  for (int s = 0; s < S; ++s) fetch_one();

  const float scale2 = a.scale * kLog2e;
  // ldmatrix rows of this lane: K (A operand, keys x dims) and V (transposed, dims x keys)
  const int krow = lane & 15, kchunk = lane >> 4;
  const int vrow = (lane & 7) + ((lane >> 4) << 3), vchunk = (lane >> 3) & 1;
  int64_t at = u0;  // begin of the CTA's current part
  while (at < u1) {
    const int64_t item0 = at - seg.k, item1 = item0 + seg.s.units, end = min(item1, u1);
    const int g0 = (seg.hc % chunks) * GH, h_kv = seg.hc / chunks;
    uint32_t q[D / 16][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int g = g0 + t * 8 + (lane >> 2);
      const __nv_bfloat16* qr = a.q + seg.b * a.q_stride_t + (int64_t(h_kv) * G + g) * a.q_stride_h;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(qr + k * 16 + (lane & 3) * 2);
        q[k][t][0] = g < G ? p[0] : 0;
        q[k][t][1] = g < G ? p[4] : 0;
      }
    }
    float o[D / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][t][e] = 0.f;
    }
    for (; u < end; u += W) {
      // a wait that runs out makes the rows NaN and stops the fetching; what is in flight
      // is still waited for
      if (in_flight > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(&bars[slot_c], phase_c))) dead = true;
        --in_flight;
      }
      const int j0 = unit_key(seg.s, int(u - item0));
      const uint32_t kb = smem_u32(ring + slot_c * 2 * R::kOperand), vb = kb + R::kOperand;
      float sc[NT][4], sc2[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][e] = sc2[t][e] = 0.f;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t af[4];
        ldsm4(kb + (k >> 2) * (kUnit * 128) + swz128(krow, ((k & 3) << 1) + kchunk), af);
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816(k & 1 ? sc2[t] : sc[t], af, q[k][t][0], q[k][t][1]);
      }
      // rows of this lane: keys j0 + lane/4 and + 8
      const bool edge = j0 + kUnit > seg.s.len || (j0 < seg.s.lo && j0 + kUnit > seg.s.sink) ||
                        (bad >> slot_c & 1) || dead;
      bool see[2] = {true, true};
      if (edge) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int j = j0 + (lane >> 2) + 8 * r;
          see[r] = j < seg.s.len && (j < seg.s.sink || j >= seg.s.lo);
        }
      }
      const bool lost = (bad >> slot_c & 1) || dead;
      uint32_t pf[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float s[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[e] = (sc[t][e] + sc2[t][e]) * scale2;
          if (edge) s[e] = see[e >> 1] ? (lost ? NAN : s[e]) : -INFINITY;
        }
        float mn[2], f[2];
        bool grew = false;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(s[c], s[c + 2]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
          mn[c] = fmaxf(m[t][c], x);
          grew |= mn[c] > m[t][c];
          f[c] = mn[c] == -INFINITY ? 0.f : mn[c];
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float keep = fast_exp2(m[t][c] - f[c]);
            m[t][c] = mn[c];
            l[t][c] *= keep;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
              o[d][t][c] *= keep;
              o[d][t][c + 2] *= keep;
            }
          }
        }
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = fast_exp2(s[e] - f[e & 1]);
          l[t][e & 1] += p[e];
        }
        pf[t][0] = movm_t(pack_bf16(p[0], p[1]));
        pf[t][1] = movm_t(pack_bf16(p[2], p[3]));
      }
      // keys that are not seen must not reach the product, whatever their V holds
      uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
      if (edge) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = j0 + (lane & 3) * 2 + e;
          const uint32_t half = e ? 0xffff0000u : 0xffffu;
          if (!(j < seg.s.len && (j < seg.s.sink || j >= seg.s.lo))) keep0 &= ~half;
          if (!(j + 8 < seg.s.len && (j + 8 < seg.s.sink || j + 8 >= seg.s.lo))) keep1 &= ~half;
        }
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t af[4];
        ldsm4_t(vb + (d >> 2) * (kUnit * 128) + swz128(vrow, ((d & 3) << 1) + vchunk), af);
        if (edge) {
          af[0] &= keep0;
          af[1] &= keep0;
          af[2] &= keep1;
          af[3] &= keep1;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) mma16816(o[d][t], af, pf[t][0], pf[t][1]);
      }
      __syncwarp();  // every lane has read the slot
      slot_c = slot_c + 1 == S ? 0 : slot_c + 1;
      if (slot_c == 0) phase_c ^= 1;
      fetch_one();
    }
    // ---- join the warps' parts ---------------------------------------------------
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[t][c] += __shfl_xor_sync(0xffffffffu, l[t][c], w);
        if (lane < 4) {
          s_m[warp * GH + t * 8 + lane * 2 + c] = m[t][c];
          s_l[warp * GH + t * 8 + lane * 2 + c] = l[t][c];
        }
      }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int g = t * 8 + (lane & 3) * 2 + c;
        float top = -INFINITY;
        for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w * GH + g]);
        const float f = fast_exp2(m[t][c] - (top == -INFINITY ? 0.f : top));
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          o[d][t][c] *= f;
          o[d][t][c + 2] *= f;
        }
      }
    const bool alone = at == item0 && end == item1;
    const int64_t item = int64_t(seg.b) * Hc + seg.hc;
    if (tid == 0 && at == item0) ws.ctas[item * 2] = blockIdx.x;
    if (tid == 0 && end == item1) ws.ctas[item * 2 + 1] = blockIdx.x;
    const int part = int(blockIdx.x) * 2 + (at == item0 ? 1 : 0);
    // The sum over the warps of dims d0 .. d0 + n - 1, which lie in buf [W][GH][n + 4].
    auto add_up = [&](const float* buf, int d0, int n) {
      for (int i = tid; i < GH * n; i += kThreads) {
        const int g = i / n, d = i % n;
        float acc = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) acc += buf[(w * GH + g) * (n + 4) + d];
        if (!alone) {
          ws.o[(size_t(part) * GH + g) * D + d0 + d] = acc;
        } else if (g0 + g < G) {
          a.out[(int64_t(seg.b) * a.Hq + int64_t(h_kv) * G + g0 + g) * D + d0 + d] =
              __float2bfloat16_rn(acc * s_inv[g]);
        }
      }
    };
    if (tid < GH) {  // 1 / l of the joined heads
      float top = -INFINITY, sum = 0.f;
      for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w * GH + tid]);
      for (int w = 0; w < W; ++w)
        sum += s_l[w * GH + tid] * fast_exp2(s_m[w * GH + tid] - (top == -INFINITY ? 0.f : top));
      s_inv[tid] = 1.f / sum;
      if (!alone) {
        ws.ml[(size_t(part) * GH + tid) * 2] = top;
        ws.ml[(size_t(part) * GH + tid) * 2 + 1] = sum;
      }
    }
    if (end == u1) {  // nothing is on its way any more: all dims at once, in the ring
      float* buf = reinterpret_cast<float*>(smem);
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            buf[(warp * GH + t * 8 + (lane & 3) * 2 + (e & 1)) * (D + 4) + d * 16 + (lane >> 2) + 8 * (e >> 1)] = o[d][t][e];
      __syncthreads();
      add_up(buf, 0, D);
    } else {
#pragma unroll
      for (int d0 = 0; d0 < D; d0 += kJoinDims) {
#pragma unroll
        for (int dd = 0; dd < kJoinDims / 16; ++dd)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s_join[(warp * GH + t * 8 + (lane & 3) * 2 + (e & 1)) * kJoinPitch + dd * 16 +
                     (lane >> 2) + 8 * (e >> 1)] = o[d0 / 16 + dd][t][e];
        __syncthreads();
        add_up(s_join, d0, kJoinDims);
        __syncthreads();
      }
    }
    walk(a, Hc, seg, int(end - at));
    at = end;
    __syncthreads();  // s_m and s_l are free again
  }
}

// One CTA per (sequence, query head): joins the parts of an item that several CTAs
// computed, in CTA order, and writes the rows that have no keys.
__global__ void __launch_bounds__(256) combine_kernel(const AttnArgs a, void* ws_raw, int GH) {
  const int b = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, tid = threadIdx.x;
  const int D = a.kv.D, G = a.Hq / a.kv.Hkv, chunks = (G + GH - 1) / GH, Hc = a.kv.Hkv * chunks;
  const int g = h % G, hc = h / G * chunks + g / GH, gl = g % GH;
  __nv_bfloat16* out = a.out + (int64_t(b) * a.Hq + h) * D;
  const DecodeWs ws = decode_ws(ws_raw, GH, D);
  // (kv_lens is older than the main kernel, which has waited for whatever wrote it)
  const int len = a.kv.kv_lens[b];
  const bool none = seq_geo(a, b).units == 0;
  pdl_wait();
  if (none) {
    bool over;
    kv_len_of(len, a.kv.max_pages, a.kv.page_shift, &over);
    for (int d = tid; d < D; d += 256) out[d] = __float2bfloat16_rn(over ? NAN : 0.f);
    return;
  }
  const int2 range = reinterpret_cast<const int2*>(ws.ctas)[int64_t(b) * Hc + hc];
  const int c0 = range.x, c1 = range.y;
  if (c0 == c1) return;  // written by that CTA
  auto part_of = [&](int c) { return size_t(2 * c + (c == c0)) * GH + gl; };
  // (m, l) of all parts, a thread each, while O is on its way
  __shared__ float2 s_ml[kDecodeCtas];
  __shared__ float s_top[8];
  float top = -INFINITY;
  if (c0 + tid <= c1) {
    s_ml[tid] = reinterpret_cast<const float2*>(ws.ml)[part_of(c0 + tid)];
    top = s_ml[tid].x;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) s_top[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) top = fmaxf(top, s_top[k]);
  const float base = top == -INFINITY ? 0.f : top;
  // D/4 threads of 16 bytes, the CTAs' parts dealt out over the 1024/D groups of them
  __shared__ float s_sum[16];
  __shared__ float4 s_o[256];
  const int lanes = D / 4, group = tid / lanes, groups = 256 / lanes, d4 = tid % lanes;
  float sum = 0.f;
  float4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int c = c0 + group; c <= c1; c += groups) {
    const float2 ml = s_ml[c - c0];
    const float f = fast_exp2(ml.x - base);
    const float4 x = reinterpret_cast<const float4*>(ws.o + part_of(c) * D)[d4];
    sum += ml.y * f;
    acc.x += x.x * f;
    acc.y += x.y * f;
    acc.z += x.z * f;
    acc.w += x.w * f;
  }
  s_o[tid] = acc;
  if (d4 == 0) s_sum[group] = sum;
  __syncthreads();
  if (group == 0) {
    for (int k = 1; k < groups; ++k) {
      const float4 x = s_o[k * lanes + d4];
      acc.x += x.x;
      acc.y += x.y;
      acc.z += x.z;
      acc.w += x.w;
      sum += s_sum[k];
    }
    const __nv_bfloat162 y0 = __floats2bfloat162_rn(acc.x / sum, acc.y / sum);
    const __nv_bfloat162 y1 = __floats2bfloat162_rn(acc.z / sum, acc.w / sum);
    reinterpret_cast<__nv_bfloat162*>(out)[d4 * 2] = y0;
    reinterpret_cast<__nv_bfloat162*>(out)[d4 * 2 + 1] = y1;
  }
}

template <int D, int NT>
cudaError_t launch_one(const AttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, void* ws,
                       cudaStream_t st) {
  // no more CTAs than the tables' width leaves work for
  const int G = a.Hq / a.kv.Hkv, chunks = (G + 8 * NT - 1) / (8 * NT);
  const int64_t items = int64_t(a.kv.B) * a.kv.Hkv * chunks;
  const int64_t units = (int64_t(a.kv.max_pages) << a.kv.page_shift) / kUnit * items;
  const int64_t most = std::max((units + Ring<D>::kWarps - 1) / Ring<D>::kWarps, items);
  cudaError_t e = launch_dependent(attn_decode_kernel<D, NT>, dim3(unsigned(std::min<int64_t>(most, kDecodeCtas))),
                                   Ring<D>::kWarps * 32, decode_smem<D, NT>(), 1, st, mk, mv, a, ws);
  if (e != cudaSuccess) return e;
  return launch_dependent(combine_kernel, dim3(unsigned(a.kv.B) * a.Hq), 256, 0, 1, st, a, ws, 8 * NT);
}

template <int D, int NT> cudaError_t init_one() {
  return cudaFuncSetAttribute(attn_decode_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              decode_smem<D, NT>());
}

// A box: 16 keys of one page and head.
bool page_map(CUtensorMap* map, const PagedKV& kv, const __nv_bfloat16* base,
                   int64_t page_stride, int rows) {
  const uint64_t D = kv.D, ps = uint64_t(1) << kv.page_shift;
  const uint64_t dims[5] = {64, ps, D / 64, uint64_t(kv.Hkv), uint64_t(kv.n_pages)};
  const uint64_t strides[4] = {D * 2, 128, ps * D * 2, uint64_t(page_stride) * 2};
  const uint32_t box[5] = {64, uint32_t(rows), uint32_t(D / 64), 1, 1};
  return make_tmap_bf16_nd(map, base, 5, dims, strides, box);
}

// Groups of up to 8 heads fill one instruction; wider ones take two at a time, so that K and V are
// fetched half as often (64 sequences of up to 4000 keys, 16 heads a group of 256: 77 us, 90 in
// eights; 8 heads a group: 60, 71 in sixteens).
int heads_per_item(int G) { return G <= 8 ? 8 : 16; }

}  // namespace

size_t attn_decode_ws_bytes(int B, int Hq, int Hkv, int D) {
  const int heads = heads_per_item(Hq / Hkv), chunks = (Hq / Hkv + heads - 1) / heads;
  return size_t(2) * kDecodeCtas * heads * (D + 2) * sizeof(float) +
         size_t(B) * Hkv * chunks * 2 * sizeof(int);
}

cudaError_t attn_decode_init() {
  cudaError_t e;
  if ((e = init_one<64, 1>()) != cudaSuccess || (e = init_one<64, 2>()) != cudaSuccess ||
      (e = init_one<128, 1>()) != cudaSuccess || (e = init_one<128, 2>()) != cudaSuccess ||
      (e = init_one<256, 1>()) != cudaSuccess || (e = init_one<256, 2>()) != cudaSuccess)
    return e;
  return cudaSuccess;
}

cudaError_t launch_attn_decode(const AttnArgs& args, void* ws, cudaStream_t st) {
  AttnArgs a = args;
  if (a.T == 0) return cudaSuccess;
  CUtensorMap mk{}, mv{};
  if (a.kv.n_pages == 0) a.kv.max_pages = 0;  // no page: every sequence with keys gets NaN
  if (a.kv.max_pages > 0 && (!page_map(&mk, a.kv, a.kv.k, a.kv.k_page_stride, kUnit) ||
                             !page_map(&mv, a.kv, a.kv.v, a.kv.v_page_stride, kUnit)))
    return cudaErrorInvalidValue;
  const bool wide = heads_per_item(a.Hq / a.kv.Hkv) > 8;
  switch (a.kv.D) {
    case 64: return wide ? launch_one<64, 2>(a, mk, mv, ws, st) : launch_one<64, 1>(a, mk, mv, ws, st);
    case 128: return wide ? launch_one<128, 2>(a, mk, mv, ws, st) : launch_one<128, 1>(a, mk, mv, ws, st);
    default: return wide ? launch_one<256, 2>(a, mk, mv, ws, st) : launch_one<256, 1>(a, mk, mv, ws, st);
  }
}

}  // namespace pmoe
