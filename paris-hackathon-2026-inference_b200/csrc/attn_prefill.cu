// Attention of packed prompts and prompt chunks over the paged cache, on the tensor cores.
//   o = sum_j softmax_j(scale q.k_j) v_j over the keys that each row sees.
//
// One CTA per (128 rows of one sequence, key/value head).  The rows are tokens x the G
// query heads that share the head, so one pass over K and V serves all of them.  Keys come in
// tiles of 128:
//   S = Q K^T         128 x 128, operands in shared memory, S in TMEM
//   P = 2^(S c - m)   a thread per row reads its S from TMEM and writes P (bf16) over it
//   O += P V          A = P from TMEM, B = V from shared memory (dims contiguous), O in TMEM
// The running maximum m of a row moves only when a tile's maximum exceeds it by more than 8
// (in powers of two): weights then stay below 2^8, exact to the same relative rounding, and O
// is rescaled rarely.  With two S buffers the product of tile j + 1 runs while the
// weights of tile j are computed.
//
// Warps 0-3: softmax and epilogue (row = thread); warp 4: TMA; warp 5: MMA.  K and V travel
// in 16 KiB chunks through one ring: K as 128 keys x 64 dims, V as 16384 / 2D keys x D dims.
//
// Values that a row does not see must not reach its sum even where they are not finite, but
// 0 x inf is NaN: in tiles at an edge of some row's sight, V rows that nobody sees or that
// hold a non-finite number are zeroed in shared memory, and the latter are added to the rows
// that see them one by one.
#include "paged.cuh"
#include "pmoe_tc.cuh"

namespace pmoe {

namespace {

constexpr int kRows = 128, kTile = 128, kChunk = 16384;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGrow = 8.f;  // powers of two that a row's maximum may lag behind

template <int D> struct Cfg {
  static constexpr int kS = D == 256 ? 2 : 1;           // S buffers
  static constexpr int kSlots = D == 256 ? 10 : D == 128 ? 4 : 5;
  static constexpr int kCtas = D == 256 ? 1 : 2;        // CTAs per SM
  static constexpr int kCols = D == 256 ? 512 : 256;    // TMEM columns
  static constexpr int kKc = D / 64;                    // K chunks of a tile
  static constexpr int kVr = kChunk / (2 * D);          // keys of a V chunk
  static constexpr int kVc = kTile / kVr;               // V chunks of a tile
  static constexpr int kSmem = 1024 + kRows * D * 2 + kSlots * kChunk;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int row, int cg,
                                        int h, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(cg), "r"(h), "r"(page),
      "r"(smem_u32(bar))
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], A bf16 pairs in 32-bit columns.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  return r;
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&p);
}
// V chunk [D/64][kVr keys][128 bytes], swizzled, as the B operand with dims contiguous: next
// 64 dims `group` bytes on (leading), next 8 keys 1024 bytes on (stride).
__device__ __forceinline__ uint64_t sdesc_mn_sw128(uint32_t saddr, uint32_t group) {
  uint64_t d = 0;
  d |= uint64_t((saddr & 0x3FFFFu) >> 4);
  d |= uint64_t(group >> 4) << 16;
  d |= uint64_t(1024 >> 4) << 32;
  d |= uint64_t(1) << 46;
  d |= uint64_t(2) << 61;
  return d;
}
// bar.red over the softmax warps: whether any thread says yes.
__device__ __forceinline__ bool softmax_any(bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(uint32_t(x))
      : "memory");
  return r != 0;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// Block x's rows: slots of a sequence begin at cu[b] / tokens + b, which leaves each
// sequence at least its number of tiles.
struct TileOf {
  int b, t0, n, p0, len;  // sequence, first packed row, tokens, index of the first, keys
  bool over;
};
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int per, int x, TileOf* o) {
  const int B = a.kv.B;
  if (x < a.cu_q[0] / per) return false;
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] / per + mid <= x) lo = mid; else hi = mid;
  }
  const int c0 = a.cu_q[lo], c1 = min(a.cu_q[lo + 1], a.T);
  const int i = x - (c0 / per + lo);
  if (c0 < 0 || i < 0 || i > (c1 - c0 - 1) / per || c1 <= c0) return false;
  o->b = lo;
  o->t0 = c0 + i * per;
  o->n = min(per, c1 - o->t0);
  o->len = kv_len_of(a.kv.kv_lens[lo], a.kv.max_pages, a.kv.page_shift, &o->over);
  o->p0 = o->len - (c1 - o->t0);
  return true;
}

template <int D>
__global__ void __launch_bounds__(192, Cfg<D>::kCtas) attn_prefill_kernel(
    const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
    const AttnArgs a) {
  using C = Cfg<D>;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* s_q = smem;                    // [D/64][128 rows][128 bytes], swizzled
  char* s_ring = smem + kRows * D * 2;
  __shared__ uint64_t full[C::kSlots], empty[C::kSlots], s_full[C::kS], p_ready[C::kS], pv_done[2], q_ready;
  __shared__ uint32_t s_tmem;
  __shared__ int s_first;              // tile 0 adds to O (set to zero before) instead of setting it
  __shared__ uint32_t s_bad[4];        // keys of the tile whose V row is not finite

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.Hq / a.kv.Hkv, per = kRows / G;
  const int h = blockIdx.x % a.kv.Hkv;
  const int x = int(gridDim.x / a.kv.Hkv) - 1 - int(blockIdx.x / a.kv.Hkv);  // late tiles, the longest, first
  TileOf tile;
  if (!find_tile(a, per, x, &tile)) return;

  // keys that some row sees: [0, sink_any) and [lo_any, last]
  const int p_last = tile.p0 + tile.n - 1, p_first = max(tile.p0, 0);
  int lo_any = 0, sink_any = 0, lo_max = 0, sink_all = 0;
  int n_tiles = 0, ns = 0, w0 = 0;
  if (p_last >= 0 && !tile.over) {
    visible_keys(p_first, a.window, a.sinks, &lo_any, &sink_all);
    visible_keys(p_last, a.window, a.sinks, &lo_max, &sink_any);
    ns = (sink_any + kTile - 1) / kTile;
    w0 = max(lo_any / kTile, ns);
    n_tiles = ns + p_last / kTile + 1 - w0;
  }
  auto tile_key = [&](int j) { return (j < ns ? j : w0 + j - ns) * kTile; };

  if (warp == 5) {
    tmem_alloc(&s_tmem, C::kCols);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < C::kS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
    }
    mbar_init(&pv_done[0], 1);
    mbar_init(&pv_done[1], 1);
    mbar_init(&q_ready, 4);
    s_first = 0;
    mbar_fence_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm_o = s_tmem, tm_s = s_tmem + D;  // O [D columns], then the S buffers

  if (warp == 4) {
    // ---- TMA: K0, (K1, V0), (K2, V1) ... with two S buffers, K0, V0, K1, V1 ... with one
    int seq = 0;
    bool ok = true;
    int page[2] = {-1, -1};  // lane i: page of the tile's i-th page, of the tiles j and j + 1
    const int ps = 1 << a.kv.page_shift, per_tile = max(1, kTile / ps);
    auto pages_of = [&](int j) {
      const int k0 = tile_key(j);
      return j < n_tiles && lane < per_tile ? page_of(a.kv, tile.b, k0 + lane * ps) : -1;
    };
    auto slot_open = [&]() {
      const int s = seq % C::kSlots;
      if (seq >= C::kSlots) ok = ok && warp_wait(&empty[s], (seq / C::kSlots - 1) & 1);
      return s;
    };
    auto load_k = [&](int j, int mine) {
      const int k0 = tile_key(j), rows = min(ps, kTile);
      const int at = mine < 0 ? a.kv.n_pages : mine, row = ps > kTile ? k0 & (ps - 1) : 0;
      for (int c = 0; c < C::kKc && ok; ++c, ++seq) {
        const int s = slot_open();
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], kChunk);
        __syncwarp();
        if (lane < per_tile)
          tma_box(smem_u32(s_ring + s * kChunk) + lane * rows * 128, &map_k, row, c, h, at, &full[s]);
      }
    };
    auto load_v = [&](int j, int mine) {
      const int rows = min(ps, C::kVr), boxes = C::kVr / rows;
      for (int c = 0; c < C::kVc && ok; ++c, ++seq) {
        const int s = slot_open();
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], kChunk);
        __syncwarp();
        // box i: rows of dims group i % (D/64)
        const int i = lane, cg = i % (D / 64), r = i / (D / 64) * rows;
        const int key = c * C::kVr + r;  // in the tile
        const int pg = __shfl_sync(0xffffffffu, mine, min(key >> a.kv.page_shift, 31));
        if (i < boxes * (D / 64))
          tma_box(smem_u32(s_ring + s * kChunk) + cg * C::kVr * 128 + r * 128, &map_v,
                  key & (ps - 1), cg, h, pg < 0 ? a.kv.n_pages : pg, &full[s]);
      }
    };
    page[0] = pages_of(0);
    if (n_tiles > 0) load_k(0, page[0]);
    for (int j = 0; j < n_tiles && ok; ++j) {
      page[1] = pages_of(j + 1);
      if (C::kS == 2 && j + 1 < n_tiles) load_k(j + 1, page[1]);
      load_v(j, page[0]);
      if (C::kS == 1 && j + 1 < n_tiles) load_k(j + 1, page[1]);
      page[0] = page[1];
    }
    if (!ok)  // a wait ran out: let the copies land before the CTA ends
      for (int q = max(0, seq - C::kSlots); q < seq; ++q)
        mbar_wait(&full[q % C::kSlots], (q / C::kSlots) & 1);
  } else if (warp == 5) {
    // ---- MMA, one thread
    if (lane == 0 && n_tiles > 0) {
      constexpr uint32_t idesc_s = idesc_bf16_f32(kRows, kTile);
      constexpr uint32_t idesc_o = idesc_bf16_f32(kRows, D) | 1u << 16;  // B with dims contiguous
      int seq = 0;
      bool ok = mbar_wait(&q_ready, 0);
      auto qk = [&](int j) {
        for (int c = 0; c < C::kKc && ok; ++c, ++seq) {
          const int s = seq % C::kSlots;
          ok = mbar_wait(&full[s], (seq / C::kSlots) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ka = smem_u32(s_ring + s * kChunk), qa = smem_u32(s_q) + c * kRows * 128;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_bf16(tm_s + (j % C::kS) * kTile, sdesc_k_sw128(qa + k * 32),
                      sdesc_k_sw128(ka + k * 32), idesc_s, c > 0 || k > 0);
          umma_commit(&empty[s]);
        }
        if (ok) umma_commit(&s_full[j % C::kS]);
      };
      auto pv = [&](int j) {
        ok = ok && mbar_wait(&p_ready[j % C::kS], (j / C::kS) & 1);
        if (!ok) return;
        tc_fence_after();
        const bool add = j > 0 || *(volatile int*)&s_first;
        for (int c = 0; c < C::kVc && ok; ++c, ++seq) {
          const int s = seq % C::kSlots;
          ok = mbar_wait(&full[s], (seq / C::kSlots) & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t va = smem_u32(s_ring + s * kChunk);
#pragma unroll
          for (int k = 0; k < C::kVr / 16; ++k)
            umma_ts(tm_o, tm_s + (j % C::kS) * kTile + (c * C::kVr + k * 16) / 2,
                    sdesc_mn_sw128(va + k * 2048, C::kVr * 128), idesc_o, add || c > 0 || k > 0);
          umma_commit(&empty[s]);
        }
        if (ok) umma_commit(&pv_done[j & 1]);
      };
      if (C::kS == 2 && ok) qk(0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        if (C::kS == 2) {
          if (j + 1 < n_tiles) qk(j + 1);
        } else {
          qk(j);
        }
        if (ok) pv(j);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: thread = row
    const uint32_t tl = uint32_t(warp) << 21;  // this warp's TMEM lanes
    const int tok = tid / G, g = tid % G;
    const bool row_live = tok < per && tok < tile.n;
    const int p = row_live ? tile.p0 + tok : -1;  // < 0: sees nothing
    int lo = 0, sink = 0;
    if (p >= 0) visible_keys(p, a.window, a.sinks, &lo, &sink);
    bool ok = true;
    if (n_tiles > 0) {
      // Q to shared memory, a warp per row; a negative scale turns its sign
      constexpr int kLanes = D / 8;
      const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
      for (int r0 = warp * 32; r0 < warp * 32 + 32; r0 += 32 / kLanes) {
        const int r = r0 + lane / kLanes, rl = lane % kLanes, rt = r / G;
        uint4 v{0, 0, 0, 0};
        if (rt < per && rt < tile.n) {
          v = *reinterpret_cast<const uint4*>(a.q + (tile.t0 + rt) * a.q_stride_t +
                                              (int64_t(h) * G + r % G) * a.q_stride_h + 8 * rl);
          v.x ^= flip;
          v.y ^= flip;
          v.z ^= flip;
          v.w ^= flip;
        }
        *reinterpret_cast<uint4*>(s_q + (rl >> 3) * kRows * 128 + swz128(r, rl & 7)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready);
    }
    // a page that is missing where some row looks: every tile is checked key by key
    bool hole = false;
    {
      const int sh = a.kv.page_shift;
      if (n_tiles > 0) {
        for (int i = tid; i < (sink_any + (1 << sh) - 1) >> sh; i += 128)
          hole |= page_of(a.kv, tile.b, i << sh) < 0;
        for (int i = (lo_any >> sh) + tid; i <= p_last >> sh; i += 128)
          hole |= page_of(a.kv, tile.b, i << sh) < 0;
      }
      hole = softmax_any(hole);
    }
    const float c2 = fabsf(a.scale) * kLog2e;
    float m = -INFINITY, l = 0.f;  // m in units of S
    // The product P V of tile j has ended.  Tiles alternate between two barriers: the one of
    // tile j - 2 is known to have ended whenever tile j is asked for.
    auto wait_pv = [&](int j) {
      ok = ok && warp_wait(&pv_done[j & 1], (j >> 1) & 1);
      tc_fence_after();
    };
    // A wait that runs out makes the warp's rows NaN; it goes on through the tiles without
    // waiting, as the others may stand at the warps' common barrier.
    for (int j = 0; j < n_tiles; ++j) {
      const int k0 = tile_key(j), buf = j % C::kS;
      const uint32_t ts = tm_s + tl + buf * kTile;
      ok = ok && warp_wait(&s_full[buf], (j / C::kS) & 1);
      tc_fence_after();
      // every live row sees every key of the tile?
      const bool edge = hole || tile.p0 < 0 || k0 + kTile - 1 > tile.p0 ||
                        (k0 < lo_max && k0 + kTile > sink_all);
      if (edge) {
        // S with what the row does not see at -inf, back to TMEM: a pass of its own keeps the
        // tests out of the common path (one per element there made its code miss the
        // instruction cache: 45 us a tile instead of 2)
#pragma unroll 1
        for (int c = 0; c < kTile; c += 16) {
          uint32_t r[16];
          tmem_ld16(ts + c, r);
          tmem_ld_wait();
          const int j0 = k0 + c;
          const uint32_t off = hole && page_of(a.kv, tile.b, j0) < 0 ? 0x7fffffffu : 0u;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int jj = j0 + e;
            const bool see = jj <= p && (jj < sink || jj >= lo);
            r[e] = see ? r[e] | off : 0xff800000u;
          }
          tmem_st16(ts + c, r);
        }
        tmem_st_wait();
      }
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kTile; c += 32) {
        uint32_t r[32];
        tmem_ld32(ts + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) top = fmaxf(top, __uint_as_float(r[e]));
      }
      // the maximum follows when it lags by more than kGrow (always from -inf)
      const bool grow = (top - m) * c2 > kGrow || (m == -INFINITY && top > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        const float old = m;
        m = fmaxf(m, top);
        const float keep = old == -INFINITY ? 0.f : ex2((old - m) * c2);
        l *= keep;
        if (j > 0) {
          wait_pv(j - 1);
#pragma unroll 1
          for (int d = 0; d < D; d += 16) {
            uint32_t r[16];
            tmem_ld16(tm_o + tl + d, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * keep);
            tmem_st16(tm_o + tl + d, r);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : m * c2;
#pragma unroll
      for (int c = 0; c < kTile; c += 32) {
        uint32_t r[32], w[16];
        tmem_ld32(ts + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float p0 = ex2(fmaf(__uint_as_float(r[e]), c2, -base));
          const float p1 = ex2(fmaf(__uint_as_float(r[e + 1]), c2, -base));
          l += p0 + p1;
          w[e / 2] = pack_bf16(p0, p1);
        }
        tmem_st16(ts + c / 2, w);  // over columns that have been read
      }
      tmem_st_wait();
      if (edge) {
        // V of this tile: thread = key
        const int vseq = C::kS == 2 ? C::kKc + (j + 1 < n_tiles ? C::kKc : 0) + j * (C::kKc + C::kVc)
                                    : C::kKc + j * (C::kKc + C::kVc);
        const int q = vseq + tid / C::kVr, s = q % C::kSlots;
        for (int c = 0; c < C::kVc && ok; ++c)
          ok = warp_wait(&full[(vseq + c) % C::kSlots], ((vseq + c) / C::kSlots) & 1);
        char* row = s_ring + s * kChunk + (tid % C::kVr) * 128;
        const int jj = k0 + tid;
        const bool seen = jj <= p_last && (jj < sink_any || jj >= lo_any);
        bool bad = false;
        if (ok && seen)
#pragma unroll 4
          for (int i = 0; i < D / 8; ++i) {  // 16-byte pieces, each lane from its own bank on
            const uint4 v = *reinterpret_cast<const uint4*>(row + (i >> 3) * C::kVr * 128 + (((i + lane) & 7) << 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x2 = (&v.x)[e];
              bad |= (x2 & 0x7f80u) == 0x7f80u || (x2 & 0x7f800000u) == 0x7f800000u;
            }
          }
        if (ok && (!seen || bad)) {
          for (int i = 0; i < D / 8; ++i)
            *reinterpret_cast<uint4*>(row + (i >> 3) * C::kVr * 128 + (((i + lane) & 7) << 4)) = uint4{0, 0, 0, 0};
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        const uint32_t some = __ballot_sync(0xffffffffu, bad);
        if (lane == 0) s_bad[warp] = some;
        if (softmax_any(bad)) {
          // add these keys to the rows that see them, before the tile's product
          if (j > 0) wait_pv(j - 1);
          if (j == 0) {
            const uint32_t zero[16] = {};
            for (int d = 0; d < D; d += 16) tmem_st16(tm_o + tl + d, zero);
            tmem_st_wait();
            if (tid == 0) *(volatile int*)&s_first = 1;
          }
          for (int w = 0; w < 4 && ok; ++w) {
            uint32_t left = s_bad[w];
            while (left) {
              const int key = w * 32 + __ffs(left) - 1;
              left &= left - 1;
              const uint32_t pw = tmem_ld1(ts + key / 2);
              tmem_ld_wait();
              const float pk = __uint_as_float(key & 1 ? pw & 0xffff0000u : pw << 16);
              const int jk = k0 + key;
              const bool mine = jk <= p && (jk < sink || jk >= lo);
              const int page = page_of(a.kv, tile.b, jk);
              const __nv_bfloat16* vr = a.kv.v + max(page, 0) * a.kv.v_page_stride +
                                        ((int64_t(h) << a.kv.page_shift) + (jk & ((1 << a.kv.page_shift) - 1))) * D;
              for (int d = 0; d < D; d += 16) {
                uint32_t r[16];
                tmem_ld16(tm_o + tl + d, r);
                tmem_ld_wait();
                if (mine && page >= 0)
#pragma unroll
                  for (int e = 0; e < 16; ++e)
                    r[e] = __float_as_uint(fmaf(pk, __bfloat162float(vr[d + e]), __uint_as_float(r[e])));
                tmem_st16(tm_o + tl + d, r);
              }
              tmem_st_wait();
            }
          }
          softmax_any(false);  // s_bad is free again
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[buf]);
    }
    if (n_tiles > 0) wait_pv(n_tiles - 1);
    // ---- epilogue: O / l
    __nv_bfloat16* out = a.out + (int64_t(tile.t0 + tok) * a.Hq + int64_t(h) * G + g) * D;
    const bool zero = p < 0 || n_tiles == 0;
    const float inv = 1.f / l;
#pragma unroll 1
    for (int d = 0; d < D; d += 16) {
      uint32_t r[16];
      if (n_tiles > 0) {
        tmem_ld16(tm_o + tl + d, r);
        tmem_ld_wait();
      }
      if (row_live) {
        uint4 y[2];
        uint32_t* w = reinterpret_cast<uint32_t*>(y);
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          float y0 = 0.f, y1 = 0.f;
          if (tile.over || !ok) {
            y0 = y1 = NAN;
          } else if (!zero) {
            y0 = __uint_as_float(r[e]) * inv;
            y1 = __uint_as_float(r[e + 1]) * inv;
          }
          w[e / 2] = pack_bf16(y0, y1);
        }
        reinterpret_cast<uint4*>(out + d)[0] = y[0];
        reinterpret_cast<uint4*>(out + d)[1] = y[1];
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 5) tmem_dealloc(s_tmem, C::kCols);
}

// Rows behind the last sequence (and before the first) get zeros.
__global__ void __launch_bounds__(256) tail_rows_kernel(const AttnArgs a) {
  const int64_t row = int64_t(a.Hq) * a.kv.D / 8;  // 16-byte pieces of a packed row
  const int lo = max(a.cu_q[0], 0), hi = max(a.cu_q[a.kv.B], lo);
  uint4* out = reinterpret_cast<uint4*>(a.out);
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < int64_t(min(lo, a.T)) * row; i += int64_t(gridDim.x) * 256)
    out[i] = uint4{0, 0, 0, 0};
  for (int64_t i = min(hi, a.T) * row + int64_t(blockIdx.x) * 256 + threadIdx.x; i < a.T * row; i += int64_t(gridDim.x) * 256)
    out[i] = uint4{0, 0, 0, 0};
}

bool page_map(CUtensorMap* map, const PagedKV& kv, const __nv_bfloat16* base, int64_t page_stride,
              int rows) {
  const uint64_t D = kv.D, ps = uint64_t(1) << kv.page_shift;
  const uint64_t dims[5] = {64, ps, D / 64, uint64_t(kv.Hkv), uint64_t(kv.n_pages)};
  const uint64_t strides[4] = {D * 2, 128, ps * D * 2, uint64_t(page_stride) * 2};
  const uint32_t box[5] = {64, uint32_t(rows), 1, 1, 1};
  return make_tmap_bf16_nd(map, base, 5, dims, strides, box);
}

template <int D>
cudaError_t launch_one(const AttnArgs& a, cudaStream_t st) {
  using C = Cfg<D>;
  const int ps = 1 << a.kv.page_shift, per = kRows / (a.Hq / a.kv.Hkv);
  CUtensorMap mk{}, mv{};
  if (a.kv.max_pages > 0 &&
      (!page_map(&mk, a.kv, a.kv.k, a.kv.k_page_stride, ps < kTile ? ps : kTile) ||
       !page_map(&mv, a.kv, a.kv.v, a.kv.v_page_stride, ps < C::kVr ? ps : C::kVr)))
    return cudaErrorInvalidValue;
  const int64_t tiles = int64_t(a.T) / per + a.kv.B;  // slots of find_tile
  if (tiles * a.kv.Hkv > 0x7fffffffLL) return cudaErrorInvalidValue;
  attn_prefill_kernel<D><<<unsigned(tiles * a.kv.Hkv), 192, C::kSmem, st>>>(mk, mv, a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  tail_rows_kernel<<<16, 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t attn_prefill_init() {
  cudaError_t e = cudaFuncSetAttribute(attn_prefill_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<64>::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(attn_prefill_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<128>::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(attn_prefill_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<256>::kSmem);
  return e;
}

cudaError_t launch_attn_prefill(const AttnArgs& args, cudaStream_t st) {
  AttnArgs a = args;
  if (a.T == 0) return cudaSuccess;
  if (a.kv.n_pages == 0) a.kv.max_pages = 0;  // no page: every row with keys gets NaN
  switch (a.kv.D) {
    case 64: return launch_one<64>(a, st);
    case 128: return launch_one<128>(a, st);
    default: return launch_one<256>(a, st);
  }
}

}  // namespace pmoe
