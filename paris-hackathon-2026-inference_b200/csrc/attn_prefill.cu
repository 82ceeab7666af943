// Attention of packed prompts and prompt chunks over the paged cache, on the tensor cores.
//   o = sum_j softmax_j(scale q.k_j) v_j over the keys that each row sees.
//
// One CTA, or a pair of CTAs, per (128 rows of one sequence for each CTA, key/value head).  The
// rows are tokens x the G query heads that share the head, so one pass over K and V serves
// all of them.  Keys come in tiles of 128:
//   S = Q K^T         128 x 128, operands in shared memory, S in TMEM
//   P = 2^(S c - m)   a thread per row takes its S from TMEM into registers, which frees S for
//                     the next tile's product at once, and writes P (bf16) to TMEM
//   O += P V          A = P from TMEM, B = V from shared memory (dims contiguous), O in TMEM
// Two groups of four softmax warps take the even and the odd tiles, each with a P buffer of its
// own, so that one group's exponentials run beside the other's maxima and beside the products.
// The running maximum m of a row passes from group to group through shared memory.  It moves
// only when a tile's maximum exceeds it by more than 8 (in powers of two): weights then stay
// below 2^8, exact to the same relative rounding, and O is rescaled rarely.
//
// In a pair each CTA fetches half of every tile (64 of the keys of K, half the dims of V) and the
// products read both halves (cta_group::2): a lone CTA asks for 128 KiB of K and V per 2048
// tensor cycles at D = 256, more than its 160 KiB ring hides at L2 latency.
//
// Warps 0-7: softmax and epilogue; warps 8 and 9: TMA of K (and Q) and of V, each through a ring
// of 16 KiB chunks; warps 10 and 11: the products S and P V (a pair's first CTA issues for
// both, and both CTAs' copies report to its barriers); warps 12-15 clean V where rows do not
// see all of it.
//
// Few rows: the keys are split over several CTAs (gridDim.y), whose parts join_kernel joins.
//
// Values that a row does not see must not reach its sum even where they are not finite, but
// 0 x inf is NaN: in tiles that are cut by some row's sight, V rows that nobody sees or that
// hold a non-finite number are zeroed in shared memory, and the latter are added to the rows
// that see them one by one.  Warps of their own do this as the tile lands: in the softmax warps it
// cost prompts of 4096 and 2531 tokens, 32/4 heads of 128, 260 us instead of 224 (215 with no
// cleaning at all).
//
// Bound by the tensor cores for long prompts at D = 256: 8192 tokens of 16/2 heads 383 us, 20
// calls in a graph (550 GFLOP, 1.43 PFLOP/s, 83 % of a matrix product's best; under the power cap
// of a long run 447), a tile of a pair 2100 cycles where the products alone need 2048.  At D = 128
// and 64 by a row's softmax: 2000 cycles a tile and group, 1024 of them the exponential unit (219 us
// for the 4096 and 2531 tokens above, 0.87 PFLOP/s; 203 at D = 64).  Short calls by a block's fixed
// 7.5 us: 3.5 until the first S, 2.7 from the last product to the end, 1.2 between blocks.
#include <algorithm>
#include <cfloat>

#include "paged.cuh"
#include "pmoe_tc.cuh"

namespace pmoe {

namespace {

constexpr int kRows = 128, kTile = 128, kThreads = 512, kChunk = 16384;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kCuts = 8;      // tiles with keys that some rows do not see, at a time
// Registers of a thread: the launch's, which init_one checks, dealt out to the roles (a sum above
// the launch's would wait for ever).  The softmax warps hold a row of S.
constexpr int kRegs = 128, kRegsSoftmax = 200, kRegsIssue = 64, kRegsClean = 48;
static_assert(256 * kRegsSoftmax + 128 * kRegsIssue + 128 * kRegsClean <= kThreads * kRegs, "");
constexpr float kGrow = 8.f;  // powers of two that a row's maximum may lag behind

template <int D, bool PAIR> struct Cfg {
  static constexpr int kN = PAIR ? 2 : 1;               // CTAs that share a tile
  static constexpr int kS = D == 256 ? 1 : 2;           // S buffers: 512 columns of TMEM hold
                                                        // O [D], S [kS][128], P [2][64]
  static constexpr int kSlots = (229376 - kRows * D * 2) / (2 * kChunk);  // of each ring
  // K chunk: [kKg groups of 64 dims][kKr keys][128 bytes]; V chunk: [kVg][kVr keys][128 bytes]
  static constexpr int kKr = kTile / kN, kKg = kChunk / (kKr * 128), kKc = D / (64 * kKg);
  static constexpr int kVg = D / (64 * kN), kVr = kChunk / (kVg * 128), kVc = kTile / kVr;
  static constexpr int kSmem = 1024 + kRows * D * 2 + 2 * kSlots * kChunk;
  static_assert(kKc * kChunk * kN == kTile * D * 2 && kVc == kKc, "");
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two 32-bit operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
// Boxes of the cache and of Q; `bar` is a shared::cluster address (a pair's copies may complete
// on the first CTA's barrier).
template <bool PAIR>
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int row, int cg,
                                        int h, int page, uint32_t bar) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(cg), "r"(h), "r"(page), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row), "r"(cg), "r"(h), "r"(page), "r"(bar)
        : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tma_load_q(uint32_t dst, const CUtensorMap* map, int d, int head,
                                           int token, uint32_t bar) {
  if (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(d), "r"(head), "r"(token), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(d), "r"(head), "r"(token), "r"(bar)
        : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}
// Shared-memory descriptors in two words: the low one holds the address and the leading
// offset and steps with plain 32-bit additions; the high one (stride 1024 bytes, version 1,
// 128-byte swizzle) is the same for all operands here.
constexpr uint32_t kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t leading) {
  return (saddr & 0x3FFFFu) >> 4 | (leading >> 4) << 16;
}
// D[tmem] (+)= A[smem] * B[smem]; with a TS prefix A is in TMEM, bf16 pairs in 32-bit columns.
#define PMOE_UMMA(GROUP, ADECL, AOP, AVAL)                                              \
  asm volatile(                                                                               \
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"                                             \
      "setp.ne.b32 p, %4, 0;\n\t" ADECL                                                       \
      "mov.b64 b, {%2, %5};\n\t"                                                              \
      "tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], " AOP ", b, %3, p;\n\t}" ::"r"(d),    \
      "r"(AVAL), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescHi)                            \
      : "memory")
template <bool PAIR>
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if (PAIR)
    PMOE_UMMA("2", "mov.b64 a, {%1, %5};\n\t", "a", a);
  else
    PMOE_UMMA("1", "mov.b64 a, {%1, %5};\n\t", "a", a);
}
template <bool PAIR>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if (PAIR)
    PMOE_UMMA("2", "", "[%1]", a);
  else
    PMOE_UMMA("1", "", "[%1]", a);
}
#undef PMOE_UMMA
template <bool PAIR> __device__ __forceinline__ void commit(uint64_t* bar) {
  if (PAIR)
    umma_commit_pair_both(bar);
  else
    umma_commit(bar);
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
// Whether any of the barrier's n threads says yes.
__device__ __forceinline__ bool bar_any(int id, int n, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "bar.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(n), "r"(uint32_t(x))
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void bar_arrive(int id, int n) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory");
}
// Arrive on a barrier of the MMA warps.  What it announces is in TMEM (wait::ld, wait::st and the
// tcgen05 fence order it); nothing else has been written, so no release: at cluster scope it
// would wait for all of the thread's stores (1276 cycles a tile, measured).
template <bool PAIR> __device__ __forceinline__ void tmem_signal(uint64_t* bar) {
  if (PAIR)
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                     mapa_shared(smem_u32(bar), 0))
                 : "memory");
  else
    mbar_arrive(bar);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, uint32_t x) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(x) : "memory");
}
// The n lowest bits (n <= 0: none, n >= 32: all).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}
// Whether a 32-bit word holds a bf16 that is not finite.
__device__ __forceinline__ bool nonfinite2(uint32_t x) {
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

// Block x's rows: slots of a sequence begin at cu[b] / tokens + b, which leaves each
// sequence at least its number of tiles.
struct TileOf {
  int b, t0, n, p0, len;  // sequence, first packed row, tokens, index of the first, keys
  bool over;
};
// (A whole warp calls this.)
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int per, int x, TileOf* o) {
  const int32_t* cu = a.cu_q;
  const int lo = last_at_or_before(a.kv.B, x, [=](int b) { return cu[b] / per + b; });
  if (lo < 0) return false;
  // (cu_q may count rows that the call does not have)
  const int c0 = a.cu_q[lo], end = a.cu_q[lo + 1], c1 = min(end, a.T), len = a.kv.kv_lens[lo];
  const int i = x - (c0 / per + lo);
  if (c0 < 0 || c1 <= c0 || i < 0 || i > (c1 - c0 - 1) / per) return false;
  o->b = lo;
  o->t0 = c0 + i * per;
  o->n = min(per, c1 - o->t0);
  o->len = kv_len_of(len, a.kv.max_pages, a.kv.page_shift, &o->over);
  o->p0 = o->len - (end - o->t0);
  return true;
}

// Rows of no sequence, before cu_q[0] and from cu_q[B] on, get zeros (all blocks of the grid
// share them).
__device__ __forceinline__ void zero_rows(const AttnArgs& a, int first, int end) {
  const int lo = min(max(first, 0), a.T), hi = min(max(end, lo), a.T);
  if (lo == 0 && hi == a.T) return;
  const int64_t row = int64_t(a.Hq) * a.kv.D / 8;  // 16-byte pieces of a packed row
  const int64_t id = (int64_t(blockIdx.y) * gridDim.x + blockIdx.x) * kThreads + threadIdx.x;
  const int64_t step = int64_t(gridDim.x) * gridDim.y * kThreads;
  uint4* out = reinterpret_cast<uint4*>(a.out);
  for (int64_t i = id; i < lo * row; i += step) out[i] = uint4{0, 0, 0, 0};
  for (int64_t i = hi * row + id; i < a.T * row; i += step) out[i] = uint4{0, 0, 0, 0};
}

// Parts of a split call: O [D/4][128 rows][4] of (block x, split y), not yet divided (a thread
// has a row, so rows lie side by side), then each row's (m, l), m in powers of two.
struct Parts {
  float* o;
  float2* ml;
};
__host__ __device__ inline Parts parts_of(void* ws, int64_t blocks, int D) {
  float* o = static_cast<float*>(ws);
  return {o, reinterpret_cast<float2*>(o + blocks * kRows * D)};
}
template <int D> __device__ __forceinline__ float4* part_row(const Parts& p, int64_t part, int row) {
  return reinterpret_cast<float4*>(p.o) + part * (kRows * D / 4) + row;
}

template <int D, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) attn_prefill_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
    const __grid_constant__ CUtensorMap map_v, const AttnArgs a, void* ws) {
  using C = Cfg<D, PAIR>;
  extern __shared__ char smem_raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* s_q = smem;                    // [D/64][128 rows][128 bytes], swizzled
  char* s_k = smem + kRows * D * 2;    // the rings
  char* s_v = s_k + C::kSlots * kChunk;
  // full: a chunk has landed, in both CTAs (the first CTA's barrier counts), and is clean.
  // Tiles that are cut (cut_of): cut_full: of their u-th chunk of V at u % 8: this CTA's part has
  // landed; p_cut: of the e-th tile at e % 8: its weights are written; bad_known at e % 2: s_bad is
  // there, from both CTAs.  (The rings hold 6 chunks at most, so that chunk u + 8 is fetched, and
  // tile e + 8 met, after tile e's product, which waits for all who use these.)
  __shared__ uint64_t k_full[C::kSlots], k_empty[C::kSlots], v_full[C::kSlots], v_empty[C::kSlots];
  __shared__ uint64_t cut_full[kCuts], p_cut[kCuts], bad_known[2];
  __shared__ uint64_t s_full[2], s_free[C::kS], p_ready[2][2], pv_done[2], q_full;
  __shared__ uint32_t s_tmem;
  __shared__ int s_first;              // tile 0 adds to O (set to zero before) instead of setting it
  __shared__ uint32_t s_bad[2][D / 64][4];  // keys of a cut tile whose V, in those 64 dims, is not
                                            // finite and not seen by all rows
  __shared__ float s_m[kRows];

  // (shuffled, so that the compiler sees one value per warp and keeps the roles' addresses
  // in uniform registers)
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int rank = PAIR ? int(cluster_ctarank()) : 0;
  const int G = a.Hq / a.kv.Hkv, per = kRows / G;
  const int block = blockIdx.x / C::kN, blocks = gridDim.x / C::kN;
  const int h = block % a.kv.Hkv;
  const int x = blocks / a.kv.Hkv - 1 - block / a.kv.Hkv;  // late tiles, the longest, first
  pdl_wait();
  const int cu_first = a.cu_q[0], cu_end = a.cu_q[a.kv.B];
  TileOf tile;
  if (!find_tile(a, per * C::kN, x, &tile)) {  // both CTAs of a pair, or none
    zero_rows(a, cu_first, cu_end);
    return;
  }

  // keys that some row sees: [0, sink_any) and [lo_any, p_last]
  const int p_last = tile.p0 + tile.n - 1, p_first = max(tile.p0, 0);
  int lo_any = 0, sink_any = 0, lo_max = 0, sink_all = 0;
  int n_tiles = 0, ns = 0, w0 = 0, j_lo = 0;
  if (p_last >= 0 && !tile.over) {
    visible_keys(p_first, a.window, a.sinks, &lo_any, &sink_all);
    visible_keys(p_last, a.window, a.sinks, &lo_max, &sink_any);
    ns = (sink_any + kTile - 1) / kTile;
    w0 = max(lo_any / kTile, ns);
    n_tiles = ns + p_last / kTile + 1 - w0;
    if (gridDim.y > 1) {  // this CTA's share of the keys
      j_lo = int(int64_t(n_tiles) * blockIdx.y / gridDim.y);
      n_tiles = int(int64_t(n_tiles) * (blockIdx.y + 1) / gridDim.y) - j_lo;
    }
  }
  auto tile_key = [&](int j) {
    j += j_lo;
    return (j < ns ? j : w0 + j - ns) * kTile;
  };

  auto cut_of = [&](int j) {  // may some row not see some key of the tile?
    const int k0 = tile_key(j);
    return tile.p0 < 0 || k0 + kTile - 1 > tile.p0 || (k0 < lo_max && k0 + kTile > sink_all);
  };

  if (warp == 10) {
    if (PAIR) {
      tmem_alloc_pair(&s_tmem, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&s_tmem, 512);
      tmem_relinquish();
    }
  }
  if (tid == 0) {
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 4 * C::kN);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < kCuts; ++i) {
      mbar_init(&cut_full[i], 1);
      mbar_init(&p_cut[i], 4);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&bad_known[i], 4 * C::kN);
    for (int i = 0; i < C::kS; ++i) mbar_init(&s_free[i], 4 * C::kN);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i][0], 4 * C::kN);
      mbar_init(&p_ready[i][1], 4 * C::kN);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(&q_full, 1);
    s_first = 0;
    mbar_fence_init();
  }
  tc_fence_before();
  if (PAIR)
    cluster_sync_all();
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tm_o = __shfl_sync(0xffffffffu, s_tmem, 0), tm_p = tm_o + D, tm_s = tm_p + 128;

  if (warp >= 12) {
    // ---- V of the cut tiles: a thread has 64 dims of a key of each chunk.  A wait that runs out in
    // one warp stops all four, at the barrier that they next meet at: a warp that left by itself
    // would keep the others there.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsClean));
    const int line = tid & 127, row = line % C::kVr, wc = warp & 3;
    const int of = rank * C::kVg + wc * 32 / C::kVr;  // 64 dims of D
    bool ok = true;
    for (int j = 0, e = 0; j < n_tiles; ++j) {
      if (!cut_of(j)) continue;
      const int k0 = tile_key(j);
      uint32_t(*bad_at)[4] = s_bad[e & 1];
      bool any = false;
      for (int c = 0; c < C::kVc; ++c) {
        const int u = e * C::kVc + c;
        // (one warp polls: four took issue slots from the softmax warps)
        if (wc == 0) ok = ok && warp_wait(&cut_full[u % kCuts], (u / kCuts) & 1);
        ok = !bar_any(6, 128, !ok);
        if (!ok) break;
        const int jj = k0 + c * C::kVr + row;
        const bool some = jj <= p_last && (jj < sink_any || jj >= lo_any);
        const bool all = jj <= tile.p0 && (jj >= lo_max || jj < sink_all);
        uint4* v = reinterpret_cast<uint4*>(s_v + (j * C::kVc + c) % C::kSlots * kChunk + line * 128);
        bool bad = false;
        if (some && !all) {  // (lines begin in the same bank)
#pragma unroll 4
          for (int i = 0; i < 8; ++i) {
            const uint4 x = v[(i + lane) & 7];
            bad |= nonfinite2(x.x) || nonfinite2(x.y) || nonfinite2(x.z) || nonfinite2(x.w);
          }
        }
        if (!some || bad)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[(i + lane) & 7] = uint4{0, 0, 0, 0};
        const uint32_t who = __ballot_sync(0xffffffffu, bad);
        if (lane == 0) {
          uint32_t* word = &bad_at[of][(c * C::kVr + wc * 32 % C::kVr) / 32];
          if (PAIR) {
            st_cluster(mapa_shared(smem_u32(word), 0), who);
            st_cluster(mapa_shared(smem_u32(word), 1), who);
          } else {
            *word = who;
          }
        }
        any |= who != 0;
      }
      if (!ok) break;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (PAIR) {  // what either CTA found: the product adds both halves of the dims to both's rows
        if (lane == 0)
          for (int cta = 0; cta < 2; ++cta) mbar_arrive_cluster(mapa_shared(smem_u32(&bad_known[e & 1]), cta));
        ok = __all_sync(0xffffffffu, mbar_wait_cluster(&bad_known[e & 1], (e >> 1) & 1));
        for (int w = 0; w < D / 16; ++w) any |= *(volatile uint32_t*)&bad_at[w / 4][w % 4] != 0;
      } else {
        any = bar_any(6, 128, any);
      }
      if (ok && any) {
        // What was taken out because not all rows see it and it is not finite: added to the
        // rows that do (thread = row from here), between the products of tiles j - 1 and j.
        ok = warp_wait(&p_cut[e % kCuts], (e / kCuts) & 1);
        // (the barrier's use before, tile j - 3, has ended: the weights were written after j - 2's)
        if (j > 0) ok = ok && warp_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1);
        tc_fence_after();
        const uint32_t tl = uint32_t(wc) << 21, o = tm_o + tl, tp = tm_p + tl + (j & 1) * 64;
        const int tok = rank * per + line / G;
        const int p = line / G < per && tok < tile.n ? tile.p0 + tok : -1;
        int lo = 0, sink = 0;
        if (p >= 0) visible_keys(p, a.window, a.sinks, &lo, &sink);
        if (j == 0) {
          const uint32_t zero[16] = {};
          for (int d = 0; d < D; d += 16) tmem_st16(o + d, zero);
          tmem_st_wait();
          if (line == 0) *(volatile int*)&s_first = 1;
        }
        for (int w = 0; w < 4 && ok; ++w) {
          uint32_t left = 0;
          for (int x = 0; x < D / 64; ++x) left |= bad_at[x][w];
          while (left) {
            const int bit = __ffs(left) - 1, key = w * 32 + bit, jk = k0 + key;
            left &= left - 1;
            const uint32_t pw = tmem_ld1(tp + key / 2);
            tmem_ld_wait();
            const float pk = __uint_as_float(key & 1 ? pw & 0xffff0000u : pw << 16);
            const int page = page_of(a.kv, tile.b, jk);
            const bool mine = page >= 0 && jk <= p && (jk < sink || jk >= lo);
            const __nv_bfloat16* vr = a.kv.v + max(page, 0) * a.kv.v_page_stride +
                                      ((int64_t(h) << a.kv.page_shift) + (jk & ((1 << a.kv.page_shift) - 1))) * D;
            for (int d = 0; d < D; d += 16) {
              if (!(bad_at[d / 64][w] >> bit & 1)) continue;  // left in the product
              uint32_t x[16];
              tmem_ld16(o + d, x);
              tmem_ld_wait();
              if (mine)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  x[i] = __float_as_uint(fmaf(pk, __bfloat162float(vr[d + i]), __uint_as_float(x[i])));
              tmem_st16(o + d, x);
            }
            tmem_st_wait();
          }
        }
        tc_fence_before();
        __syncwarp();
      }
      if (ok && lane == 0)
        for (int c = 0; c < C::kVc; ++c) {
          uint64_t* bar = &v_full[(j * C::kVc + c) % C::kSlots];
          if (PAIR)
            mbar_arrive_cluster(mapa_shared(smem_u32(bar), 0));
          else
            mbar_arrive(bar);
        }
      __syncwarp();
      ++e;
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (warp < 10) {
      // ---- TMA of one operand
      const bool is_v = warp == 9;
      uint64_t* full = is_v ? v_full : k_full;
      uint64_t* empty = is_v ? v_empty : k_empty;
      const uint32_t ring = smem_u32(is_v ? s_v : s_k);
      const uint32_t first_full = mapa_shared(smem_u32(full), 0);  // the first CTA's barriers
      const int sh = a.kv.page_shift, ps = 1 << sh, per_tile = kTile >> sh;
      // this CTA's part of a tile: K: half the keys in a pair; V: half the dims
      const int keys = is_v ? C::kVr : C::kKr, groups = is_v ? C::kVg : C::kKg;
      const int rows = min(ps, keys), grp = lane % groups, r = lane / groups * rows;  // this lane's box
      if (!is_v && n_tiles > 0) {
        // Q: rows = tokens x heads, as they lie.  Rows behind the tile's tokens are other
        // tokens' or zeros, and their results are not used.
        if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&q_full, C::kN * per * G * D * 2);
        __syncwarp();
        if (lane < D / 64)
          tma_load_q<PAIR>(smem_u32(s_q + lane * kRows * 128), &map_q, lane * 64, h * G,
                           tile.t0 + rank * per, mapa_shared(smem_u32(&q_full), 0));
      }
      auto pages_of = [&](int j) {  // lane i: the tile's i-th page
        return j < n_tiles && lane < per_tile ? page_of(a.kv, tile.b, tile_key(j) + lane * ps) : -1;
      };
      int next = pages_of(0), slot = 0, use = 0, cuts = 0;
      bool ok = true;
      int seq = 0;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int page = next;
        next = pages_of(j + 1);
        const bool cut = is_v && cut_of(j);
        for (int c = 0; c < C::kKc; ++c, ++seq) {
          if (use > 0) ok = warp_wait(&empty[slot], (use - 1) & 1);
          if (!ok) break;
          uint64_t* landed = &cut_full[cuts % kCuts];
          cuts += cut;
          if (lane == 0) {
            if (cut) {
              mbar_arrive_expect_tx(landed, kChunk);
            } else if (rank == 0) {
              mbar_expect_tx(&full[slot], C::kN * kChunk);
              mbar_arrive_n(&full[slot], is_v ? 4 * C::kN : 1);
            }
          }
          __syncwarp();
          const int key = (is_v ? c * C::kVr : rank * C::kKr) + r;  // in the tile
          const int cg = (is_v ? rank * C::kVg : c * C::kKg) + grp;
          const int at = __shfl_sync(0xffffffffu, page, min(key >> sh, 31));
          if (r < keys)
            tma_box<PAIR>(ring + slot * kChunk + (grp * keys + r) * 128, is_v ? &map_v : &map_k,
                          key & (ps - 1), cg, h, at < 0 ? a.kv.n_pages : at,  // no page: zeros
                          cut ? smem_u32(landed) : first_full + slot * 8);
          slot = slot + 1 == C::kSlots ? 0 : slot + 1;
          use += slot == 0;
        }
      }
      if (!ok) {  // a wait ran out: let the copies land before the CTA ends
        for (int q = max(0, seq - C::kSlots); q < seq; ++q)
          if (rank == 0 && !(is_v && cut_of(q / C::kVc)))
            mbar_wait(&full[q % C::kSlots], (q / C::kSlots) & 1);
        for (int u = max(0, cuts - C::kSlots); u < cuts; ++u) mbar_wait(&cut_full[u % kCuts], (u / kCuts) & 1);
      }
    } else {
      // ---- the products: a warp each for S and P V walks and waits, one lane issues.  (A warp
      // of its own for each: one warp for both spent 3300 cycles a tile on waits and issue, the
      // tensor cores 2048.  The whole warp, so that the addresses are uniform: issued from one
      // lane's branch, with descriptors built one by one, a product took 130 to 310 cycles to
      // issue.)  The waits acquire at CTA scope also for what the pair's other CTA signals:
      // these warps themselves read none of that data (the tensor cores do, after the other CTA's
      // own waits and proxy fences), and a cluster-scope acquire costs some 400 cycles.
      if (rank == 0 && n_tiles > 0) {
        int slot = 0, phase = 0;
        bool ok = true;
        auto chunk_next = [&]() {
          slot = slot + 1 == C::kSlots ? 0 : slot + 1;
          phase ^= slot == 0;
        };
        if (warp == 10) {
          // A negative scale turns the sign of Q (bit 13).
          const uint32_t idesc = idesc_bf16_f32(kRows * C::kN, kTile) | (a.scale < 0.f ? 1u << 13 : 0u);
          const uint32_t ring = smem_u32(s_k), q_lo = desc_lo(smem_u32(s_q), 0);
          ok = warp_wait(&q_full, 0);
          for (int j = 0; j < n_tiles && ok; ++j) {
            const int buf = j % C::kS;
            const uint32_t d = tm_s + buf * kTile;
            if (j >= C::kS) ok = warp_wait(&s_free[buf], (j / C::kS - 1) & 1);
#pragma unroll 1
            for (int c = 0; c < C::kKc; ++c) {
              ok = ok && warp_wait(&k_full[slot], phase);
              tc_fence_after();
              if (!ok) break;
              const uint32_t qa = q_lo + c * C::kKg * kRows * 8, ka = desc_lo(ring + slot * kChunk, 0);
              if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4 * C::kKg; ++k)
                  umma_ss<PAIR>(d, qa + (k >> 2) * kRows * 8 + (k & 3) * 2,
                                ka + (k >> 2) * C::kKr * 8 + (k & 3) * 2, idesc, k > 0 ? 1 : c > 0);
                commit<PAIR>(&k_empty[slot]);
                if (c == C::kKc - 1) commit<PAIR>(&s_full[j & 1]);
              }
              __syncwarp();
              chunk_next();
            }
          }
        } else {
          constexpr uint32_t idesc = idesc_bf16_f32(kRows * C::kN, D) | 1u << 16;  // B: dims contiguous
          const uint32_t ring = smem_u32(s_v);
          for (int j = 0; j < n_tiles && ok; ++j) {
            const uint32_t p = tm_p + (j & 1) * 64;
            uint32_t add = 1;
#pragma unroll 1
            for (int c = 0; c < C::kVc; ++c) {
              ok = ok && warp_wait(&v_full[slot], phase);
              const uint32_t v_lo = desc_lo(ring + slot * kChunk, C::kVr * 128);
              constexpr int kHalves = C::kVr == kTile ? 2 : 1, kSteps = C::kVr / 16 / kHalves;
#pragma unroll 1
              for (int half = 0; half < kHalves; ++half) {
                // the first 64 keys' weights come before the others'
                const int k0 = c * C::kVr + half * kTile / 2;
                if (k0 == 0 || k0 == kTile / 2)
                  ok = ok && warp_wait(&p_ready[j & 1][k0 > 0], (j >> 1) & 1);
                tc_fence_after();
                if (!ok) break;
                if (k0 == 0) add = j > 0 || *(volatile int*)&s_first;
                if (elect_one()) {
#pragma unroll
                  for (int k = 0; k < kSteps; ++k)
                    umma_ts<PAIR>(tm_o, p + k0 / 2 + k * 8, v_lo + (half * kSteps + k) * 128, idesc,
                                  k > 0 || k0 > 0 ? 1u : add);
                  if (half == kHalves - 1) {
                    commit<PAIR>(&v_empty[slot]);
                    if (c == C::kVc - 1) commit<PAIR>(&pv_done[j & 1]);
                  }
                }
                __syncwarp();
              }
              if (!ok) break;
              chunk_next();
            }
          }
        }
      }
      __syncwarp();
    }
  } else {
    // ---- softmax: group = warps 0-3 or 4-7, thread = row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int grp = warp >> 2, wq = warp & 3, row = tid & 127;
    const uint32_t tl = uint32_t(wq) << 21;  // this warp's TMEM lanes
    const int tok = rank * per + row / G, g = row % G;
    const bool row_live = row / G < per && tok < tile.n;
    const int p = row_live ? tile.p0 + tok : -1;  // < 0: sees nothing
    int lo = 0, sink = 0;
    if (p >= 0) visible_keys(p, a.window, a.sinks, &lo, &sink);
    bool ok = true;
    // a page that is missing where some row looks: every tile is checked key by key
    bool hole = false;
    {
      const int sh = a.kv.page_shift;
      if (n_tiles > 0) {
        for (int i = tid; i < (sink_any + (1 << sh) - 1) >> sh; i += 256)
          hole |= page_of(a.kv, tile.b, i << sh) < 0;
        for (int i = (lo_any >> sh) + tid; i <= p_last >> sh; i += 256)
          hole |= page_of(a.kv, tile.b, i << sh) < 0;
      }
      hole = bar_any(1, 256, hole);
    }
    // (never 0, which would make NaN of the -inf that stands for what a row does not see)
    float c2 = fabsf(a.scale) * kLog2e;
    if (c2 < FLT_MIN) c2 = FLT_MIN;
    float m = -INFINITY, l = 0.f;  // m in units of S; l relative to m
    // The product P V of tile j has ended.  Tiles alternate between two barriers, and a barrier's
    // parity tells two uses apart: tile j may be asked for only once tile j - 2's product is known
    // to have ended.  (This group waits for tile j - 2 in every tile j; products end in order.)
    auto wait_pv = [&](int j) {
      ok = ok && warp_wait(&pv_done[j & 1], (j >> 1) & 1);
      tc_fence_after();
    };
    // A wait that runs out makes the warp's rows NaN; it goes on through the tiles without
    // waiting, as the others may stand at the groups' barriers.
    int cuts = 0;
    for (int j = grp; j < n_tiles; j += 2) {
      const int k0 = tile_key(j);
      const int buf = j % C::kS;
      const uint32_t ts = tm_s + tl + buf * kTile, tp = tm_p + tl + grp * 64;
      cuts += j > 0 && cut_of(j - 1);
      const int e_cut = cuts;
      const bool cut = cut_of(j);
      cuts += cut;
      ok = ok && warp_wait(&s_full[grp], (j >> 1) & 1);
      tc_fence_after();
      uint32_t r[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, r[c]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) tmem_signal<PAIR>(&s_free[buf]);
      if (cut || hole) {
        // What the row does not see at -inf, as bits of the tile's keys: 0..hi but not
        // [a, b).  (A comparison per element took 7000 cycles a tile, most of it fetching code.)
        const int hi = p - k0, ka = sink - k0, kb = lo - k0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t see = low_bits(hi + 1 - 32 * c) & (low_bits(ka - 32 * c) | ~low_bits(kb - 32 * c));
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(see >> e & 1)) r[c][e] = 0xff800000u;
        }
        if (hole) {  // keys without a page: NaN where they are seen
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (page_of(a.kv, tile.b, k0 + c * 16) < 0)
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                uint32_t& x = r[c >> 1][(c & 1) * 16 + e];
                x = x == 0xff800000u ? x : 0x7fffffffu;
              }
        }
      }
      float top;
      {
        float t[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) t[e] = __uint_as_float(r[0][e]);
#pragma unroll
        for (int e = 4; e < 128; ++e) t[e & 3] = fmaxf(t[e & 3], __uint_as_float(r[e >> 5][e & 31]));
        top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
      }
      // the maximum as the other group left it; it follows the tile's when it lags by more
      // than kGrow (always from -inf)
      float m_now = -INFINITY;
      if (j > 0) {
        named_bar_sync(2 + grp, 256);
        m_now = s_m[row];
      }
      const bool grow = (top - m_now) * c2 > kGrow || (m_now == -INFINITY && top > -INFINITY);
      const bool grows = __any_sync(0xffffffffu, grow);
      const float m_was = m_now;
      if (grows) {
        m_now = fmaxf(m_now, top);
        s_m[row] = m_now;
      }
      if (j == 0) s_m[row] = m_now;
      if (j + 1 < n_tiles) bar_arrive(3 - grp, 256);
      if (grows && j > 0) {
        const float keep = m_was == -INFINITY ? 0.f : ex2((m_was - m_now) * c2);
        if (j >= 2) wait_pv(j - 2);  // (which also ends tile j - 3's, before j - 1 on its barrier)
        wait_pv(j - 1);
#pragma unroll 1
        for (int d = 0; d < D; d += 16) {
          uint32_t x[16];
          tmem_ld16(tm_o + tl + d, x);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * keep);
          tmem_st16(tm_o + tl + d, x);
        }
      }
      if (m != m_now) {  // this group's sum follows, whichever group moved the maximum
        l *= m == -INFINITY ? 0.f : ex2((m - m_now) * c2);
        m = m_now;
      }
      const float base = m == -INFINITY ? 0.f : m * c2;
      const float2 cc = make_float2(c2, c2), bb = make_float2(-base, -base);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          float2 y = fma2(make_float2(__uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1])), cc, bb);
          y.x = ex2(y.x);
          y.y = ex2(y.y);
          sum = add2(sum, y);
          w[e / 2] = pack_bf16(y.x, y.y);
        }
        if (c == 0 && j >= 2) wait_pv(j - 2);  // this group's P buffer is free
        tmem_st16(tp + c * 16, w);
        if (c == 1) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) tmem_signal<PAIR>(&p_ready[grp][0]);
        }
      }
      l += sum.x + sum.y;
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (cut) mbar_arrive(&p_cut[e_cut % kCuts]);
        tmem_signal<PAIR>(&p_ready[grp][1]);
      }
    }
    if (n_tiles > 1) wait_pv(n_tiles - 2);
    if (n_tiles > 0) wait_pv(n_tiles - 1);
    // ---- the groups' sums, each brought to the last maximum (in the place of Q, which is done)
    float* s_l = reinterpret_cast<float*>(s_q);
    named_bar_sync(1, 256);
    const float m_end = n_tiles > 0 ? s_m[row] : -INFINITY;
    s_l[grp * kRows + row] = !ok ? NAN : l * (m == m_end ? 1.f : m == -INFINITY ? 0.f : ex2((m - m_end) * c2));
    named_bar_sync(1, 256);
    const float total = s_l[row] + s_l[kRows + row];
    // (not earlier: join_kernel's CTAs would crowd onto the few SMs that have no CTA of this kernel)
    pdl_trigger();
    // ---- epilogue: O / l, half the dims each
    const bool zero = p < 0, lost = tile.over || !ok;
    const int d0 = grp * (D / 2);
    if (gridDim.y > 1) {
      const int64_t part = int64_t(blockIdx.x) * gridDim.y + blockIdx.y;
      const Parts parts = parts_of(ws, int64_t(gridDim.x) * gridDim.y, D);
      if (row_live && grp == 0)
        parts.ml[part * kRows + row] = make_float2(m_end == -INFINITY ? -INFINITY : m_end * c2, lost ? NAN : total);
      float4* out = part_row<D>(parts, part, row);
#pragma unroll 1
      for (int d = d0; d < d0 + D / 2 && n_tiles > 0; d += 32) {
        uint32_t r[32];
        tmem_ld32(tm_o + tl + d, r);
        tmem_ld_wait();
        if (row_live)
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(out + (d + e) / 4 * kRows) = uint4{r[e], r[e + 1], r[e + 2], r[e + 3]};
      }
    } else {
      __nv_bfloat16* out = a.out + (int64_t(tile.t0 + tok) * a.Hq + int64_t(h) * G + g) * D + d0;
      const float inv = lost ? NAN : zero ? 0.f : 1.f / total;
#pragma unroll
      for (int d = 0; d < D / 2; d += 32) {  // 64 bytes of a row at a time
        uint32_t x[32];
        if (n_tiles > 0) {
          tmem_ld32(tm_o + tl + d0 + d, x);
          tmem_ld_wait();
        }
        if (row_live) {
          uint4 y[4];
          uint32_t* w = reinterpret_cast<uint32_t*>(y);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            // (a row that sees nothing: 0 whatever its columns hold)
            const float y0 = zero && !lost ? 0.f : __uint_as_float(x[e]) * inv;
            const float y1 = zero && !lost ? 0.f : __uint_as_float(x[e + 1]) * inv;
            w[e / 2] = pack_bf16(lost ? NAN : y0, lost ? NAN : y1);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) reinterpret_cast<uint4*>(out + d)[e] = y[e];
        }
      }
    }
    tc_fence_before();
  }
  zero_rows(a, cu_first, cu_end);
  if (PAIR) {
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while its peer may still signal it
    if (warp == 10) tmem_dealloc_pair(s_tmem, 512);
  } else {
    __syncthreads();
    if (warp == 10) tmem_dealloc(s_tmem, 512);
  }
}

// Joins the parts of a split call: a thread has 16 dims of a row, so that a warp's loads lie side
// by side in the parts and each thread writes a whole 32-byte sector.
template <int D>
__global__ void __launch_bounds__(2 * kRows) join_kernel(const AttnArgs a, void* ws, int splits) {
  const int G = a.Hq / a.kv.Hkv, per = kRows / G, row = threadIdx.x % kRows;
  const int d0 = blockIdx.y * 32 + threadIdx.x / kRows * 16;
  const int block = blockIdx.x, h = block % a.kv.Hkv;
  const int x = int(gridDim.x) / a.kv.Hkv - 1 - block / a.kv.Hkv;
  TileOf tile;
  // (the lengths are older than the main kernel, which has waited for whatever wrote them)
  const bool any = find_tile(a, per, x, &tile);
  pdl_wait();
  if (!any || row >= tile.n * G) return;
  const Parts parts = parts_of(ws, int64_t(gridDim.x) * splits, D);
  const float2* ml = parts.ml + int64_t(block) * splits * kRows + row;
  const float4* o = part_row<D>(parts, int64_t(block) * splits, row) + d0 / 4 * kRows;
  float top = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s * kRows].x);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  float4 acc[4] = {};
#pragma unroll 2
  for (int s = 0; s < splits; ++s, o += kRows * D / 4) {
    const float2 m = ml[s * kRows];
    if (m.x == -INFINITY && m.y == 0.f) continue;  // no key there: its O may be unwritten
    const float f = ex2(m.x - base);
    sum += m.y * (m.x == -INFINITY ? 1.f : f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 y = o[e * kRows];
      acc[e].x += f * y.x;
      acc[e].y += f * y.y;
      acc[e].z += f * y.z;
      acc[e].w += f * y.w;
    }
  }
  const int tok = row / G;
  const bool zero = tile.p0 + tok < 0;
  const float inv = 1.f / sum;
  uint32_t y[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float4 v = acc[e];
    y[2 * e] = pack_bf16(zero ? 0.f : v.x * inv, zero ? 0.f : v.y * inv);
    y[2 * e + 1] = pack_bf16(zero ? 0.f : v.z * inv, zero ? 0.f : v.w * inv);
  }
  if (tile.over)
    for (int e = 0; e < 8; ++e) y[e] = pack_bf16(NAN, NAN);
  uint4* out = reinterpret_cast<uint4*>(
      a.out + (int64_t(tile.t0 + tok) * a.Hq + int64_t(h) * G + row % G) * D + d0);
  out[0] = uint4{y[0], y[1], y[2], y[3]};
  out[1] = uint4{y[4], y[5], y[6], y[7]};
}

bool page_map(CUtensorMap* map, const PagedKV& kv, const __nv_bfloat16* base, int64_t page_stride,
              int rows) {
  const uint64_t D = kv.D, ps = uint64_t(1) << kv.page_shift;
  const uint64_t dims[5] = {64, ps, D / 64, uint64_t(kv.Hkv), uint64_t(kv.n_pages)};
  const uint64_t strides[4] = {D * 2, 128, ps * D * 2, uint64_t(page_stride) * 2};
  const uint32_t box[5] = {64, ps < uint64_t(rows) ? uint32_t(ps) : uint32_t(rows), 1, 1, 1};
  return make_tmap_bf16_nd(map, base, 5, dims, strides, box);
}

// How a call runs: rows in pairs of CTAs, or in single CTAs, which may split the keys.
struct Plan {
  bool pair;
  int splits;
  int64_t slots;  // of find_tile
};
// Slots that find_tile uses: floor(cu / per) + ceil(n / per) <= ceil((cu + n) / per).
int64_t slots_of(int T, int B, int per) { return (int64_t(T) + per - 1) / per + B - 1; }
// `keys`: the most that a row may see, by the table's width and the window.  (The lengths are on
// the device.  A table is as wide as its cache's longest sequence may get, so that few rows on few
// keys take parts that hold nothing: their CTAs set up and leave, and the join walks them.  On
// a table 32768 tokens wide 64 new tokens took 14.5 us, on one as wide as they are 10.7; 64 on
// 836 keys 16.6 and 15.6; 300 new 15.0 and 12.9; 64 on 30000 keys, and 32 prompts, the same.)
//
// Split: while the parts still fit on the GPU at once (300 tokens on 8000 keys: 152 CTAs took 66 us
// where 114 took 46), and no further than a part's tiles and the join cost the same: a tile takes
// about 1.2 us, joining one more part 0.4, so sqrt(3 tiles) parts.  64 tokens on 8000 keys, 2
// heads of 256: 95 us whole, 25 in 13 parts, 37 in 24; one token on 30000 keys: 328 whole, 34 in
// 24 parts, 47 in 74.  Below 6 tiles the join costs what it saves (16 times up to 8 tokens on up
// to 600 keys: 15.1 whole, 15.4 in 2; 4 heads of 128: 11.2 and 14.1).  All on tables as wide as
// the longest sequence.
//
// Pairs: at D = 256, where sequences have two CTAs' rows: one prompt of 2048 tokens 39 us, 42 in
// single CTAs, of 8192 back to back 446 and 462; up to 16 tokens each for 64 sequences on up to
// 4000 keys 106 in pairs, 78 in single CTAs.  At D = 128 a lone CTA hides its copies: 4096 and 2531
// tokens of 32/4 heads of 128 took 1 to 8 % longer in pairs.
Plan plan_of(int T, int B, int Hq, int Hkv, int D, int64_t keys) {
  const int per = kRows / (Hq / Hkv);
  const int64_t slots = slots_of(T, B, per), rows = (int64_t(T) + per - 1) / per;
  const int64_t tiles = (keys + kTile - 1) / kTile;
  const int64_t most = 148 / (std::max<int64_t>(rows, B) * Hkv);
  int splits = 1;
  while (tiles >= 6 && splits < most && int64_t(splits + 1) * (splits + 1) <= 3 * tiles) ++splits;
  if (splits > 1) return {false, splits, slots};
  const bool pair = D == 256 && rows >= 2 * int64_t(B);
  return {pair, 1, pair ? slots_of(T, B, 2 * per) : slots};
}

template <int D, bool PAIR>
cudaError_t launch_one(const AttnArgs& a, const Plan& plan, void* ws, cudaStream_t st) {
  using C = Cfg<D, PAIR>;
  CUtensorMap mq{}, mk{}, mv{};
  const uint32_t G = uint32_t(a.Hq / a.kv.Hkv);
  const uint64_t q_dims[3] = {uint64_t(D), uint64_t(a.Hq), uint64_t(a.T)};
  const uint64_t q_strides[2] = {uint64_t(a.Hq > 1 ? a.q_stride_h : D) * 2,
                                 uint64_t(a.T > 1 ? a.q_stride_t : int64_t(a.Hq) * D) * 2};
  const uint32_t q_box[3] = {64, G, kRows / G};
  if (!make_tmap_bf16_nd(&mq, a.q, 3, q_dims, q_strides, q_box)) return cudaErrorInvalidValue;
  if (a.kv.max_pages > 0 && (!page_map(&mk, a.kv, a.kv.k, a.kv.k_page_stride, C::kKr) ||
                             !page_map(&mv, a.kv, a.kv.v, a.kv.v_page_stride, C::kVr)))
    return cudaErrorInvalidValue;
  const int64_t blocks = plan.slots * a.kv.Hkv;
  if (blocks * C::kN > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaError_t e = launch_dependent(attn_prefill_kernel<D, PAIR>,
                                   dim3(unsigned(blocks * C::kN), unsigned(plan.splits)), kThreads,
                                   C::kSmem, C::kN, st, mq, mk, mv, a, ws);
  if (e != cudaSuccess || plan.splits == 1) return e;
  return launch_dependent(join_kernel<D>, dim3(unsigned(blocks), D / 32), 2 * kRows, 0, 1, st, a, ws,
                          plan.splits);
}

template <int D, bool PAIR> cudaError_t init_one() {
  // the registers that the roles share out are those of the launch
  cudaFuncAttributes f{};
  const cudaError_t e = cudaFuncGetAttributes(&f, attn_prefill_kernel<D, PAIR>);
  if (e != cudaSuccess) return e;
  if (f.numRegs != kRegs) return cudaErrorInvalidDeviceFunction;
  return cudaFuncSetAttribute(attn_prefill_kernel<D, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Cfg<D, PAIR>::kSmem);
}

}  // namespace

cudaError_t attn_prefill_init() {
  cudaError_t e;
  if ((e = init_one<64, false>()) != cudaSuccess || (e = init_one<128, false>()) != cudaSuccess ||
      (e = init_one<256, false>()) != cudaSuccess || (e = init_one<256, true>()) != cudaSuccess)
    return e;
  return cudaSuccess;
}

size_t attn_prefill_ws_bytes(int T, int B, int Hq, int Hkv, int D, int64_t keys) {
  const Plan p = plan_of(T, B, Hq, Hkv, D, keys);
  return p.splits == 1 ? 0 : size_t(p.slots) * Hkv * p.splits * kRows * (D + 2) * sizeof(float);
}

cudaError_t launch_attn_prefill(const AttnArgs& args, void* ws, cudaStream_t st) {
  AttnArgs a = args;
  if (a.T == 0) return cudaSuccess;
  int64_t keys = int64_t(a.kv.max_pages) << a.kv.page_shift;
  if (a.window > 0)  // (a window's tiles may begin and end inside, the sinks' end inside)
    keys = std::min(keys, int64_t(a.window) + a.sinks + 3 * kTile);
  const Plan p = plan_of(a.T, a.kv.B, a.Hq, a.kv.Hkv, a.kv.D, keys);
  if (a.kv.n_pages == 0) a.kv.max_pages = 0;  // no page: every row with keys gets NaN
  switch (a.kv.D) {
    case 64: return launch_one<64, false>(a, p, ws, st);
    case 128: return launch_one<128, false>(a, p, ws, st);
    default: return p.pair ? launch_one<256, true>(a, p, ws, st) : launch_one<256, false>(a, p, ws, st);
  }
}

}  // namespace pmoe
