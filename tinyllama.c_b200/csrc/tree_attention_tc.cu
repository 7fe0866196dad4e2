// Attention of drafted tokens on the 5th-generation tensor cores (sm_100a): bfloat16, heads of 64 and 128.
//
// The mathematics is tree_attention.cu's.  A tile is 128 pairs of a drafted row and one of the G query heads that share a key/value head,
// 128 / G rows with all of their heads, and a block takes two such tiles with every key tile that it fetches: 2 operations a pair and
// byte of keys and values, so it is bound by HBM up to some 250 pairs (measured peaks, 1,648 TFLOP/s over 6,553 GB/s).
// Queries come by TMA as boxes of {64 columns, G heads, 128 / G rows}, key tiles as boxes of 64 rows from the pages or, the drafts', from
// the projections' own rows.  One agent warp starts the copies, one issues O += P V (M 128, N hd, K 64; V an MN-major operand), and two issue
// S = Q K^T (M 128, N 64, K hd; operands as in the prompts' kernel, attention_prefill_tc.cu): such a product keeps the thread that issues
// it for the 540 cycles that it runs, and 600 more go by in waits and commits before the thread's next (one agent for the scores of both row
// tiles took 2,300 cycles a key tile, one for all products 3,400).  Two groups of four worker warps have a score
// buffer, two buffers of weights and an output accumulator each, all in tensor memory (a thread a row): they take one row tile each, or, of a
// request with one row tile, every second key tile; either way products alternate between the groups, and step u is group u % 2's.
// The weights P = 2^(s - m) go to the second product from tensor memory too, which
// leaves shared memory to four key and six value tiles on their way (160 KB: HBM's latency at a block's share of its bandwidth is some 70 KB).
// The weights are bfloat16 (the sums l add them up before that): each is off by 2^-8 of itself at most, which leaves results 0.0021 to 0.0023 of their size
// from 64 bits where 32-bit weights, with the output rounded once, leave 0.0017; two such operands, high and low part, would double the second product.
// A block takes a piece of an item, or an equal share of all requests' key tiles (see tree_attention.cuh); keys are masked by a bit per (row, draft); and values that some
// row of the tile does not see are looked over first, since 0 x NaN is NaN on the tensor cores: rows past the keys' end become
// zeros, and a value that is no number becomes 0 and is added, at the end, to the rows that do see it.
// Every wait on an mbarrier is bounded (codes 61-69 of the error word), as in the prompts' kernel.
#include "tree_attention.cuh"
#include "mbarrier.cuh"
#include "tcgen05.cuh"

int tlc_tensor_map_bf16_nd(const void* p, int rank, const unsigned long long* dims, const unsigned long long* strides, const unsigned* box,
                           CUtensorMap* out);

namespace {

constexpr int BM = 128, BN = TLC_PAGE;
constexpr int KS = 4, VS = 6;            // stages of the K and V rings: scores are made two tiles ahead, so keys leave earlier
constexpr int WORKERS = 256, THREADS = WORKERS + 128, NG = 2;
constexpr float TAU = 8.0f;              // how far (in powers of two) a row's maximum may run ahead of its reference
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(WORKERS) : "memory"); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float ex2_quick(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// two 32-bit operations at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// a bfloat16 pair's halves that are infinite or NaN become 0; whether there was one
__device__ __forceinline__ bool make_finite(uint32_t& w) {
  bool odd = false;
  if ((w & 0x7f80u) == 0x7f80u) { w &= 0xffff0000u; odd = true; }
  if ((w & 0x7f800000u) == 0x7f800000u) { w &= 0x0000ffffu; odd = true; }
  return odd;
}

// D += A B with A (128 rows, 16 columns of 16-bit values, two to a 32-bit column) in tensor memory
__device__ __forceinline__ void umma_a_in_tmem(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <int HD>
struct TreeSmem {
  static constexpr int Q_SLAB = BM * 128, Q = 0, Q_TILE = (HD / 64) * Q_SLAB;
  static constexpr int X = Q;                             // [2][NG][128] floats: the groups' reference maxima and sums, when the queries have been used
  static constexpr int K_SLAB = BN * 128, K_STAGE = (HD / 64) * K_SLAB, K = Q + 2 * Q_TILE;
  static constexpr int V_STAGE = HD * 128, V = K + KS * K_STAGE;
  static constexpr int BARS = V + VS * V_STAGE;           // mbarriers, tmem slot, dead flag
  static constexpr int N_BARS = 1 + 2 * KS + 2 * VS + 12;
  static constexpr int TOTAL = BARS + N_BARS * 8 + 16 + 1024;
};
static_assert(TreeSmem<128>::TOTAL <= 227 * 1024 - 512, "shared memory of a block");

template <int HD, bool CAPPED>
__global__ void __launch_bounds__(THREADS, 1)
tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_kn,
                         const __grid_constant__ CUtensorMap map_vn, TreeArgs a, float cap_in, float cap_out, ErrWords* err) {
  asm volatile("griddepcontrol.launch_dependents;");
  using L_ = TreeSmem<HD>;
  constexpr uint32_t T_O = 2 * BN, T_P = T_O + 2 * HD, TCOLS = 512;     // tensor memory: the groups' scores, outputs, weights (BN / 2 columns a buffer)
  static_assert(T_P + 2 * BN <= TCOLS, "tensor memory");
  extern __shared__ uint8_t tree_tc_raw[];
  uint8_t* sm = (uint8_t*)(((uintptr_t)tree_tc_raw + 1023) & ~(uintptr_t)1023);
  float* xch = reinterpret_cast<float*>(sm + L_::X);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L_::BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + L_::N_BARS);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int s_last_pos, s_odd;                       // the tile's largest position; whether a value was no number
  const uint32_t sm0 = smem_u32(sm);
  const uint32_t bar_q = smem_u32(bars);
  auto k_full = [&](int s) { return smem_u32(bars + 1 + s); };
  auto k_empty = [&](int s) { return smem_u32(bars + 1 + KS + s); };
  auto v_full = [&](int s) { return smem_u32(bars + 1 + 2 * KS + s); };
  auto v_empty = [&](int s) { return smem_u32(bars + 1 + 2 * KS + VS + s); };
  auto s_full = [&](int i) { return smem_u32(bars + 1 + 2 * KS + 2 * VS + i); };
  auto s_free = [&](int i) { return smem_u32(bars + 1 + 2 * KS + 2 * VS + 2 + i); };
  auto p_ready = [&](int w, int buffer) { return smem_u32(bars + 1 + 2 * KS + 2 * VS + 4 + 2 * w + buffer); };
  auto pv_done = [&](int w, int buffer) { return smem_u32(bars + 1 + 2 * KS + 2 * VS + 8 + 2 * w + buffer); };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long wait_limit = mbar_wait_limit(err);
  if (tid == 0) *dead = 0;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TCOLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 8 && lane < 5) {
    const CUtensorMap* const m = lane == 0 ? &map_q : lane == 1 ? &map_k : lane == 2 ? &map_v : lane == 3 ? &map_kn : &map_vn;
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
  }
  tlc_wait(a.v_new, a.v_pages, a.block_table, a.slots, a.start, a.cu, a.positions, a.mask, a.out, a.part_o, a.part_ml, a.splits);
  if (warp == 9) {                                        // every worker warp arrives once on s_free and p_ready, two agents on k_empty, one on the rest
    for (int i = lane; i < L_::N_BARS; i += 32) {
      const int own = i - (1 + 2 * KS + 2 * VS);
      mbar_init(bar_q + 8 * i, own >= 2 && own < 8 ? 4 : i >= 1 + KS && i < 1 + 2 * KS ? 2 : 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  const TreeTake take = tree_plan<THREADS>(a, blockIdx.x, reinterpret_cast<int*>(sm));
  int b = take.b, item = take.item, kt0 = take.tile, todo = take.todo;
  TreeSeq s = take.s;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint32_t bar, uint32_t parity, int code) {
    if (mbar_try(bar, parity) || *dead) return;
    if (!mbar_wait(bar, parity, err, code, wait_limit)) *dead = 1;
  };
  const int G = a.G, NI = tree_div(BM, G);                // drafted rows of a tile
  const float scale_log2 = a.scale * LOG2E;
  // Barriers are made once: what each agent counts goes on from segment to segment.  done: key tiles of earlier segments; used0, used1:
  // how often a group's buffers have been used in them.
  int done = 0, used0 = 0, used1 = 0, segment = 0;
#pragma unroll 1
  for (; todo > 0; segment++) {
  const bool first_segment = segment == 0;
  while (item >= a.KV * s.row_tiles) { item -= a.KV * s.row_tiles; s = tree_seq(a, ++b); }
  const int g = tree_div(item, s.row_tiles), i0 = (item - g * s.row_tiles) * 2 * NI;
  const int n = min(s.key_tiles - kt0, todo);             // key tiles of this segment
  const int rows = min(2 * NI, s.n - i0);
  const bool pair = rows > NI;                            // two row tiles: a group each; else every second key tile for each group
  if (tid == 0) {
    s_last_pos = 0;
    s_odd = 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");         // (the queries' memory has held statistics and results)
  }
  __syncthreads();
  if (a.window > 0) {
    for (int i = tid; i < rows; i += THREADS) atomicMax(&s_last_pos, a.positions[s.t0 + i0 + i]);
    __syncthreads();
  }

  if (warp >= WORKERS / 32) {
    const int role = warp - WORKERS / 32;
    constexpr uint32_t DESC_HI = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);      // see smem_desc
    auto desc_lo = [](uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | (1u << 16); };
    if (role == 0) {
      // the copies: the warp reads 32 entries of the block table at a time, its first lane starts the copies
      if (lane == 0) {
        mbar_expect_tx(bar_q, (pair ? 2 : 1) * (HD / 64) * NI * G * 128);
        for (int w = 0; w < (pair ? 2 : 1); w++)
          for (int c = 0; c < HD / 64; c++) tma_load_3d(sm0 + L_::Q + w * L_::Q_TILE + c * L_::Q_SLAB, &map_q, bar_q, 64 * c, g * G, s.t0 + i0 + w * NI);
      }
      const int* table = a.block_table + (size_t)(s.context_tiles > 0 ? a.slots[b] : 0) * a.max_pages;
      int entry = 0;
      for (int t = 0; t < n; t++) {
        const int kt = kt0 + t;
        if (t % 32 == 0 && kt + lane < s.context_tiles) entry = table[s.first_tile + kt + lane];
        const int page = __shfl_sync(0xffffffffu, entry, t % 32);
        const bool draft = kt >= s.context_tiles;
        // (a page that is none: behind the map's last row, which reads as zeros)
        const int row = draft ? s.t0 + (kt - s.context_tiles) * BN : ((page >= 0 && page < a.n_pages ? page * a.KV + g : a.n_pages * a.KV)) * BN;
        {
          const int st = (done + t) % KS;
          if (done + t >= KS) wait(k_empty(st), (uint32_t)(((done + t) / KS - 1) & 1), 66);       // S of the tile KS before is done
          if (lane == 0) {
            mbar_expect_tx(k_full(st), L_::K_STAGE);
            for (int c = 0; c < HD / 64; c++)
              tma_load_2d(sm0 + L_::K + st * L_::K_STAGE + c * L_::K_SLAB, draft ? &map_kn : &map_k, k_full(st), (draft ? g * HD : 0) + 64 * c, row);
          }
        }
        {
          const int st = (done + t) % VS;
          if (done + t >= VS) wait(v_empty(st), (uint32_t)(((done + t) / VS - 1) & 1), 67);       // P V of the tile VS before is done
          if (lane == 0) {
            mbar_expect_tx(v_full(st), L_::V_STAGE);
            for (int c = 0; c < HD / 64; c++)
              tma_load_2d(sm0 + L_::V + st * L_::V_STAGE + c * L_::K_SLAB, draft ? &map_vn : &map_v, v_full(st), (draft ? g * HD : 0) + 64 * c, row);
          }
        }
        __syncwarp();
      }
      // the last arrivals on the stages' barriers (the products' commits), which nothing else waits for: after
      // them the segment's products are done and no barrier has anything pending
      for (int t = max(0, n - KS); t < n; t++) wait(k_empty((done + t) % KS), (uint32_t)(((done + t) / KS) & 1), 66);
      for (int t = max(0, n - VS); t < n; t++) wait(v_empty((done + t) % VS), (uint32_t)(((done + t) / VS) & 1), 67);
    } else if (lane == 0) {
      constexpr uint32_t idesc_s = instr_desc(BM, BN), idesc_o = instr_desc(BM, HD) | (1u << 16);             // V is MN-major: hd runs along its rows
      const int steps = pair ? 2 * n : n;                 // step u: group u % 2, key tile u / 2 of a pair, else u
      if (role < 3) {
        const int w = role - 1;
        wait(bar_q, (uint32_t)(segment & 1), 61);
        const uint32_t q_lo = desc_lo(sm0 + L_::Q + (pair ? w * L_::Q_TILE : 0));
#pragma unroll 1
        for (int u = w; u < steps; u += 2) {
          const int tile = done + (pair ? u >> 1 : u), st = tile % KS, all = (u >> 1) + (w ? used1 : used0);
          wait(k_full(st), (uint32_t)((tile / KS) & 1), 62);
          if (all > 0) wait(s_free(w), (uint32_t)((all - 1) & 1), 63);               // the workers hold the scores before in registers
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t k_lo = desc_lo(sm0 + L_::K + st * L_::K_STAGE);
#pragma unroll
          for (int c = 0; c < HD / 64; c++)
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              umma_halves(tmem + (uint32_t)(w * BN), q_lo + (uint32_t)((c * L_::Q_SLAB + kk * 32) >> 4), k_lo + (uint32_t)((c * L_::K_SLAB + kk * 32) >> 4),
                          DESC_HI, idesc_s, (c > 0 || kk > 0) ? 1u : 0u);
          umma_commit(s_full(w));
          umma_commit(k_empty(st));                       // (two arrivals: the agents' of a pair, else both by the one whose tile it is)
          if (!pair) mbar_arrive(k_empty(st));
        }
      } else
#pragma unroll 1
      for (int u = 0; u < steps; u++) {
        const int w = u & 1, tile = done + (pair ? u >> 1 : u), st = tile % VS, use = u >> 1, all = use + (w ? used1 : used0);
        if (!pair || w == 0) wait(v_full(st), (uint32_t)((tile / VS) & 1), 65);
        wait(p_ready(w, all & 1), (uint32_t)(all / 2 & 1), 64);                                   // the step's weights are in tensor memory
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t v_lo = (desc_lo(sm0 + L_::V + st * L_::V_STAGE) & 0xFFFFu) | ((uint32_t)(L_::K_SLAB >> 4) << 16);
#pragma unroll
        for (int kk = 0; kk < 4; kk++)
          umma_a_in_tmem(tmem + T_O + (uint32_t)(w * HD), tmem + T_P + (uint32_t)((2 * w + (all & 1)) * (BN / 2) + kk * 8), v_lo + (uint32_t)(kk * (16 * 128 >> 4)), DESC_HI,
                         idesc_o, (use > 0 || kk > 0) ? 1u : 0u);
        umma_commit(pv_done(w, all & 1));
        if (!pair || w == 1) umma_commit(v_empty(st));
      }
    }
    __syncwarp();
  } else {
    // ---- the workers: thread (quarter, lane) of a group owns pair r of the tile: row i0 + r / G, head r % G of the group.  It holds all 64 scores of a
    // key tile and its row of the group's output. ----
    const int wg = warp >> 2, quarter = warp & 3, r = 32 * quarter + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int first_row = i0 + (pair ? wg * NI : 0), i = first_row + r / G;            // the row among the request's drafts
    const int live_rows = min(NI, s.n - first_row) * G;
    const bool live = r < live_rows;
    const int t = s.t0 + (live ? i : 0);
    const int lo_r = a.window > 0 ? a.positions[t] - a.window + 1 : 0;                 // the first position it sees
    const int lo_most = a.window > 0 ? s_last_pos - a.window + 1 : 0;
    const uint32_t s_at = tmem + lanes + (uint32_t)(wg * BN);
    const uint32_t o_at = tmem + lanes + T_O + (uint32_t)(wg * HD), p_at = tmem + lanes + T_P + (uint32_t)(wg * BN);
    float m_ref = -INFINITY, l = 0.f;                     // the maximum the numerators refer to (scaled, log2), the sum
    int mine = 0;                                         // tiles this group has done, and in earlier segments
    const int used = wg ? used1 : used0;
    for (int j = pair ? 0 : wg; j < n; j += pair ? 1 : NG, mine++) {
      const bool draft = kt0 + j >= s.context_tiles;
      const int base = draft ? (kt0 + j - s.context_tiles) * BN : (s.first_tile + kt0 + j) * BN;      // a draft's index, or a position
      const int keys = (draft ? s.n : s.context) - base;
      const bool edge = draft || keys < BN || base < lo_most;       // some row of the tile may not see some key of it
      uint32_t seen_lo = 0xffffffffu, seen_hi = 0xffffffffu;
      if (edge) {
        if (draft) {
          const int word = base >> 5;
          if (a.mask) {
            const int* bits = a.mask + (size_t)t * a.words;
            seen_lo = word < a.words ? (uint32_t)bits[word] : 0u;
            seen_hi = word + 1 < a.words ? (uint32_t)bits[word + 1] : 0u;
          } else {                                        // a chain: the rows up to its own
            const int upto = i - base + 1;
            seen_lo = upto >= 32 ? 0xffffffffu : upto > 0 ? (1u << upto) - 1 : 0u;
            seen_hi = upto >= 64 ? 0xffffffffu : upto > 32 ? (1u << (upto - 32)) - 1 : 0u;
          }
          if (a.window > 0) {
            const int* at = a.positions + s.t0 + base;
            for (int c = 0; c < min(keys, BN); c++)
              if (at[c] < lo_r) { if (c < 32) seen_lo &= ~(1u << c); else seen_hi &= ~(1u << (c - 32)); }
          }
        } else if (lo_r > base) {
          const int from = min(lo_r - base, BN);
          seen_lo = from >= 32 ? 0u : 0xffffffffu << from;
          seen_hi = from >= 64 ? 0u : from > 32 ? 0xffffffffu << (from - 32) : 0xffffffffu;
        }
        if (keys < 32) seen_lo &= keys > 0 ? (1u << keys) - 1 : 0u;
        if (keys < 64) seen_hi &= keys > 32 ? (1u << (keys - 32)) - 1 : 0u;
      }
      if (!live) seen_lo = seen_hi = 0u;
      uint32_t sr[64];
      wait(s_full(wg), (uint32_t)((used + mine) & 1), 68);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      __syncwarp();
      tmem_ld32_nowait(s_at, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
      tmem_ld32_nowait(s_at + 32u, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free(wg));             // the scores are in registers: the buffer may take the next
      const int all = used + mine;
      const bool p_free = all < 2 || mbar_try(pv_done(wg, all & 1), (uint32_t)((all / 2 - 1) & 1));       // the weights of two steps before have been used
      if constexpr (CAPPED) {
        // a capped score: s <- cap tanh(s scale / cap), left divided by the scale (what follows multiplies by it);
        // tanh(x) = 1 - 2 / (e^(2x) + 1), cap_in = 2 log2(e) scale / cap, cap_out = cap / scale.  Off by some 2^-21 of the cap, since scores far below it
        // are a difference of 1s: caps of more than 1,024 go to the other kernel.
#pragma unroll
        for (int c = 0; c < 64; c++) {
          const float e = ex2_quick(__uint_as_float(sr[c]) * cap_in);
          sr[c] = __float_as_uint(fmaf(-cap_out, __fdividef(2.0f, e + 1.0f), cap_out));
        }
      }
      // (hidden before the scale, which is above 0: 0 x -inf would be NaN, and a negative one would make them the largest)
      if (__any_sync(0xffffffffu, (seen_lo & seen_hi) != 0xffffffffu)) {
#pragma unroll
        for (int c = 0; c < 64; c++)
          if (!((c < 32 ? seen_lo >> c : seen_hi >> (c - 32)) & 1u)) sr[c] = 0xff800000u;     // -inf
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 64; c++) mx4[c % 4] = fmaxf(mx4[c % 4], __uint_as_float(sr[c]));
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * scale_log2;
      // the reference maximum moves only when the true one has run ahead of it by more than 2^TAU
      const bool grow = mx > m_ref + TAU || (m_ref == -INFINITY && mx > -INFINITY);
      if (__any_sync(0xffffffffu, grow)) {
        float factor = 1.f;
        if (grow) {
          factor = m_ref == -INFINITY ? 0.f : ex2_quick(m_ref - mx);
          m_ref = mx;
          l *= factor;
        }
        if (mine > 0) {
          wait(pv_done(wg, (all - 1) & 1), (uint32_t)((all - 1) / 2 & 1), 69);        // every product into this output so far is done
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          __syncwarp();
#pragma unroll 1
          for (int c = 0; c < HD / 32; c++) {
            uint32_t o[32];
            tmem_ld32(o_at + (uint32_t)(32 * c), o);
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st32(o_at + (uint32_t)(32 * c), o);
          }
        }
      }
      const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
      float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 32; c++) {
        float2 x = fma2(make_float2(__uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1])), make_float2(scale_log2, scale_log2), make_float2(neg, neg));
        x.x = ex2_quick(x.x);
        x.y = ex2_quick(x.y);
        sums[c % 2] = add2(sums[c % 2], x);
        pk[c] = pack_bf16(x.x, x.y);
      }
      const float2 sum = add2(sums[0], sums[1]);
      l += sum.x + sum.y;
      if (!p_free) wait(pv_done(wg, all & 1), (uint32_t)((all / 2 - 1) & 1), 69);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      __syncwarp();
      tmem_st32(p_at + (uint32_t)((all & 1) * (BN / 2)), pk);
      if (edge && !(pair && wg == 1)) {                     // (of a pair the first group: both products come after it)
        // the tile's values: rows past the keys' end become zeros, and so does what is no number (it is looked at again at the end)
        wait(v_full((done + j) % VS), (uint32_t)(((done + j) / VS) & 1), 65);
        uint4* const v = reinterpret_cast<uint4*>(sm + L_::V + (done + j) % VS * L_::V_STAGE);
        bool odd = false;
#pragma unroll
        for (int e = 0; e < HD / 16; e++) {
          const int at = e * 128 + r;                     // pieces of 16 bytes, eight a key, the 64-column halves one after the other
          if (at / 8 % BN >= keys) v[at] = make_uint4(0u, 0u, 0u, 0u);
          else {
            uint4 w = v[at];
            const bool x = make_finite(w.x), y = make_finite(w.y), z = make_finite(w.z), u = make_finite(w.w);
            if (x || y || z || u) { v[at] = w; odd = true; }
          }
        }
        if (odd) s_odd = 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();                                         // the warp's rows of P are written and fenced
      if (lane == 0) mbar_arrive(p_ready(wg, all & 1));
    }
    // ---- the end: a pair's groups have a result each, else the two meet: O = (O_0 2^(m_0 - m) + O_1 2^(m_1 - m)) / (l_0 2^(m_0 - m) + l_1 2^(m_1 - m)) ----
    if (mine > 0) wait(pv_done(wg, (used + mine - 1) & 1), (uint32_t)((used + mine - 1) / 2 & 1), 69);
    float m0 = m_ref, m1 = -INFINITY, l0 = l, l1 = 0.f;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    workers_sync();
    if (!pair) {                                          // (every product with the queries is done: their memory takes the statistics)
      xch[wg * BM + r] = m_ref;
      xch[(NG + wg) * BM + r] = l;
      workers_sync();
      m0 = xch[r]; m1 = xch[BM + r]; l0 = xch[NG * BM + r]; l1 = xch[(NG + 1) * BM + r];
      workers_sync();                                     // (read, before it takes results)
    }
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const bool whole = n == s.key_tiles;                  // else the sums stay unnormalised: another kernel adds the segments
    const int h = g * G + r % G;
    const bool with_sink = a.sink && whole;
    const float sv = with_sink && a.sink_values ? a.sink_values[live ? h : 0] * LOG2E : 0.f;
    const float m_keys = fmaxf(m0, m1), m_all = with_sink ? fmaxf(m_keys, sv) : m_keys;
    const float w0 = m0 == -INFINITY ? 0.f : ex2_quick(m0 - m_all), w1 = m1 == -INFINITY ? 0.f : ex2_quick(m1 - m_all);
    const float l_keys = l0 * w0 + l1 * w1;
    const bool none = l0 == 0.f && l1 == 0.f;             // it sees nothing
    const float inv = whole ? 1.0f / (l_keys + (with_sink ? ex2_quick(sv - m_all) : 0.f)) : 1.0f;
    const float f0 = w0 * inv, f1 = w1 * inv;
    const bool second = !pair && n > 1;                   // the second group had a tile at all (else its accumulator was never written)
    const int slot = first_segment ? 0 : 1, part_row = (pair ? wg * NI * G : 0) + r;
    if (!whole && live && (pair || wg == 0)) *tree_part_ml(a, blockIdx.x, slot, part_row) = make_float2(m_all, l_keys);
    const bool odd = s_odd != 0;
    // where the pieces of 16 bytes that the lane stores belong: rows 8 q + lane / 4 of the warp's
    __nv_bfloat16* to[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
      const int at = min(32 * quarter + q * 8 + (lane >> 2), BM - 1);
      to[q] = (__nv_bfloat16*)a.out + (size_t)(s.t0 + first_row + at / G) * a.out_ld + (size_t)(g * G + at % G) * HD + 8 * (lane & 3);
    }
    __syncwarp();
#pragma unroll 1
    for (int c = 0; c < (pair ? HD / 32 : HD / 64); c++) {               // 32 output columns at a time: of a pair all, else the group's half
      const int col = (pair ? 0 : wg * (HD / 2)) + 32 * c;
      uint32_t o[32];
      float acc[32];
      tmem_ld32(tmem + lanes + T_O + (uint32_t)((pair ? wg * HD : 0) + col), o);
#pragma unroll
      for (int e = 0; e < 32; e++) acc[e] = __uint_as_float(o[e]) * f0;
      if (second) {
        tmem_ld32(tmem + lanes + T_O + (uint32_t)(HD + col), o);
#pragma unroll
        for (int e = 0; e < 32; e++) acc[e] = fmaf(__uint_as_float(o[e]), f1, acc[e]);
      }
#pragma unroll
      for (int e = 0; e < 32; e++) acc[e] = none ? 0.f : acc[e];
      if (!whole) {
        if (live) {
          float4* const p = tree_part(a, blockIdx.x, slot, col / 4, part_row);
#pragma unroll
          for (int q = 0; q < 8; q++) p[q * (2 * BM)] = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
        }
      } else {
        // through 2 KB of the queries' memory of the warp's own, pieces of 16 bytes in turned order, so that a store covers whole sectors
        uint8_t* const mem = sm + L_::Q + warp * 2048;
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; q++)
          *reinterpret_cast<uint4*>(mem + lane * 64 + ((q ^ (lane >> 1 & 3)) << 4)) =
              make_uint4(pack_bf16(acc[8 * q], acc[8 * q + 1]), pack_bf16(acc[8 * q + 2], acc[8 * q + 3]), pack_bf16(acc[8 * q + 4], acc[8 * q + 5]),
                         pack_bf16(acc[8 * q + 6], acc[8 * q + 7]));
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const int row = q * 8 + (lane >> 2), piece = lane & 3, at = 32 * quarter + row;
          const uint4 x = *reinterpret_cast<const uint4*>(mem + row * 64 + ((piece ^ (row >> 1 & 3)) << 4));
          if (at < live_rows) *reinterpret_cast<uint4*>(to[q] + col) = x;
        }
      }
    }
    if (odd) {
      // values that are no numbers, into the results of the rows that see them (a positive weight times NaN or infinity is that again).
      // In line and without unrolling: a function of its own, with the arguments in memory, costs every launch 1.5 us.
      __syncwarp();                                       // (a row's result was stored by several lanes of its warp)
      __nv_bfloat16* const result = (__nv_bfloat16*)a.out + (size_t)t * a.out_ld + (size_t)h * HD;
      const int col = pair ? 0 : wg * (HD / 2), cols = pair ? HD : HD / 2;
#pragma unroll 1
      for (int j = live ? 0 : n; j < n; j++) {
        const bool draft = kt0 + j >= s.context_tiles;
        const int base = draft ? (kt0 + j - s.context_tiles) * BN : (s.first_tile + kt0 + j) * BN;
        const int keys = min(BN, (draft ? s.n : s.context) - base);
        const int page = draft ? 0 : a.block_table[(size_t)a.slots[b] * a.max_pages + base / BN];
        if (!(draft || keys < BN || base < lo_most) || page < 0 || page >= a.n_pages) continue;
        const __nv_bfloat16* v = draft ? (const __nv_bfloat16*)a.v_new + (size_t)(s.t0 + base) * a.ld_v + (size_t)g * HD
                                       : (const __nv_bfloat16*)a.v_pages + ((size_t)page * a.KV + g) * BN * HD;
#pragma unroll 1
        for (int k = 0; k < keys; k++, v += draft ? a.ld_v : HD) {
          if (!(draft ? tree_sees(a, s.t0, i, base + k) : base + k >= lo_r)) continue;
#pragma unroll 1
          for (int d = col; d < col + cols; d++) {
            const float f = __bfloat162float(v[d]);
            if (isfinite(f)) continue;
            if (whole) result[d] = __float2bfloat16_rn(__bfloat162float(result[d]) + f);
            else reinterpret_cast<float*>(tree_part(a, blockIdx.x, slot, d / 4, part_row))[d % 4] += f;
          }
        }
      }
    }
  }
  // every agent is done with the segment: its copies have landed, its products have completed (the workers read
  // their last results, the loader saw the last commits), tensor memory and shared memory may be written again
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  todo -= n;
  kt0 = 0;
  item++;
  done += n;
  used0 += pair ? n : (n + 1) >> 1;
  used1 += pair ? n : n >> 1;
  }
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TCOLS) : "memory");
}

template <int HD, bool CAPPED> int run(const TreeArgs& a, cudaStream_t stream) {
  auto* const kernel = tree_attention_tc_kernel<HD, CAPPED>;
  static OncePerDevice ready;
  if (!ready.done([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TreeSmem<HD>::TOTAL); }))
    return tlc_fail(-2, "tree_attention(tcgen05): cannot reserve shared memory");
  const int G = a.H / a.KV, NI = BM / G;
  CUtensorMap mq, mk, mv, mkn, mvn;
  const unsigned long long dims[3] = {HD, (unsigned long long)a.H, (unsigned long long)a.T}, strides[2] = {HD * 2, (unsigned long long)a.ld_q * 2};
  const unsigned box[3] = {64, (unsigned)G, (unsigned)NI};
  if (int rc = tlc_tensor_map_bf16_nd(a.q, 3, dims, strides, box, &mq)) return rc;
  const long long page_rows = (long long)a.n_pages * a.KV * BN;
  if (int rc = tlc_tensor_map_bf16(a.k_pages, page_rows, HD, HD, 64, BN, &mk)) return rc;
  if (int rc = tlc_tensor_map_bf16(a.v_pages, page_rows, HD, HD, 64, BN, &mv)) return rc;
  if (int rc = tlc_tensor_map_bf16(a.k_new, a.T, a.KV * HD, a.ld_k, 64, BN, &mkn)) return rc;
  if (int rc = tlc_tensor_map_bf16(a.v_new, a.T, a.KV * HD, a.ld_v, 64, BN, &mvn)) return rc;
  tlc_launch(kernel, dim3(a.blocks), dim3(THREADS), (size_t)TreeSmem<HD>::TOTAL, stream, mq, mk, mv, mkn, mvn, a,
             a.softcap > 0.f ? 2.0f * LOG2E * a.scale / a.softcap : 0.f, a.softcap > 0.f ? a.softcap / a.scale : 0.f, tlc_error_words());
  TLC_CHECK_LAUNCH("tree_attention(tcgen05)");
  return 0;
}

}  // namespace

bool tlc_tree_attention_tc_takes(int dtype, int aligned, int H, int KV, int hd, long long n_pages) {
  return dtype == TLC_BF16 && aligned && (hd == 64 || hd == 128) && H / KV <= BM && n_pages * KV * BN < (1ll << 31) - BN && tlc_error_words_here() != nullptr;
}

int tlc_tree_attention_tc(const TreeArgs& a, cudaStream_t stream) {
  if (a.softcap > 0.f) return a.hd == 64 ? run<64, true>(a, stream) : run<128, true>(a, stream);
  return a.hd == 64 ? run<64, false>(a, stream) : run<128, false>(a, stream);
}
