// Products in 8-bit integers of many rows on the 5th-generation tensor cores: pairs of blocks (clusters of two) on tiles of 256 weight
// rows x NB = 128 or 256 activation rows, D[n, m] = sum_k w[n, k] a[m, k] by tcgen05.mma.cta_group::2 (kind::i8, M = 256, N = NB, K = 32).
//
// A pair keeps the tensor cores fed where a block alone cannot: each block stages its 128 weight rows and NB / 2 of the activation
// rows (128 values of K a stage, copied by TMA with the 128-byte swizzle) and both halves serve both, so a block moves (128 + NB / 2)
// rows in for 128 x NB products a value of K.  The block of rank 0 issues the products; each block finds its 128 weight rows of the
// result in the lanes of its own tensor memory.  Two accumulators (2 x NB columns) let the results of one tile leave under the
// products of the next; blocks are persistent and pairs walk the tiles.
//
// A lane holds one weight row, so its scale and bias stay in a register and neighbouring lanes write neighbouring columns of a row of
// the result.  Gated products have the gate and up rows of 8 features in neighbouring groups of 8 lanes (load_weights): of two
// activation rows the gate's lanes finish one and the up projection's lanes the other.  Sixteen warps take the results out, sixteen
// rows at a time, what they need beside the sums asked for a tile ahead.
//
// What bounds it: the way of the operands from the L2 into shared memory.  The products of a stage take 512 clocks (the unit's 4.5 POP/s),
// 32 KB come in at some 47 bytes a clock and SM (11 TB/s over the GPU), so a stage takes 700; without copies the largest case would
// take 172 us, without results 205, it takes 250 to 270.  Over many milliseconds the power limit holds the clock at 1.5 GHz
// (2.4 POP/s; bfloat16 products 1.24 GHz, 1.34).  8,192 x 2,560 -> 16,384 260 us, 2.6 POP/s; 2,048 x 2,048 -> 8,240 31 us (four rounds of 74
// pairs for 3.57); gated 1,031 x 2,560 -> 2 x 8,192 42 us, a fifth of it for the last seven rows.
//
// Tiles of 128 activation rows are for groups of up to 110: the weights come in once for a group either way, the rows' stages are
// half as long and eight of them fit.
//
// Waits are bounded (codes 55-59); after one that ran out both blocks of a pair go to their common end.
#include "gemm_int8_tc.cuh"
#include <algorithm>
#include <atomic>

namespace {

constexpr int EPI_WARPS = 16, THREADS = 64 + 32 * EPI_WARPS;      // loader warp, issuer warp, the results' warps (four a quarter of the lanes)

template <int NB> struct Wide {
  static constexpr int STAGES = NB == 256 ? 6 : 8;
  static constexpr int W_BYTES = I8_ROWS * I8_K, X_BYTES = NB / 2 * I8_K;
  static constexpr int TILES = STAGES * (W_BYTES + X_BYTES);
  static constexpr int N_BARS = 2 * STAGES + 4;
  static constexpr int TOTAL = TILES + N_BARS * 8 + 16 + 4 * NB * 3 * 4 + 1024;     // ..., where tensor memory lies, the rows' numbers (and the groups' offsets)
};

template <typename TO, int NB, bool GLU, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 1)
int8_wide_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Int8Args p,
                 int n_tiles, ErrWords* err) {
  asm volatile("griddepcontrol.launch_dependents;");
  using S = Wide<NB>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t wide_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)wide_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* x_tiles = smem + STAGES * S::W_BYTES;
  uint64_t* bars = (uint64_t*)(smem + S::TILES);
  uint32_t* tmem_slot = (uint32_t*)(bars + S::N_BARS);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
  const uint32_t acc_full0 = smem_u32(bars + 2 * STAGES), acc_empty0 = smem_u32(bars + 2 * STAGES + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long wait_limit = mbar_wait_limit(err);
  const uint32_t rank = cluster_rank();
  const int walker = (int)blockIdx.x >> 1, walkers = (int)gridDim.x >> 1;
  const int num_k = (p.K + I8_K - 1) / I8_K;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
    for (int s = 0; s < 2; s++) { mbar_init(acc_full0 + 8 * s, 1); mbar_init(acc_empty0 + 8 * s, 2 * EPI_WARPS); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * NB) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cluster_sync();                                       // the other block's mbarriers are initialised too
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  // Tiles: without groups the activation rows' tiles run fastest (pairs that run together share weights in the L2), with them the
  // weight rows' (a group has few tiles of activation rows).
  int* offsets = reinterpret_cast<int*>(tmem_slot + 4 + 12 * NB);      // (the groups' offsets, a copy)
  const int m_tiles = GROUPED ? 1 : (p.M + NB - 1) / NB;
  int total = m_tiles * n_tiles;
  if (GROUPED) {
    const int* from = p.offsets;
    tlc_wait(from);
    for (int e = threadIdx.x; e <= p.E; e += THREADS) offsets[e] = from[e];
    __syncthreads();
    int tiles = 0;
    for (int e = lane; e < p.E; e += 32) tiles += (offsets[e + 1] - offsets[e] + NB - 1) / NB;
    total = __reduce_add_sync(0xffffffffu, tiles) * n_tiles;
  }
  struct Place { int group, row0, rows, n; };
  auto place = [&](int tile) {
    Place at;
    if constexpr (GROUPED) {
      at.group = at.row0 = at.rows = 0;
      int8_group_tile(tile / n_tiles, NB, offsets, p.E, &at.group, &at.row0, &at.rows);
      at.n = tile % n_tiles;
    } else {
      at.group = 0;
      at.n = tile / m_tiles;
      at.row0 = (tile - at.n * m_tiles) * NB;
      at.rows = min(NB, p.M - at.row0);
    }
    at.n = at.n * 2 * I8_ROWS + (int)rank * I8_ROWS;    // its first weight row (gated: of the interleaved ones) in this block
    return at;
  };

  if (warp == 0) {                                      // ---- copies (one lane issues them) ----
    int it = 0;
    bool ok = true, waited = GROUPED;
    // a pair's copies count on the mbarriers of the block of rank 0, whose issuer waits for them
    const uint32_t full_bar0 = cluster_address(full0, 0);
    int pending = 0;                                    // first stages whose activations are held back until the kernel before is through
    const int first = min(STAGES, num_k);               // (all of them in the first tile)
    for (int tile = walker; tile < total && ok; tile += walkers) {
      const Place at = place(tile);
      const int m0 = at.row0 + (int)rank * (NB / 2);
      if (lane == 0) {
        for (int k = 0; k < num_k; k++, it++) {
          const int s = it % STAGES;
          ok = mbar_wait(empty0 + 8 * s, ((it / STAGES) & 1) ^ 1, err, 55, wait_limit);
          if (!ok) break;
          if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * (S::W_BYTES + S::X_BYTES));
          load_weights<GLU, true>(smem_u32(smem + s * S::W_BYTES), &map_w, full_bar0 + 8 * s, k * I8_K, at.n, at.group);
          if (!waited) {
            pending++;
            if (pending < first) continue;
            asm volatile("griddepcontrol.wait;" ::: "memory");
            waited = true;
            for (int j = 0; j < pending; j++)
              tma_load_2d_pair(smem_u32(x_tiles + j * S::X_BYTES), &map_x, full_bar0 + 8 * j, j * I8_K, m0);
            continue;
          }
          tma_load_2d_pair(smem_u32(x_tiles + s * S::X_BYTES), &map_x, full_bar0 + 8 * s, k * I8_K, m0);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      it = __shfl_sync(0xffffffffu, it, 0);
    }
    if (lane == 0 && rank == 0 && (!ok || *(volatile int*)&err->flag != 0)) {
      // something went wrong: let the copies still in flight land (a pair's count on these mbarriers)
      for (int i = max(0, it - STAGES); i < it; i++)
        mbar_wait(full0 + 8 * (i % STAGES), (i / STAGES) & 1, err, 56, wait_limit);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {                       // ---- products ----
      constexpr uint32_t idesc = int8_desc(2 * I8_ROWS, NB);
      int it = 0, local = 0;
      bool ok = true;
      for (int tile = walker; tile < total && ok; tile += walkers, local++) {
        const int as = local & 1;
        ok = mbar_wait(acc_empty0 + 8 * as, ((local >> 1) & 1) ^ 1, err, 57, wait_limit);     // both blocks have taken this half out
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem + (uint32_t)(as * NB);
        for (int k = 0; k < num_k; k++, it++) {
          const int s = it % STAGES;
          ok = mbar_wait(full0 + 8 * s, (it / STAGES) & 1, err, 58, wait_limit);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t w_addr = smem_u32(smem + s * S::W_BYTES), x_addr = smem_u32(x_tiles + s * S::X_BYTES);
#pragma unroll
          for (int kk = 0; kk < I8_K / I8_MMA_K; kk++)
            int8_mma_pair(d, smem_desc(w_addr + kk * I8_MMA_K), smem_desc(x_addr + kk * I8_MMA_K), idesc, (k > 0 || kk > 0) ? 1u : 0u);
          umma_commit_pair(empty0 + 8 * s);             // the slot is free in both blocks once these products have read it
        }
        if (ok) umma_commit_pair(acc_full0 + 8 * as);
      }
    }
  } else {                                              // ---- results ----
    const int quarter = warp & 3, share = (warp - 2) >> 2;
    const int row = quarter * 32 + lane;                // weight row of the block's tile
    constexpr int CHUNKS = NB / (8 * EPI_WARPS), MINE = 32 * CHUNKS;      // activation rows a warp takes, 32 CHUNKS of them
    constexpr int PIECE = 16;                           // ..., so many at a time
    int local = 0;
    bool ok = true;
    const float* a_scale = p.a_scale;
    const int* order = p.order;
    const float* wts = p.wts;
    TO* out = reinterpret_cast<TO*>(p.out);
    tlc_wait(out, a_scale, order, wts);                 // `out` may still be read or written by the kernel before
    // this warp's activation rows: scales, where their results go, the pairs' weights
    float* scales = reinterpret_cast<float*>(tmem_slot + 4) + (warp - 2) * (MINE * (GROUPED ? 3 : 1));
    int* to = reinterpret_cast<int*>(scales + MINE);
    float* pw = scales + 2 * MINE;
    const bool is_up = GLU && (lane & 8);
    // what a tile needs beside its sums, asked for a tile ahead: this lane's column's scale and bias, this warp's rows' numbers
    Place at, next;
    float cs, cb, n_cs = 0.f, n_cb = 0.f, n_rs[CHUNKS], n_pw[CHUNKS];
    int n_to[CHUNKS];
    auto column = [&](const Place& t) { return GLU ? (t.n >> 1) + ((row >> 4) << 3) + (row & 7) : t.n + row; };
    auto fetch = [&](int tile) {
      next = place(tile);
      const int col = column(next);
      const bool in = col < p.N;
      n_cs = in ? p.w_scale[(size_t)next.group * p.w_rows + (is_up ? p.N : 0) + col] : 0.f;
      n_cb = in && p.colbias ? p.colbias[(is_up ? p.N : 0) + col] : 0.f;
#pragma unroll
      for (int c = 0; c < CHUNKS; c++) {
        const int m = share * MINE + c * 32 + lane;
        const bool there = m < next.rows;
        n_rs[c] = there ? a_scale[next.row0 + m] : 0.f;
        if (GROUPED) {
          const int pair = there ? order[next.row0 + m] : 0;
          n_pw[c] = there ? wts[pair] : 0.f;
          n_to[c] = p.scatter ? pair : next.row0 + m;
        }
      }
    };
    if (walker < total) fetch(walker);
    for (int tile = walker; tile < total && ok; tile += walkers, local++) {
      const int as = local & 1;
      at = next;
      cs = n_cs;
      cb = n_cb;
      const int col = column(at);                       // of the result
      const bool in = col < p.N, inside = (GLU ? (at.n + I8_ROWS) / 2 : at.n + I8_ROWS) <= p.N;
      __syncwarp();                                     // (the last tile's numbers have been read)
#pragma unroll
      for (int c = 0; c < CHUNKS; c++) {
        const int m = c * 32 + lane;
        scales[m] = GROUPED && p.w_out ? n_rs[c] * n_pw[c] : n_rs[c];
        if (GROUPED) {
          to[m] = n_to[c];
          pw[m] = p.w_in ? n_pw[c] : 1.0f;
        }
      }
      __syncwarp();
      if (tile + walkers < total) fetch(tile + walkers);
      ok = mbar_wait(acc_full0 + 8 * as, (local >> 1) & 1, err, 59, wait_limit);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(as * NB + share * MINE);
      uint32_t r[PIECE];
      tmem_ld16_nowait(acc, r);
#pragma unroll 1                                        // (a piece's code stays near the scheduler)
      for (int m1 = 0; m1 < MINE; m1 += PIECE) {
        const int m0 = share * MINE + m1, left = at.rows - m0;                   // activation rows of this piece
        tmem_wait16(r);
        float v[PIECE];
#pragma unroll
        for (int j = 0; j < PIECE; j += 4) {
          const float4 rs = *reinterpret_cast<const float4*>(scales + m1 + j);
          v[j] = int8_value((int)r[j], rs.x, cs, cb);
          v[j + 1] = int8_value((int)r[j + 1], rs.y, cs, cb);
          v[j + 2] = int8_value((int)r[j + 2], rs.z, cs, cb);
          v[j + 3] = int8_value((int)r[j + 3], rs.w, cs, cb);
        }
        if (m1 + PIECE < MINE) {
          tmem_ld16_nowait(acc + (uint32_t)(m1 + PIECE), r);                     // the next piece, under this one's stores
        } else {                                        // all taken out: the accumulator goes back to the issuer's block
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(cluster_address(acc_empty0 + 8 * as, 0));
        }
        if (left <= 0) continue;
        // where this lane writes row j + mine of the piece: the rows' own places, or one row after the other
        TO* base = out + (size_t)(at.row0 + m0) * p.ldo + col;
        auto leave = [&](const bool whole) {            // whole: every row and column of the piece is there
          if constexpr (GLU) {
            const int mine = is_up ? 1 : 0;
            TO* t = base + (size_t)mine * p.ldo;
            auto gated = [&](const auto act_of) {
#pragma unroll
              for (int j = 0; j < PIECE; j += 2) {      // of rows j and j + 1 the gate's lanes finish the first, the up projection's the second
                const float other = __shfl_xor_sync(0xffffffffu, is_up ? v[j] : v[j + 1], 8);
                const float y = act_of(is_up ? other : v[j], is_up ? v[j + 1] : other, j + mine);
                if (whole || (in && j + mine < left)) t[(unsigned)(j * p.ldo)] = from_f32<TO>(y);
              }
            };
            if (p.act == TLC_ACT_SILU && !(GROUPED && p.w_in)) gated([&](float g, float u, int) { return int8_silu(g, u); });
            else gated([&](float g, float u, int j) { return int8_gated(p, GROUPED && p.w_in, GROUPED ? pw[m1 + j] : 1.0f, g, u); });
          } else if constexpr (GROUPED) {
#pragma unroll
            for (int j = 0; j < PIECE; j += 4) {
              const int4 rows = *reinterpret_cast<const int4*>(to + m1 + j);
              const int place_of[4] = {rows.x, rows.y, rows.z, rows.w};
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (whole || (in && j + e < left)) out[(size_t)place_of[e] * p.ldo + col] = from_f32<TO>(v[j + e]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < PIECE; j++)
              if (whole || (in && j < left)) base[(unsigned)(j * p.ldo)] = from_f32<TO>(v[j]);
          }
        };
        if (!GLU && p.mode == I8_ACT) {
#pragma unroll
          for (int j = 0; j < PIECE; j++) v[j] = int8_gated(p, GROUPED && p.w_in, GROUPED ? pw[m1 + j] : 1.0f, v[j], 0.f);
        } else if (!GLU && !GROUPED && p.mode == I8_ADD) {
          float old[PIECE];                             // (all in flight before the first is added)
#pragma unroll
          for (int j = 0; j < PIECE; j++) old[j] = in && j < left ? to_f32(base[(unsigned)(j * p.ldo)]) : 0.f;
#pragma unroll
          for (int j = 0; j < PIECE; j++) v[j] += old[j];
        }
        if (left >= PIECE && inside) leave(true);
        else leave(false);
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cluster_sync();                                       // neither block's memories are in use by the other any more
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * NB) : "memory");
}

template <typename TO, int NB, bool GLU, bool GROUPED>
int launch(const Int8Args& p, long long tiles, int n_tiles, int pairs, cudaStream_t stream) {
  using S = Wide<NB>;
  static std::atomic<bool> set{false};
  if (!set) {
    if (cudaFuncSetAttribute(int8_wide_kernel<TO, NB, GLU, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             S::TOTAL + (GROUPED ? (TLC_INT8_GROUPS + 1) * (int)sizeof(int) : 0)) != cudaSuccess)
      return tlc_fail(-2, "linear_int8: cannot reserve %d bytes of shared memory", S::TOTAL);
    set = true;
  }
  CUtensorMap mw, mx;
  if (int rc = tlc_int8_maps(p, NB / 2, &mw, &mx)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)std::min<long long>(tiles, pairs));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = S::TOTAL + (GROUPED ? ((size_t)p.E + 1) * sizeof(int) : 0);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = g_tlc_pdl ? 2 : 1;
  tlc_launch_config(cfg, int8_wide_kernel<TO, NB, GLU, GROUPED>, mw, mx, p, n_tiles, tlc_error_words());
  TLC_CHECK_LAUNCH("linear_int8 (pairs)");
  return 0;
}

template <typename TO, int NB>
int launch_of(const Int8Args& p, int pairs, cudaStream_t stream) {
  const int n_tiles = ((p.mode == I8_GLU ? 2 : 1) * p.N + 2 * I8_ROWS - 1) / (2 * I8_ROWS);
  const long long tiles = (long long)n_tiles * (p.offsets ? p.M / NB + std::min(p.M, p.E) : (p.M + NB - 1) / NB);    // (grouped: an upper bound)
  if (p.mode == I8_GLU)
    return p.offsets ? launch<TO, NB, true, true>(p, tiles, n_tiles, pairs, stream) : launch<TO, NB, true, false>(p, tiles, n_tiles, pairs, stream);
  return p.offsets ? launch<TO, NB, false, true>(p, tiles, n_tiles, pairs, stream) : launch<TO, NB, false, false>(p, tiles, n_tiles, pairs, stream);
}

}  // namespace

// nb: activation rows of a tile (128 or 256); pairs: how many pairs of blocks run at once.
int tlc_int8_wide(const Int8Args& p, int out_dtype, int nb, int pairs, cudaStream_t stream) {
  if (nb == 128) return out_dtype == TLC_F32 ? launch_of<float, 128>(p, pairs, stream) : launch_of<__nv_bfloat16, 128>(p, pairs, stream);
  return out_dtype == TLC_F32 ? launch_of<float, 256>(p, pairs, stream) : launch_of<__nv_bfloat16, 256>(p, pairs, stream);
}
