// Products in 8-bit integers of up to 128 rows (or groups of that size) on the 5th-generation tensor cores, the weights on the
// 128-row side of tcgen05.mma (kind::i8, K = 32 an instruction, exact 32-bit sums): D[n, m] = sum_k w[n, k] a[m, k], a tile of 128
// weight rows x NB = 16, 32, 64 or 128 activation rows in 128 lanes x NB columns of tensor memory.
//
// The time is the time to stream the weights once, so the K-steps of a tile are shared among the up to 8 blocks of a cluster where
// there are fewer tiles than places on the SMs (2048 rows of weights are 16 tiles).  Every block copies its [128, 128] tiles of
// weights and [NB, 128] tiles of activations by TMA into a ring of stages, leaves its integer sums [NB][128] in shared memory, and
// block r of the cluster adds up its share of the activation rows over all blocks through distributed shared memory; integers add up
// exactly, in whatever order.  Then scales, bias, activation or sum: a warp a row, a lane four weight rows.
//
// What bounds it: the weights' stream where there are enough of them (64 rows of 2,560 -> 16,384 12.0 us, 42 MB at 3.5 TB/s; 37 rows of
// experts, 134 MB, 26 us, 5.1 TB/s), else the way in and out: set-up, first bytes, the cluster's meeting, stores (24 rows of 8,192 -> 2,560
// 7.2 us, 21 MB; 32 of 2,048 -> 8,240 6.5, 17 MB).  Two blocks an SM keep 190 to 220 KB on their way.
//
// Gated products find a feature's gate and up row 8 lanes of tensor memory apart, because the copy interleaves them so
// (load_weights).  Waits are bounded (codes 51-54); a block whose wait ran out still meets its cluster.
#include "gemm_int8_tc.cuh"
#include <algorithm>
#include <atomic>

namespace {

constexpr int THREADS = 192;            // loader warp, issuer warp, four warps for the results

template <int NB> struct Few {
  static constexpr int STAGES = NB == 16 ? 6 : NB == 32 ? 5 : NB == 64 ? 4 : 3;      // two blocks an SM
  static constexpr int W_BYTES = I8_ROWS * I8_K, X_BYTES = NB * I8_K;
  static constexpr int TILES = STAGES * (W_BYTES + X_BYTES);
  static constexpr int N_BARS = 2 * STAGES + 1;
  static constexpr int TOTAL = TILES + N_BARS * 8 + 32 + 3 * NB * 4 + 1024;      // ..., where tensor memory lies, the rows' numbers
  static_assert(NB * I8_ROWS * 4 <= TILES, "the sums take the stages' place");
};

__device__ __forceinline__ const int* in_rank(const int* p, int rank) {
  unsigned long long q;
  asm("mapa.u64 %0, %1, %2;" : "=l"(q) : "l"((unsigned long long)(uintptr_t)p), "r"(rank));
  return reinterpret_cast<const int*>((uintptr_t)q);
}
__device__ __forceinline__ void four_of(const float* p, int n, int N, float none, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = p && n + i < N ? p[n + i] : none;
}

template <typename TO, int NB, bool GLU, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 2)
int8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Int8Args p,
                int split, int n_tiles, ErrWords* err) {
  asm volatile("griddepcontrol.launch_dependents;");
  using S = Few<NB>;
  constexpr int STAGES = S::STAGES, CW = NB < 32 ? 16 : 32, TCOLS = NB < 32 ? 32 : NB;
  extern __shared__ uint8_t few_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)few_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* x_tiles = smem + STAGES * S::W_BYTES;
  int* part = reinterpret_cast<int*>(smem);
  uint64_t* bars = (uint64_t*)(smem + S::TILES);
  uint32_t* tmem_slot = (uint32_t*)(bars + S::N_BARS);
  // the tile's activation rows: scale, where the result goes, the pair's weight
  float* row_scale = reinterpret_cast<float*>(tmem_slot + 4);
  int* row_to = reinterpret_cast<int*>(row_scale + NB);
  float* row_weight = row_scale + 2 * NB;
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES), acc_full = smem_u32(bars + 2 * STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  int group = 0, row0 = 0, rows = p.M;
  const int tile = (int)blockIdx.x / split;
  if (GROUPED) {
    const int* offsets = p.offsets;
    tlc_wait(offsets);                                      // (which weights it takes depends on the routing)
    if (!int8_group_tile(tile / n_tiles, NB, offsets, p.E, &group, &row0, &rows)) return;    // (the whole cluster)
  } else {
    row0 = tile / n_tiles * NB;
    rows = min(NB, p.M - row0);
  }
  const long long wait_limit = mbar_wait_limit(err);
  const int rank = split > 1 ? (int)cluster_rank() : 0;     // clusters are runs of `split` consecutive blocks
  const int n0 = (tile % n_tiles) * I8_ROWS;                // of the weight rows (gated: interleaved, two a feature)
  const int num_k = (p.K + I8_K - 1) / I8_K, k_per = (num_k + split - 1) / split;
  const int k_begin = min(num_k, rank * k_per), n_k = min(num_k, k_begin + k_per) - k_begin;      // (the last ranks may have none)

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; s++) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
    mbar_init(acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TCOLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {                                        // ---- copies ----
      // the first stages' weights do not depend on the kernel before and are asked for ahead of the wait on it
      bool ok = true, waited = false;
      int issued = 0;
      for (int i = 0; i < n_k && ok; i++) {
        const int s = i % STAGES, k = (k_begin + i) * I8_K;
        if (i >= STAGES) ok = mbar_wait(empty0 + 8 * s, (uint32_t)(((i - STAGES) / STAGES) & 1), err, 51, wait_limit);
        if (!ok) break;
        mbar_expect_tx(full0 + 8 * s, S::W_BYTES + S::X_BYTES);
        load_weights<GLU, false>(smem_u32(smem + s * S::W_BYTES), &map_w, full0 + 8 * s, k, n0, group);
        issued = i + 1;
        if (!waited) {
          if (i < min(n_k, STAGES) - 1) continue;
          asm volatile("griddepcontrol.wait;" ::: "memory");
          waited = true;
          for (int j = 0; j < i; j++)
            tma_load_2d(smem_u32(x_tiles + j * S::X_BYTES), &map_x, full0 + 8 * j, (k_begin + j) * I8_K, row0);
        }
        tma_load_2d(smem_u32(x_tiles + s * S::X_BYTES), &map_x, full0 + 8 * s, k, row0);
      }
      if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");
      if (!ok || *(volatile int*)&err->flag != 0) {
        // something went wrong: let the copies still in flight land before the block goes on to its end
        for (int i = max(0, issued - STAGES); i < issued; i++)
          mbar_wait(full0 + 8 * (i % STAGES), (uint32_t)((i / STAGES) & 1), err, 54, wait_limit);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {                                        // ---- products ----
      constexpr uint32_t idesc = int8_desc(I8_ROWS, NB);
      bool ok = true;
      for (int i = 0; i < n_k; i++) {
        const int s = i % STAGES;
        ok = mbar_wait(full0 + 8 * s, (uint32_t)((i / STAGES) & 1), err, 52, wait_limit);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t w_addr = smem_u32(smem + s * S::W_BYTES), x_addr = smem_u32(x_tiles + s * S::X_BYTES);
#pragma unroll
        for (int kk = 0; kk < I8_K / I8_MMA_K; kk++)
          int8_mma(tmem, smem_desc(w_addr + kk * I8_MMA_K), smem_desc(x_addr + kk * I8_MMA_K), idesc, (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(empty0 + 8 * s);
      }
      if (ok && n_k > 0) umma_commit(acc_full);
      else if (n_k == 0) mbar_arrive(acc_full);             // no K-steps: the sums are zeros
    }
  } else {                                                  // ---- results, warps 2..5 ----
    const int quarter = warp & 3;                           // a warp may touch lanes 32 * (warp % 4) .. + 31 only
    const int row = quarter * 32 + lane;                    // weight row of the tile
    // Block r finishes its share of the activation rows: a warp every fourth of them, a lane four weight rows.
    const int rows_per = (NB + split - 1) / split, m_begin = rank * rows_per, m_end = min(min(rows, NB), m_begin + rows_per);
    const int n = n0 + 4 * lane;                            // of this lane's four weight rows
    const int c0 = GLU ? (n0 >> 1) + ((lane >> 2) << 3) + (lane & 1) * 4 : n;        // first result column of its four
    const bool writes = GLU ? !(lane & 2) && c0 < p.N : n < p.N;
    const size_t s0 = (size_t)group * p.w_rows + (GLU && (lane & 2) ? p.N : 0);      // its rows' first scale, less the column
    float cs[4], cb[4];
    four_of(p.w_scale + s0, c0, p.N, 0.f, cs);
    four_of(p.colbias ? p.colbias + (GLU && (lane & 2) ? p.N : 0) : nullptr, c0, p.N, 0.f, cb);
    const float* a_scale = p.a_scale;
    TO* out = reinterpret_cast<TO*>(p.out);
    const int* order = p.order;
    const float* wts = p.wts;
    tlc_wait(a_scale, out, order, wts);                     // `out` may still be read or written by the kernel before
    if (row < min(rows, NB)) {
      float rs = a_scale[row0 + row], w = 1.0f;
      int to = row0 + row;
      if (GROUPED) {
        const int pair = order[row0 + row];
        w = wts[pair];
        if (p.w_out) rs *= w;
        if (p.scatter) to = pair;
      }
      row_scale[row] = rs;
      row_to[row] = to;
      row_weight[row] = w;
    }
    mbar_wait(acc_full, 0, err, 53, wait_limit);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
    for (int c = 0; c < NB / CW; c++) {
      uint32_t r[CW];
      __syncwarp();
      tmem_ldn(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(c * CW), r);
#pragma unroll
      for (int j = 0; j < CW; j++) part[(c * CW + j) * I8_ROWS + row] = n_k > 0 ? (int)r[j] : 0;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("bar.sync 1, 128;" ::: "memory");          // the rows' numbers, and this block's sums
    if (split > 1) {                                        // ... and those of the others of the cluster
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    const int* src[8];
#pragma unroll
    for (int q = 0; q < 8; q++) src[q] = (split > 1 ? in_rank(part, min(q, split - 1)) : part) + 4 * lane;
    const bool vec = c0 + 4 <= p.N && ((size_t)p.ldo * sizeof(TO)) % (4 * sizeof(TO)) == 0 && (uintptr_t)out % (4 * sizeof(TO)) == 0;
#pragma unroll 1
    for (int m = m_begin + quarter; m < m_end; m += 4) {
      const float rs = row_scale[m], pw = GROUPED && p.w_in ? row_weight[m] : 1.0f;
      TO* o = out + (size_t)row_to[m] * p.ldo + c0;
      int4 x[8];
#pragma unroll
      for (int q = 0; q < 8; q++) x[q] = q < split ? *reinterpret_cast<const int4*>(src[q] + m * I8_ROWS) : make_int4(0, 0, 0, 0);
      int sum[4] = {0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < 8; q++) { sum[0] += x[q].x; sum[1] += x[q].y; sum[2] += x[q].z; sum[3] += x[q].w; }
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; i++) v[i] = int8_value(sum[i], rs, cs[i], cb[i]);
      if (GLU) {                                            // the up rows sit two lanes above their gate rows
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float u = __shfl_down_sync(0xffffffffu, v[i], 2);
          v[i] = int8_gated(p, GROUPED && p.w_in, pw, v[i], u);
        }
      } else if (p.mode == I8_ACT) {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = int8_gated(p, GROUPED && p.w_in, pw, v[i], 0.f);
      } else if (p.mode == I8_ADD) {
#pragma unroll
        for (int i = 0; i < 4; i++) if (writes && c0 + i < p.N) v[i] += to_f32(o[i]);
      }
      if (!writes) continue;
      if (vec) {
        if constexpr (sizeof(TO) == 4) {
          *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
          *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const unsigned*>(&lo), *reinterpret_cast<const unsigned*>(&hi));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) if (c0 + i < p.N) o[i] = from_f32<TO>(v[i]);
      }
    }
  }
  __syncwarp();                                             // the loader's and the issuer's warps are whole again
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  if (split > 1) {
    if (warp < 2) {                                         // (the other warps met above)
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
    // no block leaves while another may still read its sums
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TCOLS) : "memory");
}

template <typename TO, int NB, bool GLU, bool GROUPED>
int launch(const Int8Args& p, int token_tiles, int split, cudaStream_t stream) {
  using S = Few<NB>;
  static std::atomic<bool> set{false};
  if (!set) {
    if (cudaFuncSetAttribute(int8_few_kernel<TO, NB, GLU, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL) != cudaSuccess)
      return tlc_fail(-2, "linear_int8: cannot reserve %d bytes of shared memory", S::TOTAL);
    set = true;
  }
  CUtensorMap mw, mx;
  if (int rc = tlc_int8_maps(p, NB, &mw, &mx)) return rc;
  const int n_tiles = ((GLU ? 2 : 1) * p.N + I8_ROWS - 1) / I8_ROWS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * token_tiles * split));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = S::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (split > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = split;
    attr[na].val.clusterDim.y = 1;
    attr[na++].val.clusterDim.z = 1;
  }
  if (g_tlc_pdl) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  tlc_launch_config(cfg, int8_few_kernel<TO, NB, GLU, GROUPED>, mw, mx, p, split, n_tiles, tlc_error_words());
  TLC_CHECK_LAUNCH("linear_int8 (few rows)");
  return 0;
}

template <typename TO, int NB>
int launch_of(const Int8Args& p, int token_tiles, int split, cudaStream_t stream) {
  if (p.mode == I8_GLU)
    return p.offsets ? launch<TO, NB, true, true>(p, token_tiles, split, stream) : launch<TO, NB, true, false>(p, token_tiles, split, stream);
  return p.offsets ? launch<TO, NB, false, true>(p, token_tiles, split, stream) : launch<TO, NB, false, false>(p, token_tiles, split, stream);
}

}  // namespace

// The maps of a product's operands: rows of 128 values of K with the 128-byte swizzle, zeros past K and past the last row.
int tlc_int8_maps(const Int8Args& p, int box_rows, CUtensorMap* weights, CUtensorMap* rows) {
  const unsigned long long ld = p.ldw, E = p.offsets ? p.E : 1;
  if (p.mode == I8_GLU) {
    const unsigned long long dims[5] = {(unsigned long long)p.K, 8, 2, (unsigned long long)p.N / 8, E};
    const unsigned long long strides[4] = {ld, (unsigned long long)p.N * ld, 8 * ld, 2 * (unsigned long long)p.N * ld};
    const unsigned box[5] = {I8_K, 8, 2, I8_ROWS / 16, 1};
    if (int rc = tlc_tensor_map_int8(p.w, 5, dims, strides, box, weights)) return rc;
  } else {
    const unsigned long long dims[3] = {(unsigned long long)p.K, (unsigned long long)p.N, E};
    const unsigned long long strides[2] = {ld, (unsigned long long)p.N * ld};
    const unsigned box[3] = {I8_K, I8_ROWS, 1};
    if (int rc = tlc_tensor_map_int8(p.w, 3, dims, strides, box, weights)) return rc;
  }
  const unsigned long long dims[2] = {(unsigned long long)p.K, (unsigned long long)p.M}, strides[1] = {(unsigned long long)p.lda};
  const unsigned box[2] = {I8_K, (unsigned)box_rows};
  return tlc_tensor_map_int8(p.a, 2, dims, strides, box, rows);
}

// Blocks a tile: as many (1, 2, 4, 8) as bring the grid to two blocks an SM, each with two K-steps or more.
int tlc_int8_few_split(long long tiles, int num_k, int sms) {
  int split = 1;
  while (split < 8 && tiles * split * 2 <= 2 * sms && num_k / (split * 2) >= 2) split *= 2;
  return split;
}

// nb: activation rows of a tile (16, 32, 64 or 128).
int tlc_int8_few(const Int8Args& p, int out_dtype, int nb, int sms, cudaStream_t stream) {
  const int token_tiles = p.offsets ? p.M / nb + std::min(p.M, p.E) : (p.M + nb - 1) / nb;     // (grouped: an upper bound)
  const long long tiles = (long long)(((p.mode == I8_GLU ? 2 : 1) * p.N + I8_ROWS - 1) / I8_ROWS) * token_tiles;
  const int split = tlc_int8_few_split(tiles, (p.K + I8_K - 1) / I8_K, sms);
#define TLC_I8_NB(TO_) (nb == 16 ? launch_of<TO_, 16>(p, token_tiles, split, stream) : nb == 32 ? launch_of<TO_, 32>(p, token_tiles, split, stream) \
                        : nb == 64 ? launch_of<TO_, 64>(p, token_tiles, split, stream) : launch_of<TO_, 128>(p, token_tiles, split, stream))
  return out_dtype == TLC_F32 ? TLC_I8_NB(float) : TLC_I8_NB(__nv_bfloat16);
#undef TLC_I8_NB
}
