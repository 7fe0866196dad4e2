// The tensor-core forms of the products in 8-bit integers: what their kernels share.
#pragma once
#include "gemm_int8.cuh"
#include "mbarrier.cuh"
#include "tcgen05.cuh"

constexpr int I8_K = 128;               // K of a stage: 128 values = 128 bytes, one row of the swizzle
constexpr int I8_MMA_K = 32;            // K of one tcgen05.mma with 8-bit operands
constexpr int I8_ROWS = 128;            // weight rows of a block's tile

// Instruction descriptor, kind::i8: D format s32 (bits 4-5 = 2), A and B signed 8-bit (bits 7-9 = 1, 10-12 = 1), both K-major, no
// saturation (bit 3 = 0), N >> 3 in 17-22, M >> 4 in 24-28.
__host__ __device__ constexpr uint32_t int8_desc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void int8_mma(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void int8_mma_pair(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(da), "l"(db), "r"(idesc), "r"(accumulate)
      : "memory");
}

// A tile of 128 weight rows x 128 values.  Plain: rows n .. n + 127 of group e, map {K, N, E}.  Gated: the rows interleaved by the
// copy itself, 8 gate rows, then their 8 up rows, and so on for 64 features from f on: map {K, 8, 2, F / 8, E}, box {128, 8, 2, 8, 1}.
// PAIR: the bytes count on an mbarrier of the cluster's shared window.
template <bool GLU, bool PAIR>
__device__ __forceinline__ void load_weights(uint32_t dst, const CUtensorMap* map, uint32_t bar, int k, int n, int e) {
  if constexpr (GLU) {
    const int f8 = n >> 4;                              // n counts interleaved rows
    if constexpr (PAIR)
      asm volatile("cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %4, %5, %6}], [%2];"
                   ::"r"(dst), "l"(map), "r"(bar), "r"(k), "r"(0), "r"(f8), "r"(e) : "memory");
    else
      asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %4, %5, %6}], [%2];"
                   ::"r"(dst), "l"(map), "r"(bar), "r"(k), "r"(0), "r"(f8), "r"(e) : "memory");
  } else {
    if constexpr (PAIR)
      asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                   ::"r"(dst), "l"(map), "r"(bar), "r"(k), "r"(n), "r"(e) : "memory");
    else
      asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                   ::"r"(dst), "l"(map), "r"(bar), "r"(k), "r"(n), "r"(e) : "memory");
  }
}

// Waits for the loads from tensor memory; what they brought counts as written here, so that nothing uses it earlier.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// Which group's which rows the tile-th tile of `rows_a_tile` sorted rows covers: a warp adds up the groups' tiles, 32 groups at a
// time.  Returns false past the last tile.  (All lanes get the results.)
__device__ __forceinline__ bool int8_group_tile(int tile, int rows_a_tile, const int* offsets, int E, int* group, int* row0, int* rows) {
  const int lane = threadIdx.x & 31;
  for (int e0 = 0; e0 < E; e0 += 32) {
    const int e = min(e0 + lane, E), from = offsets[e], to = offsets[min(e + 1, E)];     // (past E: no rows)
    const int tiles = (to - from + rows_a_tile - 1) / rows_a_tile;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += below;
    }
    const unsigned past = __ballot_sync(0xffffffffu, sum > tile);
    if (past) {
      const int who = __ffs(past) - 1;
      *group = e0 + who;
      const int begin = __shfl_sync(0xffffffffu, from, who) + (tile - __shfl_sync(0xffffffffu, sum - tiles, who)) * rows_a_tile;
      *row0 = begin;
      *rows = min(rows_a_tile, __shfl_sync(0xffffffffu, to, who) - begin);
      return true;
    }
    tile -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return false;
}

// gemm_tcgen05.cu: a tensor map of 8-bit values in boxes with the 128-byte swizzle; dims, strides (bytes, of dims 1 ..), box: rank values.
int tlc_tensor_map_int8(const void* p, int rank, const unsigned long long* dims, const unsigned long long* strides, const unsigned* box,
                        CUtensorMap* out);
// The two operands' maps; box_rows: activation rows of a copy.
int tlc_int8_maps(const Int8Args& p, int box_rows, CUtensorMap* weights, CUtensorMap* rows);
