// Products in 8-bit integers of up to 16 rows, the weights' way from HBM straight into the registers of mma.sync.
//
// A block makes 16 columns of the result (gated: 8 features, their gate rows and their up rows) for all activation rows, its warps share K:
// a warp takes 256 of its values at a time, a lane 16 bytes of every 64 of two weight rows.  Integer sums do not depend on their order,
// so K is permuted to suit: the four lanes that hold a row's parts of m16n8k32 hold 16 neighbouring values each of weights and of
// activations, which are two of its steps; nothing is shuffled and only whole 16-byte pieces are loaded.  The warps' sums meet in
// shared memory.
//
// What bounds it: the weights are asked for before the wait on the kernel before, all of them where the blocks find a place at once (64
// registers a thread: 19 MB on the way over the GPU), so that after the wait the rows come from the L2, eight products a warp are made
// and the sums meet; that way is what is left of a decode step's product (8 rows of 2,048 -> 2,048 2.1 us, of which the 4 MB are 0.65; of
// 2,048 -> 8,240 3.9, 17 MB at 4.4 TB/s; of 2,048 -> 65,536 22.6, 134 MB at 5.9 TB/s; 12 rows of 2,048 -> 8,240 5.1).  Through rings
// of shared memory and the tensor cores' memory the same take 3.6, 6.0, 26.1 and 6.1.
#include "gemm_int8.cuh"
#include <algorithm>
#include <atomic>

namespace {

constexpr int PIECES = 4, SPAN = 64 * PIECES, MOST = 16;       // pieces of 64 values a warp has on their way; warps at most

__device__ __forceinline__ void multiply(int (&c)[4], int a0, int a1, int a2, int a3, int b0, int b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT: eights of activation rows.
template <typename TO, int NT, bool GLU>
__global__ void __launch_bounds__(32 * MOST, 2)
int8_thin_kernel(Int8Args p) {
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr int C = GLU ? 8 : 16;
  __shared__ int sums[MOST][NT][4][32];
  extern __shared__ __align__(16) int4 thin_rows[];         // [warp][NT][PIECES][lane]: what the lane itself multiplies
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int K = p.K, n0 = blockIdx.x * C;
  const int8_t* rows[2];                                  // (past the last column: that one again)
  rows[0] = p.w + (size_t)min(n0 + g, p.N - 1) * p.ldw;
  rows[1] = p.w + (size_t)(GLU ? p.N + min(n0 + g, p.N - 1) : min(n0 + 8 + g, p.N - 1)) * p.ldw;
  const int k0 = SPAN * warp + 16 * t;
  int4 w[2][PIECES];
#pragma unroll
  for (int j = 0; j < PIECES; j++)
#pragma unroll
    for (int r = 0; r < 2; r++) w[r][j] = k0 + 64 * j < K ? int8_weights(rows[r], k0 + 64 * j, K) : make_int4(0, 0, 0, 0);
  // thread m C + c finishes column c of row m
  const int c = threadIdx.x % C, m = threadIdx.x / C, n = n0 + c;
  const bool finishes = m < p.M && n < p.N;
  float cs = 0.f, cb = 0.f, us = 0.f, ub = 0.f;
  if (finishes) {
    cs = p.w_scale[n];
    if (p.colbias) cb = p.colbias[n];
    if (GLU) {
      us = p.w_scale[p.N + n];
      if (p.colbias) ub = p.colbias[p.N + n];
    }
  }
  const int8_t* x = p.a;
  const float* a_scale = p.a_scale;
  TO* out = reinterpret_cast<TO*>(p.out);
  tlc_wait(x, a_scale, out);
  const bool whole = (((uintptr_t)x | (uintptr_t)p.lda) & 15) == 0;
  // the rows: of eight a lane's parts come to its registers, of sixteen to its places in shared memory (in registers beside the weights
  // the second eight would wait for the first)
  int4 a[PIECES];
  int4* mine = thin_rows + warp * (NT * PIECES * 32) + lane;
#pragma unroll
  for (int i = 0; i < NT; i++)
#pragma unroll
    for (int j = 0; j < PIECES; j++) {
      const int k = k0 + 64 * j, row = g + 8 * i;
      const int8_t* from = x + (size_t)row * p.lda;
      int4* to = NT == 1 ? &a[j] : mine + 32 * (PIECES * i + j);
      if (NT > 1 && k + 16 <= K && row < p.M && whole)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from + k) : "memory");
      else
        *to = k < K && row < p.M ? int8_row(from, k, K, whole) : make_int4(0, 0, 0, 0);
    }
  float old = 0.f, rs = 0.f;
  if (finishes) {
    out += (size_t)m * p.ldo + n;
    rs = a_scale[m];
    if (!GLU && p.mode == I8_ADD) old = to_f32(*out);
  }
  if (NT > 1) asm volatile("cp.async.wait_all;" ::: "memory");
  int acc[NT][4] = {};
#pragma unroll
  for (int i = 0; i < NT; i++) {
#pragma unroll
    for (int j = 0; j < PIECES; j++) {
      if (NT > 1) a[j] = mine[32 * (PIECES * i + j)];
      multiply(acc[i], w[0][j].x, w[1][j].x, w[0][j].y, w[1][j].y, a[j].x, a[j].y);
      multiply(acc[i], w[0][j].z, w[1][j].z, w[0][j].w, w[1][j].w, a[j].z, a[j].w);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) sums[warp][i][r][lane] = acc[i][r];
  }
  __syncthreads();
  if (!finishes) return;
  // column c, row m of a product of 16 x 8: lane 4 (c % 8) + m / 2, its number 2 (c / 8) + m % 2
  const int from = 4 * (c & 7) + (m & 7) / 2, reg = 2 * (c >> 3) + (m & 1);
  int sum = 0, up = 0;
  for (int i = 0; i < warps; i++) {
    sum += sums[i][m >> 3][reg][from];
    if (GLU) up += sums[i][m >> 3][reg + 2][from];
  }
  float v = int8_value(sum, rs, cs, cb);
  if (GLU) v = int8_gated(p, false, 1.0f, v, int8_value(up, rs, us, ub));
  else if (p.mode == I8_ADD) v += old;
  *out = from_f32<TO>(v);
}

template <typename TO, int NT, bool GLU>
int launch(const Int8Args& p, cudaStream_t stream) {
  constexpr int C = GLU ? 8 : 16;
  const int warps = std::max(8 * NT * C / 32, (p.K + SPAN - 1) / SPAN);      // (a thread for every result, too)
  const int smem = NT == 1 ? 0 : warps * NT * PIECES * 32 * (int)sizeof(int4);      // 64 KB at most
  if (NT > 1) {
    static std::atomic<unsigned long long> raised{0};       // a bit a device: the limit is the device's, and this kernel runs on any
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (!(raised & bit)) {
      const int most = MOST * NT * PIECES * 32 * (int)sizeof(int4);
      if (cudaFuncSetAttribute(int8_thin_kernel<TO, NT, GLU>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
        return tlc_fail(-2, "linear_int8: cannot reserve %d bytes of shared memory", most);
      raised |= bit;
    }
  }
  tlc_launch(int8_thin_kernel<TO, NT, GLU>, dim3((p.N + C - 1) / C), dim3(32 * warps), smem, stream, p);
  TLC_CHECK_LAUNCH("linear_int8 (up to 16 rows)");
  return 0;
}
template <typename TO, int NT>
int launch_of(const Int8Args& p, cudaStream_t stream) {
  return p.mode == I8_GLU ? launch<TO, NT, true>(p, stream) : launch<TO, NT, false>(p, stream);
}

}  // namespace

// Rows as integers; the weights' rows on 16-byte boundaries; M <= 16, K <= TLC_INT8_THIN.
int tlc_int8_thin(const Int8Args& p, int out_dtype, cudaStream_t stream) {
  if (out_dtype == TLC_F32) return p.M <= 8 ? launch_of<float, 1>(p, stream) : launch_of<float, 2>(p, stream);
  return p.M <= 8 ? launch_of<__nv_bfloat16, 1>(p, stream) : launch_of<__nv_bfloat16, 2>(p, stream);
}
