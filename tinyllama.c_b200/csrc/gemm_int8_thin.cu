// Products in 8-bit integers of up to 8 rows, the weights' way from HBM straight into the registers of mma.sync.
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
// 2,048 -> 8,240 3.9, 17 MB at 4.4 TB/s; of 2,048 -> 65,536 22.6, 134 MB at 5.9 TB/s).  Through rings of shared memory and the tensor
// cores' memory the same take 3.6, 6.0 and 26.1.
#include "gemm_int8.cuh"
#include <algorithm>

namespace {

constexpr int PIECES = 4, SPAN = 64 * PIECES, MOST = 16;       // pieces of 64 values a warp has on their way; warps at most

__device__ __forceinline__ void multiply(int (&c)[4], int a0, int a1, int a2, int a3, int b0, int b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename TO, bool GLU>
__global__ void __launch_bounds__(32 * MOST, 2)
int8_thin_kernel(Int8Args p) {
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr int C = GLU ? 8 : 16;
  __shared__ int sums[MOST][4][32];
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
    for (int r = 0; r < 2; r++) w[r][j] = k0 + 64 * j < K ? sixteen(rows[r], k0 + 64 * j, K, true) : make_int4(0, 0, 0, 0);
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
  int4 a[PIECES];
#pragma unroll
  for (int j = 0; j < PIECES; j++)
    a[j] = k0 + 64 * j < K && g < p.M ? sixteen(x + (size_t)g * p.lda, k0 + 64 * j, K, whole) : make_int4(0, 0, 0, 0);
  float old = 0.f, rs = 0.f;
  if (finishes) {
    out += (size_t)m * p.ldo + n;
    rs = a_scale[m];
    if (!GLU && p.mode == I8_ADD) old = to_f32(*out);
  }
  int acc[4] = {};
#pragma unroll
  for (int j = 0; j < PIECES; j++) {
    multiply(acc, w[0][j].x, w[1][j].x, w[0][j].y, w[1][j].y, a[j].x, a[j].y);
    multiply(acc, w[0][j].z, w[1][j].z, w[0][j].w, w[1][j].w, a[j].z, a[j].w);
  }
#pragma unroll
  for (int r = 0; r < 4; r++) sums[warp][r][lane] = acc[r];
  __syncthreads();
  if (!finishes) return;
  // column c, row m of a product of 16 x 8: lane 4 (c % 8) + m / 2, its number 2 (c / 8) + m % 2
  const int from = 4 * (c & 7) + m / 2, reg = 2 * (c >> 3) + (m & 1);
  int sum = 0, up = 0;
  for (int i = 0; i < warps; i++) {
    sum += sums[i][reg][from];
    if (GLU) up += sums[i][reg + 2][from];
  }
  float v = int8_value(sum, rs, cs, cb);
  if (GLU) v = int8_gated(p, false, 1.0f, v, int8_value(up, rs, us, ub));
  else if (p.mode == I8_ADD) v += old;
  *out = from_f32<TO>(v);
}

template <typename TO, bool GLU>
int launch(const Int8Args& p, cudaStream_t stream) {
  constexpr int C = GLU ? 8 : 16;
  const int warps = std::max(8 * C / 32, (p.K + SPAN - 1) / SPAN);      // (a thread for every result, too)
  tlc_launch(int8_thin_kernel<TO, GLU>, dim3((p.N + C - 1) / C), dim3(32 * warps), 0, stream, p);
  TLC_CHECK_LAUNCH("linear_int8 (up to 8 rows)");
  return 0;
}

}  // namespace

// Rows as integers; the weights' rows on 16-byte boundaries; M <= 8, K <= TLC_INT8_THIN.
int tlc_int8_thin(const Int8Args& p, int out_dtype, cudaStream_t stream) {
  if (out_dtype == TLC_F32) return p.mode == I8_GLU ? launch<float, true>(p, stream) : launch<float, false>(p, stream);
  return p.mode == I8_GLU ? launch<__nv_bfloat16, true>(p, stream) : launch<__nv_bfloat16, false>(p, stream);
}
