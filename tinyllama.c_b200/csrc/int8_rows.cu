// Rows rounded to 8-bit integers, one scale a row:
//   s_t = max_k |v_tk| / 127,   q_tk = rint(v_tk / s_t)   (so |q| <= 127),
// where v is the row itself or its RMS norm, v_tk = x_tk w_k / sqrt(mean_k x_tk^2 + eps).  These are the operands of the products in
// gemm_int8.cu; a weight matrix is rounded the same way, a scale per output channel.
//
// The norm's factor r = 1 / sqrt(mean + eps) is the same for a whole row and cancels in v / s, so the integers are those of
// p = x w and only the scale is multiplied by r: the row's sum of squares and its largest |p| come from one trip through the
// block, and a row is read once (up to 16,384 values a block keeps it in registers).
//
// The largest magnitude is a maximum of bit patterns without their sign: an infinity or a NaN is larger than every number there,
// and a row that holds one gets the scale NaN and zeros, so that whatever is multiplied by it is NaN.  A row of zeros (or of values
// below 127 x 2^-126) gets the scale 0.  Both divisions are IEEE's, not products with a reciprocal: with a largest magnitude of
// 127 x 2^j, as one bfloat16 row in 128 has, v / s is often a half exactly, and the rounding to even should see it.
#include "common.cuh"

namespace {

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

// Eight values from column k on, zeros past K; vec: rows start on 16-byte boundaries, and so does every eighth column.
template <typename T> __device__ __forceinline__ void row8(const T* x, int k, int K, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= K) return load8(x + k, v);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = k + i < K ? to_f32(x[k + i]) : 0.f;
}
__device__ __forceinline__ void store8(int8_t* q, int k, int K, bool vec, const int (&n)[8]) {
  if (vec && k + 8 <= K) {
    uint2 o = make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 4; i++) { o.x |= (uint32_t)(n[i] & 255) << (8 * i); o.y |= (uint32_t)(n[4 + i] & 255) << (8 * i); }
    *reinterpret_cast<uint2*>(q + k) = o;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) if (k + i < K) q[k + i] = (int8_t)n[i];
}

// A block a row.  NI: pieces of eight values that a thread keeps in registers (0: it reads the row a second time).
// order: row i of the result is row order[i] / top of x (the sorted pairs of a routing).
template <typename T, int NI, bool NORM>
__global__ void __launch_bounds__(512)
int8_rows_kernel(const T* __restrict__ x, int ldx, int K, const float* __restrict__ w, float eps, int8_t* __restrict__ q, int ldq,
                 float* __restrict__ scale, const int* __restrict__ order, int top, int vec_x, int vec_q, int vec_w) {
  tlc_pdl(x, q, scale, order);
  __shared__ unsigned red_max[16];
  __shared__ float red_sum[16];
  const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nw = blockDim.x >> 5;
  const T* xr = x + (size_t)(order ? order[row] / top : row) * ldx;
  int8_t* qr = q + (size_t)row * ldq;
  constexpr int N = NI > 0 ? NI : 1;
  float v[N][8];
  unsigned largest = 0;
  float sum = 0.f;
  auto fetch = [&](int c, float (&u)[8]) {                    // p of piece c, and what it adds to the row's statistics
    row8(xr, 8 * c, K, vec_x, u);
    if (NORM) {
      float g[8];
      row8(w, 8 * c, K, vec_w, g);
#pragma unroll
      for (int i = 0; i < 8; i++) { sum += u[i] * u[i]; u[i] *= g[i]; }
    }
  };
  const int pieces = (K + 7) >> 3;
  if (NI > 0) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int c = tid + j * blockDim.x;
      if (c < pieces) {
        fetch(c, v[j]);
#pragma unroll
        for (int i = 0; i < 8; i++) largest = max(largest, __float_as_uint(v[j][i]) & 0x7fffffffu);
      }
    }
  } else {
    for (int c = tid; c < pieces; c += blockDim.x) {
      fetch(c, v[0]);
#pragma unroll
      for (int i = 0; i < 8; i++) largest = max(largest, __float_as_uint(v[0][i]) & 0x7fffffffu);
    }
  }
  largest = __reduce_max_sync(0xffffffffu, largest);
  if (NORM) sum = warp_sum(sum);
  if (lane == 0) { red_max[warp] = largest; if (NORM) red_sum[warp] = sum; }
  __syncthreads();
  largest = __reduce_max_sync(0xffffffffu, lane < nw ? red_max[lane] : 0u);
  const float s = __fdiv_rn(__uint_as_float(largest), 127.0f);
  const bool finite = largest < 0x7f800000u, some = finite && s >= 1.17549435e-38f;
  if (tid < 32) {
    float r = 1.0f;
    if (NORM) r = rsqrtf(warp_sum(lane < nw ? red_sum[lane] : 0.f) / (float)K + eps);
    if (lane == 0) scale[row] = !finite ? __uint_as_float(0x7fc00000u) : some ? s * r : 0.f;
  }
  auto leave = [&](int c, const float (&u)[8]) {
    int n[8];
#pragma unroll
    for (int i = 0; i < 8; i++) n[i] = some ? __float2int_rn(__fdiv_rn(u[i], s)) : 0;
    store8(qr, 8 * c, K, vec_q, n);
  };
  if (NI > 0) {
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int c = tid + j * blockDim.x;
      if (c < pieces) leave(c, v[j]);
    }
  } else {
    for (int c = tid; c < pieces; c += blockDim.x) { fetch(c, v[0]); leave(c, v[0]); }
  }
}

__global__ void int8_boundary_kernel() {}

template <typename T, bool NORM>
int rows_of(const T* x, int ldx, int T_, int K, const float* w, float eps, int8_t* q, int ldq, float* scale, const int* order, int top,
            cudaStream_t stream) {
  const int vec_x = (uintptr_t)x % 16 == 0 && ((size_t)ldx * sizeof(T)) % 16 == 0, vec_q = (uintptr_t)q % 8 == 0 && ldq % 8 == 0;
  const int vec_w = NORM && (uintptr_t)w % 16 == 0;
  const int pieces = (K + 7) / 8;
  const int threads = pieces <= 128 ? 128 : pieces <= 256 ? 256 : 512;
#define TLC_ROWS(NI_) tlc_launch(int8_rows_kernel<T, NI_, NORM>, dim3(T_), dim3(threads), 0, stream, x, ldx, K, w, eps, q, ldq, scale, \
                                 order, top, vec_x, vec_q, vec_w)
  if (pieces <= threads) TLC_ROWS(1);
  else if (pieces <= 2 * threads) TLC_ROWS(2);
  else if (pieces <= 4 * threads) TLC_ROWS(4);
  else TLC_ROWS(0);
#undef TLC_ROWS
  TLC_CHECK_LAUNCH("rows_int8");
  return 0;
}

}  // namespace

extern "C" int tlc_rows_int8(const void* x, int x_dtype, int ldx, int T_, int K, const float* norm_weight, float eps, void* q, int ldq,
                             float* scale, const int* order, int top, int boundary, cudaStream_t stream) {
  if (T_ == 0) return 0;
  TLC_REQUIRE(T_ > 0 && K > 0 && ldx >= K && ldq >= K && top >= 1, "rows_int8: bad sizes T=%d K=%d ldx=%d ldq=%d top=%d", T_, K, ldx, ldq, top);
  TLC_DISPATCH_DTYPE(x_dtype, T, {
    const int rc = norm_weight ? rows_of<T, true>((const T*)x, ldx, T_, K, norm_weight, eps, (int8_t*)q, ldq, scale, order, top, stream)
                               : rows_of<T, false>((const T*)x, ldx, T_, K, nullptr, 0.f, (int8_t*)q, ldq, scale, order, top, stream);
    if (rc) return rc;
  })
  if (boundary) {       // weights: whatever follows on the stream may fetch them ahead of its wait on the kernel before it
    tlc_launch_step_boundary(int8_boundary_kernel, dim3(1), dim3(1), 0, stream);
    TLC_CHECK_LAUNCH("rows_int8 (boundary)");
  }
  return 0;
}
