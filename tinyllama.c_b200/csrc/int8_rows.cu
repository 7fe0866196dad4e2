// Rows rounded to 8-bit integers, one scale a row:
//   s_t = max_k |v_tk| / 127,   q_tk = rint(v_tk / s_t)   (so |q| <= 127),
// where v is the row itself or its RMS norm, v_tk = x_tk w_k / sqrt(mean_k x_tk^2 + eps).  These are the operands of the products in
// gemm_int8.cu; a weight matrix is rounded the same way, a scale per output channel.
//
// The norm's factor r = 1 / sqrt(mean + eps) is the same for a whole row and cancels in v / s, so the integers are those of
// p = x w and only the scale is multiplied by r: the row's sum of squares and its largest |p| come from one trip through the
// row's warps, and a row is read once (up to 24,576 values stay in registers).
//
// Few rows: as many threads a row as it has pieces of eight values, for the shortest way through (1 x 2,048 1.3 us).  Rows that fill the
// GPU: several pieces a thread and several rows a block, so that enough loads are on their way: 8,192 x 2,560 bfloat16 values 12.5 us
// (63 MB, 5.0 TB/s), 16,384 x 1,024 float values 12.6 us (6.7 TB/s); a block a row took 27.5 and 18.6.
//
// Rows that do not come in whole pieces on 16-byte boundaries are read value by value, and a second time for their integers: 1 x 2,043 1.9 us,
// 24 x 8,187 3.7, 333 x 2,555 floats 5.2 (2.4 in pieces), 8,192 x 2,555 32, 16,384 x 1,019 floats 44.  So is a row of zeros, of an infinity or
// a NaN, or of the smallest scales (int8_usual).
//
// The largest magnitude is a maximum of bit patterns without their sign: an infinity or a NaN is larger than every number there,
// and a row that holds one gets the scale NaN and zeros, so that whatever is multiplied by it is NaN.  A row of zeros (or of values
// below 127 x 2^-126) gets the scale 0.  Both divisions are IEEE's, not products with a reciprocal: with a largest magnitude of
// 127 x 2^j, as one bfloat16 row in 128 has, v / s is often a half exactly, and the rounding to even should see it.
#include "int8_round.cuh"
#include <algorithm>

namespace {

// Eight values from column k on, zeros past K, in any layout.
template <typename T> __device__ __forceinline__ void row8(const T* x, int k, int K, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = k + i < K ? to_f32(x[k + i]) : 0.f;
}
__device__ __forceinline__ void store8(int8_t* q, int k, int K, uint2 n) {
#pragma unroll
  for (int i = 0; i < 8; i++) if (k + i < K) q[k + i] = (int8_t)((i < 4 ? n.x : n.y) >> (8 * (i & 3)));
}

// `warps` warps a row, blockDim / (32 warps) rows a block.  NI > 0: rows of pieces that start on 16-byte boundaries, at most NI a
// thread, which keeps them in registers; 0: any layout and length, and the row is read a second time.  order: row i of the result is
// row order[i] / top of x (a routing's sorted pairs).  PLACED: row i of x becomes the rows place[top i] .. place[top i + top - 1] of the
// result (the same pairs from the other side: a row is read and rounded once).
template <typename T, int NI, bool NORM, bool PLACED>
__global__ void __launch_bounds__(512)
int8_rows_kernel(const T* __restrict__ x, int ldx, int rows, int K, const float* __restrict__ w, float eps, int8_t* __restrict__ q, int ldq,
                 float* __restrict__ scale, const int* __restrict__ order, const int* __restrict__ place, int top, int warps) {
  tlc_pdl(x, q, scale, order, place);
  __shared__ unsigned red_max[16];
  __shared__ float red_sum[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = warp / warps * warps, tid = threadIdx.x - 32 * first, threads = 32 * warps;     // of the row's warps
  const int row = blockIdx.x * ((blockDim.x >> 5) / warps) + warp / warps;
  const bool there = row < rows;
  const T* xr = x + (size_t)(there ? (order ? order[row] / top : row) : 0) * ldx;
  const int copies = PLACED ? top : 1;
  auto to = [&](int copy) { return PLACED ? place[(size_t)row * top + copy] : row; };
  int8_t* qr = q + (size_t)row * ldq;
  const int pieces = (K + 7) >> 3;
  constexpr int N = NI > 0 ? NI : 1;
  Piece<T> raw[N];
  Piece<float> gain[NORM ? N : 1];
  float magnitude = 0.f, sum = 0.f;
  auto weigh = [&](float (&u)[8], const float (&g)[8], bool counts) {        // p of a piece, and what it adds to the row's statistics
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (NORM) {
        if (counts) sum += u[i] * u[i];
        u[i] *= g[i];
      }
      magnitude = larger(magnitude, u[i]);
    }
  };
  if constexpr (NI > 0) {
#pragma unroll
    for (int j = 0; j < N; j++) {                             // (past the last piece: that piece again)
      const int c = min(tid + j * threads, pieces - 1);
      raw[j].load(xr + 8 * c);
      if constexpr (NORM) gain[j].load(w + 8 * c);
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
      float u[8], g[8] = {};
      raw[j].numbers(u);
      if constexpr (NORM) gain[j].numbers(g);
      weigh(u, g, tid + j * threads < pieces);
    }
  } else {
    for (int c = tid; c < pieces; c += threads) {
      float u[8], g[8] = {};
      row8(xr, 8 * c, K, u);
      if (NORM) row8(w, 8 * c, K, g);
      weigh(u, g, true);
    }
  }
  unsigned largest = __reduce_max_sync(0xffffffffu, __float_as_uint(magnitude));
  if (NORM) sum = warp_sum(sum);
  if (warps > 1) {
    if (lane == 0) { red_max[warp] = largest; if (NORM) red_sum[warp] = sum; }
    __syncthreads();
    largest = __reduce_max_sync(0xffffffffu, lane < warps ? red_max[first + lane] : 0u);
    if (NORM) sum = warp_sum(lane < warps ? red_sum[first + lane] : 0.f);
  }
  if (!there) return;
  bool some;
  const float s = int8_scale(largest, &some);
  if (tid == 0) {
    const float r = NORM ? rsqrtf(sum / (float)K + eps) : 1.0f;
    const float told = int8_told(largest, some, s * r);
    for (int i = 0; i < copies; i++) scale[to(i)] = told;
  }
  const bool usual = int8_usual(largest, s);
  if (NI == 0 || !usual) {                                   // from memory again, a value at a time
    const float lift = usual ? 1.0f : INT8_LIFT, lifted = s * lift, inv = __frcp_rn(lifted);
    for (int c = tid; c < pieces; c += threads) {
      float u[8], g[8] = {};
      row8(xr, 8 * c, K, u);
      if (NORM) row8(w, 8 * c, K, g);
#pragma unroll
      for (int i = 0; i < 8; i++) u[i] = (NORM ? u[i] * g[i] : u[i]) * lift;
      const uint2 bytes = some ? eight_nearest(u, lifted, inv) : make_uint2(0u, 0u);
      for (int i = 0; i < copies; i++) store8(PLACED ? q + (size_t)to(i) * ldq : qr, 8 * c, K, bytes);
    }
  } else if constexpr (NI > 0) {
    const float inv = __frcp_rn(s);
    uint2 bytes[PLACED ? N : 1];
#pragma unroll
    for (int j = 0; j < N; j++) {
      const int c = tid + j * threads;
      if (!PLACED && c >= pieces) break;
      float u[8];
      raw[j].numbers(u);
      if constexpr (NORM) {
        float g[8];
        gain[j].numbers(g);
#pragma unroll
        for (int i = 0; i < 8; i++) u[i] *= g[i];
      }
      const uint2 b = eight_nearest(u, s, inv);
      if constexpr (PLACED) bytes[j] = b;
      else *reinterpret_cast<uint2*>(qr + 8 * c) = b;
    }
    if constexpr (PLACED) {
#pragma unroll 1
      for (int i = 0; i < copies; i++) {
        int8_t* o = q + (size_t)to(i) * ldq;
#pragma unroll
        for (int j = 0; j < N; j++) {
          const int c = tid + j * threads;
          if (c < pieces) *reinterpret_cast<uint2*>(o + 8 * c) = bytes[j];
        }
      }
    }
  }
}

__global__ void int8_boundary_kernel() {}

__global__ void __launch_bounds__(256) int8_places_kernel(const int* __restrict__ order, int n, int* __restrict__ place) {
  tlc_pdl(order, place);
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) place[order[i]] = i;
}

template <typename T, bool NORM, bool PLACED = false>
int rows_of(const T* x, int ldx, int T_, int K, const float* w, float eps, int8_t* q, int ldq, float* scale, const int* order, const int* place, int top,
            cudaStream_t stream) {
  const bool whole = (uintptr_t)x % 16 == 0 && ((size_t)ldx * sizeof(T)) % 16 == 0 && (uintptr_t)q % 8 == 0 && ldq % 8 == 0 && K % 8 == 0 &&
                     (!NORM || (uintptr_t)w % 16 == 0);
  const int pieces = (K + 7) / 8;
  // a thread's pieces: one for few rows, or from 592 rows (four blocks an SM) on 64 or 96 bytes of it at most.  One, four, six pieces:
  // 128 x 2,048 (bfloat16) 1.4, 1.7, 1.7 us; 1,024 x 2,560 3.7, 3.5, 3.7; 8,192 x 2,560 18.7, 13.4, 12.3
  const int per_thread = T_ < 592 ? 1 : sizeof(T) == 2 ? 6 : 4;
  const int warps = std::min(16, (pieces + 32 * per_thread - 1) / (32 * per_thread));
  const int block_rows = T_ < 592 ? 1 : std::max(1, 8 / warps), threads = 32 * warps * block_rows;
#define TLC_ROWS(NI_) tlc_launch(int8_rows_kernel<T, NI_, NORM, PLACED>, dim3((T_ + block_rows - 1) / block_rows), dim3(threads), 0, stream, x, \
                                 ldx, T_, K, w, eps, q, ldq, scale, order, place, top, warps)
  if (!whole) TLC_ROWS(0);
  else if (pieces <= 32 * warps) TLC_ROWS(1);
  else if (pieces <= 64 * warps) TLC_ROWS(2);
  else if (pieces <= 128 * warps) TLC_ROWS(4);
  else if (pieces <= 192 * warps) TLC_ROWS(6);
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
    const int rc = norm_weight ? rows_of<T, true>((const T*)x, ldx, T_, K, norm_weight, eps, (int8_t*)q, ldq, scale, order, nullptr, top, stream)
                               : rows_of<T, false>((const T*)x, ldx, T_, K, nullptr, 0.f, (int8_t*)q, ldq, scale, order, nullptr, top, stream);
    if (rc) return rc;
  })
  if (boundary) {       // weights: whatever follows on the stream may fetch them ahead of its wait on the kernel before it
    tlc_launch_step_boundary(int8_boundary_kernel, dim3(1), dim3(1), 0, stream);
    TLC_CHECK_LAUNCH("rows_int8 (boundary)");
  }
  return 0;
}

// The rows of a routing's sorted pairs: row i of q is row order[i] / top of x [T, K].  place: room for T * top integers.  From 1,024 pairs on
// every row is rounded once and written `top` times, by the pairs' places, instead of once for every pair (16,384 pairs of 4,096 rows
// of 2,048 values: 20.5 us, 12 with the places, which take 2 of them).
int tlc_rows_int8_pairs(const void* x, int x_dtype, int ldx, int T_, int K, void* q, int ldq, float* scale, const int* order, int top, int* place,
                        cudaStream_t stream) {
  const int pairs = T_ * top;
  const bool by_place = top > 1 && pairs >= 1024;
  if (by_place) {
    tlc_launch(int8_places_kernel, dim3((pairs + 255) / 256), dim3(256), 0, stream, order, pairs, place);
    TLC_CHECK_LAUNCH("rows_int8 (places)");
  }
  TLC_DISPATCH_DTYPE(x_dtype, T, {
    if (by_place) return rows_of<T, false, true>((const T*)x, ldx, T_, K, nullptr, 0.f, (int8_t*)q, ldq, scale, nullptr, place, top, stream);
    return rows_of<T, false>((const T*)x, ldx, pairs, K, nullptr, 0.f, (int8_t*)q, ldq, scale, order, nullptr, top, stream);
  })
}
