// Products in 8-bit integers of one row, or two that are still to be rounded, on the CUDA cores; rows in 16 or 32 bits are rounded in
// the same kernel.
//
// The weights are streamed once, a lane 16 bytes of every 512 of a weight row; dp4a multiplies them with the activation row, which every
// block keeps as integers in shared memory, and a warp reduction adds the lanes' sums, exactly.  Every block rounds the row for itself (it
// is small and comes from the L2): a decode step's product is one launch, without room for the integers.  The first pieces of the
// weights are asked for before the wait on the kernel before; where one item a warp covers the matrix that is all of them, the scales
// and biases too, so that after the wait no load from HBM is left.
//
// What bounds it: for small matrices the way from launch to last store (2,048 -> 2,048 2.1 us, of which the 4 MB are 0.65; rounded by
// one kernel and multiplied by another 2.8), then the weights' stream (8,240 x 2,048 3.7 us, 17 MB at 4.6 TB/s; 4.5 so).  Items that come
// one after another in a warp cost a wait each (two rows at a time, four or five items a warp: 5.2 us there).
#include "gemm_int8.cuh"
#include "int8_round.cuh"
#include <algorithm>

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ __forceinline__ int dot16(int4 a, int4 b, int c) { return __dp4a(a.w, b.w, __dp4a(a.z, b.z, __dp4a(a.y, b.y, __dp4a(a.x, b.x, c)))); }

// The block's copy of the MR rows: integers in xs [MR][ld], zeros from K on, and their scales.
template <int MR>
__device__ __forceinline__ void stage(const int8_t* x, int, const float* a_scale, int K, int8_t* xs, int ld, unsigned*, float (&scale)[MR]) {
  static_assert(MR == 1, "integers come by themselves");
  scale[0] = *a_scale;
  for (int k = 16 * threadIdx.x; k < ld; k += 16 * THREADS) *reinterpret_cast<int4*>(xs + k) = int8_row(x, k, K, (uintptr_t)x % 16 == 0);
  __syncthreads();
}
template <int MR, typename T>
__device__ __forceinline__ void stage(const T* x, int ldx, const float*, int K, int8_t* xs, int ld, unsigned* red, float (&scale)[MR]) {
  const bool whole = (uintptr_t)x % 16 == 0 && (MR == 1 || (size_t)ldx * sizeof(T) % 16 == 0);
  const int pieces = ld / 8, lane = threadIdx.x & 31;
  auto piece = [&](int m, int c, float (&v)[8]) {
    const T* p = x + (size_t)m * ldx + 8 * c;
    if (whole && 8 * c + 8 <= K) {
      Piece<T> raw;
      raw.load(p);
      raw.numbers(v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = 8 * c + i < K ? to_f32(p[i]) : 0.f;
    }
  };
#pragma unroll
  for (int m = 0; m < MR; m++) {
    float magnitude = 0.f;
    for (int c = threadIdx.x; c < pieces; c += THREADS) {
      float v[8];
      piece(m, c, v);
#pragma unroll
      for (int i = 0; i < 8; i++) magnitude = larger(magnitude, v[i]);
    }
    const unsigned most = __reduce_max_sync(0xffffffffu, __float_as_uint(magnitude));
    if (lane == 0) red[m * WARPS + (threadIdx.x >> 5)] = most;
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MR; m++) {
    bool some;
    const unsigned largest = __reduce_max_sync(0xffffffffu, red[m * WARPS + (lane & (WARPS - 1))]);
    const float s = int8_scale(largest, &some), inv = __frcp_rn(s);
    scale[m] = int8_told(largest, some, s);
    int8_t* to = xs + (size_t)m * ld;
    if (int8_usual(largest, s)) {
      for (int c = threadIdx.x; c < pieces; c += THREADS) {
        float v[8];
        piece(m, c, v);
        *reinterpret_cast<uint2*>(to + 8 * c) = eight_nearest(v, s, inv);
      }
    } else {
      for (int c = threadIdx.x; c < pieces; c += THREADS) {
        uint2 n = make_uint2(0u, 0u);
        if (some) {
          float v[8];
          piece(m, c, v);
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] *= INT8_LIFT;
          n = eight_nearest(v, s * INT8_LIFT, __frcp_rn(s * INT8_LIFT));
        }
        *reinterpret_cast<uint2*>(to + 8 * c) = n;
      }
    }
  }
  __syncthreads();
}

// MR: activation rows, one or two.  R: weight rows that a warp takes at a time, an item (gated: R / 2 features, their gate rows and then their up rows); A: pieces of 512
// bytes of every one of them that are on their way together; ONCE: a warp has one item at most and A pieces are its rows.
// GROUPED: blocks of blockIdx.y take the pair of that number, row pair / per_row of x times the weights of expert ids[pair].
template <typename TX, typename TO, int MR, int R, int A, bool ONCE, bool GLU, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 2)
int8_skinny_kernel(const TX* __restrict__ x, Int8Args p, const int* __restrict__ ids, int per_row) {
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr int C = GLU ? R / 2 : R;                      // columns of the result an item makes
  extern __shared__ __align__(16) int8_t skinny_rows[];
  __shared__ unsigned red[MR * WARPS];
  const int lane = threadIdx.x & 31, K = p.K, ld = (K + 15) & ~15;
  const int warps = gridDim.x * WARPS, items = (p.N + C - 1) / C;
  // a warp's items: one from each block in turn, so that few items spread over all SMs
  int item = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
  const float* wts = p.wts;
  TO* out = reinterpret_cast<TO*>(p.out);
  float share = 1.0f;
  if (GROUPED) {
    tlc_wait(x, ids, wts, out);                           // (which weights it takes depends on the routing)
    const int pair = blockIdx.y, expert = ids[pair];
    if (expert >= p.E) return;                            // an output of the router without weights
    p.w += (size_t)expert * p.w_rows * p.ldw;
    p.w_scale += (size_t)expert * p.w_rows;
    x += (size_t)(pair / per_row) * p.lda;
    out += (size_t)pair * p.ldo;
    share = wts[pair];
  }
  int4 w[R][A];
  auto fetch = [&](int item, int k0) {                    // (past the last column: that one again)
#pragma unroll
    for (int j = 0; j < A; j++)
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int k = k0 + 512 * j + 16 * lane, n = min(C * item + (GLU ? r % C : r), p.N - 1) + (GLU && r >= C ? p.N : 0);
        w[r][j] = k < K ? int8_weights(p.w + (size_t)n * p.ldw, k, K) : make_int4(0, 0, 0, 0);
      }
  };
  // lane m C + c finishes column c of row m of the item; its scales and biases come with the weights
  const int m_mine = lane / C, c_mine = lane % C;
  float cs, cb, us, ub;
  auto column = [&](int item) {
    const int n = C * item + c_mine;
    const bool in = n < p.N && m_mine < MR;
    cs = in ? p.w_scale[n] : 0.f;
    cb = in && p.colbias ? p.colbias[n] : 0.f;
    us = GLU && in ? p.w_scale[p.N + n] : 0.f;
    ub = GLU && in && p.colbias ? p.colbias[p.N + n] : 0.f;
  };
  if (item < items) {
    fetch(item, 0);
    column(item);
  }
  const float* a_scale = p.a_scale;
  if (!GROUPED) tlc_wait(x, a_scale, out);
  float scales[MR];
  stage<MR>(x, p.lda, a_scale, K, skinny_rows, ld, red, scales);
  const float scale = MR > 1 && m_mine > 0 ? scales[MR - 1] : scales[0];
  if (m_mine < MR) out += (size_t)m_mine * p.ldo;
  for (; item < items; item += warps) {
    const int n = C * item + c_mine, next = item + warps;
    const bool writes = m_mine < MR && n < p.N;
    const float old = !GLU && p.mode == I8_ADD && writes ? to_f32(out[n]) : 0.f;
    int acc[R][MR] = {};
    auto multiply = [&](const int4 (&w)[R][A], int k0) {
#pragma unroll
      for (int j = 0; j < A; j++) {
        if (k0 + 512 * j >= K) break;
        const int k = min(k0 + 512 * j + 16 * lane, ld - 16);           // (where the row has ended, w is zeros)
#pragma unroll
        for (int m = 0; m < MR; m++) {
          const int4 a = *reinterpret_cast<const int4*>(skinny_rows + (size_t)m * ld + k);
#pragma unroll
          for (int r = 0; r < R; r++) acc[r][m] = dot16(w[r][j], a, acc[r][m]);
        }
      }
    };
    if constexpr (ONCE) {
      multiply(w, 0);
    } else {
      for (int k0 = 0; k0 < K; k0 += 512 * A) {
        int4 now[R][A];
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int j = 0; j < A; j++) now[r][j] = w[r][j];
        // the next pieces, of this item or the next one, under these pieces' products
        if (k0 + 512 * A < K) fetch(item, k0 + 512 * A);
        else if (next < items) fetch(next, 0);
        multiply(now, k0);
      }
    }
    int mine = 0, up = 0;
#pragma unroll
    for (int m = 0; m < MR; m++)
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int sum = __reduce_add_sync(0xffffffffu, acc[r][m]);
        if (lane == m * C + r % C) { if (GLU && r >= C) up = sum; else mine = sum; }
      }
    if (writes) {
      const float rs = GROUPED && p.w_out ? scale * share : scale, pw = GROUPED && p.w_in ? share : 1.0f;
      float v = int8_value(mine, rs, cs, cb);
      if (GLU) v = int8_gated(p, GROUPED && p.w_in, pw, v, int8_value(up, rs, us, ub));
      else if (p.mode == I8_ACT) v = int8_gated(p, GROUPED && p.w_in, pw, v, 0.f);
      else if (p.mode == I8_ADD) v += old;
      out[n] = from_f32<TO>(v);
    }
    if constexpr (ONCE) break;
    if (next < items) column(next);
  }
}

template <typename TX, typename TO, int MR, bool GLU, bool GROUPED>
int launch(const void* x, const Int8Args& p, const int* ids, int per_row, int sms, cudaStream_t stream) {
  const size_t smem = (size_t)MR * ((p.K + 15) & ~15);    // (TLC_INT8_SKINNY at most)
  const int places = GROUPED ? std::max(1, 2 * sms / p.M) : 2 * sms, rows = GLU ? 2 * p.N : p.N;
  const long long warps = (long long)places * WARPS;
#define TLC_SKINNY(R_, A_, ONCE_) \
  tlc_launch(int8_skinny_kernel<TX, TO, MR, R_, A_, ONCE_, GLU, GROUPED>, dim3(std::min((rows + WARPS * R_ - 1) / (WARPS * R_), places), GROUPED ? p.M : 1), \
             dim3(THREADS), smem, stream, (const TX*)x, p, ids, per_row)
  // one item a warp, all of it on its way before the wait on the kernel before, where that takes no more than 16 pieces.  Microseconds so
  // and two rows and four pieces at a time: 2,048 -> 8,240 3.7, 5.2; 2,048 -> 2 x 4,096 3.4, 5.2; 4,096 -> 2,048 3.0, 3.9.
  // (2,048 -> 2,048 by the row, 3.0 for 2.1: half as many warps leave the next kernel room to fetch its weights meanwhile.)
  bool done = false;
  if constexpr (!GROUPED) {
    if (p.K <= 2048 && rows > 2 * warps && rows <= 4 * warps) TLC_SKINNY(4, 4, true), done = true;
    if constexpr (!GLU && MR == 1)
      if (p.K > 2048 && p.K <= 4096 && rows <= warps) TLC_SKINNY(1, 8, true), done = true;
  }
  if (!done) TLC_SKINNY(2, 4, false);
#undef TLC_SKINNY
  TLC_CHECK_LAUNCH("linear_int8 (one row)");
  return 0;
}

template <typename TX, typename TO, int MR, bool GROUPED>
int launch_of(const void* x, const Int8Args& p, const int* ids, int per_row, int sms, cudaStream_t stream) {
  return p.mode == I8_GLU ? launch<TX, TO, MR, true, GROUPED>(x, p, ids, per_row, sms, stream) : launch<TX, TO, MR, false, GROUPED>(x, p, ids, per_row, sms, stream);
}
template <typename TO, bool GROUPED>
int launch_from(const void* x, int x_dtype, const Int8Args& p, const int* ids, int per_row, int sms, cudaStream_t stream) {
  if constexpr (!GROUPED) {
    if (x_dtype == TLC_I8) return launch_of<int8_t, TO, 1, false>(x, p, ids, per_row, sms, stream);
    if (p.M == 2)
      return x_dtype == TLC_F32 ? launch_of<float, TO, 2, false>(x, p, ids, per_row, sms, stream) : launch_of<__nv_bfloat16, TO, 2, false>(x, p, ids, per_row, sms, stream);
  }
  return x_dtype == TLC_F32 ? launch_of<float, TO, 1, GROUPED>(x, p, ids, per_row, sms, stream)
                            : launch_of<__nv_bfloat16, TO, 1, GROUPED>(x, p, ids, per_row, sms, stream);
}

}  // namespace

// x: one row of K values, float, bfloat16 or integers (with their scale in p.a_scale), or two rows of float or bfloat16.
int tlc_int8_skinny(const void* x, int x_dtype, const Int8Args& p, int out_dtype, int sms, cudaStream_t stream) {
  return out_dtype == TLC_F32 ? launch_from<float, false>(x, x_dtype, p, nullptr, 1, sms, stream) : launch_from<__nv_bfloat16, false>(x, x_dtype, p, nullptr, 1, sms, stream);
}

// p.M pairs, each a product of its own: row pair / per_row of x (float or bfloat16), the weights of expert ids[pair], row `pair` of the result.
int tlc_int8_skinny_pairs(const void* x, int x_dtype, const Int8Args& p, const int* ids, int per_row, int out_dtype, int sms, cudaStream_t stream) {
  return out_dtype == TLC_F32 ? launch_from<float, true>(x, x_dtype, p, ids, per_row, sms, stream)
                              : launch_from<__nv_bfloat16, true>(x, x_dtype, p, ids, per_row, sms, stream);
}
