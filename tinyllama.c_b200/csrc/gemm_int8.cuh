// What the kernels of the products in 8-bit integers share: the operands, and the groups (experts) of a grouped product.
#pragma once
#include "common.cuh"

// out[m, n] (+)= a_scale[m] * w_scale[n] * sum_k a[m, k] w[n, k] + colbias[n], or gated: act(y[m, n]) * y[m, F + n] for a w of 2 F
// rows (the gate's, then the up projection's).  Grouped (offsets not NULL): rows offsets[e] .. offsets[e + 1] - 1 of a are multiplied
// by the rows e * w_rows .. of w; order [rows] is the pair (row of the step * top + choice) of every row, wts [pairs] the pairs'
// weights.
struct Int8Args {
  const int8_t* a; const float* a_scale;
  const int8_t* w; const float* w_scale;
  void* out; const float* colbias;
  int lda, ldw, ldo, M, N, K;           // N: columns of the result (gated: F, w has 2 F rows)
  int w_rows;                           // rows of w, or of one group's
  int mode;                             // I8_*
  int act, w_in;                        // gated / I8_ACT: the activation; w_in: the pair's weight multiplies the products before it
  float limit, alpha;
  const int* offsets; const int* order; const float* wts;
  int E;
  int scatter, w_out;                   // result rows go where order says, times the pair's weight
};
constexpr int TLC_INT8_SKINNY = 8192;     // values of one row, at most, in the kernel of one or two rows
constexpr int TLC_INT8_TWO = 2048;        // ... of each of two (ops.linear_int8 brings room for longer ones at once)
constexpr int TLC_INT8_THIN = 4096;       // values of a row in the kernel of up to 16 rows, at most: 256 for each of 16 warps
constexpr int TLC_INT8_GROUPS = 4096;     // at most (as a routing)
enum { I8_PLAIN = 0, I8_ADD = 1, I8_ACT = 2, I8_GLU = 3 };

// 16 values of a row from k on, zeros past K.  Weights (rows on 16-byte boundaries) come through the read-only way; activations, which an
// earlier kernel may still have been writing when this one started, by ordinary loads (whole: the row is on a 16-byte boundary).  Past the
// L1 they would cost the blocks of an SM, which read the same rows, half a microsecond of four.
__device__ __forceinline__ int4 int8_bytes(const int8_t* p, int k, int K) {
  int v[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; i++) if (k + i < K) v[i >> 2] |= (int)(uint8_t)p[k + i] << (8 * (i & 3));
  return make_int4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ int4 int8_weights(const int8_t* p, int k, int K) {
  return k + 16 <= K ? __ldg(reinterpret_cast<const int4*>(p + k)) : int8_bytes(p, k, K);
}
__device__ __forceinline__ int4 int8_row(const int8_t* p, int k, int K, bool whole) {
  return whole && k + 16 <= K ? *reinterpret_cast<const int4*>(p + k) : int8_bytes(p, k, K);
}

// One result from its integer sum.  Both scales in 32 bits, one after the other: their product alone may leave the range.  The
// operations are spelled out, so that every kernel rounds alike and a result does not depend on which one made it.
__device__ __forceinline__ float int8_value(int sum, float row_scale, float col_scale, float bias) {
  return __fmaf_rn(__fmul_rn(__int2float_rn(sum), row_scale), col_scale, bias);
}

// A gated activation as all kernels here make it; w: the pair's weight on gate and up, where it goes there.  SiLU is g / (1 + 2^(-g log2 e)) by
// the special-function unit's power and reciprocal.  The product g log2 e is rounded before the power, so the error of the result grows
// with |g| where g is negative: (4 + 1.2 |g|) 2^-24 of it at most, measured (9 at g = -10, 63 at -80), 4 where g is positive.  From
// g = -87.4 down (results of 1e-36) it is 0.  A result in 16 bits is rounded to 2^-8 after that; the 32-bit paths elsewhere (silu_f) keep
// the slower form.
__device__ __forceinline__ float int8_silu(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return __fmul_rn(__fmul_rn(g, r), u);
}
__device__ __forceinline__ float int8_gated(const Int8Args& p, bool weighted, float w, float g, float u) {
  if (weighted) {
    g = __fmul_rn(g, w);
    u = __fmul_rn(u, w);
  }
  return p.act == TLC_ACT_SILU ? int8_silu(g, u) : moe_pair_act<true>(p.act, 1, p.limit, p.alpha, 1.0f, g, u);
}
