// Rounding rows to 8-bit integers: the pieces that the kernels share (int8_rows.cu, gemm_int8_skinny.cu).
#pragma once
#include "common.cuh"

// Eight values as they lie in memory (a 16- or 32-byte piece), and as numbers: apart, so that all of a thread's loads are on their way
// before the first is looked at.
template <typename T> struct Piece;
template <> struct Piece<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ __forceinline__ void numbers(float (&v)[8]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
};
template <> struct Piece<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void numbers(float (&v)[8]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
};
// The larger magnitude; a NaN stays.
__device__ __forceinline__ float larger(float m, float v) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v)));
  return m;
}
// Eight integers nearest to the quotients v / s (halves to even) as bytes, inv = 1 / s correctly rounded.  A first quotient v inv is
// mended by its remainder, which a fused multiply-add gives exactly, times inv (Markstein, IBM Journal of Research and Development 34,
// 1990): the IEEE quotient, without the general division's cases, which do not arise here (s is no denormal and |v / s| <= 127).
// The remainder of a quotient of 1/2 or more comes in steps of 2^-47 of s's power of two or more, so it is exact down to s = 2^-102; rows of
// smaller scales come multiplied by 2^64 (int8_usual), which changes no quotient.  Adding 1.5 * 2^23 rounds it to an integer and
// leaves that in the sum's low bits; conversions would go through the special-function unit, at a quarter of the rate.
__device__ __forceinline__ uint2 eight_nearest(const float (&v)[8], float s, float inv) {
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float first = __fmul_rn(v[i], inv), quotient = __fmaf_rn(__fmaf_rn(-first, s, v[i]), inv, first);
    b[i] = __float_as_uint(__fadd_rn(quotient, 12582912.0f));
  }
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// A row's scale from the bits of its largest magnitude; `some`: whether its integers are not all zero.
__device__ __forceinline__ float int8_scale(unsigned largest, bool* some) {
  const float s = __fdiv_rn(__uint_as_float(largest), 127.0f);
  *some = largest < 0x7f800000u && s >= 1.17549435e-38f;
  return s;
}
// Rows of numbers, not all zero, whose scale is 2^-100 or more.  Of a row with a smaller scale the quotients are taken of 2^64 times its
// values and 2^64 times its scale, exactly (see eight_nearest).
__device__ __forceinline__ bool int8_usual(unsigned largest, float s) { return largest < 0x7f800000u && s >= 7.8886091e-31f; }
constexpr float INT8_LIFT = 18446744073709551616.0f;
// ... as it is told: NaN where the row holds an infinity or a NaN.
__device__ __forceinline__ float int8_told(unsigned largest, bool some, float s) {
  return largest >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : some ? s : 0.f;
}
