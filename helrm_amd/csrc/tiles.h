// tiles.h -- device functions that the products share: matrix instructions,
// activations, the pieces of a softmax, the parts of a float32.
#pragma once
#include "cleartext.h"
#include "products.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16;

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
template <class T> struct Vec8;
template <> struct Vec8<__bf16> { typedef bf16x8 type; };
template <> struct Vec8<_Float16> { typedef f16x8 type; };

// a = act(g) and d = act'(g) of four values
__device__ __forceinline__ void act4(int act, const float* c, const float g[4], float a[4], float d[4]) {
  if (act == ACT_SILU) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-g[e]));   // (within 1 ulp)
      a[e] = g[e] * s;
      d[e] = s * (1.0f + g[e] * (1.0f - s));
    }
  } else if (act == ACT_GELU) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float cdf = 0.5f * (1.0f + erff(g[e] * 0.70710678118654752f));
      a[e] = g[e] * cdf;
      d[e] = cdf + g[e] * __expf(-0.5f * g[e] * g[e]) * 0.39894228040143268f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      a[e] = ((c[3] * g[e] + c[2]) * g[e] + c[1]) * g[e] + c[0];
      d[e] = (3.0f * c[3] * g[e] + 2.0f * c[2]) * g[e] + c[1];
    }
  }
}

// (maximum, sum of exponentials about it) of two pieces of a row, (-inf, 0) for
// one that holds nothing above -inf.  A NaN is in the sum and stays there.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(m, a.y + b.y);
  return make_float2(m, a.y * __expf(a.x - m) + b.y * __expf(b.x - m));
}

// The parts of a float32 value, x = x0 + x1 + x2.  x0 is x (1 - 2^-9) rounded:
// what 8 bits hold is its own first part, and no finite x has an infinite one
// (the largest float32 rounds to infinity).  So x1 is up to 1.5 2^-8 of x and
// x2 up to 2^-16; both are NaN of an infinite x.
__device__ __forceinline__ void split3(float v, __bf16 out[3]) {
  out[0] = (__bf16)(v * 0x1.ffp-1f);
  const float r = v - (float)out[0];
  out[1] = (__bf16)r;
  out[2] = (__bf16)(r - (float)out[1]);
}

// A sum of parts' products as what the first parts' are corrected by.  Those
// alone know what an infinite factor or an overflow comes to: the other parts
// are NaN or of either sign there, and the correction is left out.
__device__ __forceinline__ float settled(float v) { return fabsf(v) < INFINITY ? v : 0.0f; }
__device__ __forceinline__ f32x4 settled(f32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = settled(v[e]);
  return v;
}

}  // namespace
