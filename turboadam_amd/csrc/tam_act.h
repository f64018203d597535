// tam_act.h -- the activations of linear and gated layers, and their slopes.
#ifndef TAM_ACT_H
#define TAM_ACT_H

#include <math.h>

#include <type_traits>

#include "tam_ops.h"

#define TAM_ACT_MAX TAM_ACT_SILU

// ---------------------------------------------------------------------------
// activations (fp32)
// ---------------------------------------------------------------------------
// gelu_tanh: 0.5 z (1 + tanh u) = z sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3)
#define TAM_GELU_2U 1.5957691216057308f
#define TAM_GELU_C 0.044715f

// FAST (16-bit results): the hardware's 2^x and reciprocal, 1 ulp each, 4 instructions
// for about 30: 2^-20 of the result at |x| < 16. At 8192 x 768 x 3072 the epilogue's
// arithmetic took longer than its stores.
template <bool FAST>
__device__ __forceinline__ float tam_sigmoid(float x) {
  if constexpr (FAST)
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * x));
  else
    return 1.0f / (1.0f + expf(-x));
}

template <bool FAST>
__device__ __forceinline__ float tam_act(float z, uint32_t act) {
  switch (act) {
    case TAM_ACT_RELU: return z < 0.0f ? 0.0f : z;  // a NaN stays
    case TAM_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
    case TAM_ACT_GELU_TANH: return z * tam_sigmoid<FAST>(TAM_GELU_2U * __builtin_fmaf(TAM_GELU_C * z * z, z, z));
    case TAM_ACT_SILU: return z * tam_sigmoid<FAST>(z);
    default: return z;
  }
}

// Past +-128 the smooth activations' slopes are 0 and 1 in fp32, and so they are at
// the infinities: a z that the layer's type cannot hold (below -65504 in fp16, where y is
// a finite 0) or whose cube passes fp32's range would give 0 * inf as a factor, so `near`
// is the factor. (One instruction, which loses a NaN: that comes from s or e.)
template <bool FAST>
__device__ __forceinline__ float tam_act_slope(float z, uint32_t act) {
  const float near = __builtin_amdgcn_fmed3f(z, -128.0f, 128.0f);
  switch (act) {
    case TAM_ACT_RELU: return z > 0.0f ? 1.0f : (z == z ? 0.0f : z);
    case TAM_ACT_GELU: {
      const float e = FAST ? __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z) : expf(-0.5f * z * z);
      return __builtin_fmaf(near * 0.39894228040143268f, e, 0.5f * (1.0f + erff(z * 0.70710678118654752f)));
    }
    case TAM_ACT_GELU_TANH: {
      const float s = tam_sigmoid<FAST>(TAM_GELU_2U * __builtin_fmaf(TAM_GELU_C * z * z, z, z));
      return __builtin_fmaf(near * s * (1.0f - s), TAM_GELU_2U * __builtin_fmaf(3.0f * TAM_GELU_C * near, near, 1.0f), s);
    }
    case TAM_ACT_SILU: {
      const float s = tam_sigmoid<FAST>(z);
      return s * __builtin_fmaf(near, 1.0f - s, 1.0f);
    }
    default: return 1.0f;
  }
}

// Eight of them, with one look at which it is.
template <bool FAST>
__device__ __forceinline__ void tam_act8(const float (&z)[8], uint32_t act, float (&y)[8]) {
  auto each = [&](auto which) {
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = tam_act<FAST>(z[j], decltype(which)::value);
  };
  switch (act) {
    case TAM_ACT_RELU: return each(std::integral_constant<uint32_t, TAM_ACT_RELU>());
    case TAM_ACT_GELU: return each(std::integral_constant<uint32_t, TAM_ACT_GELU>());
    case TAM_ACT_GELU_TANH: return each(std::integral_constant<uint32_t, TAM_ACT_GELU_TANH>());
    case TAM_ACT_SILU: return each(std::integral_constant<uint32_t, TAM_ACT_SILU>());
    default: return each(std::integral_constant<uint32_t, TAM_ACT_NONE>());
  }
}

#endif  // TAM_ACT_H
