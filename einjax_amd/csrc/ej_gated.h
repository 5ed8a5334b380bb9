// Activations of the gated products and their derivatives, in fp32.
//
//   silu       g p,          p = 1 / (1 + exp(-g))
//   gelu       g Phi(g),     Phi(g) = erfc(-g / sqrt 2) / 2
//   gelu_tanh  g p(2 z),     z = sqrt(2 / pi) (g + 0.044715 g^3): 0.5 g (1 + tanh z)
//
// FINE: the library's exp and division.  Otherwise the hardware's exp2 and
// reciprocal (each within one unit in the last place, and the argument's
// rounding, |g| 2^-24 relative in all), for results that are rounded to 16
// bits.
#pragma once

#include "ej_internal.h"

namespace ej {

// 1 / (1 + exp(-v)); 0 where exp(-v) overflows.
template <bool FINE>
__device__ inline float sigmoid(float v) {
  if constexpr (FINE) return 1.f / (1.f + expf(-v));
  else return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.44269504f));
}

// 1 - sigmoid(v), without cancellation.
template <bool FINE>
__device__ inline float sigmoid_of_minus(float v) {
  return sigmoid<FINE>(-v);
}

// 2 z of gelu_tanh
__device__ inline float gelu_twice_z(float g) { return g * (1.59576912f + 0.0713548163f * g * g); }

template <bool FINE>
struct Silu {
  __device__ inline float operator()(float g) const { return g * sigmoid<FINE>(g); }
  __device__ static inline void both(float g, float *value, float *slope) {
    const float p = sigmoid<FINE>(g);
    *value = g * p;
    *slope = p + g * p * sigmoid_of_minus<FINE>(g);
  }
};

template <bool FINE>
struct Gelu {
  __device__ inline float operator()(float g) const { return 0.5f * g * erfcf(g * -0.707106781f); }
  __device__ static inline void both(float g, float *value, float *slope) {
    const float p = 0.5f * erfcf(g * -0.707106781f);
    *value = g * p;
    *slope = p + g * (0.39894228f * expf(-0.5f * g * g));
  }
};

template <bool FINE>
struct GeluTanh {
  __device__ inline float operator()(float g) const { return g * sigmoid<FINE>(gelu_twice_z(g)); }
  __device__ static inline void both(float g, float *value, float *slope) {
    const float z = gelu_twice_z(g), p = sigmoid<FINE>(z);
    *value = g * p;
    // the second term is below 2^-126 beyond 16, where g^3 may pass fp32's range
    const float s = p * sigmoid_of_minus<FINE>(z);
    *slope = s > 0.f ? p + g * s * (1.59576912f + 0.214064449f * g * g) : p;
  }
};

// f with the activation's function object.
template <bool FINE, class F>
__device__ inline void by_activation(int activation, F f) {
  if (activation == EJ_SILU) f(Silu<FINE>());
  else if (activation == EJ_GELU) f(Gelu<FINE>());
  else f(GeluTanh<FINE>());
}

}  // namespace ej
