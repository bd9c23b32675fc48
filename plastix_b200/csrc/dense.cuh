// Shared by dense.cu and the products that it runs.
#pragma once

#include "norm.cuh"

namespace plx {

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == PLX_ACT_SIGMOID) return sigmoid(z).a;
  else if constexpr (ACT == PLX_ACT_TANH) return tanhf(z);
  else if constexpr (ACT == PLX_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  else if constexpr (ACT == PLX_ACT_SILU) return z * sigmoid(z).a;
  else if constexpr (ACT == PLX_ACT_GELU)
    return z * (0.5f * erfcf(z * -0.70710678118654752f));
  else return z;
}
// The same for results of 16 bits, in fewer instructions. Relative errors: sigmoids
// (9 + 1.3 |z|) 2^-24 (the exponent's argument is rounded), tanh 8e-6 (at 0.02, where 1 -
// e begins to cancel), GELU's Phi 1e-5 for |z| < 10 and 1e-4 beyond (where it is below
// 1e-23).
template <int ACT>
__device__ __forceinline__ float act_value16(float z) {
  if constexpr (ACT == PLX_ACT_SIGMOID) {
    return rcp_approx(1.0f + exp2_approx(z * -kLog2e));
  } else if constexpr (ACT == PLX_ACT_SILU) {
    return z * rcp_approx(1.0f + exp2_approx(z * -kLog2e));
  } else if constexpr (ACT == PLX_ACT_TANH) {
    // (1 - e) / (1 + e), e = exp(-2 |z|); near 0, where that cancels, z - z^3 / 3
    const float a = fabsf(z), e = exp2_approx(a * (-2.0f * kLog2e));
    const float far = copysignf((1.0f - e) * rcp_approx(1.0f + e), z);
    return a < 0.02f ? fmaf(z * z * z, -1.0f / 3.0f, z) : far;
  } else if constexpr (ACT == PLX_ACT_GELU) {
    // Phi(-|z|) = exp(-z^2 / 2) times a polynomial in t = 1 / (1 + 0.3 |z|) without a
    // constant, fitted for the least relative error over |z| <= 10
    const float t = rcp_approx(fmaf(fabsf(z), 0.3f, 1.0f));
    float q = -0.08074618130922318f;
    q = fmaf(q, t, 0.22719280421733856f);
    q = fmaf(q, t, -0.029975734651088715f);
    q = fmaf(q, t, 0.1514199823141098f);
    q = fmaf(q, t, 0.11184987425804138f);
    q = fmaf(q, t, 0.1202608123421669f);
    q *= t * exp2_approx(z * z * (-0.5f * kLog2e));
    return z * (z < 0.0f ? q : 1.0f - q);
  } else {
    return act_value<ACT>(z);
  }
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == PLX_ACT_SIGMOID) {
    const Sigmoid s = sigmoid(z);
    return s.a * s.keep;
  } else if constexpr (ACT == PLX_ACT_TANH) {
    const float t = tanhf(z);
    return fmaf(-t, t, 1.0f);
  } else if constexpr (ACT == PLX_ACT_RELU) {
    return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
  } else if constexpr (ACT == PLX_ACT_SILU) {
    const Sigmoid s = sigmoid(z);
    return s.a * fmaf(z, s.keep, 1.0f);
  } else if constexpr (ACT == PLX_ACT_GELU) {
    const float pdf = 0.39894228040143268f * exp2_approx(-0.5f * kLog2e * z * z);
    return fmaf(z, pdf, 0.5f * erfcf(z * -0.70710678118654752f));
  } else {
    return 1.0f;
  }
}

// Runs f with the activation as a constant.
template <typename F>
int with_act(int act, F f) {
  using std::integral_constant;
  switch (act) {
    case PLX_ACT_SIGMOID: return f(integral_constant<int, PLX_ACT_SIGMOID>{});
    case PLX_ACT_TANH: return f(integral_constant<int, PLX_ACT_TANH>{});
    case PLX_ACT_RELU: return f(integral_constant<int, PLX_ACT_RELU>{});
    case PLX_ACT_SILU: return f(integral_constant<int, PLX_ACT_SILU>{});
    case PLX_ACT_GELU: return f(integral_constant<int, PLX_ACT_GELU>{});
    default: return f(integral_constant<int, PLX_ACT_IDENTITY>{});
  }
}

// One operand of a product over k: value (i, k) is p[i * ld + k] (k_major) or
// p[k * ld + i]. 32-bit values come as three planes of bfloat16 whose sum they are,
// `plane` bytes apart.
struct Operand {
  const void* p;
  int64_t ld, plane;
  bool k_major;
};

// What becomes of the sums z[i][j] of a product: y = act(z + bias[j]) + residual.
// factor: of float16 operands, what z is multiplied by before (NULL: nothing).
struct Finish {
  int param_dtype, act;
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* y;
  int64_t ldy;
  float* pre;  // z + bias, [rows][cols]
  const float* factor;
};

// y[i][j] for i < rows, j < cols: sums over k < depth of a(i, k) b(j, k).
struct Product {
  uint32_t rows, cols, depth;
  Operand a, b;
  Finish f;
};

// Operands start at, and have strides of, multiples of 16 bytes; residual and result
// are of type dtype.
int product_tensor(plx_ctx* ctx, int dtype, const Product& p);

}  // namespace plx
