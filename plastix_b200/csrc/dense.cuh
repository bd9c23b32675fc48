// Shared by dense.cu and the products that it runs.
#pragma once

#include "norm.cuh"

namespace plx {

// sigmoid(g) and 1 - sigmoid(g), neither by a difference that cancels.
struct Squash {
  float a, keep;
};
__device__ __forceinline__ Squash squash(float g) {
  const float e = exp2_approx(-fabsf(g) * kLog2e), d = 1.0f + e;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  r = fmaf(r, fmaf(-d, r, 1.0f), r);
  const float er = e * r;
  return g < 0.0f ? Squash{er, r} : Squash{r, er};
}

template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == PLX_ACT_SIGMOID) return squash(z).a;
  else if constexpr (ACT == PLX_ACT_TANH) return tanhf(z);
  else if constexpr (ACT == PLX_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  else if constexpr (ACT == PLX_ACT_SILU) return z * squash(z).a;
  else if constexpr (ACT == PLX_ACT_GELU)
    return z * (0.5f + 0.5f * erff(z * 0.70710678118654752f));
  else return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == PLX_ACT_SIGMOID) {
    const Squash s = squash(z);
    return s.a * s.keep;
  } else if constexpr (ACT == PLX_ACT_TANH) {
    const float t = tanhf(z);
    return fmaf(-t, t, 1.0f);
  } else if constexpr (ACT == PLX_ACT_RELU) {
    return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
  } else if constexpr (ACT == PLX_ACT_SILU) {
    const Squash s = squash(z);
    return s.a * fmaf(z, s.keep, 1.0f);
  } else if constexpr (ACT == PLX_ACT_GELU) {
    const float pdf = 0.39894228040143268f * exp2_approx(-0.5f * kLog2e * z * z);
    return fmaf(z, pdf, 0.5f + 0.5f * erff(z * 0.70710678118654752f));
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
// p[k * ld + i].
struct Operand {
  const void* p;
  int64_t ld;
  bool k_major;
};

// What becomes of the sums z[i][j] of a product: y = act(z + bias[j]) + residual.
struct Finish {
  int param_dtype, act;
  const void* bias;
  const void* residual;
  int64_t ldr;
  void* y;
  int64_t ldy;
  float* pre;  // z + bias, [rows][cols]
};

// y[i][j] for i < rows, j < cols: sums over k < depth of a(i, k) b(j, k).
struct Product {
  uint32_t rows, cols, depth;
  Operand a, b;
  Finish f;
};

int product_f32(plx_ctx* ctx, int dtype, const Product& p);
// 16-bit types; operands start at, and have strides of, multiples of 16 bytes.
int product_tensor(plx_ctx* ctx, int dtype, const Product& p);

}  // namespace plx
