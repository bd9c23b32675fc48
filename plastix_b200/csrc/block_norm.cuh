// Shared by block_norm.cu (forward) and block_norm_backward.cu.
#pragma once

#include "norm.cuh"

namespace plx {

struct BlockNorm {
  uint32_t rows, n;
  float inv_n, scale, eps;
  int gate;
  bool layer, post, sigmoid, param_f32;
  const void *x, *o, *gate_values;
  int64_t ldx, ldo, ldg;
  const void *post_weight, *post_bias, *pre_weight, *pre_bias;
  // forward
  void *r, *u;
  int64_t ldr, ldu;
  float4* stats_out;
  // backward
  const void *dr, *du;
  int64_t lddr, lddu;
  const float4* stats;  // mean and rstd of o, of r
  void *dx, *d_o, *dgate;
  int64_t lddx, lddo, lddg;
  float* partial;  // column sums
};

int check_block_norm(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                     const plx_block_norm_params* p);
BlockNorm block_norm_of(uint64_t rows, uint32_t n, const plx_block_norm_params* p);

// sigmoid(g) and 1 - sigmoid(g), neither by a difference that cancels.
struct Sigmoid {
  float a, keep;
};
__device__ __forceinline__ Sigmoid sigmoid(float g) {
  const float e = exp2_approx(-fabsf(g) * kLog2e), d = 1.0f + e;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  r = fmaf(r, fmaf(-d, r, 1.0f), r);
  const float er = e * r;
  return g < 0.0f ? Sigmoid{er, r} : Sigmoid{r, er};
}

// Pieces of a row, STEP values apart; 0 past its end.
template <int STEP, int NV, int V, typename T>
__device__ __forceinline__ void load_row(const T* from, int left, Pack<T, V> (&q)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j * STEP < left) {
      q[j] = load_pack<T, V>(from + j * STEP);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) q[j].v[e] = from_f32<T>(0.0f);
    }
  }
}

template <int STEP, typename P, int NV, int V>
__device__ __forceinline__ void affine(float (&v)[NV * V], const P* w, const P* b, uint32_t c0,
                                       int left) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j * STEP >= left) continue;
    if (w) {
      const Pack<P, V> q = load_pack<P, V>(w + c0 + j * STEP);
#pragma unroll
      for (int e = 0; e < V; ++e) v[j * V + e] *= to_f32(q.v[e]);
    }
    if (b) {
      const Pack<P, V> q = load_pack<P, V>(b + c0 + j * STEP);
#pragma unroll
      for (int e = 0; e < V; ++e) v[j * V + e] += to_f32(q.v[e]);
    }
  }
}

// The values of a row, made from what is read (rows that no registers hold).
template <typename T, typename P>
struct RowOf {
  const BlockNorm& a;
  int64_t row;
  float m1, s1, m2, s2;
  __device__ __forceinline__ RowOf(const BlockNorm& b, int64_t r) : a(b), row(r) {}
  __device__ __forceinline__ float affine(float h, const void* w, const void* b, uint32_t i) const {
    if (w) h *= to_f32(((const P*)w)[i]);
    if (b) h += to_f32(((const P*)b)[i]);
    return h;
  }
  __device__ __forceinline__ float o(uint32_t i) const {
    return to_f32(((const T*)a.o)[row * a.ldo + i]);
  }
  __device__ __forceinline__ float h1(uint32_t i) const { return a.post ? (o(i) - m1) * s1 : o(i); }
  __device__ __forceinline__ float p(uint32_t i) const {
    return a.post ? affine(h1(i), a.post_weight, a.post_bias, i) : o(i);
  }
  // The gate and its derivative.
  __device__ __forceinline__ float gate(uint32_t i, float& slope) const {
    slope = 1.0f;
    if (a.gate == PLX_BLOCK_GATE_NONE) return 1.0f;
    const float g = a.gate == PLX_BLOCK_GATE_UNITS
                        ? to_f32(((const P*)a.gate_values)[i])
                        : to_f32(((const T*)a.gate_values)[row * a.ldg + i]);
    if (!a.sigmoid) return g;
    const Sigmoid s = sigmoid(g);
    slope = s.a * s.keep;
    return s.a;
  }
  __device__ __forceinline__ float r(uint32_t i) const {
    float slope;
    const float g = gate(i, slope);
    return fmaf(g, p(i), a.scale * to_f32(((const T*)a.x)[row * a.ldx + i]));
  }
};

// Values that can be read together in every array of a call.
template <typename T, typename P>
uint32_t block_piece(const BlockNorm& a, std::initializer_list<const void*> rows,
                     std::initializer_list<int64_t> strides) {
  uint64_t at = 0, ld = 0, w = 0;
  for (const void* p : rows) at |= reinterpret_cast<uintptr_t>(p);
  for (int64_t s : strides) ld |= (uint64_t)s;
  const uint64_t g = reinterpret_cast<uintptr_t>(a.gate_values);
  if (a.gate == PLX_BLOCK_GATE_VALUES) {
    at |= g;
    ld |= (uint64_t)a.ldg;
  } else {
    w |= g;
  }
  for (const void* p : {a.post_weight, a.post_bias, a.pre_weight, a.pre_bias})
    w |= reinterpret_cast<uintptr_t>(p);
  return piece_values(a.n, sizeof(T), {(const void*)at}, {(int64_t)ld}, (const void*)w, nullptr,
                      sizeof(P));
}

}  // namespace plx
