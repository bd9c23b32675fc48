// Shared by norm.cu (layer norm forward) and norm_backward.cu.
#pragma once

#include "rows.cuh"

namespace plx {

// V consecutive values in one access (16 bytes where V * sizeof(T) is 16; V
// float weights beside 8 half-width values are two accesses).
template <typename T, int V>
struct alignas(V * sizeof(T) >= 16 ? 16 : V * sizeof(T)) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}

// Sum over the TPR threads that share a row, the same in each of them. `red`
// holds two halves used in turn, so one barrier a sum is enough.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float* red, int& turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = warp_sum(v[k]);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    float* r = red + turn * W * K;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) r[(threadIdx.x >> 5) * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = r[k];
#pragma unroll
      for (int w = 1; w < W; ++w) s = __fadd_rn(s, r[w * K + k]);
      v[k] = s;
    }
  }
}

inline int check_norm(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, int param_dtype) {
  PLX_CHECK_ARG(ctx, "ctx is required");
  PLX_CHECK_ARG(valid_dtype(dtype), "dtype %d is none of PLX_F32, PLX_BF16, PLX_F16", dtype);
  PLX_CHECK_ARG(n > 0 && n < (1u << 31), "n = %u is out of range", n);
  if (rows >= (1ull << 31))
    return set_error(PLX_ERR_CAPACITY, "%llu rows: fewer than 2^31 are supported",
                     (unsigned long long)rows);
  PLX_CHECK_ARG(param_dtype == PLX_F32 || param_dtype == dtype,
                "param_dtype %d is neither PLX_F32 nor the rows' dtype %d", param_dtype, dtype);
  return PLX_OK;
}

// Whether rows can be read in 16-byte pieces: no piece crosses a row's end.
inline bool whole_pieces(uint32_t n, size_t elem, std::initializer_list<const void*> ptrs,
                         std::initializer_list<int64_t> strides) {
  const uint32_t v = 16 / (uint32_t)elem;
  if (n % v) return false;
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  for (int64_t s : strides)
    if (s % v) return false;
  return true;
}

}  // namespace plx
