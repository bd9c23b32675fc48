// Shared by norm.cu (layer norm forward) and norm_backward.cu.
#pragma once

#include <type_traits>

#include "chunk_copy.h"
#include "rows.cuh"

namespace plx {

// V consecutive values in one access (16 bytes where V * sizeof(T) is 16; V
// float weights beside 8 half-width values are two accesses).
template <typename T, int V>
struct alignas(V * sizeof(T) >= 16 ? 16 : V * sizeof(T)) Pack {
  T v[V];
};

// All a thread's values of a row at once, in 32 bits.
template <int NV, int V, typename T>
__device__ __forceinline__ void widen(const Pack<T, V> (&q)[NV], float (&f)[NV * V]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) f[j * V + e] = to_f32(q[j].v[e]);
}

// Values e and e + 1 of a piece, rounded together.
template <typename T, int V>
__device__ __forceinline__ void put_pair(Pack<T, V>& q, int e, F2 v) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    *reinterpret_cast<__nv_bfloat162*>(&q.v[e]) = __floats2bfloat162_rn(v.x, v.y);
  } else if constexpr (std::is_same_v<T, __half>) {
    *reinterpret_cast<__half2*>(&q.v[e]) = __floats2half2_rn(v.x, v.y);
  } else {
    q.v[e] = v.x;
    q.v[e + 1] = v.y;
  }
}
template <typename T, int V>
__device__ __forceinline__ F2 pair_of(const Pack<T, V>& q, int e) {
  return pack2(to_f32(q.v[e]), to_f32(q.v[e + 1]));
}

// H pairs of results as NV pieces of a row: piece j goes j * STEP values on
// from `to`, where that is less than `left`.
template <int STEP, int NV, int V, typename T>
__device__ __forceinline__ void store_row(T* to, int left, const F2 (&v)[NV * V / 2]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j * STEP >= left) continue;
    Pack<T, V> out;
    if constexpr (V == 1) {
      out.v[0] = from_f32<T>(j & 1 ? v[j / 2].y : v[j / 2].x);
    } else {
#pragma unroll
      for (int e = 0; e < V; e += 2) put_pair(out, e, v[(j * V + e) / 2]);
    }
    *reinterpret_cast<Pack<T, V>*>(to + j * STEP) = out;
  }
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}

// Rows of 16-bit values of which not even two can be read together: sixteen-byte
// chunks go to shared memory whole and the values are read from there. A
// chunk's bytes outside its row are of the rows beside it or of what lies
// between them and are not used; nothing outside the array is touched.
template <typename T, int TPR, int NV>
struct Staged {
  static_assert(sizeof(T) == 2, "for 16-bit values");
  static constexpr int bytes = (TPR * NV * 2 + 31) / 16 * 16;  // a row, at any offset

  static __device__ __forceinline__ uint32_t offset(const T* row) {
    return (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u);
  }
  // Starts the copies of this thread's chunks of row r of an array.
  static __device__ __forceinline__ void fetch(char* to, const T* array, int64_t ld, uint32_t rows,
                                               uint32_t n, uint32_t r, uint32_t lane) {
    const T* row = array + r * ld;
    const uint32_t off = offset(row), end = off + 2 * n;
    const char* from = reinterpret_cast<const char*>(row) - off;
    const bool near = near_edge(r, rows);
    for (uint32_t c = lane * 16; c < end; c += TPR * 16) {
      ChunkCopy k{0u, 16u, true};
      if (near) {
        const uint64_t at = reinterpret_cast<uintptr_t>(row);
        const uint64_t first = reinterpret_cast<uintptr_t>(array);
        k = chunk_copy(at - off + c, at, at + 2 * n, first,
                       first + ((rows - 1) * ld + n) * sizeof(T));
      }
      if (k.whole) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(to + c)),
                     "l"(from + c), "r"(k.to)
                     : "memory");
      } else {
        for (uint32_t e = c + k.from; e < c + k.to; e += 2)
          *reinterpret_cast<T*>(to + e) = *reinterpret_cast<const T*>(from + e);
      }
    }
  }
  // This thread's values (0 past the row's end).
  static __device__ __forceinline__ void read(const char* at, const T* row, uint32_t n,
                                              uint32_t lane, Pack<T, 1> (&q)[NV]) {
    const T* v = reinterpret_cast<const T*>(at + offset(row)) + lane;
    const int left = (int)n - (int)lane;
#pragma unroll
    for (int j = 0; j < NV; ++j) q[j].v[0] = j * TPR < left ? v[j * TPR] : from_f32<T>(0.0f);
  }
};

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

// Two sums at once: half of the warp carries each, so that they cost five
// exchanges and not ten. Else as row_sum.
template <int TPR>
__device__ __forceinline__ F2 row_sum2(F2 v, float* red, int& turn) {
  const uint32_t lane = threadIdx.x & 31;
  const bool upper = lane & 16;
  float a = upper ? v.y : v.x;
  a += __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
#pragma unroll
  for (int d = 8; d; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;  // 4 to 32
    float* r = red + turn * W * 2;
    turn ^= 1;
    if ((lane & 15) == 0) r[(upper ? W : 0) + (threadIdx.x >> 5)] = a;
    __syncthreads();
    const uint32_t k = lane & 15;
    a = k < W ? r[(upper ? W : 0) + k] : 0.0f;
    if (W > 16) a += r[(upper ? W : 0) + 16 + k];
#pragma unroll
    for (int d = W < 16 ? W / 2 : 8; d; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
    if (W < 16) a = __shfl_sync(0xffffffffu, a, lane & 16);
  }
  const float b = __shfl_xor_sync(0xffffffffu, a, 16);
  return upper ? pack2(b, a) : pack2(a, b);
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

// How many values, of 16 bytes down to one value, can be read together: no
// piece crosses a row's end, and every one is aligned. The weights may be of
// another size.
inline uint32_t piece_values(uint32_t n, size_t elem, std::initializer_list<const void*> rows,
                             std::initializer_list<int64_t> strides, const void* weight,
                             const void* bias, size_t param) {
  uint64_t all = n;
  for (int64_t s : strides) all |= (uint64_t)s;
  uint64_t at = 0, wat = 0;
  for (const void* p : rows) at |= reinterpret_cast<uintptr_t>(p);
  wat |= reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias);
  uint32_t v = 16 / (uint32_t)elem;
  while (v > 1 && (all % v || at % (v * elem) || wat % std::min<size_t>(16, v * param))) v /= 2;
  return v;
}

}  // namespace plx
