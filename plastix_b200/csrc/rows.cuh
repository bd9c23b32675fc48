// Shared pieces of the row operators (norm.cu, norm_backward.cu, log_probs.cu,
// distill.cu): element types, pairs of values, reductions in a fixed order and
// asynchronous copies.
#pragma once

#include <atomic>
#include <initializer_list>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace plx {

inline bool valid_dtype(int dtype) {
  return dtype == PLX_F32 || dtype == PLX_BF16 || dtype == PLX_F16;
}

inline size_t dtype_bytes(int dtype) { return dtype == PLX_F32 ? 4 : 2; }

// Arrays start at a multiple of their elements' size.
inline int check_aligned(size_t elem, std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    PLX_CHECK_ARG(reinterpret_cast<uintptr_t>(p) % elem == 0,
                  "array %p is not aligned to its elements of %zu bytes", p, elem);
  return PLX_OK;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Runs f with a value of the C++ type that `dtype` names.
template <typename F>
int with_dtype(int dtype, F f) {
  if (dtype == PLX_F32) return f(float{});
  if (dtype == PLX_BF16) return f(__nv_bfloat16{});
  return f(__half{});
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
// ---- two 32-bit values at once (one instruction each) ----------------------
using F2 = float2;
__device__ __forceinline__ F2 pack2(float a, float b) { return make_float2(a, b); }
__device__ __forceinline__ void unpack2(F2 v, float& a, float& b) {
  a = v.x;
  b = v.y;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { return __ffma2_rn(a, b, c); }

// NaN wins, as in the arithmetic that follows it.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}

// Block-wide sum, the same value in every thread, added in a fixed order. `red`
// holds one float per warp; the barrier at the head lets it be used again at once.
template <int WARPS>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) s = __fadd_rn(s, red[w]);
  return s;
}

// From global to shared memory without a register in between.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst_smem, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst_smem)), "l"(src)
                 : "memory");
  else  // 4 or 8
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_addr(dst_smem)), "l"(src),
                 "n"(BYTES)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// 2^x by the special-function unit (relative error about 2^-22; 0 for
// arguments below -126).
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

}  // namespace plx

// Lets a kernel use `bytes` of dynamic shared memory, asking the driver once a
// device. `KERNEL` makes the memory of that the kernel's own.
template <auto KERNEL>
cudaError_t allow_shared(int device, int bytes) {
  static std::atomic<uint64_t> asked{0};
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (asked.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Makes a context's device current for one call and puts the caller's back.
struct DeviceGuard {
  int before = -1;
  cudaError_t err;
  explicit DeviceGuard(int device) {
    err = cudaGetDevice(&before);
    if (err == cudaSuccess && before != device)
      err = cudaSetDevice(device);
    else
      before = -1;
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
};
