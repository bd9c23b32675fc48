// Layer norm of rows of unit activations, forward and backward.
//   mu = mean x; rstd = 1/sqrt(mean (x-mu)^2 + eps); h = (x-mu) rstd; y = h w + b
//   dx = rstd (w dy - mean(w dy) - h mean(w dy h)); dw = sum_rows dy h; db = sum_rows dy
// Statistics, gradients of the weights and everything between load and store
// are in 32 bits. The weights' gradients are added in a fixed order (no
// atomics), so a call gives the same bits every time.
#include "rows.cuh"

namespace plx {
namespace {

constexpr int kThreads = 256;

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads)
k_norm_fwd(uint32_t n, const T* __restrict__ x, int64_t ldx, const P* __restrict__ w,
           const P* __restrict__ b, float eps, T* __restrict__ y, int64_t ldy,
           float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[kThreads / 32];
  const int64_t r = blockIdx.x;
  const T* xr = x + r * ldx;
  T* yr = y + r * ldy;
  float s = 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) s += to_f32(xr[i]);
  const float mu = block_sum<kThreads / 32>(s, red) / (float)n;
  s = 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const float d = to_f32(xr[i]) - mu;
    s = fmaf(d, d, s);
  }
  const float rs = 1.0f / sqrtf(block_sum<kThreads / 32>(s, red) / (float)n + eps);
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const float h = (to_f32(xr[i]) - mu) * rs;
    yr[i] = from_f32<T>(fmaf(h, w ? to_f32(w[i]) : 1.0f, b ? to_f32(b[i]) : 0.0f));
  }
  if (threadIdx.x == 0) {
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads)
k_norm_dx(uint32_t n, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
          const float* __restrict__ mean, const float* __restrict__ rstd,
          const P* __restrict__ w, T* __restrict__ dx, int64_t lddx) {
  __shared__ float red[kThreads / 32];
  const int64_t r = blockIdx.x;
  const T* dyr = dy + r * lddy;
  const T* xr = x + r * ldx;
  const float mu = mean[r], rs = rstd[r];
  float s1 = 0.0f, s2 = 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const float g = to_f32(dyr[i]) * (w ? to_f32(w[i]) : 1.0f);
    s1 += g;
    s2 = fmaf(g, (to_f32(xr[i]) - mu) * rs, s2);
  }
  const float c1 = block_sum<kThreads / 32>(s1, red) / (float)n;
  const float c2 = block_sum<kThreads / 32>(s2, red) / (float)n;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const float g = to_f32(dyr[i]) * (w ? to_f32(w[i]) : 1.0f);
    const float h = (to_f32(xr[i]) - mu) * rs;
    dx[r * lddx + i] = from_f32<T>(rs * (g - c1 - h * c2));
  }
}

// Columns' sums over one of `groups` contiguous runs of rows:
// partial[group][0][i] = sum dy h, partial[group][1][i] = sum dy.
template <typename T>
__global__ void __launch_bounds__(kThreads)
k_norm_dw_partial(uint64_t rows, uint32_t n, const T* __restrict__ dy, int64_t lddy,
                  const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean,
                  const float* __restrict__ rstd, float* __restrict__ partial) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  const uint64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float sw = 0.0f, sb = 0.0f;
  for (uint64_t r = r0; r < r1; ++r) {
    const float g = to_f32(dy[(int64_t)r * lddy + i]);
    sw = fmaf(g, (to_f32(x[(int64_t)r * ldx + i]) - mean[r]) * rstd[r], sw);
    sb += g;
  }
  partial[(uint64_t)blockIdx.y * 2 * n + i] = sw;
  partial[(uint64_t)blockIdx.y * 2 * n + n + i] = sb;
}

template <typename P>
__global__ void __launch_bounds__(kThreads)
k_norm_dw_join(uint32_t groups, uint32_t n, const float* __restrict__ partial, P* __restrict__ dw,
               P* __restrict__ db) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  float sw = 0.0f, sb = 0.0f;
  for (uint32_t g = 0; g < groups; ++g) {
    sw += partial[(uint64_t)g * 2 * n + i];
    sb += partial[(uint64_t)g * 2 * n + n + i];
  }
  if (dw) dw[i] = from_f32<P>(sw);
  if (db) db[i] = from_f32<P>(sb);
}

// Runs of rows whose column sums are taken apart: enough to fill the device,
// few enough that joining them costs little beside reading the rows.
uint32_t norm_groups(uint64_t rows) {
  return (uint32_t)std::min<uint64_t>(std::max<uint64_t>(rows / 16, 1), 256);
}

int check_rows(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype) {
  PLX_CHECK_ARG(ctx, "ctx is required");
  PLX_CHECK_ARG(valid_dtype(dtype), "dtype %d is none of PLX_F32, PLX_BF16, PLX_F16", dtype);
  PLX_CHECK_ARG(n > 0 && n < (1u << 31), "n = %u is out of range", n);
  if (rows >= (1ull << 31))
    return set_error(PLX_ERR_CAPACITY, "%llu rows: fewer than 2^31 are supported",
                     (unsigned long long)rows);
  return PLX_OK;
}

int check_param_dtype(int param_dtype, int dtype) {
  PLX_CHECK_ARG(param_dtype == PLX_F32 || param_dtype == dtype,
                "param_dtype %d is neither PLX_F32 nor the rows' dtype %d", param_dtype, dtype);
  return PLX_OK;
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" int plx_layer_norm(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, const void* x,
                              int64_t ldx, int param_dtype, const void* weight, const void* bias,
                              float eps, void* y, int64_t ldy, float* mean, float* rstd) {
  if (int rc = check_rows(ctx, rows, n, dtype)) return rc;
  if (int rc = check_param_dtype(param_dtype, dtype)) return rc;
  PLX_CHECK_ARG(eps >= 0.0f && eps < INFINITY, "eps = %g has to be finite and not negative", eps);
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(x && y, "x and y are required");
  PLX_CHECK_ARG(ldx >= (int64_t)n || rows == 1, "ldx = %lld is less than n", (long long)ldx);
  PLX_CHECK_ARG(ldy >= (int64_t)n || rows == 1, "ldy = %lld is less than n", (long long)ldy);
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      k_norm_fwd<T, P><<<(unsigned)rows, kThreads, 0, ctx->stream>>>(
          n, (const T*)x, ldx, (const P*)weight, (const P*)bias, eps, (T*)y, ldy, mean, rstd);
      PLX_LAUNCH_CHECK("k_norm_fwd");
      return PLX_OK;
    };
    return param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}

extern "C" size_t plx_layer_norm_scratch_bytes(uint64_t rows, uint32_t n) {
  return (size_t)norm_groups(rows) * 2 * n * sizeof(float);
}

extern "C" int plx_layer_norm_backward(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                                       const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                       const float* mean, const float* rstd, int param_dtype,
                                       const void* weight, void* dx, int64_t lddx, void* dweight,
                                       void* dbias, void* scratch, size_t scratch_bytes) {
  if (int rc = check_rows(ctx, rows, n, dtype)) return rc;
  if (int rc = check_param_dtype(param_dtype, dtype)) return rc;
  const bool sums = dweight || dbias;
  PLX_CHECK_ARG(!sums || (scratch && scratch_bytes >= plx_layer_norm_scratch_bytes(rows, n)),
                "the weights' gradients need %zu bytes of scratch, got %zu",
                plx_layer_norm_scratch_bytes(rows, n), scratch ? scratch_bytes : (size_t)0);
  PLX_CHECK_ARG(!sums || (reinterpret_cast<uintptr_t>(scratch) & 15u) == 0,
                "scratch has to be 16-byte aligned");
  if (rows) {
    PLX_CHECK_ARG(dy && x && mean && rstd, "dy, x, mean and rstd are required");
    PLX_CHECK_ARG(rows == 1 || (ldx >= (int64_t)n && lddy >= (int64_t)n && (!dx || lddx >= (int64_t)n)),
                  "a row stride is less than n");
  }
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      if (rows && dx) {
        k_norm_dx<T, P><<<(unsigned)rows, kThreads, 0, ctx->stream>>>(
            n, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, (const P*)weight, (T*)dx, lddx);
        PLX_LAUNCH_CHECK("k_norm_dx");
      }
      if (sums) {
        const uint32_t groups = norm_groups(rows), cols = (n + kThreads - 1) / kThreads;
        k_norm_dw_partial<T><<<dim3(cols, groups), kThreads, 0, ctx->stream>>>(
            rows, n, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, (float*)scratch);
        PLX_LAUNCH_CHECK("k_norm_dw_partial");
        k_norm_dw_join<P><<<cols, kThreads, 0, ctx->stream>>>(groups, n, (const float*)scratch,
                                                            (P*)dweight, (P*)dbias);
        PLX_LAUNCH_CHECK("k_norm_dw_join");
      }
      return PLX_OK;
    };
    return param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}
