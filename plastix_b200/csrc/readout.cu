// What a row of output units answers, and how it learns from a teacher:
//   log probabilities of given outputs, entropy, best alternatives, their gradient
//   distillation from a teacher's top outputs, loss and gradient
// With M the row's largest logit and d_i = scale (x_i - M):
//   s = sum exp d_i; lse = scale M + log s; logp_i = d_i - log s;
//   entropy = log s - (sum exp(d_i) d_i) / s
// Subtracting M before scaling is exact where it matters (near M), so large
// common offsets cost no accuracy. All sums are in 32 bits.
#include "rows.cuh"

namespace plx {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// A value and its index as one number: larger values first, NaN above all,
// the lower index first among equals (-0 equals 0).
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t i) {
  uint32_t b = __float_as_uint(v + 0.0f);
  b = v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
  return (uint64_t)b << 32 | (0xffffffffu - i);
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = max(v, red[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
k_log_probs(uint32_t n, const T* __restrict__ x, int64_t ld, const int32_t* __restrict__ target,
            float scale, uint32_t top, float* __restrict__ logp, float* __restrict__ lse,
            float* __restrict__ entropy, int32_t* __restrict__ top_ids,
            float* __restrict__ top_logp, int32_t* __restrict__ status) {
  __shared__ float red[kWarps];
  __shared__ uint64_t redk[kWarps];
  const int64_t r = blockIdx.x;
  const T* xr = x + r * ld;
  const float c = scale * kLog2e;
  float m = -INFINITY;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) m = max_nan(m, to_f32(xr[i]));
  m = block_max<kWarps>(m, red);
  const bool none = m == -INFINITY;  // every output masked
  float s = 0.0f, t = 0.0f;
  for (uint32_t i = threadIdx.x; i < n && !none; i += kThreads) {
    const float d = to_f32(xr[i]) - m, e = exp2_approx(d * c);
    s += e;
    if (e > 0.0f) t = fmaf(e, d, t);
  }
  s = block_sum<kWarps>(s, red);
  t = block_sum<kWarps>(t, red);
  const float ls = logf(s);
  if (threadIdx.x == 0) {
    lse[r] = none ? -INFINITY : fmaf(scale, m, ls);
    if (entropy) entropy[r] = none ? 0.0f : ls - scale * (t / s);
    if (logp) {
      const int32_t at = target[r];
      if (at < -1 || at >= (int64_t)n) record_status(status, kStatusBadOutput);
      logp[r] = at < 0 || at >= (int64_t)n ? 0.0f
                : none                     ? -INFINITY
                                           : scale * (to_f32(xr[at]) - m) - ls;
    }
  }
  uint64_t below = ~0ull;
  for (uint32_t k = 0; k < top; ++k) {
    uint64_t best = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t key = rank_key(to_f32(xr[i]), i);
      if (key < below) best = max(best, key);
    }
    below = best = block_max_u64(best, redk);
    if (threadIdx.x == 0) {
      const uint32_t i = 0xffffffffu - (uint32_t)best;
      top_ids[r * top + k] = (int32_t)i;
      top_logp[r * top + k] = none ? -INFINITY : scale * (to_f32(xr[i]) - m) - ls;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
k_log_probs_bwd(uint32_t n, const T* x, int64_t ld, const int32_t* __restrict__ target,
                float scale, const float* __restrict__ lse, const float* __restrict__ entropy,
                const float* __restrict__ grad_logp, const float* __restrict__ grad_entropy,
                T* dx, int64_t ldd) {
  const int64_t r = blockIdx.x;
  const float z = lse[r];
  const int32_t at = target ? target[r] : -1;
  const float g = grad_logp && at >= 0 && at < (int64_t)n ? grad_logp[r] : 0.0f;
  const float gh = grad_entropy ? grad_entropy[r] : 0.0f;
  const float h = grad_entropy ? entropy[r] : 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
    const float v = to_f32(x[r * ld + i]);
    const float l = fmaf(v, scale, -z);
    const float p = z == -INFINITY ? 0.0f : exp2_approx(l * kLog2e);
    float d = p == 0.0f ? 0.0f : -p * fmaf(gh, l + h, g);
    if ((int32_t)i == at) d += g;
    dx[r * ldd + i] = from_f32<T>(d * scale);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
k_distill(uint32_t n, const T* x, int64_t ld, uint32_t k, const int32_t* __restrict__ ids,
          const float* __restrict__ values, int kind, float tau, float inv_tau,
          const float* __restrict__ weight, float* __restrict__ loss, T* dx, int64_t ldd,
          int32_t* __restrict__ status) {
  __shared__ float red[kWarps];
  __shared__ int32_t sid[PLX_DISTILL_MAX_K];
  __shared__ float sq[PLX_DISTILL_MAX_K], slog[PLX_DISTILL_MAX_K], sx[PLX_DISTILL_MAX_K];
  const int64_t r = blockIdx.x;
  const T* xr = x + r * ld;
  T* dr = dx ? dx + r * ldd : nullptr;
  // The teacher's row: one thread an entry.
  const uint32_t j = threadIdx.x;
  int32_t id = j < k ? ids[r * k + j] : -1;
  if (id < -1 || id >= (int64_t)n) {
    record_status(status, kStatusBadOutput);
    id = -1;
  }
  float lq = id < 0 ? -INFINITY : values[r * k + j];
  if (kind == PLX_TEACHER_LOGITS) {
    const float most = block_max<kWarps>(lq, red);
    lq = most == -INFINITY ? -INFINITY : (lq - most) * inv_tau;
    lq -= logf(block_sum<kWarps>(expf(lq), red));
  }
  const float q = id < 0 || lq == -INFINITY ? 0.0f : expf(lq);
  if (j < k) {
    sid[j] = id;
    sq[j] = q;
    slog[j] = lq;
  }
  const float qsum = block_sum<kWarps>(id < 0 ? 0.0f : q, red);
  const float w = weight ? weight[r] : 1.0f;
  if (w == 0.0f || qsum == 0.0f) {  // the row does not count, whatever it holds
    if (threadIdx.x == 0) loss[r] = 0.0f;
    for (uint32_t i = threadIdx.x; i < n && dr; i += kThreads) dr[i] = from_f32<T>(0.0f);
    return;
  }
  const float c = inv_tau * kLog2e;
  float m = -INFINITY;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) m = max_nan(m, to_f32(xr[i]));
  m = block_max<kWarps>(m, red);
  const bool none = m == -INFINITY;
  float s = 0.0f;
  for (uint32_t i = threadIdx.x; i < n && !none; i += kThreads)
    s += exp2_approx((to_f32(xr[i]) - m) * c);
  s = block_sum<kWarps>(s, red);
  float term = 0.0f;
  if (id >= 0) {
    const float d = none ? -INFINITY : (to_f32(xr[id]) - m) * inv_tau - logf(s);
    sx[j] = d;
    if (q != 0.0f) term = q * (lq - d);
  }
  term = block_sum<kWarps>(term, red);
  if (threadIdx.x == 0) loss[r] = w * tau * tau * term;
  if (!dr) return;
  const float a = w * tau, f = none ? 0.0f : a * qsum / s;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads)
    dr[i] = from_f32<T>(none ? 0.0f : f * exp2_approx((to_f32(xr[i]) - m) * c));
  __syncthreads();
  if (id >= 0) {  // an output named twice is written by its first entry
    float both = 0.0f;
    bool first = true;
    for (uint32_t i = 0; i < k; ++i)
      if (sid[i] == id) {
        both += sq[i];
        if (i < j) first = false;
      }
    if (first) dr[id] = from_f32<T>(a * (qsum * expf(sx[j]) - both));
  }
}

int check_logits(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, const void* logits,
                 int64_t ld, float scale, const char* what) {
  PLX_CHECK_ARG(ctx, "ctx is required");
  PLX_CHECK_ARG(valid_dtype(dtype), "dtype %d is none of PLX_F32, PLX_BF16, PLX_F16", dtype);
  PLX_CHECK_ARG(n > 0 && n < (1u << 31), "n = %u is out of range", n);
  if (rows >= (1ull << 31))
    return set_error(PLX_ERR_CAPACITY, "%llu rows: fewer than 2^31 are supported",
                     (unsigned long long)rows);
  PLX_CHECK_ARG(scale > 0.0f && scale < INFINITY, "%s = %g has to be positive and finite", what,
                scale);
  PLX_CHECK_ARG(rows == 0 || logits, "logits is required");
  PLX_CHECK_ARG(rows <= 1 || ld >= (int64_t)n, "the logits' row stride %lld is less than n",
                (long long)ld);
  return PLX_OK;
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" int plx_log_probs(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                             const void* logits, int64_t ld, const int32_t* target, float scale,
                             uint32_t top, float* logp, float* lse, float* entropy,
                             int32_t* top_ids, float* top_logp) {
  if (int rc = check_logits(ctx, rows, n, dtype, logits, ld, scale, "scale")) return rc;
  PLX_CHECK_ARG(top <= n, "top = %u exceeds the %u outputs of a row", top, n);
  if (top > PLX_TOP_MAX)
    return set_error(PLX_ERR_CAPACITY, "top = %u: at most %d are supported", top, PLX_TOP_MAX);
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(lse, "lse is required");
  PLX_CHECK_ARG(!target == !logp, "target and logp go together");
  PLX_CHECK_ARG(!top || (top_ids && top_logp), "top_ids and top_logp are required");
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_log_probs<T><<<(unsigned)rows, kThreads, 0, ctx->stream>>>(
        n, (const T*)logits, ld, target, scale, top, logp, lse, entropy, top_ids, top_logp,
        ctx->d_status);
    PLX_LAUNCH_CHECK("k_log_probs");
    return PLX_OK;
  });
}

extern "C" int plx_log_probs_backward(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                                      const void* logits, int64_t ld, const int32_t* target,
                                      float scale, const float* lse, const float* entropy,
                                      const float* grad_logp, const float* grad_entropy,
                                      void* dlogits, int64_t ldd) {
  if (int rc = check_logits(ctx, rows, n, dtype, logits, ld, scale, "scale")) return rc;
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(grad_logp || grad_entropy, "grad_logp or grad_entropy is required");
  PLX_CHECK_ARG(!grad_logp || target, "grad_logp needs target");
  PLX_CHECK_ARG(!grad_entropy || entropy, "grad_entropy needs entropy");
  PLX_CHECK_ARG(lse && dlogits, "lse and dlogits are required");
  PLX_CHECK_ARG(rows == 1 || ldd >= (int64_t)n, "the gradient's row stride is less than n");
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_log_probs_bwd<T><<<(unsigned)rows, kThreads, 0, ctx->stream>>>(
        n, (const T*)logits, ld, target, scale, lse, entropy, grad_logp, grad_entropy,
        (T*)dlogits, ldd);
    PLX_LAUNCH_CHECK("k_log_probs_bwd");
    return PLX_OK;
  });
}

extern "C" int plx_distill(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, const void* logits,
                           int64_t ld, uint32_t k, const int32_t* teacher_ids,
                           const float* teacher_values, int teacher_kind, float temperature,
                           const float* row_weight, float* loss, void* dlogits, int64_t ldd) {
  if (int rc = check_logits(ctx, rows, n, dtype, logits, ld, temperature, "temperature"))
    return rc;
  PLX_CHECK_ARG(1.0f / temperature < INFINITY, "temperature = %g is too small", temperature);
  PLX_CHECK_ARG(teacher_kind == PLX_TEACHER_LOGITS || teacher_kind == PLX_TEACHER_LOG_PROBS,
                "teacher_kind %d is neither PLX_TEACHER_LOGITS nor PLX_TEACHER_LOG_PROBS",
                teacher_kind);
  PLX_CHECK_ARG(k > 0, "k has to be positive");
  if (k > PLX_DISTILL_MAX_K)
    return set_error(PLX_ERR_CAPACITY, "k = %u: at most %d entries a row are supported", k,
                     PLX_DISTILL_MAX_K);
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(teacher_ids && teacher_values && loss,
                "teacher_ids, teacher_values and loss are required");
  PLX_CHECK_ARG(!dlogits || rows == 1 || ldd >= (int64_t)n,
                "the gradient's row stride is less than n");
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    k_distill<T><<<(unsigned)rows, kThreads, 0, ctx->stream>>>(
        n, (const T*)logits, ld, k, teacher_ids, teacher_values, teacher_kind, temperature,
        1.0f / temperature, row_weight, loss, (T*)dlogits, ldd, ctx->d_status);
    PLX_LAUNCH_CHECK("k_distill");
    return PLX_OK;
  });
}
