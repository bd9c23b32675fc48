// A fully connected layer on rows, and its gradients.
//   z = x W^T + b;  y = act(z) + residual
//   dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum over rows of dz
// Three products over one kernel each (their operands differ in which of their
// dimensions is contiguous), and one pass that makes dz and the sums of its
// columns. z is kept in 32 bits: its rounding would go into every gradient. dz is
// rounded to the rows' type, which the products take; that is as much as one
// rounding of the gradients themselves.
#include "dense.cuh"

namespace plx {
namespace {

constexpr uint32_t kGroups = 128;  // runs of rows whose column sums are joined

// dz of one of gridDim.y runs of rows and the sums of its columns: a lane V
// columns, a warp every eighth row.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256)
k_dense_dz(uint32_t rows, uint32_t m, uint32_t run, const T* dy, int64_t lddy,
           const float* __restrict__ pre, T* dz, int64_t lddz, float* __restrict__ partial) {
  __shared__ float joined[8][32 * V];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t c = (blockIdx.x * 32 + lane) * V;
  const uint32_t r0 = blockIdx.y * run, r1 = min(r0 + run, rows);
  float sum[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sum[e] = 0.0f;
  if (c < m)
    for (uint32_t r = r0 + warp; r < r1; r += 8) {
      const Pack<T, V> g = load_pack<T, V>(dy + r * lddy + c);
      Pack<float, V> z;
      if (ACT != PLX_ACT_IDENTITY) z = load_pack<float, V>(pre + (uint64_t)r * m + c);
      Pack<T, V> out;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float d = to_f32(g.v[e]);
        if (ACT != PLX_ACT_IDENTITY) d *= act_slope<ACT>(z.v[e]);
        sum[e] += d;
        out.v[e] = from_f32<T>(d);
      }
      if (dz) *reinterpret_cast<Pack<T, V>*>(dz + r * lddz + c) = out;
    }
  if (!partial) return;
#pragma unroll
  for (int e = 0; e < V; ++e) joined[warp][lane * V + e] = sum[e];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < 32 * V; i += 256) {
    float s = joined[0][i];
#pragma unroll
    for (int w = 1; w < 8; ++w) s += joined[w][i];
    if (blockIdx.x * 32 * V + i < m)
      partial[(uint64_t)blockIdx.y * m + blockIdx.x * 32 * V + i] = s;
  }
}

template <typename P>
__global__ void __launch_bounds__(256)
k_dense_db(uint32_t groups, uint32_t m, const float* __restrict__ partial, P* __restrict__ db) {
  __shared__ float part[8][32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < m)
    for (uint32_t g = warp; g < groups; g += 8) s += partial[(uint64_t)g * m + c];
  part[warp][lane] = s;
  __syncthreads();
  if (warp || c >= m) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) s += part[w][lane];
  db[c] = from_f32<P>(s);
}

int check_dense(const plx_ctx* ctx, uint64_t rows, uint32_t n, uint32_t m, int dtype,
                int param_dtype, int act) {
  PLX_CHECK_ARG(ctx, "ctx is required");
  PLX_CHECK_ARG(valid_dtype(dtype), "dtype %d is none of PLX_F32, PLX_BF16, PLX_F16", dtype);
  PLX_CHECK_ARG(n > 0 && n < (1u << 31), "n = %u is out of range", n);
  PLX_CHECK_ARG(m > 0 && m < (1u << 31), "m = %u is out of range", m);
  if (rows >= (1ull << 31))
    return set_error(PLX_ERR_CAPACITY, "%llu rows: fewer than 2^31 are supported",
                     (unsigned long long)rows);
  PLX_CHECK_ARG(param_dtype == PLX_F32 || param_dtype == dtype,
                "param_dtype %d is neither PLX_F32 nor the rows' dtype %d", param_dtype, dtype);
  PLX_CHECK_ARG(act >= PLX_ACT_IDENTITY && act <= PLX_ACT_GELU, "act %d is none of PLX_ACT_*", act);
  return PLX_OK;
}

int product(plx_ctx* ctx, int dtype, const Product& p) { return product_f32(ctx, dtype, p); }

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// dz and the column sums' groups, in scratch.
struct BackwardScratch {
  uint64_t lddz, dz_bytes, sums_bytes;
  BackwardScratch(uint64_t rows, uint32_t m, int dtype) {
    lddz = round_up(m, 8);
    dz_bytes = round_up(rows * lddz * dtype_bytes(dtype), 256);
    sums_bytes = round_up((uint64_t)kGroups * m * 4, 256);
  }
};

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" size_t plx_dense_scratch_bytes(uint64_t rows, uint32_t n, uint32_t m, int dtype,
                                          int backward) {
  (void)n;
  if (!backward || !valid_dtype(dtype)) return 0;
  const BackwardScratch s(rows, m, dtype);
  return s.dz_bytes + s.sums_bytes;
}

extern "C" int plx_dense(plx_ctx* ctx, uint64_t rows, uint32_t n, uint32_t m, int dtype,
                         const void* x, int64_t ldx, const void* weight, int64_t ldw,
                         int param_dtype, const void* bias, int act, const void* residual,
                         int64_t ldr, void* y, int64_t ldy, float* pre, void* scratch,
                         size_t scratch_bytes) {
  if (int rc = check_dense(ctx, rows, n, m, dtype, param_dtype, act)) return rc;
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(x && weight && y, "x, weight and y are required");
  PLX_CHECK_ARG(ldw >= (int64_t)n || m == 1, "ldw = %lld is less than n", (long long)ldw);
  PLX_CHECK_ARG(rows == 1 || (ldx >= (int64_t)n && ldy >= (int64_t)m &&
                              (!residual || ldr >= (int64_t)m)),
                "a row stride is less than the row");
  const size_t need = plx_dense_scratch_bytes(rows, n, m, dtype, 0);
  PLX_CHECK_ARG(need == 0 || (scratch && scratch_bytes >= need),
                "%zu bytes of scratch are needed, got %zu", need,
                scratch ? scratch_bytes : (size_t)0);
  PLX_CHECK_ARG(aligned16(scratch), "scratch has to be 16-byte aligned");
  if (int rc = check_aligned(dtype_bytes(dtype), {x, weight, residual, y})) return rc;
  if (int rc = check_aligned(dtype_bytes(param_dtype), {bias})) return rc;
  if (int rc = check_aligned(4, {pre})) return rc;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  Product p = {};
  p.rows = (uint32_t)rows;
  p.cols = m;
  p.depth = n;
  p.a = {x, ldx, true};
  p.b = {weight, ldw, true};
  p.f = {param_dtype, act, bias, residual, ldr, y, ldy, pre};
  return product(ctx, dtype, p);
}

extern "C" int plx_dense_backward(plx_ctx* ctx, uint64_t rows, uint32_t n, uint32_t m, int dtype,
                                  const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                  const void* weight, int64_t ldw, int act, const float* pre,
                                  void* dx, int64_t lddx, void* dweight, int64_t lddw,
                                  int param_dtype, void* dbias, void* scratch,
                                  size_t scratch_bytes) {
  if (int rc = check_dense(ctx, rows, n, m, dtype, param_dtype, act)) return rc;
  if (rows) {
    PLX_CHECK_ARG(dy, "dy is required");
    PLX_CHECK_ARG(!dx || weight, "dx needs weight");
    PLX_CHECK_ARG(!dweight || x, "dweight needs x");
    PLX_CHECK_ARG(act == PLX_ACT_IDENTITY || pre, "pre is required");
    PLX_CHECK_ARG(rows == 1 || (lddy >= (int64_t)m && (!dweight || ldx >= (int64_t)n) &&
                                (!dx || lddx >= (int64_t)n)),
                  "a row stride is less than the row");
  }
  PLX_CHECK_ARG(m == 1 || ((!dx || ldw >= (int64_t)n) && (!dweight || lddw >= (int64_t)n)),
                "a row stride of weight or dweight is less than n");
  const size_t need = plx_dense_scratch_bytes(rows, n, m, dtype, 1);
  PLX_CHECK_ARG(scratch && scratch_bytes >= need, "%zu bytes of scratch are needed, got %zu", need,
                scratch ? scratch_bytes : (size_t)0);
  PLX_CHECK_ARG(aligned16(scratch), "scratch has to be 16-byte aligned");
  if (int rc = check_aligned(dtype_bytes(dtype), {dy, x, weight, dx, dweight})) return rc;
  if (int rc = check_aligned(dtype_bytes(param_dtype), {dbias})) return rc;
  if (int rc = check_aligned(4, {pre})) return rc;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  const BackwardScratch s(rows, m, dtype);
  void* dz = scratch;
  float* partial = (float*)((char*)scratch + s.dz_bytes);
  const bool own = act != PLX_ACT_IDENTITY && (dx || dweight);  // dz is not dy
  uint32_t groups = 0;
  if (rows && (own || dbias)) {
    const uint32_t run = (uint32_t)std::max<uint64_t>(8, (rows + kGroups - 1) / kGroups);
    groups = (uint32_t)((rows + run - 1) / run);
    int rc = with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      return with_act(act, [&](auto a) {
        constexpr int ACT = decltype(a)::value, W = 16 / sizeof(T);
        auto go = [&](auto v_c) {
          constexpr int V = decltype(v_c)::value;
          k_dense_dz<T, V, ACT><<<dim3((m + 32 * V - 1) / (32 * V), groups), 256, 0, ctx->stream>>>(
              (uint32_t)rows, m, run, (const T*)dy, rows > 1 ? lddy : 0, pre,
              own ? (T*)dz : nullptr, (int64_t)s.lddz, dbias ? partial : nullptr);
        };
        const bool wide = m % W == 0 && (rows == 1 || lddy % W == 0) && aligned16(dy) &&
                          (ACT == PLX_ACT_IDENTITY || aligned16(pre));
        if (wide) go(std::integral_constant<int, W>{});
        else go(std::integral_constant<int, 1>{});
        PLX_LAUNCH_CHECK("k_dense_dz");
        return PLX_OK;
      });
    });
    if (rc != PLX_OK) return rc;
  }
  if (dbias) {
    auto join = [&](auto p) {
      using P = decltype(p);
      k_dense_db<P><<<(m + 31) / 32, 256, 0, ctx->stream>>>(groups, m, partial, (P*)dbias);
      PLX_LAUNCH_CHECK("k_dense_db");
      return PLX_OK;
    };
    if (int rc = param_dtype == PLX_F32 ? join(float{}) : with_dtype(dtype, join)) return rc;
  }
  const void* d = own ? dz : dy;
  const int64_t ldd = own ? (int64_t)s.lddz : lddy;
  if (dx && rows) {
    Product p = {};
    p.rows = (uint32_t)rows;
    p.cols = n;
    p.depth = m;
    p.a = {d, ldd, true};
    p.b = {weight, ldw, false};
    p.f = {dtype, PLX_ACT_IDENTITY, nullptr, nullptr, 0, dx, lddx, nullptr};
    if (int rc = product(ctx, dtype, p)) return rc;
  }
  if (dweight) {
    Product p = {};
    p.rows = m;
    p.cols = n;
    p.depth = (uint32_t)rows;
    p.a = {d, ldd, false};
    p.b = {x, ldx, false};
    p.f = {dtype, PLX_ACT_IDENTITY, nullptr, nullptr, 0, dweight, lddw, nullptr};
    if (int rc = product(ctx, dtype, p)) return rc;
  }
  return PLX_OK;
}
