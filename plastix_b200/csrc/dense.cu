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

uint64_t round_up(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

// Rows of 16-bit values that the tensor copies do not take (their start or stride
// is no multiple of 16 bytes) are copied to some that they do.
__global__ void __launch_bounds__(256)
k_dense_pack(uint32_t rows, uint32_t n, const uint16_t* __restrict__ from, int64_t ld,
             uint16_t* __restrict__ to, int64_t ldto) {
  const uint32_t c = (blockIdx.x * 32 + (threadIdx.x & 31)) * 8;
  if (c >= n) return;
  for (uint32_t r = blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8) {
    const uint16_t* at = from + r * ld + c;
    uint16_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < n ? at[e] : 0;
    *reinterpret_cast<uint4*>(to + r * ldto + c) = *reinterpret_cast<const uint4*>(v);
  }
}

bool packed(const void* p, int64_t ld, uint64_t rows, int dtype) {
  return dtype == PLX_F32 || (aligned16(p) && (rows <= 1 || ld % 8 == 0));
}
// Bytes of a packed copy, whose rows are round_up(n, 8) apart.
uint64_t pack_bytes(uint64_t rows, uint32_t n) { return round_up(rows * round_up(n, 8) * 2, 256); }

// Makes rows of values an operand; `at` is where a copy goes, and is moved past it.
int operand(plx_ctx* ctx, int dtype, const void* p, int64_t ld, uint64_t rows, uint32_t n,
            bool k_major, char** at, Operand* out) {
  *out = {p, ld, k_major};
  if (dtype == PLX_F32) return PLX_OK;
  if (packed(p, ld, rows, dtype)) {
    if (rows <= 1) out->ld = (int64_t)round_up(n, 8);
    return PLX_OK;
  }
  out->p = *at;
  out->ld = (int64_t)round_up(n, 8);
  const dim3 grid((n + 255) / 256, (unsigned)std::min<uint64_t>((rows + 7) / 8, 4096));
  k_dense_pack<<<grid, 256, 0, ctx->stream>>>((uint32_t)rows, n, (const uint16_t*)p, ld,
                                              (uint16_t*)*at, out->ld);
  PLX_LAUNCH_CHECK("k_dense_pack");
  *at += pack_bytes(rows, n);
  return PLX_OK;
}

int product(plx_ctx* ctx, int dtype, Product p) {
  if (p.rows == 1) p.f.ldy = p.f.ldr = (int64_t)round_up(p.cols, 8);  // strides of one row
  return dtype == PLX_F32 ? product_f32(ctx, dtype, p) : product_tensor(ctx, dtype, p);
}

// dz and the column sums' groups, at the head of a backward call's scratch.
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
                                          int backward, int aligned) {
  if (!valid_dtype(dtype) || n == 0 || m == 0) return 0;
  uint64_t bytes = 0;
  if (backward) {
    const BackwardScratch s(rows, m, dtype);
    bytes = s.dz_bytes + s.sums_bytes;
  }
  if (!aligned && dtype != PLX_F32)
    bytes += pack_bytes(rows, n) + pack_bytes(m, n) + (backward ? pack_bytes(rows, m) : 0);
  return bytes;
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
  const size_t need =
      plx_dense_scratch_bytes(rows, n, m, dtype, 0,
                              packed(x, ldx, rows, dtype) && packed(weight, ldw, m, dtype));
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
  char* at = (char*)scratch;
  if (int rc = operand(ctx, dtype, x, ldx, rows, n, true, &at, &p.a)) return rc;
  if (int rc = operand(ctx, dtype, weight, ldw, m, n, true, &at, &p.b)) return rc;
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
  const bool own = act != PLX_ACT_IDENTITY && (dx || dweight);  // dz is not dy
  const size_t need = plx_dense_scratch_bytes(
      rows, n, m, dtype, 1,
      (!dweight || packed(x, ldx, rows, dtype)) && (!dx || packed(weight, ldw, m, dtype)) &&
          (own || !(dx || dweight) || packed(dy, lddy, rows, dtype)));
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
  char* at = (char*)scratch + s.dz_bytes + s.sums_bytes;
  Operand d = {dz, (int64_t)s.lddz, true};
  if (!own && rows && (dx || dweight))
    if (int rc = operand(ctx, dtype, dy, lddy, rows, m, true, &at, &d)) return rc;
  if (dx && rows) {
    Product p = {};
    p.rows = (uint32_t)rows;
    p.cols = n;
    p.depth = m;
    p.a = d;
    if (int rc = operand(ctx, dtype, weight, ldw, m, n, false, &at, &p.b)) return rc;
    p.f = {dtype, PLX_ACT_IDENTITY, nullptr, nullptr, 0, dx, lddx, nullptr};
    if (int rc = product(ctx, dtype, p)) return rc;
  }
  if (dweight && rows == 0) {
    PLX_TRY_CUDA(cudaMemset2DAsync(dweight, (size_t)(m > 1 ? lddw : n) * dtype_bytes(dtype), 0,
                                   (size_t)n * dtype_bytes(dtype), m, ctx->stream));
  } else if (dweight) {
    Product p = {};
    p.rows = m;
    p.cols = n;
    p.depth = (uint32_t)rows;
    d.k_major = false;
    p.a = d;
    if (int rc = operand(ctx, dtype, x, ldx, rows, n, false, &at, &p.b)) return rc;
    p.f = {dtype, PLX_ACT_IDENTITY, nullptr, nullptr, 0, dweight, lddw, nullptr};
    if (int rc = product(ctx, dtype, p)) return rc;
  }
  return PLX_OK;
}
