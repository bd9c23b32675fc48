// A fully connected layer on rows, and its gradients.
//   z = x W^T + b;  y = act(z) + residual
//   dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum over rows of dz
// Products on the tensor cores (product_tensor.cu; the three differ in which of their
// operands' dimensions is contiguous), and one pass that makes dz and the sums of its
// columns. z is kept in 32 bits: its rounding would go into every gradient. dz is
// rounded to 16-bit rows' type, which the products take (two products of parts would
// take the unrounded one, at twice the time): half a step of every dz, besides the half
// step of every stored gradient, relative to the sum of the products' magnitudes. As
// float16 it is a power of two times larger, so that the largest dy is in [2^13, 2^14):
// what a dz below 6e-5 would lose, and one above 65,504 overflow by (slopes reach 1.13),
// stays; what the type cuts off is below 2^-38 of the largest dy. (Looking for the
// largest dy first takes 10 us of 445 forwards and backwards of 8,192 x 4,096 x 2,048.)
// 32-bit values are cut into three bfloat16 values whose sum they are, toward zero, so
// that all have one sign: up to 2^-7 and 2^-15 of the value beside the first. Of the nine
// products of parts six are made; what is left out makes a product up to 2^-21 smaller,
// 4e-8 on average (two more would make that 2^-30, and the tensor cores' work a third
// longer). A part that would be 0 is the first one times 2^-30 or 2^-40, so that an
// infinity beside it stays one (values below 2^-100 have no room for all parts, and below
// 2^-93 an infinity beside them may become NaN).
#include "dense.cuh"

namespace plx {
namespace {

constexpr uint32_t kGroups = 128;  // runs of rows whose column sums are joined

// The three parts of a 32-bit value.
__device__ __forceinline__ void cut(float v, __nv_bfloat16 (&part)[3]) {
  auto top = [](float f) { return __uint_as_float(__float_as_uint(f) & 0xffff0000u); };
  float h = top(v), m, l;
  if (fabsf(v) < INFINITY) {
    const float rest = __fsub_rn(v, h);
    m = top(rest);
    l = __fsub_rn(rest, m);
    if (m == 0.0f) m = h * 0x1p-30f;
    if (l == 0.0f) l = h * 0x1p-40f;
  } else {
    h = v != v ? v : h;
    m = l = copysignf(1.0f, v);
  }
  const float p[3] = {h, m, l};
#pragma unroll
  for (int k = 0; k < 3; ++k) part[k] = __float2bfloat16_rn(p[k]);
}
// Two neighbouring values' parts, to three planes.
__device__ __forceinline__ void put_parts(__nv_bfloat16* to, int64_t plane, float a, float b) {
  __nv_bfloat16 x[3], y[3];
  cut(a, x);
  cut(b, y);
#pragma unroll
  for (int k = 0; k < 3; ++k)
    *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<char*>(to) + k * plane) =
        __halves2bfloat162(x[k], y[k]);
}

// The largest finite |dy| of a block's rows.
template <int V>
__global__ void __launch_bounds__(1024)
k_dense_most(uint32_t rows, uint32_t m, const __half* dy, int64_t lddy, float* __restrict__ most) {
  __shared__ float warps[32];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float v = 0.0f;
  for (uint32_t r = blockIdx.x * 32 + warp; r < rows; r += gridDim.x * 32)
#pragma unroll 4
    for (uint32_t c = lane * V; c < m; c += 32 * V) {
      const Pack<__half, V> q = load_pack<__half, V>(dy + r * lddy + c);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float a = fabsf(to_f32(q.v[e]));
        if (a < INFINITY) v = fmaxf(v, a);
      }
    }
  v = warp_max(v);
  if (lane == 0) warps[warp] = v;
  __syncthreads();
  if (warp == 0) {
    v = warp_max(warps[lane]);
    if (lane == 0) most[blockIdx.x] = v;
  }
}

// What float16 dz are multiplied by, from the blocks' largest |dy| (the same in every
// thread); `factor` is its inverse, for the products' sums.
struct DzScale {
  const float* most;
  uint32_t count;  // 0: no scale
  float* factor;
};
__device__ __forceinline__ float dz_scale(const DzScale& s) {
  float v = 0.0f;
  for (uint32_t i = threadIdx.x & 31; i < s.count; i += 32) v = fmaxf(v, s.most[i]);
  v = warp_max(v);
  // of values from 2^-24 up, all normal in 32 bits: 2^13 over the power of two below
  const uint32_t power = __float_as_uint(v) & 0x7f800000u;
  const float scale = v > 0.0f ? __uint_as_float(((13u + 254u) << 23) - power) : 1.0f;
  if (s.count && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *s.factor = 1.0f / scale;
  return scale;
}

// dz of one of gridDim.y runs of rows and the sums of its columns: a lane V
// columns, a warp every eighth row.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256)
k_dense_dz(uint32_t rows, uint32_t m, uint32_t run, const T* dy, int64_t lddy,
           const float* __restrict__ pre, void* dz, int64_t lddz, int64_t plane,
           float* __restrict__ partial, const __grid_constant__ DzScale dz_scaled) {
  __shared__ float joined[8][32 * V];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr bool kScaled = std::is_same_v<T, __half> && ACT != PLX_ACT_IDENTITY;
  const float scale = kScaled ? dz_scale(dz_scaled) : 1.0f;
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
      float d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        d[e] = to_f32(g.v[e]);
        if (ACT != PLX_ACT_IDENTITY) d[e] *= act_slope<ACT>(z.v[e]);
        sum[e] += d[e];
        out.v[e] = from_f32<T>(kScaled ? d[e] * scale : d[e]);
      }
      if (!dz) continue;
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<Pack<T, V>*>((T*)dz + r * lddz + c) = out;
      } else if constexpr (V > 1) {
#pragma unroll
        for (int e = 0; e < V; e += 2)
          put_parts((__nv_bfloat16*)dz + r * lddz + c + e, plane, d[e], d[e + 1]);
      } else {
        __nv_bfloat16 part[3];
        cut(d[0], part);
#pragma unroll
        for (int k = 0; k < 3; ++k)
          *((__nv_bfloat16*)((char*)dz + k * plane) + r * lddz + c) = part[k];
      }
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

// 32-bit rows as three planes; of two arrays at once.
struct CutRows {
  const float* from;
  int64_t ld;
  uint32_t rows, n;
  __nv_bfloat16* to;
  int64_t ldto, plane;
};
__global__ void __launch_bounds__(256)
k_dense_cut(const __grid_constant__ CutRows first, const __grid_constant__ CutRows second) {
  const CutRows& q = blockIdx.z ? second : first;
  const uint32_t c = (blockIdx.x * 32 + (threadIdx.x & 31)) * 2;
  if (c >= q.n) return;
#pragma unroll 2
  for (uint32_t r = blockIdx.y * 8 + (threadIdx.x >> 5); r < q.rows; r += gridDim.y * 8) {
    const float* at = q.from + r * q.ld + c;
    put_parts(q.to + r * q.ldto + c, q.plane, at[0], c + 1 < q.n ? at[1] : 0.0f);
  }
}

// Few 32-bit rows: R of them against U units a warp, whose lanes share k and add in
// a fixed order. Reading the weights once bounds it; cutting them would read and write
// four times as much. Measured, weights of 4,096 x 4,096 out of memory (10.3 us at the copy
// rate): 1 row 21 us, 4 rows 26, 8 rows 29 (9 rows by planes 64; library 17, 54, 51, 61).
template <typename P, int R, int U, int V>
__global__ void __launch_bounds__(256)
k_dense_few(uint32_t rows, uint32_t n, uint32_t m, const float* __restrict__ x, int64_t ldx,
            const float* __restrict__ w, int64_t ldw, const __grid_constant__ Finish f) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t u0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * U;
  if (u0 >= m) return;
  float acc[R][U];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int u = 0; u < U; ++u) acc[r][u] = 0.0f;
  const float* wu[U];
#pragma unroll
  for (int u = 0; u < U; ++u) wu[u] = w + (int64_t)min(u0 + u, m - 1) * ldw;
#pragma unroll 2
  for (uint32_t k = lane * V; k < n; k += 32 * V) {
    Pack<float, V> wv[U], xv[R];
#pragma unroll
    for (int u = 0; u < U; ++u) wv[u] = load_pack<float, V>(wu[u] + k);
#pragma unroll
    for (int r = 0; r < R; ++r) xv[r] = load_pack<float, V>(x + (r < rows ? r : 0) * ldx + k);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r][u] = fmaf(xv[r].v[e], wv[u].v[e], acc[r][u]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float z = warp_sum(acc[r][u]);
      if (lane || (uint32_t)r >= rows || u0 + u >= m) continue;
      const uint32_t col = u0 + u;
      if (f.bias) z += to_f32(((const P*)f.bias)[col]);
      if (f.pre) f.pre[(uint64_t)r * m + col] = z;
      float y = z;
      switch (f.act) {
        case PLX_ACT_SIGMOID: y = act_value<PLX_ACT_SIGMOID>(z); break;
        case PLX_ACT_TANH: y = act_value<PLX_ACT_TANH>(z); break;
        case PLX_ACT_RELU: y = act_value<PLX_ACT_RELU>(z); break;
        case PLX_ACT_SILU: y = act_value<PLX_ACT_SILU>(z); break;
        case PLX_ACT_GELU: y = act_value<PLX_ACT_GELU>(z); break;
        default: break;
      }
      if (f.residual) y += ((const float*)f.residual)[r * f.ldr + col];
      ((float*)f.y)[r * f.ldy + col] = y;
    }
}
constexpr uint32_t kFew = 8;

int few_rows(plx_ctx* ctx, uint32_t rows, uint32_t n, uint32_t m, const float* x, int64_t ldx,
             const float* w, int64_t ldw, const Finish& f) {
  const bool wide = n % 4 == 0 && (rows == 1 || ldx % 4 == 0) && (m == 1 || ldw % 4 == 0) &&
                    aligned16(x) && aligned16(w);
  auto go = [&](auto r, auto u, auto v) {
    constexpr int R = decltype(r)::value, U = decltype(u)::value, V = decltype(v)::value;
    k_dense_few<float, R, U, V><<<(m + 8 * U - 1) / (8 * U), 256, 0, ctx->stream>>>(
        rows, n, m, x, rows > 1 ? ldx : 0, w, ldw, f);
    PLX_LAUNCH_CHECK("k_dense_few");
    return PLX_OK;
  };
  using std::integral_constant;
  auto width = [&](auto r, auto u) {
    return wide ? go(r, u, integral_constant<int, 4>{}) : go(r, u, integral_constant<int, 1>{});
  };
  if (rows == 1) return width(integral_constant<int, 1>{}, integral_constant<int, 2>{});
  if (rows <= 4) return width(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  return width(integral_constant<int, 8>{}, integral_constant<int, 2>{});
}

// 16-bit rows that the tensor copies take as they are.
bool packed(const void* p, int64_t ld, uint64_t rows, int dtype) {
  return dtype != PLX_F32 && aligned16(p) && (rows <= 1 || ld % 8 == 0);
}
// Bytes of what they are copied or cut to; rows are round_up(n, 8) apart.
uint64_t plane_bytes(uint64_t rows, uint32_t n) { return round_up(rows * round_up(n, 8) * 2, 256); }
uint64_t pack_bytes(uint64_t rows, uint32_t n, int dtype) {
  return plane_bytes(rows, n) * (dtype == PLX_F32 ? 3 : 1);
}

// Makes rows of values an operand; `at` is where a copy goes, and is moved past it.
// Rows to be cut are noted in `cuts`, for cut_rows.
struct Cuts {
  CutRows of[2];
  int count = 0;
};
int operand(plx_ctx* ctx, int dtype, const void* p, int64_t ld, uint64_t rows, uint32_t n,
            bool k_major, char** at, Operand* out, Cuts* cuts) {
  if (rows <= 1) ld = 0;
  if (packed(p, ld, rows, dtype)) {
    *out = {p, rows <= 1 ? (int64_t)round_up(n, 8) : ld, 0, k_major};
    return PLX_OK;
  }
  *out = {*at, (int64_t)round_up(n, 8), (int64_t)plane_bytes(rows, n), k_major};
  if (dtype == PLX_F32) {
    cuts->of[cuts->count++] = {(const float*)p, ld, (uint32_t)rows, n, (__nv_bfloat16*)*at,
                               out->ld, out->plane};
  } else {
    const dim3 grid((n + 255) / 256, (unsigned)std::min<uint64_t>((rows + 7) / 8, 4096));
    k_dense_pack<<<grid, 256, 0, ctx->stream>>>((uint32_t)rows, n, (const uint16_t*)p, ld,
                                                (uint16_t*)*at, out->ld);
    PLX_LAUNCH_CHECK("k_dense_pack");
  }
  *at += pack_bytes(rows, n, dtype);
  return PLX_OK;
}
int cut_rows(plx_ctx* ctx, const Cuts& cuts) {
  if (!cuts.count) return PLX_OK;
  const CutRows &a = cuts.of[0], &b = cuts.of[cuts.count - 1];
  const uint32_t n = std::max(a.n, b.n), rows = std::max(a.rows, b.rows);
  const dim3 grid((n + 63) / 64, std::min<uint32_t>((rows + 15) / 16, 2048), cuts.count);
  k_dense_cut<<<grid, 256, 0, ctx->stream>>>(a, b);
  PLX_LAUNCH_CHECK("k_dense_cut");
  return PLX_OK;
}

int product(plx_ctx* ctx, int dtype, Product p) {
  if (p.rows == 1) p.f.ldy = p.f.ldr = (int64_t)round_up(p.cols, 8);  // strides of one row
  return product_tensor(ctx, dtype, p);
}

// dz, the column sums' groups and, of float16, what its scale is made of, at the head of
// a backward call's scratch.
constexpr uint32_t kMost = 148;  // blocks that look for the largest |dy|, one an SM
struct BackwardScratch {
  uint64_t lddz, dz_bytes, sums_bytes, scale_bytes;
  BackwardScratch(uint64_t rows, uint32_t m, int dtype) {
    lddz = round_up(m, 8);
    dz_bytes = pack_bytes(rows, m, dtype);
    sums_bytes = round_up((uint64_t)kGroups * m * 4, 256);
    scale_bytes = dtype == PLX_F16 ? round_up((kMost + 1) * 4, 256) : 0;
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
    bytes = s.dz_bytes + s.sums_bytes + s.scale_bytes;
  }
  if (dtype == PLX_F32 && !backward && rows <= kFew) return 0;
  if (!aligned || dtype == PLX_F32)
    bytes += pack_bytes(rows, n, dtype) + pack_bytes(m, n, dtype) +
             (backward && dtype != PLX_F32 ? pack_bytes(rows, m, dtype) : 0);
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
  const Finish f = {param_dtype, act, bias, residual, ldr, y, ldy, pre, nullptr};
  if (dtype == PLX_F32 && rows <= kFew)
    return few_rows(ctx, (uint32_t)rows, n, m, (const float*)x, ldx, (const float*)weight, ldw, f);
  Product p = {};
  p.rows = (uint32_t)rows;
  p.cols = m;
  p.depth = n;
  char* at = (char*)scratch;
  Cuts cuts;
  if (int rc = operand(ctx, dtype, x, ldx, rows, n, true, &at, &p.a, &cuts)) return rc;
  if (int rc = operand(ctx, dtype, weight, ldw, m, n, true, &at, &p.b, &cuts)) return rc;
  if (int rc = cut_rows(ctx, cuts)) return rc;
  p.f = f;
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
  DzScale scale = {};
  if (rows && own && dtype == PLX_F16) {
    float* most = (float*)((char*)scratch + s.dz_bytes + s.sums_bytes);
    scale = {most, (uint32_t)std::min<uint64_t>((rows + 31) / 32, kMost), most + kMost};
    const bool wide = m % 8 == 0 && (rows == 1 || lddy % 8 == 0) && aligned16(dy);
    (wide ? k_dense_most<8> : k_dense_most<1>)<<<scale.count, 1024, 0, ctx->stream>>>(
        (uint32_t)rows, m, (const __half*)dy, rows > 1 ? lddy : 0, most);
    PLX_LAUNCH_CHECK("k_dense_most");
  }
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
              own ? dz : nullptr, (int64_t)s.lddz, (int64_t)plane_bytes(rows, m),
              dbias ? partial : nullptr, scale);
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
  char* at = (char*)scratch + s.dz_bytes + s.sums_bytes + s.scale_bytes;
  Operand d = {dz, (int64_t)s.lddz, (int64_t)plane_bytes(rows, m), true};
  if (!own && rows && (dx || dweight)) {
    char* to = dtype == PLX_F32 ? (char*)dz : at;  // parts take dz's place
    Cuts cuts;
    if (int rc = operand(ctx, dtype, dy, lddy, rows, m, true, &to, &d, &cuts)) return rc;
    if (int rc = cut_rows(ctx, cuts)) return rc;
    if (dtype != PLX_F32) at = to;
  }
  Cuts cuts;
  Operand w = {}, xs = {};
  if (dx && rows)
    if (int rc = operand(ctx, dtype, weight, ldw, m, n, false, &at, &w, &cuts)) return rc;
  if (dweight && rows)
    if (int rc = operand(ctx, dtype, x, ldx, rows, n, false, &at, &xs, &cuts)) return rc;
  if (int rc = cut_rows(ctx, cuts)) return rc;
  Product p = {};
  if (dx && rows) {
    p.rows = (uint32_t)rows;
    p.cols = n;
    p.depth = m;
    p.a = d;
    p.b = w;
    p.f = {dtype, PLX_ACT_IDENTITY, nullptr, nullptr, 0, dx, lddx, nullptr, scale.factor};
    if (int rc = product(ctx, dtype, p)) return rc;
  }
  if (dweight && rows == 0) {
    PLX_TRY_CUDA(cudaMemset2DAsync(dweight, (size_t)(m > 1 ? lddw : n) * dtype_bytes(dtype), 0,
                                   (size_t)n * dtype_bytes(dtype), m, ctx->stream));
  } else if (dweight) {
    p.rows = m;
    p.cols = n;
    p.depth = (uint32_t)rows;
    d.k_major = false;
    p.a = d;
    p.b = xs;
    p.f = {dtype, PLX_ACT_IDENTITY, nullptr, nullptr, 0, dweight, lddw, nullptr, scale.factor};
    if (int rc = product(ctx, dtype, p)) return rc;
  }
  return PLX_OK;
}
