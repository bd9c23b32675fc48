// Layer norm of rows of unit activations.
//   mu = mean x; rstd = 1/sqrt(mean (x-mu)^2 + eps); y = (x-mu) rstd w + b
// Everything between load and store is in 32 bits. The mean is off by its sum's
// roundings, which around a large value are as large as the deviations. In rows
// whose mean is more than four deviations from zero the deviations d from that
// first mean are therefore summed as well, and what they have of a mean is taken
// away: mu = first + mean d, variance = mean d^2 - (mean d)^2. A large common
// offset then costs no accuracy (rows of one value come out below 1e-5); below
// four deviations the first mean is within 5 U of a deviation for each of a
// sum's few dozen steps.
//
// Bound by memory (each value read once, written once): a row is held in
// registers by the threads that share it, a warp for rows of up to 128
// sixteen-byte pieces (no barrier), a block of 128 to 1,024 threads above. Few
// threads with many values each do best, since the two sums' exchanges cost the
// same for every thread (32,768 rows of 4,096 bf16, before the last step: 128
// threads 95 us, 256 107, 512 147), and weights that are read, applied, rounded
// and stored piece by piece (95 to 87 us: fewer registers, more blocks an SM).
// Measured (in brackets: if all rows are far from zero): those rows 89 us, 6.0
// TB/s (93; 90 each if every row summed its deviations); 8,192 rows of 16,384
// bf16 96 us, 5.6 TB/s (103); 65,536 rows of 1,024 bf16 50 us, 5.4 TB/s (52);
// 16,384 rows of 2,049 f32 (one value a load) 50 us, 5.4 TB/s (54); of 4,097 bf16
// (staged) 115 us, 2.3 TB/s (127); 1,024 rows of 65,536 bf16 (too long for
// registers, where all rows sum their deviations) 117 us, 2.3 TB/s.
#include "norm.cuh"

namespace plx {
namespace {

constexpr float kFar = 4.0f;  // deviations between a row's mean and zero

struct RowStats {
  float mean, rstd, shift;  // h = d rstd + shift
};
// From the first mean and the sums of d and d^2. rsqrtf is two units in the last
// place off at most; max_nan: a variance that rounds below 0 is 0, NaN stays.
__device__ __forceinline__ RowStats row_stats(float first, float d, float d2, float inv_n,
                                              float eps) {
  const float e = d * inv_n;
  const float rs = rsqrtf(max_nan(fmaf(-e, e, d2 * inv_n), 0.0f) + eps);
  return {first + e, rs, -e * rs};
}

template <typename T, typename P, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, TPR == 512 && V >= 4 ? 2 : 1)
k_norm(uint32_t rows, uint32_t n, const T* x, int64_t ldx, const P* __restrict__ w,
       const P* __restrict__ b, float eps, float inv_n, T* y, int64_t ldy,
       float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int ROWS = TPR == 32 ? 8 : 1;
  __shared__ float red[2 * (TPR / 32)];
  const uint32_t lane = threadIdx.x % TPR;
  const uint32_t r = blockIdx.x * ROWS + threadIdx.x / TPR;
  if (ROWS > 1 && r >= rows) return;
  const T* xr = x + r * ldx;
  // This thread's first column; the others are constants further on. A column j
  // pieces on is within the row where j * STEP < left.
  constexpr int STEP = TPR * V;
  const int left = (int)n - (int)(lane * V);
  const T* xl = xr + lane * V;
  constexpr int E = NV * V, H = E / 2;  // a thread's columns, as H pairs
  static_assert(E % 2 == 0, "columns in pairs");
  Pack<T, V> q[NV];
  if constexpr (V * sizeof(T) >= 4) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * STEP < left) {
        q[j] = load_pack<T, V>(xl + j * STEP);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) q[j].v[e] = from_f32<T>(0.0f);
      }
    }
  } else {
    using St = Staged<T, TPR, NV>;
    __shared__ uint4 stage[ROWS * St::bytes / 16];
    char* at = reinterpret_cast<char*>(stage) + threadIdx.x / TPR * St::bytes;
    St::fetch(at, x, ldx, rows, n, r, lane);
    copy_commit();
    copy_wait<0>();
    if (TPR == 32) __syncwarp();
    else __syncthreads();
    St::read(at, xr, n, lane, q);
  }
  float f[E];
  widen<NV, V>(q, f);
  F2 v[H], s2 = pack2(0.0f, 0.0f);
#pragma unroll
  for (int h = 0; h < H; ++h) {
    v[h] = pack2(f[2 * h], f[2 * h + 1]);
    s2 = add2(s2, v[h]);
  }
  int turn = 0;
  float s[1] = {s2.x + s2.y};
  row_sum<TPR>(s, red, turn);
  const float mu = s[0] * inv_n;
  const F2 minus = pack2(-mu, -mu);
#pragma unroll
  for (int h = 0; h < H; ++h) v[h] = add2(v[h], minus);
  if (n < (uint32_t)(NV * STEP))  // columns past the row's end have no deviation
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (j * STEP >= left)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int k = j * V + e;
        (k & 1 ? v[k / 2].y : v[k / 2].x) = 0.0f;
      }
  s2 = pack2(0.0f, 0.0f);
#pragma unroll
  for (int h = 0; h < H; ++h) s2 = fma2(v[h], v[h], s2);
  s[0] = s2.x + s2.y;
  row_sum<TPR>(s, red, turn);
  RowStats st = row_stats(mu, 0.0f, s[0], inv_n, eps);
  if (fabsf(mu) * st.rstd > kFar) {  // so say all threads of the row
    s2 = pack2(0.0f, 0.0f);
#pragma unroll
    for (int h = 0; h < H; ++h) s2 = add2(v[h], s2);
    float d[1] = {s2.x + s2.y};
    row_sum<TPR>(d, red, turn);
    st = row_stats(mu, d[0], s[0], inv_n, eps);
  }
  const F2 rs2 = pack2(st.rstd, st.rstd), shift2 = pack2(st.shift, st.shift);
#pragma unroll
  for (int h = 0; h < H; ++h) v[h] = fma2(v[h], rs2, shift2);
  // Weights (out of L1), rounding and storing piece by piece: few of them are
  // live at once.
  T* yl = y + r * ldy + lane * V;
  const P *wl = w + lane * V, *bl = b + lane * V;
  auto finish = [&](auto has_w, auto has_b) {
    constexpr bool W = decltype(has_w)::value, B = decltype(has_b)::value;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * STEP >= left) continue;
      Pack<P, V> pw, pb;
      if (W) pw = load_pack<P, V>(wl + j * STEP);
      if (B) pb = load_pack<P, V>(bl + j * STEP);
      Pack<T, V> out;
      if constexpr (V == 1) {
        const float a = j & 1 ? v[j / 2].y : v[j / 2].x;
        out.v[0] = from_f32<T>(fmaf(a, W ? to_f32(pw.v[0]) : 1.0f, B ? to_f32(pb.v[0]) : 0.0f));
      } else {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const F2 a = v[(j * V + e) / 2];
          put_pair(out, e,
                   W && B ? fma2(a, pair_of(pw, e), pair_of(pb, e))
                   : W    ? mul2(a, pair_of(pw, e))
                   : B    ? add2(a, pair_of(pb, e))
                          : a);
        }
      }
      *reinterpret_cast<Pack<T, V>*>(yl + j * STEP) = out;
    }
  };
  using Yes = std::true_type;
  using No = std::false_type;
  if (w && b) finish(Yes{}, Yes{});
  else if (w) finish(Yes{}, No{});
  else if (b) finish(No{}, Yes{});
  else finish(No{}, No{});
  if (lane == 0) {
    if (mean) mean[r] = st.mean;
    if (rstd) rstd[r] = st.rstd;
  }
}

// Rows too long for registers: three passes, the later two out of L2 (one value
// a thread at a time, for any alignment: rows this long are rare).
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
k_norm_long(uint32_t n, const T* x, int64_t ldx, const P* __restrict__ w,
            const P* __restrict__ b, float eps, float inv_n, T* y, int64_t ldy,
            float* __restrict__ mean, float* __restrict__ rstd) {
  __shared__ float red[32];
  const int64_t r = blockIdx.x;
  const T* xr = x + r * ldx;
  T* yr = y + r * ldy;
  float s = 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += 1024) s += to_f32(xr[i]);
  const float mu = block_sum<32>(s, red) * inv_n;
  s = 0.0f;
  float e = 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += 1024) {
    const float d = to_f32(xr[i]) - mu;
    e += d;
    s = fmaf(d, d, s);
  }
  e = block_sum<32>(e, red);
  const RowStats st = row_stats(mu, e, block_sum<32>(s, red), inv_n, eps);
  for (uint32_t i = threadIdx.x; i < n; i += 1024)
    yr[i] = from_f32<T>(fmaf(fmaf(to_f32(xr[i]) - mu, st.rstd, st.shift), w ? to_f32(w[i]) : 1.0f,
                             b ? to_f32(b[i]) : 0.0f));
  if (threadIdx.x == 0) {
    if (mean) mean[r] = st.mean;
    if (rstd) rstd[r] = st.rstd;
  }
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" int plx_layer_norm(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, const void* x,
                              int64_t ldx, int param_dtype, const void* weight, const void* bias,
                              float eps, void* y, int64_t ldy, float* mean, float* rstd) {
  if (int rc = check_norm(ctx, rows, n, dtype, param_dtype)) return rc;
  PLX_CHECK_ARG(eps >= 0.0f && eps < INFINITY, "eps = %g has to be finite and not negative", eps);
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(x && y, "x and y are required");
  PLX_CHECK_ARG(ldx >= (int64_t)n || rows == 1, "ldx = %lld is less than n", (long long)ldx);
  PLX_CHECK_ARG(ldy >= (int64_t)n || rows == 1, "ldy = %lld is less than n", (long long)ldy);
  if (int rc = check_aligned(dtype_bytes(dtype), {x, y})) return rc;
  if (int rc = check_aligned(dtype_bytes(param_dtype), {weight, bias})) return rc;
  if (int rc = check_aligned(4, {mean, rstd})) return rc;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  if (rows == 1) ldx = ldy = 0;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    auto go = [&](auto p) {
      using P = decltype(p);
      auto launch = [&](auto kernel, unsigned grid, unsigned block) {
        kernel<<<grid, block, 0, ctx->stream>>>((uint32_t)rows, n, (const T*)x, ldx,
                                                (const P*)weight, (const P*)bias, eps,
                                                1.0f / (float)n, (T*)y, ldy, mean, rstd);
      };
      const unsigned one = (unsigned)rows, eighth = (unsigned)((rows + 7) / 8);
      const uint32_t v = piece_values(n, sizeof(T), {x, y}, {ldx, ldy}, weight, bias, sizeof(P));
      auto loops = [&] {
        k_norm_long<T, P><<<one, 1024, 0, ctx->stream>>>(n, (const T*)x, ldx, (const P*)weight,
                                                         (const P*)bias, eps, 1.0f / (float)n,
                                                         (T*)y, ldy, mean, rstd);
      };
      // A row takes the first launch that holds it: fewest threads, fewest values
      // each. The next one in its place takes (134 MB of rows) 1.05 to 2.0 times as
      // long for aligned rows, 1.9 to 3.1 for pairs, and for single values 1.01
      // (2,047 f32, 256 threads of 8: 49 us and 50) to 3.3 (193 bf16, a warp: 105 and
      // 348; 2,559 f32, 256 threads of 10: 46 and 74).
      if (v == V) {
        const uint32_t pieces = n / V;
        if (pieces <= 32) launch(k_norm<T, P, V, 1, 32>, eighth, 256);
        else if (pieces <= 64) launch(k_norm<T, P, V, 2, 32>, eighth, 256);
        else if (pieces <= 128) launch(k_norm<T, P, V, 4, 32>, eighth, 256);
        else if (pieces <= 256) launch(k_norm<T, P, V, 2, 128>, one, 128);
        else if (pieces <= 512) launch(k_norm<T, P, V, 4, 128>, one, 128);
        else if (pieces <= 1024) launch(k_norm<T, P, V, 4, 256>, one, 256);
        else if (pieces <= 2048) launch(k_norm<T, P, V, 4, 512>, one, 512);
        else if (pieces <= 4096) launch(k_norm<T, P, V, 4, 1024>, one, 1024);
        else loops();
      } else if (sizeof(T) == 2 && v >= 2) {
        const uint32_t pieces = n / 2;
        if (pieces <= 256) launch(k_norm<T, P, 2, 8, 32>, eighth, 256);
        else if (pieces <= 1024) launch(k_norm<T, P, 2, 8, 128>, one, 128);
        else if (pieces <= 2048) launch(k_norm<T, P, 2, 8, 256>, one, 256);
        else if (pieces <= 4096) launch(k_norm<T, P, 2, 8, 512>, one, 512);
        else loops();
      } else if (n <= 128) launch(k_norm<T, P, 1, 4, 32>, eighth, 256);
      else if (n <= 256) launch(k_norm<T, P, 1, 8, 32>, eighth, 256);
      else if (n <= 1024) launch(k_norm<T, P, 1, 8, 128>, one, 128);
      else if (n <= 2048) launch(k_norm<T, P, 1, 8, 256>, one, 256);
      else if (n <= 2560) launch(k_norm<T, P, 1, 10, 256>, one, 256);
      else if (n <= 4096) launch(k_norm<T, P, 1, 8, 512>, one, 512);
      else if (n <= 5120) launch(k_norm<T, P, 1, 10, 512>, one, 512);
      else if (n <= 8192) launch(k_norm<T, P, 1, 16, 512>, one, 512);
      else loops();
      PLX_LAUNCH_CHECK("k_norm");
      return PLX_OK;
    };
    return param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}
