// Gradients of layer norm. With h = (x-mu) rstd and g = w dy, per row
//   dx = rstd (g - mean g - h mean(g h)),
// and over all rows dw = sum dy h, db = sum dy.
//
// Bound by memory (x and dy read once, dx written once), so the sums over rows
// are taken in the same pass: a thread owns the same columns of every row its
// block visits and carries their two sums in registers (32 bits), the next
// row's values being loaded while the current one is worked on. Blocks leave
// their sums in scratch and a second kernel adds them in a fixed order: no
// atomics, the same bits on every call.
#include <initializer_list>

#include "norm.cuh"

namespace plx {
namespace {

constexpr uint32_t kSms = 148;                // of a B200; fixes the order of the sums
constexpr uint32_t kMaxGroups = kSms * 4;     // blocks that leave column sums

template <typename T, typename P, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR)
k_norm_bwd(uint32_t rows, uint32_t n, const T* dy, int64_t lddy, const T* x,
           int64_t ldx, const float* __restrict__ mean, const float* __restrict__ rstd,
           const P* __restrict__ w, T* dx, int64_t lddx, float* __restrict__ partial) {
  constexpr int ROWS = TPR == 32 ? 8 : 1;
  __shared__ float red[4 * (TPR / 32)];
  const uint32_t lane = threadIdx.x % TPR;
  const uint32_t step = gridDim.x * ROWS;
  uint32_t r = blockIdx.x * ROWS + threadIdx.x / TPR;
  float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const uint32_t i = (j * TPR + lane) * V;
    Pack<P, V> pw;
    if (w && i < n) pw = load_pack<P, V>(w + i);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      wv[j][e] = w && i < n ? to_f32(pw.v[e]) : 1.0f;
      aw[j][e] = ab[j][e] = 0.0f;
    }
  }
  Pack<T, V> qx[NV], qg[NV];
  float mu = 0.0f, rs = 0.0f;
  auto fetch = [&](uint32_t row) {
    if (row >= rows) return;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t i = (j * TPR + lane) * V;
      if (i < n) {
        qx[j] = load_pack<T, V>(x + row * ldx + i);
        qg[j] = load_pack<T, V>(dy + row * lddy + i);
      }
    }
    mu = mean[row];
    rs = rstd[row];
  };
  fetch(r);
  int turn = 0;
  const float inv_n = 1.0f / (float)n;
  // Rows of a block-wide row end for the whole block at once; those of a warp
  // for the warp (no barrier inside).
  for (; r < rows; r += step) {
    Pack<T, V> cx[NV], cg[NV];
    const float m = mu, s = rs;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      cx[j] = qx[j];
      cg[j] = qg[j];
    }
    fetch(r + step);
    float c[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if ((j * TPR + lane) * V < n)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = to_f32(cg[j].v[e]), h = (to_f32(cx[j].v[e]) - m) * s;
          const float g = d * wv[j][e];
          aw[j][e] = fmaf(d, h, aw[j][e]);
          ab[j][e] += d;
          c[0] += g;
          c[1] = fmaf(g, h, c[1]);
        }
    }
    if (dx) {
      row_sum<TPR>(c, red, turn);
      c[0] *= inv_n;
      c[1] *= inv_n;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const uint32_t i = (j * TPR + lane) * V;
        if (i < n) {
          Pack<T, V> out;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float h = (to_f32(cx[j].v[e]) - m) * s;
            out.v[e] = from_f32<T>(s * fmaf(-h, c[1], fmaf(to_f32(cg[j].v[e]), wv[j][e], -c[0])));
          }
          *reinterpret_cast<Pack<T, V>*>(dx + r * lddx + i) = out;
        }
      }
    }
  }
  if (!partial) return;
  float* out = partial + (uint64_t)blockIdx.x * 2 * n;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t i = (j * TPR + lane) * V;
      if (i < n)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          out[i + e] = aw[j][e];
          out[n + i + e] = ab[j][e];
        }
    }
  } else {  // the eight warps' sums, added in their order
    __shared__ float joined[8][32 * NV * V];
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e)
          joined[threadIdx.x / 32][(j * 32 + lane) * V + e] = half ? ab[j][e] : aw[j][e];
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < n; i += 256) {
        float s = joined[0][i];
#pragma unroll
        for (int k = 1; k < 8; ++k) s += joined[k][i];
        out[half * n + i] = s;
      }
    }
  }
}

// Rows too long for registers: dx in two passes, the second out of L2 ...
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
k_norm_dx_long(uint32_t n, const T* dy, int64_t lddy, const T* x, int64_t ldx,
               const float* __restrict__ mean, const float* __restrict__ rstd,
               const P* __restrict__ w, T* dx, int64_t lddx) {
  __shared__ float red[32];
  const int64_t r = blockIdx.x;
  const T* dyr = dy + r * lddy;
  const T* xr = x + r * ldx;
  const float mu = mean[r], rs = rstd[r];
  float s1 = 0.0f, s2 = 0.0f;
  for (uint32_t i = threadIdx.x; i < n; i += 1024) {
    const float g = to_f32(dyr[i]) * (w ? to_f32(w[i]) : 1.0f);
    s1 += g;
    s2 = fmaf(g, (to_f32(xr[i]) - mu) * rs, s2);
  }
  const float c1 = block_sum<32>(s1, red) / (float)n;
  const float c2 = block_sum<32>(s2, red) / (float)n;
  for (uint32_t i = threadIdx.x; i < n; i += 1024) {
    const float g = to_f32(dyr[i]) * (w ? to_f32(w[i]) : 1.0f);
    const float h = (to_f32(xr[i]) - mu) * rs;
    dx[r * lddx + i] = from_f32<T>(rs * (g - c1 - h * c2));
  }
}

// ... and the column sums over one of gridDim.y runs of rows apart (before dx
// is written, which may be dy).
template <typename T>
__global__ void __launch_bounds__(256)
k_norm_dw_long(uint32_t rows, uint32_t n, const T* __restrict__ dy, int64_t lddy,
               const T* __restrict__ x, int64_t ldx, const float* __restrict__ mean,
               const float* __restrict__ rstd, float* __restrict__ partial) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float sw = 0.0f, sb = 0.0f;
  for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = to_f32(dy[(int64_t)r * lddy + i]);
    sw = fmaf(g, (to_f32(x[(int64_t)r * ldx + i]) - mean[r]) * rstd[r], sw);
    sb += g;
  }
  partial[(uint64_t)blockIdx.y * 2 * n + i] = sw;
  partial[(uint64_t)blockIdx.y * 2 * n + n + i] = sb;
}

// Adds the blocks' column sums: 32 columns a block, its 32 warps take every
// 32nd group each and are joined in order.
template <typename P>
__global__ void __launch_bounds__(1024)
k_norm_join(uint32_t groups, uint32_t n, const float* __restrict__ partial, P* __restrict__ dw,
            P* __restrict__ db) {
  __shared__ float part[32][33];
  const uint32_t col = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t i = (uint64_t)blockIdx.x * 32 + col;  // of the 2 n columns of a group
  float s = 0.0f;
  if (i < 2ull * n)
    for (uint32_t g = warp; g < groups; g += 32) s += partial[(uint64_t)g * 2 * n + i];
  part[warp][col] = s;
  __syncthreads();
  s = warp_sum(part[col][warp]);  // column `warp` of this block
  const uint64_t j = (uint64_t)blockIdx.x * 32 + warp;
  if (col == 0 && j < 2ull * n) {
    if (j < n) {
      if (dw) dw[j] = from_f32<P>(s);
    } else if (db) {
      db[j - n] = from_f32<P>(s);
    }
  }
}

uint32_t most_groups(uint64_t rows) {
  return (uint32_t)std::min<uint64_t>(std::max<uint64_t>(rows, 1), kMaxGroups);
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" size_t plx_layer_norm_scratch_bytes(uint64_t rows, uint32_t n) {
  return (size_t)most_groups(rows) * 2 * n * sizeof(float);
}

extern "C" int plx_layer_norm_backward(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                                       const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                       const float* mean, const float* rstd, int param_dtype,
                                       const void* weight, void* dx, int64_t lddx, void* dweight,
                                       void* dbias, void* scratch, size_t scratch_bytes) {
  if (int rc = check_norm(ctx, rows, n, dtype, param_dtype)) return rc;
  const bool sums = dweight || dbias;
  PLX_CHECK_ARG(!sums || (scratch && scratch_bytes >= plx_layer_norm_scratch_bytes(rows, n)),
                "the weights' gradients need %zu bytes of scratch, got %zu",
                plx_layer_norm_scratch_bytes(rows, n), scratch ? scratch_bytes : (size_t)0);
  PLX_CHECK_ARG(!sums || aligned16(scratch), "scratch has to be 16-byte aligned");
  if (rows) {
    PLX_CHECK_ARG(dy && x && mean && rstd, "dy, x, mean and rstd are required");
    PLX_CHECK_ARG(rows == 1 || (ldx >= (int64_t)n && lddy >= (int64_t)n && (!dx || lddx >= (int64_t)n)),
                  "a row stride is less than n");
  }
  if (!sums && (!rows || !dx)) return PLX_OK;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  if (rows <= 1) ldx = lddy = lddx = 0;
  float* partial = sums ? (float*)scratch : nullptr;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    auto go = [&](auto p) {
      using P = decltype(p);
      uint32_t groups = 0;
      // `each` blocks an SM; a block visits rows of the same remainder.
      auto launch = [&](auto kernel, uint32_t block, uint32_t per_block, uint32_t each) {
        groups = (uint32_t)std::min<uint64_t>((rows + per_block - 1) / per_block, kSms * each);
        if (groups == 0) return;
        kernel<<<groups, block, 0, ctx->stream>>>((uint32_t)rows, n, (const T*)dy, lddy,
                                                  (const T*)x, ldx, mean, rstd, (const P*)weight,
                                                  (T*)dx, lddx, partial);
      };
      auto loops = [&] {
        if (sums && rows) {
          groups = std::min<uint32_t>((uint32_t)rows, 64);
          k_norm_dw_long<T><<<dim3((n + 255) / 256, groups), 256, 0, ctx->stream>>>(
              (uint32_t)rows, n, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, partial);
        }
        if (dx && rows)
          k_norm_dx_long<T, P><<<(unsigned)rows, 1024, 0, ctx->stream>>>(
              n, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, (const P*)weight, (T*)dx, lddx);
      };
      if (whole_pieces(n, sizeof(T), {dy, x, dx, weight}, {lddy, ldx, lddx})) {
        const uint32_t pieces = n / V;
        if (pieces <= 32) launch(k_norm_bwd<T, P, V, 1, 32>, 256, 8, 4);
        else if (pieces <= 64) launch(k_norm_bwd<T, P, V, 2, 32>, 256, 8, 2);
        else if (pieces <= 256) launch(k_norm_bwd<T, P, V, 2, 128>, 128, 1, 4);
        else if (pieces <= 512) launch(k_norm_bwd<T, P, V, 2, 256>, 256, 1, 2);
        else if (pieces <= 1024) launch(k_norm_bwd<T, P, V, 2, 512>, 512, 1, 1);
        else if (pieces <= 2048) launch(k_norm_bwd<T, P, V, 2, 1024>, 1024, 1, 1);
        else loops();
      } else if (n <= 128) launch(k_norm_bwd<T, P, 1, 4, 32>, 256, 8, 4);
      else if (n <= 256) launch(k_norm_bwd<T, P, 1, 8, 32>, 256, 8, 4);
      else if (n <= 1024) launch(k_norm_bwd<T, P, 1, 8, 128>, 128, 1, 4);
      else if (n <= 2048) launch(k_norm_bwd<T, P, 1, 8, 256>, 256, 1, 4);
      else if (n <= 4096) launch(k_norm_bwd<T, P, 1, 8, 512>, 512, 1, 2);
      else if (n <= 8192) launch(k_norm_bwd<T, P, 1, 8, 1024>, 1024, 1, 1);
      else loops();
      PLX_LAUNCH_CHECK("k_norm_bwd");
      if (sums) {
        k_norm_join<P><<<(unsigned)((2ull * n + 31) / 32), 1024, 0, ctx->stream>>>(
            groups, n, partial, (P*)dweight, (P*)dbias);
        PLX_LAUNCH_CHECK("k_norm_join");
      }
      return PLX_OK;
    };
    return param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}
