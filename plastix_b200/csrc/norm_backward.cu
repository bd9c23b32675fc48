// Gradients of layer norm. With h = (x-mu) rstd and g = w dy, per row
//   dx = rstd (g - mean g - h mean(g h)),
// and over all rows dw = sum dy h, db = sum dy.
//
// Bound by memory (x and dy read once, dx written once), so the sums over rows
// are taken in the same pass: a thread owns the same columns of every row its
// block visits and carries their two sums in registers (32 bits), while the
// next rows are on their way into shared memory. Blocks leave
// their sums in scratch and a second kernel adds them in a fixed order: no
// atomics, the same bits on every call. Measured, both kernels: 16,384 rows of
// 4,096 bf16 69 us, 5.8 TB/s; 8,192 rows of 4,096 f32 69 us, 5.8 TB/s; 65,536
// rows of 512 bf16 38 us, 5.3 TB/s. With one row ahead, in registers, the first
// took 119 us; arithmetic on single values 98.
#include <type_traits>

#include "norm.cuh"

namespace plx {
namespace {

constexpr uint32_t kSms = 148;                // of a B200; fixes the order of the sums
constexpr uint32_t kLongest = 16384;          // row of any type that stays in registers
constexpr uint32_t kLongGroups = 64;          // runs of longer rows
// Groups of column sums, at most: as many blocks an SM as the launches below
// take for the rows of this length that have the most, whatever their type and
// alignment (each launch checks that for the longest row it is used for).
constexpr uint32_t max_groups(uint32_t n) {
  return n > kLongest ? kLongGroups : kSms * (n <= 1024 ? 8 : n <= 2048 ? 4 : n <= 5120 ? 2 : 1);
}
// Groups that `rows` rows leave, a block with `per_block` of them at a time and
// `most` blocks: eight rows a block or more, if that leaves a block an SM; what
// a block leaves to be joined costs as much as a few rows.
uint32_t groups_of(uint64_t rows, uint32_t per_block, uint32_t most) {
  const uint64_t by_rows = (rows + per_block - 1) / per_block;
  return (uint32_t)std::min<uint64_t>(
      std::min<uint64_t>(by_rows, std::max<uint64_t>(kSms, (by_rows + 7) / 8)), most);
}

// Rows under way at once, in shared memory: enough of them to keep memory busy
// beside one barrier a row. A thread reads what it copied itself, except where
// the values are too small for that (staged).
template <typename T, int V, int NV, int TPR>
struct Ring {
  static constexpr int piece = V * sizeof(T);
  static constexpr bool staged = piece < 4;
  static constexpr int block = TPR == 32 ? 256 : TPR;
  static constexpr int array_bytes =
      staged ? (TPR * NV * 2 + 31) / 16 * 16 * (block / TPR) : NV * block * piece;
  static constexpr int stage_bytes = 2 * array_bytes;  // x, dy
  static constexpr int stages = stage_bytes <= 17408 ? 4 : 3;
  static constexpr int bytes = stages * stage_bytes;
};

template <typename T, typename P, int V, int NV, int TPR, int EACH>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, EACH)
k_norm_bwd(uint32_t rows, uint32_t n, const T* dy, int64_t lddy, const T* x, int64_t ldx,
           const float* __restrict__ mean, const float* __restrict__ rstd,
           const P* __restrict__ w, T* dx, int64_t lddx, float* __restrict__ partial) {
  using R = Ring<T, V, NV, TPR>;
  constexpr int ROWS = TPR == 32 ? 8 : 1, S = R::stages, BLOCK = R::block;
  extern __shared__ uint4 ring_bytes[];  // [stage][x, dy]
  char* ring = reinterpret_cast<char*>(ring_bytes);
  __shared__ float red[4 * (TPR / 32)], stats[S][BLOCK / 32][2];
  constexpr int E = NV * V, H = E / 2;  // a thread's columns, as H pairs
  static_assert(E % 2 == 0, "columns in pairs");
  const uint32_t lane = threadIdx.x % TPR, warp = threadIdx.x / 32, wl = threadIdx.x & 31;
  const uint32_t step = gridDim.x * ROWS;
  // A column j pieces on from this thread's first one is within the row where
  // j * STEP < left.
  constexpr int STEP = TPR * V;
  const int left = (int)n - (int)(lane * V);
  uint32_t r = blockIdx.x * ROWS + threadIdx.x / TPR;
  auto slot = [&](uint32_t stage, int array, int j) {  // a piece of this thread's
    char* at = ring + stage * R::stage_bytes + array * R::array_bytes;
    return reinterpret_cast<Pack<T, V>*>(at) + j * BLOCK + threadIdx.x;
  };
  auto staged_row = [&](uint32_t stage, int array) {  // or the row that it shares
    return ring + stage * R::stage_bytes + array * R::array_bytes +
           threadIdx.x / TPR * (R::array_bytes / ROWS);
  };
  auto rows_barrier = [] {
    if (TPR == 32) __syncwarp();
    else __syncthreads();
  };
  // Columns past the row's end: weight and values are 0 and stay so.
  Pack<T, V> qx[NV], qg[NV];
  F2 wv[H], aw[H], ab[H];
  {
    float f[E];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t i = (j * TPR + lane) * V;
      Pack<P, V> pw;
      if (w && i < n) pw = load_pack<P, V>(w + i);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[j * V + e] = i >= n ? 0.0f : w ? to_f32(pw.v[e]) : 1.0f;
        qx[j].v[e] = qg[j].v[e] = from_f32<T>(0.0f);
      }
      if (!R::staged && i >= n)
        for (int s = 0; s < S; ++s) *slot(s, 0, j) = *slot(s, 1, j) = qx[j];
    }
#pragma unroll
    for (int h = 0; h < H; ++h) {
      wv[h] = pack2(f[2 * h], f[2 * h + 1]);
      aw[h] = ab[h] = pack2(0.0f, 0.0f);
    }
  }
  // Starts the copies of a row.
  auto fetch = [&](uint64_t row, uint32_t stage) {
    if (row < rows) {
      if constexpr (R::staged) {
        using St = Staged<T, TPR, NV>;
        St::fetch(staged_row(stage, 0), x, ldx, rows, n, (uint32_t)row, lane);
        St::fetch(staged_row(stage, 1), dy, lddy, rows, n, (uint32_t)row, lane);
      } else {
        const T *xr = x + row * ldx, *gr = dy + row * lddy;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (j * STEP >= left) continue;
          copy_async<R::piece>(slot(stage, 0, j), xr + lane * V + j * STEP);
          copy_async<R::piece>(slot(stage, 1, j), gr + lane * V + j * STEP);
        }
      }
      if (wl < 2) copy_async<4>(&stats[stage][warp][wl], (wl ? rstd : mean) + row);
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(r + (uint64_t)s * step, s);
  int turn = 0;
  uint32_t stage = 0;
  const float inv_n = 1.0f / (float)n;
  // Rows of a block-wide row end for the whole block at once; those of a warp
  // for the warp (no barrier inside).
  for (; r < rows; r += step) {
    float fx[E], fg[E];
    copy_wait<S - 2>();
    // Staged rows are everybody's, the statistics two lanes' of every warp; and
    // what is written next has been read by all.
    if (R::staged) rows_barrier();
    else __syncwarp();
    fetch(r + (uint64_t)(S - 1) * step, stage == 0 ? S - 1 : stage - 1);
    if constexpr (R::staged) {
      Staged<T, TPR, NV>::read(staged_row(stage, 0), x + (int64_t)r * ldx, n, lane, qx);
      Staged<T, TPR, NV>::read(staged_row(stage, 1), dy + (int64_t)r * lddy, n, lane, qg);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        qx[j] = *slot(stage, 0, j);
        qg[j] = *slot(stage, 1, j);
      }
    }
    const float m = stats[stage][warp][0], s = stats[stage][warp][1];
    stage = stage == S - 1 ? 0 : stage + 1;
    widen<NV, V>(qx, fx);
    widen<NV, V>(qg, fg);
    // With d = dy, t = d (x - mu): g = w d, g h = rstd w t, dy h = rstd t.
    F2 xm[H], c0 = pack2(0.0f, 0.0f), c1 = c0;
    const F2 minus = pack2(-m, -m), s2 = pack2(s, s);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const F2 d = pack2(fg[2 * h], fg[2 * h + 1]);
      xm[h] = add2(pack2(fx[2 * h], fx[2 * h + 1]), minus);
      const F2 t = mul2(d, xm[h]);
      aw[h] = fma2(t, s2, aw[h]);
      ab[h] = add2(d, ab[h]);
      c0 = fma2(d, wv[h], c0);
      c1 = fma2(t, wv[h], c1);
    }
    if (dx) {
      const F2 c = row_sum2<TPR>(pack2(c0.x + c0.y, c1.x + c1.y), red, turn);
      // dx = s g + ((x - mu) a + b), a = -s^2 mean(g h), b = -s mean g
      const float a = -s * s * (c.y * s * inv_n), b = -s * (c.x * inv_n);
      const F2 a2 = pack2(a, a), b2 = pack2(b, b);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const F2 g = mul2(pack2(fg[2 * h], fg[2 * h + 1]), wv[h]);
        xm[h] = fma2(g, s2, fma2(xm[h], a2, b2));
      }
      store_row<STEP, NV, V>(dx + r * lddx + lane * V, left, xm);
    }
  }
  if (!partial) return;
  float* out = partial + (uint64_t)blockIdx.x * 2 * n;
  auto column = [&](int half, int e) {
    const F2 v = half ? ab[e / 2] : aw[e / 2];
    return e & 1 ? v.y : v.x;
  };
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint32_t i = (j * TPR + lane) * V;
      if (i >= n) continue;
      if constexpr (V >= 4) {  // n and i are multiples of four
#pragma unroll
        for (int e = 0; e < V; e += 4)
          for (int half = 0; half < 2; ++half)
            *reinterpret_cast<float4*>(out + half * (uint64_t)n + i + e) =
                make_float4(column(half, j * V + e), column(half, j * V + e + 1),
                            column(half, j * V + e + 2), column(half, j * V + e + 3));
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          out[i + e] = column(0, j * V + e);
          out[n + i + e] = column(1, j * V + e);
        }
      }
    }
  } else {  // the eight warps' sums, added in their order
    __shared__ float joined[8][32 * E];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e)
          joined[threadIdx.x / 32][(j * 32 + lane) * V + e] = column(half, j * V + e);
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < n; i += 256) {
        float s = joined[0][i];
#pragma unroll
        for (int k = 1; k < 8; ++k) s += joined[k][i];
        out[half * (uint64_t)n + i] = s;
      }
    }
  }
}

// Rows too long for registers: dx in two passes, the second out of L2 (values
// one by one, for any alignment) ...
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
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the kernel before is done
  if (i < 2ull * n)
#pragma unroll 8
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

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" size_t plx_layer_norm_scratch_bytes(uint64_t rows, uint32_t n) {
  // One row a block: no launch leaves more groups. At least one, of no rows.
  return (size_t)std::max(1u, groups_of(rows, 1, max_groups(n))) * 2 * n * sizeof(float);
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
    PLX_CHECK_ARG(rows == 1 || (ldx >= (int64_t)n && lddy >= (int64_t)n &&
                                (!dx || lddx >= (int64_t)n)),
                  "a row stride is less than n");
  }
  if (int rc = check_aligned(dtype_bytes(dtype), {dy, x, dx})) return rc;
  if (int rc = check_aligned(dtype_bytes(param_dtype), {weight, dweight, dbias})) return rc;
  if (int rc = check_aligned(4, {mean, rstd})) return rc;
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
      // EACH blocks an SM; a block visits rows of the same remainder.
      auto launch = [&](auto nv_c, auto tpr_c, auto each_c, auto v_c) -> int {
        constexpr int NV = decltype(nv_c)::value, TPR = decltype(tpr_c)::value;
        constexpr int EACH = decltype(each_c)::value, VV = decltype(v_c)::value;
        using R = Ring<T, VV, NV, TPR>;
        static_assert(kSms * EACH <= max_groups(NV * TPR * VV), "max_groups");
        constexpr auto kernel = k_norm_bwd<T, P, VV, NV, TPR, EACH>;
        groups = groups_of(rows, TPR == 32 ? 8 : 1, kSms * EACH);
        if (groups == 0) return PLX_OK;
        if (R::bytes > 32 * 1024)
          PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, R::bytes));
        kernel<<<groups, R::block, R::bytes, ctx->stream>>>(
            (uint32_t)rows, n, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, (const P*)weight,
            (T*)dx, lddx, partial);
        return PLX_OK;
      };
      auto loops = [&] {
        if (sums && rows) {
          groups = std::min<uint32_t>((uint32_t)rows, kLongGroups);
          k_norm_dw_long<T><<<dim3((n + 255) / 256, groups), 256, 0, ctx->stream>>>(
              (uint32_t)rows, n, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, partial);
        }
        if (dx && rows)
          k_norm_dx_long<T, P><<<(unsigned)rows, 1024, 0, ctx->stream>>>(
              n, (const T*)dy, lddy, (const T*)x, ldx, mean, rstd, (const P*)weight, (T*)dx, lddx);
      };
      using std::integral_constant;
#define PLX_C(v) integral_constant<int, v>{}
      int rc = PLX_OK;
      const uint32_t v = piece_values(n, sizeof(T), {dy, x, dx}, {lddy, ldx, lddx}, weight,
                                      nullptr, sizeof(P));
      // A row takes the first launch that holds it. The next one in its place takes
      // (134 MB of rows) 1.03 to 4.4 times as long, but for f32 rows of exactly 128
      // or 512 values (0.92, 0.99). EACH is as many blocks as registers and shared
      // memory leave room for: half as many take up to 1.9 times as long for 16-bit
      // rows (8,191 values 143 us and 267; least for 512, 71 and 65), for f32 0.9
      // (1,024 values 70 and 66) to 1.7.
      if (v == V) {
        const uint32_t pieces = n / V;
        if (pieces <= 32) rc = launch(PLX_C(1), PLX_C(32), PLX_C(4), PLX_C(V));
        else if (pieces <= 64) rc = launch(PLX_C(2), PLX_C(32), PLX_C(2), PLX_C(V));
        else if (pieces <= 128) rc = launch(PLX_C(1), PLX_C(128), PLX_C(8), PLX_C(V));
        else if (pieces <= 256) rc = launch(PLX_C(2), PLX_C(128), PLX_C(4), PLX_C(V));
        else if (pieces <= 512) rc = launch(PLX_C(2), PLX_C(256), PLX_C(2), PLX_C(V));
        else if (pieces <= 1024) rc = launch(PLX_C(2), PLX_C(512), PLX_C(1), PLX_C(V));
        else if (pieces <= 2048) rc = launch(PLX_C(2), PLX_C(1024), PLX_C(1), PLX_C(V));
        else loops();
      } else if (sizeof(T) == 2 && v >= 2) {
        const uint32_t pieces = n / 2;
        if (pieces <= 128) rc = launch(PLX_C(4), PLX_C(32), PLX_C(4), PLX_C(2));
        else if (pieces <= 512) rc = launch(PLX_C(4), PLX_C(128), PLX_C(6), PLX_C(2));
        else if (pieces <= 1024) rc = launch(PLX_C(4), PLX_C(256), PLX_C(3), PLX_C(2));
        else if (pieces <= 2048) rc = launch(PLX_C(4), PLX_C(512), PLX_C(2), PLX_C(2));
        else if (pieces <= 4096) rc = launch(PLX_C(4), PLX_C(1024), PLX_C(1), PLX_C(2));
        else loops();
      } else if (n <= 128) rc = launch(PLX_C(4), PLX_C(32), PLX_C(4), PLX_C(1));
      else if (n <= 256) rc = launch(PLX_C(8), PLX_C(32), PLX_C(4), PLX_C(1));
      else if (n <= 1024) rc = launch(PLX_C(8), PLX_C(128), PLX_C(6), PLX_C(1));
      else if (n <= 2048) rc = launch(PLX_C(8), PLX_C(256), PLX_C(3), PLX_C(1));
      else if (n <= 4096) rc = launch(PLX_C(8), PLX_C(512), PLX_C(2), PLX_C(1));
      else if (n <= 5120) rc = launch(PLX_C(10), PLX_C(512), PLX_C(2), PLX_C(1));
      else if (n <= 8192) rc = launch(PLX_C(8), PLX_C(1024), PLX_C(1), PLX_C(1));
      else loops();
#undef PLX_C
      if (rc != PLX_OK) return rc;
      PLX_LAUNCH_CHECK("k_norm_bwd");
      if (sums) {
        // Launched while the sums are still being made; it waits for them itself.
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((2ull * n + 31) / 32));
        cfg.blockDim = dim3(1024);
        cfg.stream = ctx->stream;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = groups ? 1 : 0;
        PLX_TRY_CUDA(cudaLaunchKernelEx(&cfg, k_norm_join<P>, groups, n, (const float*)partial,
                                        (P*)dweight, (P*)dbias));
      }
      return PLX_OK;
    };
    return param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}
