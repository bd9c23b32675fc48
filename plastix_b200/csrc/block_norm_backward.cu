// Gradients of the norms around a block. With h1 = N(o), h2 = N(r), and where dr
// and du are given for r and u:
//   e = w2 du;  d = dr + rstd2 (e - [mean e] - h2 mean(e h2));  dx = scale d
//   dp = gate d;  f = w1 dp;  do = rstd1 (f - [mean f] - h1 mean(f h1))
//   dgate = d p (of every value, or summed over the rows)
//   dw2 = sum du h2, db2 = sum du, dw1 = sum dp h1, db1 = sum dp
// ([]: where the mean was taken away). p, r, h1 and h2 are made anew from x, o,
// the gate and the rows' statistics: as many bytes as reading r, without its
// rounding.
//
// Bound by memory: x, o, dr, du (and a gate of every value) read once, dx and do
// written once. The sums over rows are taken in the same pass: a thread owns the
// same columns of every row its block visits and carries their sums in registers
// (32 bits); blocks leave them in scratch and a second kernel adds them in a fixed
// order.
#include "block_norm.cuh"

namespace plx {
namespace {

constexpr int kSums = 5;  // dw2, db2, dw1, db1, dgate of units
constexpr uint32_t kMostGroups = 148 * 4;
constexpr uint32_t kLongGroups = 64;

struct SumsOut {
  void* out[kSums];
};

template <typename T, typename P, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR)
k_block_norm_bwd(const __grid_constant__ BlockNorm a) {
  constexpr int ROWS = TPR == 32 ? 8 : 1, E = NV * V, STEP = TPR * V;
  __shared__ float red[4 * (TPR / 32)];
  const uint32_t lane = threadIdx.x % TPR, c0 = lane * V;
  const int left = (int)a.n - (int)c0;
  float sums[kSums][E];
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) sums[k][e] = 0.0f;
  int turn = 0;
  for (uint32_t r = blockIdx.x * ROWS + threadIdx.x / TPR; r < a.rows; r += gridDim.x * ROWS) {
    Pack<T, V> qx[NV], qo[NV], qg[NV], qdr[NV], qdu[NV];
    load_row<STEP>((const T*)a.o + (int64_t)r * a.ldo + c0, left, qo);
    load_row<STEP>((const T*)a.x + (int64_t)r * a.ldx + c0, left, qx);
    if (a.du) load_row<STEP>((const T*)a.du + (int64_t)r * a.lddu + c0, left, qdu);
    if (a.dr) load_row<STEP>((const T*)a.dr + (int64_t)r * a.lddr + c0, left, qdr);
    if (a.gate == PLX_BLOCK_GATE_VALUES)
      load_row<STEP>((const T*)a.gate_values + (int64_t)r * a.ldg + c0, left, qg);
    const float4 st = a.stats[r];
    float h1[E], p[E], gate[E], slope[E], h2[E], d[E];
    float c[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = j * STEP < left;
      const uint32_t i = c0 + j * STEP;
      Pack<P, V> w1, b1, w2, pg;
      if (in && a.post_weight) w1 = load_pack<P, V>((const P*)a.post_weight + i);
      if (in && a.post_bias) b1 = load_pack<P, V>((const P*)a.post_bias + i);
      if (in && a.pre_weight) w2 = load_pack<P, V>((const P*)a.pre_weight + i);
      if (in && a.gate == PLX_BLOCK_GATE_UNITS)
        pg = load_pack<P, V>((const P*)a.gate_values + i);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int e = j * V + k;
        const float o = to_f32(qo[j].v[k]);
        h1[e] = a.post && in ? (o - st.x) * st.y : o;
        p[e] = h1[e];
        if (in && a.post_weight) p[e] *= to_f32(w1.v[k]);
        if (in && a.post_bias) p[e] += to_f32(b1.v[k]);
        gate[e] = slope[e] = 1.0f;
        if (in && a.gate != PLX_BLOCK_GATE_NONE) {
          gate[e] = a.gate == PLX_BLOCK_GATE_UNITS ? to_f32(pg.v[k]) : to_f32(qg[j].v[k]);
          if (a.sigmoid) {
            const Sigmoid s = sigmoid(gate[e]);
            gate[e] = s.a;
            slope[e] = s.a * s.keep;
          }
        }
        const float rv = fmaf(gate[e], p[e], a.scale * to_f32(qx[j].v[k]));
        h2[e] = in ? (rv - st.z) * st.w : 0.0f;
        d[e] = 0.0f;
        if (a.du) {
          const float du = to_f32(qdu[j].v[k]);
          sums[0][e] = fmaf(du, h2[e], sums[0][e]);
          sums[1][e] += du;
          d[e] = du;
          if (in && a.pre_weight) d[e] *= to_f32(w2.v[k]);
          c[0] += d[e];
          c[1] = fmaf(d[e], h2[e], c[1]);
        }
      }
    }
    if (a.du) {
      row_sum<TPR>(c, red, turn);
      const float e0 = a.layer ? c[0] * a.inv_n : 0.0f, e1 = c[1] * a.inv_n;
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = st.w * (d[e] - e0 - h2[e] * e1);
    }
    c[0] = c[1] = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = j * STEP < left;
      const uint32_t i = c0 + j * STEP;
      Pack<P, V> w1;
      if (in && a.post_weight) w1 = load_pack<P, V>((const P*)a.post_weight + i);
      Pack<T, V> ox, og;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int e = j * V + k;
        if (a.dr) d[e] += to_f32(qdr[j].v[k]);
        if (!in) d[e] = 0.0f;
        ox.v[k] = from_f32<T>(a.scale * d[e]);
        const float dg = d[e] * p[e] * slope[e];
        og.v[k] = from_f32<T>(dg);
        sums[4][e] += dg;
        float dp = d[e] * gate[e];
        sums[2][e] = fmaf(dp, h1[e], sums[2][e]);
        sums[3][e] += dp;
        if (in && a.post_weight) dp *= to_f32(w1.v[k]);
        d[e] = dp;
        c[0] += dp;
        c[1] = fmaf(dp, h1[e], c[1]);
      }
      if (!in) continue;
      *reinterpret_cast<Pack<T, V>*>((T*)a.dx + (int64_t)r * a.lddx + i) = ox;
      if (a.gate == PLX_BLOCK_GATE_VALUES && a.dgate)
        *reinterpret_cast<Pack<T, V>*>((T*)a.dgate + (int64_t)r * a.lddg + i) = og;
    }
    if (a.post) {
      row_sum<TPR>(c, red, turn);
      const float e0 = a.layer ? c[0] * a.inv_n : 0.0f, e1 = c[1] * a.inv_n;
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = st.y * (d[e] - e0 - h1[e] * e1);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * STEP >= left) continue;
      Pack<T, V> out;
#pragma unroll
      for (int k = 0; k < V; ++k) out.v[k] = from_f32<T>(d[j * V + k]);
      *reinterpret_cast<Pack<T, V>*>((T*)a.d_o + (int64_t)r * a.lddo + c0 + j * STEP) = out;
    }
  }
  if (!a.partial) return;
  float* out = a.partial + (uint64_t)blockIdx.x * kSums * a.n;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * STEP < left)
#pragma unroll
          for (int e = 0; e < V; ++e) out[(uint64_t)k * a.n + c0 + j * STEP + e] = sums[k][j * V + e];
  } else {  // the eight warps' sums, added in their order
    __shared__ float joined[8][32 * E];
    for (int k = 0; k < kSums; ++k) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float s = 0.0f;
#pragma unroll
          for (int q = 0; q < kSums; ++q) s = q == k ? sums[q][j * V + e] : s;
          joined[threadIdx.x / 32][(j * 32 + lane) * V + e] = s;
        }
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < a.n; i += 256) {
        float s = joined[0][i];
#pragma unroll
        for (int w = 1; w < 8; ++w) s += joined[w][i];
        out[(uint64_t)k * a.n + i] = s;
      }
    }
  }
}

// Rows too long for registers, in three passes over values made anew: the means
// of every row,
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
k_block_norm_means(const __grid_constant__ BlockNorm a, float4* __restrict__ means) {
  __shared__ float red[32];
  RowOf<T, P> row(a, blockIdx.x);
  const float4 st = a.stats[row.row];
  row.m1 = st.x, row.s1 = st.y, row.m2 = st.z, row.s2 = st.w;
  auto e_at = [&](uint32_t i) {
    const float du = to_f32(((const T*)a.du)[row.row * a.lddu + i]);
    return a.pre_weight ? du * to_f32(((const P*)a.pre_weight)[i]) : du;
  };
  float e0 = 0.0f, e1 = 0.0f, f0 = 0.0f, f1 = 0.0f;
  if (a.du) {
    for (uint32_t i = threadIdx.x; i < a.n; i += 1024) {
      const float e = e_at(i);
      e0 += e;
      e1 = fmaf(e, (row.r(i) - st.z) * st.w, e1);
    }
    e0 = block_sum<32>(e0, red) * a.inv_n;
    e1 = block_sum<32>(e1, red) * a.inv_n;
    if (!a.layer) e0 = 0.0f;
  }
  if (a.post) {
    for (uint32_t i = threadIdx.x; i < a.n; i += 1024) {
      float slope, d = 0.0f;
      if (a.du) d = st.w * (e_at(i) - e0 - (row.r(i) - st.z) * st.w * e1);
      if (a.dr) d += to_f32(((const T*)a.dr)[row.row * a.lddr + i]);
      float f = d * row.gate(i, slope);
      if (a.post_weight) f *= to_f32(((const P*)a.post_weight)[i]);
      f0 += f;
      f1 = fmaf(f, row.h1(i), f1);
    }
    f0 = block_sum<32>(f0, red) * a.inv_n;
    f1 = block_sum<32>(f1, red) * a.inv_n;
    if (!a.layer) f0 = 0.0f;
  }
  if (threadIdx.x == 0) means[row.row] = make_float4(e0, e1, f0, f1);
}

// a column's sums over one of gridDim.y runs of rows (before dx and do, which may
// be inputs, are written: `write` is false), and those.
template <typename T, typename P>
__global__ void __launch_bounds__(256)
k_block_norm_columns(const __grid_constant__ BlockNorm a, const float4* __restrict__ means,
                     bool write) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.n) return;
  float sums[kSums] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    RowOf<T, P> row(a, r);
    const float4 st = a.stats[r], m = means[r];
    row.m1 = st.x, row.s1 = st.y, row.m2 = st.z, row.s2 = st.w;
    const float h2 = (row.r(i) - st.z) * st.w, h1 = row.h1(i);
    float d = 0.0f, slope;
    if (a.du) {
      const float du = to_f32(((const T*)a.du)[row.row * a.lddu + i]);
      sums[0] = fmaf(du, h2, sums[0]);
      sums[1] += du;
      d = st.w * ((a.pre_weight ? du * to_f32(((const P*)a.pre_weight)[i]) : du) - m.x - h2 * m.y);
    }
    if (a.dr) d += to_f32(((const T*)a.dr)[row.row * a.lddr + i]);
    const float gate = row.gate(i, slope), dg = d * row.p(i) * slope, dp = d * gate;
    sums[2] = fmaf(dp, h1, sums[2]);
    sums[3] += dp;
    sums[4] += dg;
    if (!write) continue;
    float f = dp;
    if (a.post_weight) f *= to_f32(((const P*)a.post_weight)[i]);
    if (a.post) f = st.y * (f - m.z - h1 * m.w);
    ((T*)a.dx)[row.row * a.lddx + i] = from_f32<T>(a.scale * d);
    ((T*)a.d_o)[row.row * a.lddo + i] = from_f32<T>(f);
    if (a.gate == PLX_BLOCK_GATE_VALUES && a.dgate)
      ((T*)a.dgate)[row.row * a.lddg + i] = from_f32<T>(dg);
  }
  if (!write && a.partial)
    for (int k = 0; k < kSums; ++k)
      a.partial[((uint64_t)blockIdx.y * kSums + k) * a.n + i] = sums[k];
}

// Adds the blocks' column sums: 32 columns a block, its 32 warps take every 32nd
// group each and are joined in order.
template <typename P>
__global__ void __launch_bounds__(1024)
k_block_norm_join(uint32_t groups, uint32_t n, const float* __restrict__ partial,
                  const __grid_constant__ SumsOut outs) {
  __shared__ float part[32][33];
  const uint32_t col = threadIdx.x & 31, warp = threadIdx.x >> 5, k = blockIdx.y;
  P* out = (P*)outs.out[k];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the kernel before is done
  if (!out) return;
  const uint32_t i = blockIdx.x * 32 + col;
  float s = 0.0f;
  if (i < n)
#pragma unroll 8
    for (uint32_t g = warp; g < groups; g += 32) s += partial[((uint64_t)g * kSums + k) * n + i];
  part[warp][col] = s;
  __syncthreads();
  s = warp_sum(part[col][warp]);  // column `warp` of this block
  const uint32_t c = blockIdx.x * 32 + warp;
  if (col == 0 && c < n) out[c] = from_f32<P>(s);
}

uint32_t groups_of(uint64_t rows, uint32_t per_block, uint32_t most) {
  const uint64_t by_rows = (rows + per_block - 1) / per_block;
  return (uint32_t)std::min<uint64_t>(
      std::min<uint64_t>(by_rows, std::max<uint64_t>(148, (by_rows + 7) / 8)), most);
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" size_t plx_block_norm_scratch_bytes(uint64_t rows, uint32_t n) {
  // column sums of the groups, and the means of rows that no registers hold
  const uint64_t sums = (uint64_t)std::max(1u, groups_of(rows, 1, kMostGroups)) * kSums * n * 4;
  return (size_t)((sums + 15) / 16 * 16 + rows * 16);
}

extern "C" int plx_block_norm_backward(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                                       const void* dr, int64_t lddr, const void* du, int64_t lddu,
                                       const void* x, int64_t ldx, const void* o, int64_t ldo,
                                       const float* stats, const plx_block_norm_params* params,
                                       void* dx, int64_t lddx, void* d_o, int64_t lddo,
                                       void* dgate, int64_t lddg, void* dpost_weight,
                                       void* dpost_bias, void* dpre_weight, void* dpre_bias,
                                       void* scratch, size_t scratch_bytes) {
  if (int rc = check_block_norm(ctx, rows, n, dtype, params)) return rc;
  const size_t need = plx_block_norm_scratch_bytes(rows, n);
  PLX_CHECK_ARG(scratch && scratch_bytes >= need, "%zu bytes of scratch are needed, got %zu", need,
                scratch ? scratch_bytes : (size_t)0);
  PLX_CHECK_ARG(aligned16(scratch) && aligned16(stats),
                "scratch and stats have to be 16-byte aligned");
  const bool units = params->gate == PLX_BLOCK_GATE_UNITS;
  const bool values = params->gate == PLX_BLOCK_GATE_VALUES;
  if (rows) {
    PLX_CHECK_ARG(x && o && stats && dx && d_o, "x, o, stats, dx and d_o are required");
    PLX_CHECK_ARG(dr || du, "dr or du is required");
    PLX_CHECK_ARG(dx != d_o && (!values || !dgate || (dgate != dx && dgate != d_o)),
                  "two gradients are the same array");
    PLX_CHECK_ARG(rows == 1 || (ldx >= (int64_t)n && ldo >= (int64_t)n && lddx >= (int64_t)n &&
                                lddo >= (int64_t)n && (!dr || lddr >= (int64_t)n) &&
                                (!du || lddu >= (int64_t)n) &&
                                (!values || !dgate || lddg >= (int64_t)n)),
                  "a row stride is less than n");
  }
  if (int rc = check_aligned(dtype_bytes(dtype), {dr, du, x, o, dx, d_o, values ? dgate : nullptr}))
    return rc;
  if (int rc = check_aligned(dtype_bytes(params->param_dtype),
                             {dpost_weight, dpost_bias, dpre_weight, dpre_bias,
                              units ? dgate : nullptr}))
    return rc;
  SumsOut outs = {{dpre_weight, dpre_bias, params->post ? dpost_weight : nullptr,
                   params->post ? dpost_bias : nullptr, units ? dgate : nullptr}};
  bool sums = false;
  for (void* p : outs.out) sums |= p != nullptr;
  if (!rows && !sums) return PLX_OK;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  BlockNorm a = block_norm_of(rows, n, params);
  a.dr = dr;
  a.du = du;
  a.x = x;
  a.o = o;
  a.stats = (const float4*)stats;
  a.dx = dx;
  a.d_o = d_o;
  a.dgate = values ? dgate : nullptr;
  if (rows > 1) {
    a.lddr = dr ? lddr : 0;
    a.lddu = du ? lddu : 0;
    a.ldx = ldx;
    a.ldo = ldo;
    a.lddx = lddx;
    a.lddo = lddo;
    a.lddg = a.dgate ? lddg : 0;
  }
  a.partial = sums ? (float*)scratch : nullptr;
  float4* means = (float4*)((char*)scratch + need - rows * 16);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    auto go = [&](auto p) {
      using P = decltype(p);
      uint32_t groups = 0;
      auto launch = [&](auto kernel, uint32_t per_block, uint32_t each, unsigned block) {
        groups = groups_of(rows, per_block, 148 * each);
        if (groups) kernel<<<groups, block, 0, ctx->stream>>>(a);
      };
      auto loops = [&] {
        if (!rows) return;
        groups = std::min<uint32_t>((uint32_t)rows, kLongGroups);
        k_block_norm_means<T, P><<<(unsigned)rows, 1024, 0, ctx->stream>>>(a, means);
        const dim3 grid((n + 255) / 256, groups);
        if (sums) k_block_norm_columns<T, P><<<grid, 256, 0, ctx->stream>>>(a, means, false);
        k_block_norm_columns<T, P><<<grid, 256, 0, ctx->stream>>>(a, means, true);
      };
      const uint32_t v =
          block_piece<T, P>(a, {dr, du, x, o, dx, d_o, a.dgate},
                            {a.lddr, a.lddu, a.ldx, a.ldo, a.lddx, a.lddo, a.lddg});
      // A row takes the first launch that holds it.
      if (v == V) {
        constexpr int NV = 8 / V;
        if (n <= 256) launch(k_block_norm_bwd<T, P, V, NV, 32>, 8, 2, 256);
        else if (n <= 1024) launch(k_block_norm_bwd<T, P, V, NV, 128>, 1, 4, 128);
        else if (n <= 2048) launch(k_block_norm_bwd<T, P, V, NV, 256>, 1, 2, 256);
        else if (n <= 4096) launch(k_block_norm_bwd<T, P, V, NV, 512>, 1, 1, 512);
        else loops();
      } else if (sizeof(T) == 2 && v >= 2) {
        if (n <= 256) launch(k_block_norm_bwd<T, P, 2, 4, 32>, 8, 2, 256);
        else if (n <= 1024) launch(k_block_norm_bwd<T, P, 2, 4, 128>, 1, 4, 128);
        else if (n <= 2048) launch(k_block_norm_bwd<T, P, 2, 4, 256>, 1, 2, 256);
        else if (n <= 4096) launch(k_block_norm_bwd<T, P, 2, 4, 512>, 1, 1, 512);
        else loops();
      } else {
        if (n <= 256) launch(k_block_norm_bwd<T, P, 1, 8, 32>, 8, 2, 256);
        else if (n <= 1024) launch(k_block_norm_bwd<T, P, 1, 8, 128>, 1, 4, 128);
        else if (n <= 2048) launch(k_block_norm_bwd<T, P, 1, 8, 256>, 1, 2, 256);
        else if (n <= 4096) launch(k_block_norm_bwd<T, P, 1, 8, 512>, 1, 1, 512);
        else loops();
      }
      PLX_LAUNCH_CHECK("k_block_norm_bwd");
      if (sums) {
        // Launched while the sums are still being made; it waits for them itself.
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((n + 31) / 32, kSums);
        cfg.blockDim = dim3(1024);
        cfg.stream = ctx->stream;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = groups ? 1 : 0;
        PLX_TRY_CUDA(cudaLaunchKernelEx(&cfg, k_block_norm_join<P>, groups, n,
                                        (const float*)a.partial, (const SumsOut)outs));
      }
      return PLX_OK;
    };
    return params->param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}
