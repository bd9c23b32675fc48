// Norms around a block of a network: what the block gave is normalised, gated and
// added to the scaled residual, and the sum normalised for the next block.
//   p = N(o) w1 + b1 (or o);   r = scale x + gate p;   u = N(r) w2 + b2
// N: v rstd with rstd = 1/sqrt(mean v^2 + eps), or (v - mean v) rstd with the
// deviations' mean square. Everything between load and store is in 32 bits, and u
// is made of the r that has not been rounded.
//
// Bound by memory: x, o and a gate of every value are read once, r and u written
// once, so a row is held in the registers of the threads that share it (a warp up
// to 512 values, a block above).
#include "block_norm.cuh"

namespace plx {
namespace {

// What is left of a mean in deviations that a mean four times their size was
// taken from is taken away as well (the first mean is off by its sum's roundings).
constexpr float kFar = 4.0f;

template <typename T, typename P, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR)
k_block_norm(const __grid_constant__ BlockNorm a) {
  constexpr int ROWS = TPR == 32 ? 8 : 1, E = NV * V, STEP = TPR * V;
  __shared__ float red[2 * (TPR / 32)];
  const uint32_t lane = threadIdx.x % TPR, c0 = lane * V;
  const uint32_t r = blockIdx.x * ROWS + threadIdx.x / TPR;
  if (ROWS > 1 && r >= a.rows) return;
  const int left = (int)a.n - (int)c0;
  Pack<T, V> qx[NV], qo[NV], qg[NV];
  load_row<STEP>((const T*)a.o + (int64_t)r * a.ldo + c0, left, qo);
  load_row<STEP>((const T*)a.x + (int64_t)r * a.ldx + c0, left, qx);
  if (a.gate == PLX_BLOCK_GATE_VALUES)
    load_row<STEP>((const T*)a.gate_values + (int64_t)r * a.ldg + c0, left, qg);
  int turn = 0;
  // Takes the row's values to h = N(v).
  auto normalise = [&](float (&v)[E], float& mean, float& rstd) {
    float s[1];
    mean = 0.0f;
    auto squares = [&] {
      s[0] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] = fmaf(v[e], v[e], s[0]);
      row_sum<TPR>(s, red, turn);
      return rsqrtf(s[0] * a.inv_n + a.eps);
    };
    auto shift = [&] {
      s[0] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] += v[e];
      row_sum<TPR>(s, red, turn);
      const float m = s[0] * a.inv_n;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e / V * STEP < left) v[e] -= m;
      mean += m;
    };
    if (a.layer) shift();
    rstd = squares();
    if (a.layer && fabsf(mean) * rstd > kFar) {  // so say all threads of the row
      shift();
      rstd = squares();
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= rstd;
  };
  float v[E], m1 = 0.0f, s1 = 0.0f, m2, s2;
  widen<NV, V>(qo, v);
  if (a.post) {
    normalise(v, m1, s1);
    affine<STEP, P, NV, V>(v, (const P*)a.post_weight, (const P*)a.post_bias, c0, left);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j * STEP >= left) continue;
    Pack<P, V> pg;
    if (a.gate == PLX_BLOCK_GATE_UNITS)
      pg = load_pack<P, V>((const P*)a.gate_values + c0 + j * STEP);
    Pack<T, V> out;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float g = 1.0f;
      if (a.gate != PLX_BLOCK_GATE_NONE) {
        g = a.gate == PLX_BLOCK_GATE_UNITS ? to_f32(pg.v[e]) : to_f32(qg[j].v[e]);
        if (a.sigmoid) g = sigmoid(g).a;
      }
      float& w = v[j * V + e];
      w = fmaf(g, w, a.scale * to_f32(qx[j].v[e]));
      out.v[e] = from_f32<T>(w);
    }
    *reinterpret_cast<Pack<T, V>*>((T*)a.r + (int64_t)r * a.ldr + c0 + j * STEP) = out;
  }
  normalise(v, m2, s2);
  affine<STEP, P, NV, V>(v, (const P*)a.pre_weight, (const P*)a.pre_bias, c0, left);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j * STEP >= left) continue;
    Pack<T, V> out;
#pragma unroll
    for (int e = 0; e < V; ++e) out.v[e] = from_f32<T>(v[j * V + e]);
    *reinterpret_cast<Pack<T, V>*>((T*)a.u + (int64_t)r * a.ldu + c0 + j * STEP) = out;
  }
  if (lane == 0 && a.stats_out) a.stats_out[r] = make_float4(m1, s1, m2, s2);
}

// Rows too long for registers: values are made anew from what was read in each
// pass, out of L2 (one at a time, for any alignment).
template <typename T, typename P>
__global__ void __launch_bounds__(1024) k_block_norm_long(const __grid_constant__ BlockNorm a) {
  __shared__ float red[32];
  const int64_t r = blockIdx.x;
  RowOf<T, P> row(a, r);
  auto mean_of = [&](auto value) {
    float s = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.n; i += 1024) s += value(i);
    return block_sum<32>(s, red) * a.inv_n;
  };
  auto stats = [&](auto value, float& mean, float& rstd) {
    mean = 0.0f;
    if (a.layer) {
      mean = mean_of(value);
      mean += mean_of([&](uint32_t i) { return value(i) - mean; });
    }
    rstd = rsqrtf(mean_of([&](uint32_t i) {
                    const float d = value(i) - mean;
                    return d * d;
                  }) + a.eps);
  };
  row.m1 = row.s1 = 0.0f;
  float m1 = 0.0f, s1 = 0.0f;
  if (a.post) stats([&](uint32_t i) { return row.o(i); }, m1, s1);
  row.m1 = m1;
  row.s1 = s1;
  float m2, s2;
  stats([&](uint32_t i) { return row.r(i); }, m2, s2);
  for (uint32_t i = threadIdx.x; i < a.n; i += 1024) {
    const float v = row.r(i);
    ((T*)a.r)[r * a.ldr + i] = from_f32<T>(v);
    ((T*)a.u)[r * a.ldu + i] = from_f32<T>(row.affine((v - m2) * s2, a.pre_weight, a.pre_bias, i));
  }
  if (threadIdx.x == 0 && a.stats_out) a.stats_out[r] = make_float4(m1, s1, m2, s2);
}

}  // namespace

int check_block_norm(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                     const plx_block_norm_params* p) {
  PLX_CHECK_ARG(ctx && p, "ctx and params are required");
  if (int rc = check_norm(ctx, rows, n, dtype, p->param_dtype)) return rc;
  PLX_CHECK_ARG(p->kind == PLX_NORM_RMS || p->kind == PLX_NORM_LAYER,
                "kind %d is neither PLX_NORM_RMS nor PLX_NORM_LAYER", p->kind);
  PLX_CHECK_ARG(p->gate >= PLX_BLOCK_GATE_NONE && p->gate <= PLX_BLOCK_GATE_VALUES,
                "gate %d is none of PLX_BLOCK_GATE_NONE, _UNITS, _VALUES", p->gate);
  PLX_CHECK_ARG(p->scale > -INFINITY && p->scale < INFINITY, "scale = %g has to be finite",
                p->scale);
  PLX_CHECK_ARG(p->eps >= 0.0f && p->eps < INFINITY, "eps = %g has to be finite and not negative",
                p->eps);
  PLX_CHECK_ARG(p->gate == PLX_BLOCK_GATE_NONE || p->gate_values || rows == 0,
                "gate_values is required");
  PLX_CHECK_ARG(p->gate != PLX_BLOCK_GATE_VALUES || rows <= 1 || p->ldg >= (int64_t)n,
                "a row stride is less than n");
  if (int rc = check_aligned(dtype_bytes(p->param_dtype),
                             {p->post_weight, p->post_bias, p->pre_weight, p->pre_bias}))
    return rc;
  return check_aligned(
      p->gate == PLX_BLOCK_GATE_VALUES ? dtype_bytes(dtype) : dtype_bytes(p->param_dtype),
      {p->gate == PLX_BLOCK_GATE_NONE ? nullptr : p->gate_values});
}

BlockNorm block_norm_of(uint64_t rows, uint32_t n, const plx_block_norm_params* p) {
  BlockNorm a = {};
  a.rows = (uint32_t)rows;
  a.n = n;
  a.inv_n = 1.0f / (float)n;
  a.layer = p->kind == PLX_NORM_LAYER;
  a.post = p->post != 0;
  a.gate = p->gate;
  a.sigmoid = p->gate_sigmoid != 0;
  a.param_f32 = p->param_dtype == PLX_F32;
  a.scale = p->scale;
  a.eps = p->eps;
  a.gate_values = p->gate == PLX_BLOCK_GATE_NONE ? nullptr : p->gate_values;
  a.ldg = p->gate == PLX_BLOCK_GATE_VALUES && rows > 1 ? p->ldg : 0;
  a.post_weight = a.post ? p->post_weight : nullptr;
  a.post_bias = a.post ? p->post_bias : nullptr;
  a.pre_weight = p->pre_weight;
  a.pre_bias = p->pre_bias;
  return a;
}

}  // namespace plx

using namespace plx;

extern "C" int plx_block_norm(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, const void* x,
                              int64_t ldx, const void* o, int64_t ldo,
                              const plx_block_norm_params* params, void* r, int64_t ldr, void* u,
                              int64_t ldu, float* stats) {
  if (int rc = check_block_norm(ctx, rows, n, dtype, params)) return rc;
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(x && o && r && u, "x, o, r and u are required");
  PLX_CHECK_ARG(r != u, "r and u are the same array");
  PLX_CHECK_ARG(rows == 1 || (ldx >= (int64_t)n && ldo >= (int64_t)n && ldr >= (int64_t)n &&
                              ldu >= (int64_t)n),
                "a row stride is less than n");
  if (int rc = check_aligned(dtype_bytes(dtype), {x, o, r, u})) return rc;
  PLX_CHECK_ARG(aligned16(stats), "stats has to be 16-byte aligned");
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  BlockNorm a = block_norm_of(rows, n, params);
  a.x = x;
  a.o = o;
  a.r = r;
  a.u = u;
  if (rows > 1) {
    a.ldx = ldx;
    a.ldo = ldo;
    a.ldr = ldr;
    a.ldu = ldu;
  }
  a.stats_out = (float4*)stats;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    auto go = [&](auto p) {
      using P = decltype(p);
      const unsigned one = (unsigned)rows, eighth = (unsigned)((rows + 7) / 8);
      auto launch = [&](auto kernel, unsigned grid, unsigned block) {
        kernel<<<grid, block, 0, ctx->stream>>>(a);
      };
      const uint32_t v = block_piece<T, P>(a, {x, o, r, u}, {a.ldx, a.ldo, a.ldr, a.ldu});
      // A row takes the first launch that holds it.
      if (v == V) {
        constexpr int NV = 16 / V;
        if (n <= 512) launch(k_block_norm<T, P, V, NV, 32>, eighth, 256);
        else if (n <= 2048) launch(k_block_norm<T, P, V, NV, 128>, one, 128);
        else if (n <= 4096) launch(k_block_norm<T, P, V, NV, 256>, one, 256);
        else if (n <= 8192) launch(k_block_norm<T, P, V, NV, 512>, one, 512);
        else if (n <= 16384) launch(k_block_norm<T, P, V, NV, 1024>, one, 1024);
        else launch(k_block_norm_long<T, P>, one, 1024);
      } else if (sizeof(T) == 2 && v >= 2) {
        if (n <= 512) launch(k_block_norm<T, P, 2, 8, 32>, eighth, 256);
        else if (n <= 2048) launch(k_block_norm<T, P, 2, 8, 128>, one, 128);
        else if (n <= 4096) launch(k_block_norm<T, P, 2, 8, 256>, one, 256);
        else if (n <= 8192) launch(k_block_norm<T, P, 2, 8, 512>, one, 512);
        else launch(k_block_norm_long<T, P>, one, 1024);
      } else {
        if (n <= 256) launch(k_block_norm<T, P, 1, 8, 32>, eighth, 256);
        else if (n <= 2048) launch(k_block_norm<T, P, 1, 16, 128>, one, 128);
        else if (n <= 4096) launch(k_block_norm<T, P, 1, 16, 256>, one, 256);
        else if (n <= 8192) launch(k_block_norm<T, P, 1, 16, 512>, one, 512);
        else launch(k_block_norm_long<T, P>, one, 1024);
      }
      PLX_LAUNCH_CHECK("k_block_norm");
      return PLX_OK;
    };
    return params->param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}
