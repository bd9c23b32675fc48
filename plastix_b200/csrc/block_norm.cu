// Norms around a block of a network: what the block gave is normalised, gated and
// added to the scaled residual, and the sum normalised for the next block.
//   p = N(o) w1 + b1 (or o);   r = scale x + gate p;   u = N(r) w2 + b2
// N: v rstd with rstd = 1/sqrt(mean v^2 + eps), or (v - mean v) rstd with the
// deviations' mean square. Everything between load and store is in 32 bits, and u
// is made of the r that has not been rounded.
//
// Bound by memory: x, o and a gate of every value are read once, r and u written
// once. A block (or a warp, for rows of up to 512 values) stays and takes every
// gridDim-th row, with the parameters of its threads' sixteen columns in registers
// and the next rows on their way into shared memory. Measured: 16,384 rows of 4,096
// bf16 with a gate of every value 107 us, 6.2 TB/s (141 with a row's loads in its own
// registers and parameters read every row); 3,001 rows of 1,001 f32 (single values)
// 24 us under the profiler.
#include "block_norm.cuh"

namespace plx {
namespace {

// What is left of a mean in deviations that a mean four times their size was
// taken from is taken away as well (the first mean is off by its sum's roundings).
constexpr float kFar = 4.0f;
template <typename T>
constexpr int kStages = sizeof(T) == 4 ? 2 : 4;

template <typename T, int V, int NV, int TPR, bool BIAS, bool VALUES, int EACH>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, EACH)
k_block_norm(const __grid_constant__ BlockNorm a) {
  using C = Columns<T, V, NV, TPR>;
  using R = BlockRing<T, V, NV, TPR, VALUES ? 3 : 2, kStages<T>>;
  constexpr int ROWS = TPR == 32 ? 8 : 1, G = C::G, HV = C::HV, H = C::H, S = R::stages;
  enum { O, X, GATE };
  extern __shared__ uint4 ring_bytes[];
  __shared__ float red[2 * (TPR / 32)];
  const uint32_t lane = threadIdx.x % TPR;
  const C c(a.n, lane * V);
  uint32_t r = blockIdx.x * ROWS + threadIdx.x / TPR;
  const uint32_t step = gridDim.x * ROWS;
  R ring;
  ring.ring = reinterpret_cast<char*>(ring_bytes);
  ring.from[O] = (const T*)a.o + (int64_t)r * a.ldo + c.c0;
  ring.from[X] = (const T*)a.x + (int64_t)r * a.ldx + c.c0;
  ring.step[O] = step * a.ldo;
  ring.step[X] = step * a.ldx;
  if constexpr (VALUES) {
    ring.from[GATE] = (const T*)a.gate_values + (int64_t)r * a.ldg + c.c0;
    ring.step[GATE] = step * a.ldg;
  }
  ring.clear(c);
  const F2 none = pack2(0.0f, 0.0f);
  F2 w1[H], w2[H], gate[VALUES ? 1 : H];
  c.param(a.post_weight, a.param_f32, w1, 1.0f);
  c.param(a.pre_weight, a.param_f32, w2, 1.0f);
  if constexpr (!VALUES) {
    c.param(a.gate == PLX_BLOCK_GATE_UNITS ? a.gate_values : nullptr, a.param_f32, gate, 1.0f);
    if (a.gate == PLX_BLOCK_GATE_UNITS && a.sigmoid)
#pragma unroll
      for (int h = 0; h < H; ++h) gate[h] = pack2(sigmoid(gate[h].x).a, sigmoid(gate[h].y).a);
  }
  T* to_r = (T*)a.r + (int64_t)r * a.ldr + c.c0;
  T* to_u = (T*)a.u + (int64_t)r * a.ldu + c.c0;
  int turn = 0;
  // The row's values less their mean (where that is taken away), and rstd.
  auto normal = [&](F2 (&v)[H], float& mean, float& rstd) {
    float s[1];
    mean = 0.0f;
    auto squares = [&] {
      F2 t = none;
#pragma unroll
      for (int h = 0; h < H; ++h) t = fma2(v[h], v[h], t);
      s[0] = t.x + t.y;
      row_sum<TPR>(s, red, turn);
      return rsqrtf(s[0] * a.inv_n + a.eps);
    };
    auto shift = [&] {
      F2 t = none;
#pragma unroll
      for (int h = 0; h < H; ++h) t = add2(v[h], t);
      s[0] = t.x + t.y;
      row_sum<TPR>(s, red, turn);
      const float m = s[0] * a.inv_n;
      const F2 minus = pack2(-m, -m);
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (c.in(g))
#pragma unroll
          for (int e = 0; e < HV; ++e) {
            F2& w = v[g * HV + e];
            w = add2(w, minus);
            if (V == 1 && !c.both(g)) w.y = 0.0f;
          }
      mean += m;
    };
    if (a.layer) shift();
    rstd = squares();
    if (a.layer && fabsf(mean) * rstd > kFar) {  // so say all threads of the row
      shift();
      rstd = squares();
    }
  };
  uint32_t stage = 0;
  if constexpr (R::used) {
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
      ring.fetch(c, r + (uint64_t)s * step < a.rows, s);
      copy_commit();
    }
  }
  for (; r < a.rows; r += step) {
    if constexpr (R::used) {
      copy_wait<S - 2>();
      ring.fetch(c, r + (uint64_t)(S - 1) * step < a.rows, stage == 0 ? S - 1 : stage - 1);
      copy_commit();
    } else {
      ring.fetch(c, true, 0);
    }
    F2 v[H];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      F2 o[HV];
      ring.get(stage, O, g, o);
#pragma unroll
      for (int e = 0; e < HV; ++e) v[g * HV + e] = o[e];
    }
    float m1 = 0.0f, s1 = 0.0f, m2, s2;
    if (a.post) {
      normal(v, m1, s1);
      const F2 by = pack2(s1, s1);
#pragma unroll
      for (int h = 0; h < H; ++h) v[h] = mul2(mul2(v[h], by), w1[h]);
      if (BIAS && a.post_bias) {
        F2 b[H];
        c.param(a.post_bias, a.param_f32, b, 0.0f);
#pragma unroll
        for (int h = 0; h < H; ++h) v[h] = add2(v[h], b[h]);
      }
    }
    const F2 scale = pack2(a.scale, a.scale);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      F2 x[HV], gv[HV], out[HV];
      ring.get(stage, X, g, x);
      if constexpr (VALUES) {
        ring.get(stage, GATE, g, gv);
        if (a.sigmoid)
#pragma unroll
          for (int e = 0; e < HV; ++e) gv[e] = pack2(sigmoid(gv[e].x).a, sigmoid(gv[e].y).a);
      }
#pragma unroll
      for (int e = 0; e < HV; ++e) {
        F2& w = v[g * HV + e];
        w = fma2(VALUES ? gv[e] : gate[VALUES ? 0 : g * HV + e], w, mul2(scale, x[e]));
        out[e] = w;
      }
      if (c.in(g)) c.put(to_r, g, out);
    }
    normal(v, m2, s2);
    const F2 by = pack2(s2, s2);
#pragma unroll
    for (int h = 0; h < H; ++h) v[h] = mul2(mul2(v[h], by), w2[h]);
    if (BIAS && a.pre_bias) {
      F2 b[H];
      c.param(a.pre_bias, a.param_f32, b, 0.0f);
#pragma unroll
      for (int h = 0; h < H; ++h) v[h] = add2(v[h], b[h]);
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      F2 out[HV];
#pragma unroll
      for (int e = 0; e < HV; ++e) out[e] = v[g * HV + e];
      if (c.in(g)) c.put(to_u, g, out);
    }
    if (lane == 0 && a.stats_out) a.stats_out[r] = make_float4(m1, s1, m2, s2);
    to_r += step * a.ldr;
    to_u += step * a.ldu;
    stage = stage == S - 1 ? 0 : stage + 1;
  }
}

// Rows too long for registers: values are made anew from what was read in each
// pass, out of L2 (one at a time, for any alignment). Measured: 4,096 rows of 12,288 bf16
// 260 us, 418 with means (62 at the copy rate).
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
      int rc = PLX_OK;
      // EACH blocks an SM.
      auto launch = [&](auto v_c, auto nv_c, auto tpr_c, auto each_c) {
        constexpr int VV = decltype(v_c)::value, NV = decltype(nv_c)::value;
        constexpr int TPR = decltype(tpr_c)::value, EACH = decltype(each_c)::value;
        constexpr unsigned per_block = TPR == 32 ? 8 : 1;
        auto with = [&](auto bias_c, auto values_c) -> int {
          constexpr bool VALUES = decltype(values_c)::value;
          using R = BlockRing<T, VV, NV, TPR, VALUES ? 3 : 2, kStages<T>>;
          constexpr auto kernel =
              k_block_norm<T, VV, NV, TPR, decltype(bias_c)::value, VALUES, EACH>;
          if (R::bytes > 32 * 1024) PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, R::bytes));
          const unsigned grid = (unsigned)std::min<uint64_t>((rows + per_block - 1) / per_block,
                                                             (uint64_t)ctx->num_sms * EACH);
          kernel<<<grid, R::threads, R::bytes, ctx->stream>>>(a);
          return PLX_OK;
        };
        using Yes = std::true_type;
        using No = std::false_type;
        const bool values = a.gate == PLX_BLOCK_GATE_VALUES;
        if (a.post_bias || a.pre_bias) rc = values ? with(Yes{}, Yes{}) : with(Yes{}, No{});
        else rc = values ? with(No{}, Yes{}) : with(No{}, No{});
      };
      const uint32_t v = block_piece<T, P>(a, {x, o, r, u}, {a.ldx, a.ldo, a.ldr, a.ldu});
      // A row takes the first launch that holds it.
      using std::integral_constant;
#define PLX_C(v) integral_constant<int, v>{}
      auto ladder = [&](auto vv, auto nv) {
        if (n <= 512) launch(vv, nv, PLX_C(32), PLX_C(2));
        else if (n <= 2048) launch(vv, nv, PLX_C(128), PLX_C(4));
        else if (n <= 4096) launch(vv, nv, PLX_C(256), PLX_C(2));
        else if (n <= 8192) launch(vv, nv, PLX_C(512), PLX_C(1));
        else k_block_norm_long<T, P><<<(unsigned)rows, 1024, 0, ctx->stream>>>(a);
      };
      if (v == V) ladder(PLX_C(V), PLX_C(16 / V));
      else if (sizeof(T) == 2 && v >= 2) ladder(PLX_C(2), PLX_C(8));
      else ladder(PLX_C(1), PLX_C(16));
#undef PLX_C
      if (rc != PLX_OK) return rc;
      PLX_LAUNCH_CHECK("k_block_norm");
      return PLX_OK;
    };
    return params->param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}
