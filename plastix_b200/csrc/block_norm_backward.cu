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
// same eight columns of every row its block visits and carries their sums in
// registers (32 bits), while the next rows are on their way into shared memory;
// what a thread needs again after a row's means are known is read there once
// more. Rows of more than 4,096 values are shared by the blocks of a cluster.
// Blocks leave their sums in scratch and a second kernel adds them in a fixed
// order. Measured: forward and backward of 16,384 rows of 4,096 bf16 248 us, 5.4 TB/s
// (1,096 with a row's loads in its own registers, which spilled; 399 with parameters
// read and gates made anew every row: 626 instructions a thread and row, now 380).
#include "block_norm.cuh"
#include "cluster.cuh"

namespace plx {
namespace {

constexpr int kSums = 5;  // dw2, dw1, dgate of units, db2, db1
constexpr uint32_t kSms = 148;  // of a B200; fixes the order of the sums
constexpr uint32_t kLongGroups = 64;
constexpr uint32_t kLong = 16384;  // values of the longest row that registers hold

struct SumsOut {
  void* out[kSums];
};

template <typename T>
constexpr int kStages = sizeof(T) == 4 ? 2 : 4;

template <typename T, int V, int NV, int TPR, int CL, bool BIAS, bool VALUES, int EACH>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, EACH)
k_block_norm_bwd(const __grid_constant__ BlockNorm a) {
  using C = Columns<T, V, NV, TPR>;
  using R = BlockRing<T, V, NV, TPR, VALUES ? 5 : 4, kStages<T>>;
  constexpr int ROWS = TPR == 32 ? 8 : 1, G = C::G, HV = C::HV, H = C::H, S = R::stages;
  constexpr int BLOCK = R::threads;
  static_assert(C::E == 8, "columns of a thread");
  enum { X, O, DR, DU, GATE };
  extern __shared__ uint4 ring_bytes[];
  __shared__ float red[4 * (TPR / 32)];
  __shared__ float4 stats[S][BLOCK / 32];
  __shared__ float2 shared_sums[2][8];
  const uint32_t lane = threadIdx.x % TPR, warp = threadIdx.x / 32;
  const uint32_t part = CL > 1 ? cluster_rank() : 0, team = blockIdx.x / CL;
  const uint32_t step = gridDim.x / CL * ROWS;
  const C c(a.n, part * (TPR * C::E) + lane * V);
  uint32_t r = team * ROWS + threadIdx.x / TPR;
  R ring;
  ring.ring = reinterpret_cast<char*>(ring_bytes);
  auto array = [&](int k, const void* p, int64_t ld) {
    ring.from[k] = p ? (const T*)p + (int64_t)r * ld + c.c0 : nullptr;
    ring.step[k] = step * ld;
  };
  array(X, a.x, a.ldx);
  array(O, a.o, a.ldo);
  array(DR, a.dr, a.lddr);
  array(DU, a.du, a.lddu);
  if constexpr (VALUES) array(GATE, a.gate_values, a.ldg);
  ring.clear(c);
  const float4* from_stats = a.stats + r;
  auto fetch = [&](bool there, uint32_t stage) {
    if constexpr (R::used) ring.fetch(c, there, stage);
    if (there && (threadIdx.x & 31) == 0) copy_async<16>(&stats[stage][warp], from_stats);
    from_stats += step;
    copy_commit();
  };
  const F2 none = pack2(0.0f, 0.0f);
  F2 w1[H], w2[H], b1[BIAS ? H : 1], gate[VALUES ? 1 : H];
  c.param(a.post_weight, a.param_f32, w1, 1.0f);
  c.param(a.pre_weight, a.param_f32, w2, 1.0f);
  if constexpr (BIAS) c.param(a.post_bias, a.param_f32, b1, 0.0f);
  if constexpr (!VALUES) {
    c.param(a.gate == PLX_BLOCK_GATE_UNITS ? a.gate_values : nullptr, a.param_f32, gate, 1.0f);
    if (a.gate == PLX_BLOCK_GATE_UNITS && a.sigmoid)
#pragma unroll
      for (int h = 0; h < H; ++h) gate[h] = pack2(sigmoid(gate[h].x).a, sigmoid(gate[h].y).a);
  }
  int turn = 0, turn2 = 0;
  // Two sums over the row.
  auto sums_of = [&](F2 v) {
    F2 s = row_sum2<TPR>(v, red, turn);
    if constexpr (CL > 1) {
      if (threadIdx.x < CL) st_peer(peer_smem(&shared_sums[turn2][part], threadIdx.x), s);
      cluster_barrier();
      s = shared_sums[turn2][0];
#pragma unroll
      for (int k = 1; k < CL; ++k) s = add2(s, shared_sums[turn2][k]);
      turn2 ^= 1;
    }
    return s;
  };
  F2 w2sum[H], w1sum[H], gsum[VALUES ? 1 : H], b2sum[BIAS ? H : 1], b1sum[BIAS ? H : 1];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    w2sum[h] = w1sum[h] = none;
    if constexpr (!VALUES) gsum[h] = none;
    if constexpr (BIAS) b2sum[h] = b1sum[h] = none;
  }
  T* to_x = (T*)a.dx + (int64_t)r * a.lddx + c.c0;
  T* to_o = (T*)a.d_o + (int64_t)r * a.lddo + c.c0;
  T* to_g = VALUES && a.dgate ? (T*)a.dgate + (int64_t)r * a.lddg + c.c0 : nullptr;
  const F2 scale = pack2(a.scale, a.scale);
  uint32_t stage = 0;
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(r + (uint64_t)s * step < a.rows, s);
  for (; r < a.rows; r += step) {
    copy_wait<S - 2>();
    __syncwarp();
    fetch(r + (uint64_t)(S - 1) * step < a.rows, stage == 0 ? S - 1 : stage - 1);
    if constexpr (!R::used) ring.fetch(c, true, 0);
    float4 st = stats[stage][warp];
    if (!a.post) st.x = 0.0f, st.y = 1.0f;  // h1 is o
    const F2 m1 = pack2(-st.x, -st.x), s1 = pack2(st.y, st.y);
    const F2 m2 = pack2(-st.z, -st.z), s2 = pack2(st.w, st.w);
    F2 h1[H], h2[H], d[H], c0 = none, c1 = none;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      F2 x[HV], o[HV], du[HV], gv[HV];
      ring.get(stage, X, g, x);
      ring.get(stage, O, g, o);
      ring.get(stage, DU, g, du);
      if constexpr (VALUES) {
        ring.get(stage, GATE, g, gv);
        if (a.sigmoid)
#pragma unroll
          for (int e = 0; e < HV; ++e) gv[e] = pack2(sigmoid(gv[e].x).a, sigmoid(gv[e].y).a);
      }
#pragma unroll
      for (int e = 0; e < HV; ++e) {
        const int h = g * HV + e;
        h1[h] = mul2(add2(o[e], m1), s1);
        F2 p = mul2(h1[h], w1[h]);
        if constexpr (BIAS) p = add2(p, b1[h]);
        const F2 rv = fma2(VALUES ? gv[e] : gate[VALUES ? 0 : h], p, mul2(scale, x[e]));
        h2[h] = mul2(add2(rv, m2), s2);
        w2sum[h] = fma2(du[e], h2[h], w2sum[h]);
        if constexpr (BIAS) b2sum[h] = add2(b2sum[h], du[e]);
        d[h] = mul2(du[e], w2[h]);
        c0 = add2(c0, d[h]);
        c1 = fma2(d[h], h2[h], c1);
      }
    }
    if (a.du) {
      const F2 c = sums_of(pack2(c0.x + c0.y, c1.x + c1.y));
      const float e0 = a.layer ? -c.x * a.inv_n : 0.0f, e1 = -c.y * a.inv_n;
      const F2 e02 = pack2(e0, e0), e12 = pack2(e1, e1);
#pragma unroll
      for (int h = 0; h < H; ++h) d[h] = mul2(s2, fma2(h2[h], e12, add2(d[h], e02)));
    }
    c0 = c1 = none;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      F2 dr[HV], gv[HV], out[HV], slope[HV];
      ring.get(stage, DR, g, dr);
      if constexpr (VALUES) {
        ring.get(stage, GATE, g, gv);
#pragma unroll
        for (int e = 0; e < HV; ++e) slope[e] = pack2(1.0f, 1.0f);
        if (a.sigmoid)
#pragma unroll
          for (int e = 0; e < HV; ++e) {
            const Sigmoid s = sigmoid(gv[e].x), t = sigmoid(gv[e].y);
            gv[e] = pack2(s.a, t.a);
            slope[e] = pack2(s.a * s.keep, t.a * t.keep);
          }
      }
      const bool in = c.in(g);
#pragma unroll
      for (int e = 0; e < HV; ++e) {
        const int h = g * HV + e;
        d[h] = add2(d[h], dr[e]);
        if (!in) d[h] = none;  // columns past the row's end have no part in what follows
        if (V == 1 && !c.both(g)) d[h].y = 0.0f;
        out[e] = mul2(scale, d[h]);
      }
      if (in) c.put(to_x, g, out);
#pragma unroll
      for (int e = 0; e < HV; ++e) {
        const int h = g * HV + e;
        F2 p = mul2(h1[h], w1[h]);
        if constexpr (BIAS) p = add2(p, b1[h]);
        if constexpr (VALUES) out[e] = mul2(mul2(d[h], p), slope[e]);
        else gsum[h] = fma2(d[h], p, gsum[h]);
        const F2 dp = mul2(d[h], VALUES ? gv[e] : gate[VALUES ? 0 : h]);
        w1sum[h] = fma2(dp, h1[h], w1sum[h]);
        if constexpr (BIAS) b1sum[h] = add2(b1sum[h], dp);
        d[h] = mul2(dp, w1[h]);
        c0 = add2(c0, d[h]);
        c1 = fma2(d[h], h1[h], c1);
      }
      if constexpr (VALUES) {
        if (in && to_g) c.put(to_g, g, out);
      }
    }
    if (a.post) {
      const F2 c = sums_of(pack2(c0.x + c0.y, c1.x + c1.y));
      const float e0 = a.layer ? -c.x * a.inv_n : 0.0f, e1 = -c.y * a.inv_n;
      const F2 e02 = pack2(e0, e0), e12 = pack2(e1, e1);
#pragma unroll
      for (int h = 0; h < H; ++h) d[h] = mul2(s1, fma2(h1[h], e12, add2(d[h], e02)));
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      F2 out[HV];
#pragma unroll
      for (int e = 0; e < HV; ++e) out[e] = d[g * HV + e];
      if (c.in(g)) c.put(to_o, g, out);
    }
    to_x += step * a.lddx;
    to_o += step * a.lddo;
    if (to_g) to_g += step * a.lddg;
    stage = stage == S - 1 ? 0 : stage + 1;
  }
  if constexpr (CL > 1) cluster_barrier();  // nobody writes to a block that has gone
  if (!a.partial) return;
  if constexpr (!VALUES) {  // the derivative of the gate, once
    if (a.gate == PLX_BLOCK_GATE_UNITS && a.sigmoid) {
      F2 raw[H];
      c.param(a.gate_values, a.param_f32, raw, 0.0f);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const Sigmoid s = sigmoid(raw[h].x), t = sigmoid(raw[h].y);
        gsum[h] = mul2(gsum[h], pack2(s.a * s.keep, t.a * t.keep));
      }
    }
  }
  float* out = a.partial + (uint64_t)team * kSums * a.n;
  constexpr int K = BIAS ? 5 : 3, STEP = C::STEP;
  auto column = [&](int k, int e) {  // of value e of the thread
    const int h = e / 2;
    F2 v = k == 0 ? w2sum[h] : k == 1 ? w1sum[h] : VALUES ? none : gsum[VALUES ? 0 : h];
    if (k > 2) v = BIAS ? (k == 3 ? b2sum[BIAS ? h : 0] : b1sum[BIAS ? h : 0]) : none;
    return e % 2 ? v.y : v.x;
  };
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j * STEP >= c.left) continue;
        float* to = out + (uint64_t)k * a.n + c.c0 + j * STEP;
        if constexpr (V >= 4) {  // n and the columns are multiples of four
#pragma unroll
          for (int e = 0; e < V; e += 4)
            *reinterpret_cast<float4*>(to + e) =
                make_float4(column(k, j * V + e), column(k, j * V + e + 1),
                            column(k, j * V + e + 2), column(k, j * V + e + 3));
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) to[e] = column(k, j * V + e);
        }
      }
  } else {  // the eight warps' sums, added in their order
    __shared__ float joined[8][32 * C::E];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) joined[warp][(j * 32 + lane) * V + e] = column(k, j * V + e);
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

// Rows too long for registers, in three passes over values made anew (2,048 rows of
// 20,000 bf16 1,306 us, 75 at the copy rate): the means of every row,
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
      sums[3] += du;
      d = st.w * ((a.pre_weight ? du * to_f32(((const P*)a.pre_weight)[i]) : du) - m.x - h2 * m.y);
    }
    if (a.dr) d += to_f32(((const T*)a.dr)[row.row * a.lddr + i]);
    const float gate = row.gate(i, slope), dg = d * row.p(i) * slope, dp = d * gate;
    sums[1] = fmaf(dp, h1, sums[1]);
    sums[4] += dp;
    sums[2] += dg;
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
      std::min<uint64_t>(by_rows, std::max<uint64_t>(kSms, (by_rows + 7) / 8)), most);
}

// Column sums of the groups that a call leaves, as many as its launch has blocks (of the
// ladder in plx_block_norm_backward).
uint64_t sums_bytes(uint64_t rows, uint32_t n) {
  const uint32_t most = n <= 1024 ? kSms * 4 : n <= 2048 ? kSms * 2 : n <= 4096 ? kSms
                        : n <= 8192 ? kSms / 2 : kSms / 4;
  const uint64_t groups =
      n > kLong ? std::min<uint64_t>(rows, kLongGroups) : groups_of(rows, 1, most);
  return (std::max<uint64_t>(1, groups) * kSums * n * 4 + 15) / 16 * 16;
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" size_t plx_block_norm_scratch_bytes(uint64_t rows, uint32_t n) {
  // and the means of rows that no registers hold
  return (size_t)(sums_bytes(rows, n) + (n > kLong ? rows * 16 : 0));
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
  PLX_CHECK_ARG(params->post || (!dpost_weight && !dpost_bias),
                "dpost_weight and dpost_bias need post");
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
  SumsOut outs = {{dpre_weight, params->post ? dpost_weight : nullptr, units ? dgate : nullptr,
                   dpre_bias, params->post ? dpost_bias : nullptr}};
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
  float4* means = (float4*)((char*)scratch + sums_bytes(rows, n));
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    auto go = [&](auto p) {
      using P = decltype(p);
      uint32_t groups = 0;
      int rc = PLX_OK;
      // EACH blocks an SM, CL blocks a row; a team visits rows of one remainder.
      auto launch = [&](auto v_c, auto nv_c, auto tpr_c, auto cl_c, auto each_c) {
        constexpr int VV = decltype(v_c)::value, NV = decltype(nv_c)::value;
        constexpr int TPR = decltype(tpr_c)::value, CL = decltype(cl_c)::value;
        constexpr int EACH = decltype(each_c)::value;
        auto with = [&](auto bias_c, auto values_c) -> int {
          constexpr bool VALUES = decltype(values_c)::value;
          using R = BlockRing<T, VV, NV, TPR, VALUES ? 5 : 4, kStages<T>>;
          constexpr auto kernel =
              k_block_norm_bwd<T, VV, NV, TPR, CL, decltype(bias_c)::value, VALUES, EACH>;
          groups = groups_of(rows, TPR == 32 ? 8 : 1, kSms * EACH / CL);
          if (groups == 0) return PLX_OK;
          if (R::bytes > 32 * 1024) PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, R::bytes));
          cudaLaunchConfig_t cfg = {};
          cfg.gridDim = dim3(groups * CL);
          cfg.blockDim = dim3(R::threads);
          cfg.dynamicSmemBytes = R::bytes;
          cfg.stream = ctx->stream;
          cudaLaunchAttribute at[1];
          at[0].id = cudaLaunchAttributeClusterDimension;
          at[0].val.clusterDim.x = CL;
          at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
          cfg.attrs = at;
          cfg.numAttrs = CL > 1 ? 1 : 0;
          PLX_TRY_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const BlockNorm)a));
          return PLX_OK;
        };
        using Yes = std::true_type;
        using No = std::false_type;
        const bool values = a.gate == PLX_BLOCK_GATE_VALUES;
        // Sums of biases where they are asked for (or biases to be applied).
        if (outs.out[3] || outs.out[4] || a.post_bias)
          rc = values ? with(Yes{}, Yes{}) : with(Yes{}, No{});
        else
          rc = values ? with(No{}, Yes{}) : with(No{}, No{});
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
      using std::integral_constant;
#define PLX_C(v) integral_constant<int, v>{}
      auto ladder = [&](auto vv, auto nv) {
        if (n <= 256) launch(vv, nv, PLX_C(32), PLX_C(1), PLX_C(2));
        else if (n <= 1024) launch(vv, nv, PLX_C(128), PLX_C(1), PLX_C(4));
        else if (n <= 2048) launch(vv, nv, PLX_C(256), PLX_C(1), PLX_C(2));
        else if (n <= 4096) launch(vv, nv, PLX_C(512), PLX_C(1), PLX_C(1));
        else if (n <= 8192) launch(vv, nv, PLX_C(512), PLX_C(2), PLX_C(1));
        else if (n <= kLong) launch(vv, nv, PLX_C(512), PLX_C(4), PLX_C(1));
        else loops();
      };
      if (v == V) ladder(PLX_C(V), PLX_C(8 / V));
      else if (sizeof(T) == 2 && v >= 2) ladder(PLX_C(2), PLX_C(4));
      else ladder(PLX_C(1), PLX_C(8));
#undef PLX_C
      if (rc != PLX_OK) return rc;
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
