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
// order.
#include "block_norm.cuh"
#include "cluster.cuh"

namespace plx {
namespace {

constexpr int kSums = 5;  // dw2, dw1, dgate of units, db2, db1
constexpr uint32_t kSms = 148;  // of a B200; fixes the order of the sums
constexpr uint32_t kMostGroups = kSms * 4;
constexpr uint32_t kLongGroups = 64;

struct SumsOut {
  void* out[kSums];
};

// Pairs of values of a parameter, of either type: V consecutive ones, or where V
// is 1 the one at i and, if there is one in the row, the one at `next`.
template <typename T, int V>
__device__ __forceinline__ void param_pairs(const void* w, bool f32, uint32_t i, uint32_t next,
                                            uint32_t n, F2 (&v)[V == 1 ? 1 : V / 2]) {
  if constexpr (V == 1) {
    const bool two = next < n;
    v[0] = f32 ? pack2(((const float*)w)[i], two ? ((const float*)w)[next] : 0.0f)
               : pack2(to_f32(((const T*)w)[i]), two ? to_f32(((const T*)w)[next]) : 0.0f);
  } else if (f32) {
    const Pack<float, V> q = load_pack<float, V>((const float*)w + i);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) v[e] = pair_of(q, 2 * e);
  } else {
    const Pack<T, V> q = load_pack<T, V>((const T*)w + i);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) v[e] = pair_of(q, 2 * e);
  }
}

// Rows under way at once, in shared memory; a thread reads what it copied itself.
// Pieces of less than four bytes go to registers.
template <typename T, int V, int NV, int TPR>
struct BlockRing {
  static constexpr int piece = V * sizeof(T);
  static constexpr bool used = piece >= 4;
  static constexpr int threads = TPR == 32 ? 256 : TPR;
  static constexpr int array_bytes = NV * threads * piece;
  static constexpr int stage_bytes = 5 * array_bytes;  // x, o, dr, du, gate
  // 512 threads an SM (in one block or more): 160 KB of its shared memory
  static constexpr int stages = sizeof(T) == 4 ? 2 : 4;
  static constexpr int bytes = used ? stages * stage_bytes : 0;
};

template <typename T, int V, int NV, int TPR, int CL, bool BIAS, int EACH>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, EACH)
k_block_norm_bwd(const __grid_constant__ BlockNorm a) {
  using R = BlockRing<T, V, NV, TPR>;
  constexpr int ROWS = TPR == 32 ? 8 : 1, E = NV * V, H = E / 2, STEP = TPR * V, S = R::stages;
  // Pairs of a piece; where pieces are single values, of two of them (G groups).
  constexpr int HV = V == 1 ? 1 : V / 2, G = V == 1 ? NV / 2 : NV, BLOCK = R::threads;
  constexpr int GSTEP = V == 1 ? 2 * STEP : STEP;
  static_assert(E == 8, "columns of a thread");
  extern __shared__ uint4 ring_bytes[];
  char* ring = reinterpret_cast<char*>(ring_bytes);
  __shared__ float red[4 * (TPR / 32)];
  __shared__ float4 stats[S][BLOCK / 32];
  __shared__ float2 shared_sums[2][8];
  const uint32_t lane = threadIdx.x % TPR, warp = threadIdx.x / 32;
  const uint32_t part = CL > 1 ? cluster_rank() : 0, team = blockIdx.x / CL;
  const uint32_t teams = gridDim.x / CL;
  const uint32_t c0 = part * (TPR * E) + lane * V;
  const int left = (int)a.n - (int)c0;
  const bool units = a.gate == PLX_BLOCK_GATE_UNITS, values = a.gate == PLX_BLOCK_GATE_VALUES;
  enum { X, O, DR, DU, GATE };
  auto slot = [&](uint32_t stage, int array, int j) {
    char* at = ring + stage * R::stage_bytes + array * R::array_bytes;
    return reinterpret_cast<Pack<T, V>*>(at) + j * BLOCK + threadIdx.x;
  };
  Pack<T, V> held[R::used ? 1 : 5][NV];  // a row's values, where no ring has them
  const T* from[5] = {(const T*)a.x, (const T*)a.o, (const T*)a.dr, (const T*)a.du,
                      values ? (const T*)a.gate_values : nullptr};
  const int64_t ld[5] = {a.ldx, a.ldo, a.lddr, a.lddu, a.ldg};
  const uint32_t step = teams * ROWS;
  uint32_t r = team * ROWS + threadIdx.x / TPR;
  auto fetch = [&](uint64_t row, uint32_t stage) {
    if (row < a.rows) {
      if constexpr (R::used) {
#pragma unroll
        for (int k = 0; k < 5; ++k)
          if (from[k])
#pragma unroll
            for (int j = 0; j < NV; ++j)
              if (j * STEP < left)
                copy_async<R::piece>(slot(stage, k, j), from[k] + (int64_t)row * ld[k] + c0 + j * STEP);
      }
      if ((threadIdx.x & 31) == 0) copy_async<16>(&stats[stage][warp], a.stats + row);
    }
    copy_commit();
  };
  // Columns past the row's end, and arrays that are not given, are 0.
  Pack<T, V> zero;
#pragma unroll
  for (int e = 0; e < V; ++e) zero.v[e] = from_f32<T>(0.0f);
  if constexpr (R::used) {
    for (int s = 0; s < S; ++s)
      for (int k = 0; k < 5; ++k)
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (!from[k] || j * STEP >= left) *slot(s, k, j) = zero;
  }
  uint32_t stage = 0;
  // Pairs of values of group j of an array of the row under way.
  auto get = [&](int array, int j, F2 (&v)[HV]) {
    auto piece = [&](int k) {
      if constexpr (R::used) return *slot(stage, array, k);
      else return held[array][k];
    };
    if constexpr (V == 1) {
      v[0] = pack2(to_f32(piece(2 * j).v[0]), to_f32(piece(2 * j + 1).v[0]));
    } else {
      const Pack<T, V> q = piece(j);
#pragma unroll
      for (int e = 0; e < HV; ++e) v[e] = pair_of(q, 2 * e);
    }
  };
  auto put = [&](void* array, int64_t lda, uint32_t row, int j, const F2 (&v)[HV]) {
    T* to = (T*)array + (int64_t)row * lda + c0 + j * GSTEP;
    if constexpr (V == 1) {
      to[0] = from_f32<T>(v[0].x);
      if (j * GSTEP + STEP < left) to[STEP] = from_f32<T>(v[0].y);
    } else {
      Pack<T, V> q;
#pragma unroll
      for (int e = 0; e < HV; ++e) put_pair(q, 2 * e, v[e]);
      *reinterpret_cast<Pack<T, V>*>(to) = q;
    }
  };
  auto param = [&](const void* w, int j, F2 (&v)[HV]) {
    const uint32_t i = c0 + j * GSTEP;
    param_pairs<T, V>(w, a.param_f32, i, i + STEP, a.n, v);
  };
  const F2 none = pack2(0.0f, 0.0f), ones = pack2(1.0f, 1.0f);
  // A piece's gate and its derivative.
  auto gate_of = [&](int j, F2 (&g)[HV], F2 (&slope)[HV]) {
    if (units) param(a.gate_values, j, g);
    else if (values) get(GATE, j, g);
    else
#pragma unroll
      for (int e = 0; e < HV; ++e) g[e] = ones;
#pragma unroll
    for (int e = 0; e < HV; ++e) {
      slope[e] = ones;
      if (a.sigmoid) {
        const Sigmoid s = sigmoid(g[e].x), t = sigmoid(g[e].y);
        g[e] = pack2(s.a, t.a);
        slope[e] = pack2(s.a * s.keep, t.a * t.keep);
      }
    }
  };
  int turn = 0, turn2 = 0;
  // Two sums over the row.
  auto sums_of = [&](F2 c) {
    F2 s = row_sum2<TPR>(c, red, turn);
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
  constexpr int HT = G * HV;  // pairs of a thread
  F2 w2sum[HT], w1sum[HT], gsum[HT], b2sum[BIAS ? HT : 1], b1sum[BIAS ? HT : 1];
#pragma unroll
  for (int h = 0; h < HT; ++h) {
    w2sum[h] = w1sum[h] = gsum[h] = none;
    if (BIAS) b2sum[h] = b1sum[h] = none;
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(r + (uint64_t)s * step, s);
  for (; r < a.rows; r += step) {
    copy_wait<S - 2>();
    __syncwarp();
    fetch(r + (uint64_t)(S - 1) * step, stage == 0 ? S - 1 : stage - 1);
    if constexpr (!R::used) {
#pragma unroll
      for (int k = 0; k < 5; ++k)
        if (from[k]) load_row<STEP>(from[k] + (int64_t)r * ld[k] + c0, left, held[k]);
        else
#pragma unroll
          for (int j = 0; j < NV; ++j) held[k][j] = zero;
    }
    const float4 st = stats[stage][warp];
    const F2 m1 = pack2(-st.x, -st.x), s1 = pack2(st.y, st.y);
    const F2 m2 = pack2(-st.z, -st.z), s2 = pack2(st.w, st.w);
    const F2 scale = pack2(a.scale, a.scale);
    F2 h1[HT], h2[HT], d[HT], c0s = none, c1s = none;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (j * GSTEP >= left) {
#pragma unroll
        for (int e = 0; e < HV; ++e) h1[j * HV + e] = h2[j * HV + e] = d[j * HV + e] = none;
        continue;
      }
      F2 x[HV], p[HV], g[HV], slope[HV], w[HV];
      get(X, j, x);
      get(O, j, p);
      if (a.post) {
#pragma unroll
        for (int e = 0; e < HV; ++e) p[e] = mul2(add2(p[e], m1), s1);
      }
#pragma unroll
      for (int e = 0; e < HV; ++e) h1[j * HV + e] = p[e];
      if (a.post_weight) {
        param(a.post_weight, j, w);
#pragma unroll
        for (int e = 0; e < HV; ++e) p[e] = mul2(p[e], w[e]);
      }
      if (BIAS && a.post_bias) {
        param(a.post_bias, j, w);
#pragma unroll
        for (int e = 0; e < HV; ++e) p[e] = add2(p[e], w[e]);
      }
      gate_of(j, g, slope);
      F2 du[HV];
      get(DU, j, du);
      if (a.pre_weight) param(a.pre_weight, j, w);
#pragma unroll
      for (int e = 0; e < HV; ++e) {
        const int h = j * HV + e;
        const F2 rv = fma2(g[e], p[e], mul2(scale, x[e]));
        h2[h] = mul2(add2(rv, m2), s2);
        w2sum[h] = fma2(du[e], h2[h], w2sum[h]);
        if (BIAS) b2sum[h] = add2(b2sum[h], du[e]);
        d[h] = a.pre_weight ? mul2(du[e], w[e]) : du[e];
        c0s = add2(c0s, d[h]);
        c1s = fma2(d[h], h2[h], c1s);
      }
    }
    if (a.du) {
      const F2 c = sums_of(pack2(c0s.x + c0s.y, c1s.x + c1s.y));
      const float e0 = a.layer ? -c.x * a.inv_n : 0.0f, e1 = -c.y * a.inv_n;
      const F2 e02 = pack2(e0, e0), e12 = pack2(e1, e1);
#pragma unroll
      for (int h = 0; h < HT; ++h) d[h] = mul2(s2, fma2(h2[h], e12, add2(d[h], e02)));
    }
    c0s = c1s = none;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (j * GSTEP >= left) {
#pragma unroll
        for (int e = 0; e < HV; ++e) d[j * HV + e] = none;
        continue;
      }
      F2 dr[HV], p[HV], g[HV], slope[HV], w[HV], out[HV];
      get(DR, j, dr);
      gate_of(j, g, slope);
      if (a.post_weight) param(a.post_weight, j, w);
#pragma unroll
      for (int e = 0; e < HV; ++e) {
        const int h = j * HV + e;
        d[h] = add2(d[h], dr[e]);
        if (V == 1 && j * GSTEP + STEP >= left) d[h].y = 0.0f;
        p[e] = a.post_weight ? mul2(h1[h], w[e]) : h1[h];
        out[e] = mul2(scale, d[h]);
      }
      put(a.dx, a.lddx, r, j, out);
      if (BIAS && a.post_bias) {
        F2 b[HV];
        param(a.post_bias, j, b);
#pragma unroll
        for (int e = 0; e < HV; ++e) p[e] = add2(p[e], b[e]);
      }
#pragma unroll
      for (int e = 0; e < HV; ++e) {
        const int h = j * HV + e;
        out[e] = mul2(mul2(d[h], p[e]), slope[e]);
        gsum[h] = add2(gsum[h], out[e]);
        F2 dp = mul2(d[h], g[e]);
        w1sum[h] = fma2(dp, h1[h], w1sum[h]);
        if (BIAS) b1sum[h] = add2(b1sum[h], dp);
        if (a.post_weight) dp = mul2(dp, w[e]);
        d[h] = dp;
        c0s = add2(c0s, dp);
        c1s = fma2(dp, h1[h], c1s);
      }
      if (a.dgate) put(a.dgate, a.lddg, r, j, out);
    }
    if (a.post) {
      const F2 c = sums_of(pack2(c0s.x + c0s.y, c1s.x + c1s.y));
      const float e0 = a.layer ? -c.x * a.inv_n : 0.0f, e1 = -c.y * a.inv_n;
      const F2 e02 = pack2(e0, e0), e12 = pack2(e1, e1);
#pragma unroll
      for (int h = 0; h < HT; ++h) d[h] = mul2(s1, fma2(h1[h], e12, add2(d[h], e02)));
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (j * GSTEP >= left) continue;
      F2 out[HV];
#pragma unroll
      for (int e = 0; e < HV; ++e) out[e] = d[j * HV + e];
      put(a.d_o, a.lddo, r, j, out);
    }
    stage = stage == S - 1 ? 0 : stage + 1;
  }
  if constexpr (CL > 1) cluster_barrier();  // nobody writes to a block that has gone
  if (!a.partial) return;
  float* out = a.partial + (uint64_t)team * kSums * a.n;
  auto column = [&](int k, int e) {  // of value e of the thread
    const int h = e / 2;
    F2 v = k == 0 ? w2sum[h] : k == 1 ? w1sum[h] : gsum[h];
    if (k > 2) v = BIAS ? (k == 3 ? b2sum[h] : b1sum[h]) : none;
    return e % 2 ? v.y : v.x;
  };
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int k = 0; k < (BIAS ? 5 : 3); ++k)
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j * STEP >= left) continue;
        float* to = out + (uint64_t)k * a.n + c0 + j * STEP;
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
    __shared__ float joined[8][32 * E];
#pragma unroll
    for (int k = 0; k < (BIAS ? 5 : 3); ++k) {
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
  float4* means = (float4*)((char*)scratch + need - rows * 16);
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
        using R = BlockRing<T, VV, NV, TPR>;
        auto with = [&](auto bias_c) -> int {
          constexpr auto kernel = k_block_norm_bwd<T, VV, NV, TPR, CL, decltype(bias_c)::value, EACH>;
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
        // Sums of biases where they are asked for (or biases to be applied).
        rc = outs.out[3] || outs.out[4] || a.post_bias ? with(std::true_type{})
                                                       : with(std::false_type{});
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
        else if (n <= 16384) launch(vv, nv, PLX_C(512), PLX_C(4), PLX_C(1));
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
