// Products of rows and weights with one multiply-add a term in 32 bits.
//
// Bound by the multiply-adds: a block makes 128 x 128 sums, a thread 8 x 8 of
// them out of shared memory, so that each value read from there serves eight
// multiply-adds (two of them an instruction).
#include "dense.cuh"

namespace plx {
namespace {

constexpr int BM = 128, BN = 128, BK = 16;

// A tile's values of one operand on their way from memory: 8 of the 128 x 16.
template <typename T>
struct TileLoad {
  float v[8];
  __device__ __forceinline__ void fetch(const Operand& o, uint32_t i0, uint32_t count, uint32_t k0,
                                        uint32_t depth) {
    const T* p = (const T*)o.p;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t i, k;
      place(o.k_major, j, i, k);
      i += i0;
      k += k0;
      v[j] = i < count && k < depth
                 ? to_f32(o.k_major ? p[(int64_t)i * o.ld + k] : p[(int64_t)k * o.ld + i])
                 : 0.0f;
    }
  }
  static __device__ __forceinline__ void place(bool k_major, int j, uint32_t& i, uint32_t& k) {
    const uint32_t t = threadIdx.x;
    if (k_major) {
      k = t % BK;
      i = t / BK + 16 * j;
    } else {
      i = t % 128;
      k = t / 128 + 2 * j;
    }
  }
  __device__ __forceinline__ void store(bool k_major, float (*to)[BM + 4]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t i, k;
      place(k_major, j, i, k);
      to[k][i] = v[j];
    }
  }
};

template <typename T, typename P, int ACT>
__global__ void __launch_bounds__(256, 2) k_product_f32(const __grid_constant__ Product p) {
  __shared__ float4 as4[2][BK][(BM + 4) / 4], bs4[2][BK][(BN + 4) / 4];
  auto as = reinterpret_cast<float(*)[BK][BM + 4]>(as4);
  auto bs = reinterpret_cast<float(*)[BK][BN + 4]>(bs4);
  const uint32_t i0 = blockIdx.y * BM, j0 = blockIdx.x * BN;
  const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  F2 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = pack2(0.0f, 0.0f);
  TileLoad<T> la, lb;
  la.fetch(p.a, i0, p.rows, 0, p.depth);
  lb.fetch(p.b, j0, p.cols, 0, p.depth);
  int turn = 0;
  for (uint32_t k0 = 0; k0 < p.depth; k0 += BK, turn ^= 1) {
    la.store(p.a.k_major, as[turn]);
    lb.store(p.b.k_major, bs[turn]);
    __syncthreads();
    if (k0 + BK < p.depth) {
      la.fetch(p.a, i0, p.rows, k0 + BK, p.depth);
      lb.fetch(p.b, j0, p.cols, k0 + BK, p.depth);
    }
#pragma unroll
    for (int k = 0; k < BK; ++k) {
      const float4 a0 = as4[turn][k][ty], a1 = as4[turn][k][16 + ty];
      const float4 b0 = bs4[turn][k][tx], b1 = bs4[turn][k][16 + tx];
      const float av[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
      const F2 bv[4] = {pack2(b0.x, b0.y), pack2(b0.z, b0.w), pack2(b1.x, b1.y),
                        pack2(b1.z, b1.w)};
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fma2(pack2(av[i], av[i]), bv[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t row = i0 + (i / 4) * 64 + ty * 4 + i % 4;
    if (row >= p.rows) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t col = j0 + (j / 4) * 64 + tx * 4 + j % 4;
      if (col >= p.cols) continue;
      float z = j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x;
      if (p.f.bias) z += to_f32(((const P*)p.f.bias)[col]);
      if (p.f.pre) p.f.pre[(uint64_t)row * p.cols + col] = z;
      float y = act_value<ACT>(z);
      if (p.f.residual) y += to_f32(((const T*)p.f.residual)[(int64_t)row * p.f.ldr + col]);
      ((T*)p.f.y)[(int64_t)row * p.f.ldy + col] = from_f32<T>(y);
    }
  }
}

}  // namespace

int product_f32(plx_ctx* ctx, int dtype, const Product& p) {
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto q) {
      using P = decltype(q);
      return with_act(p.f.act, [&](auto act) {
        const dim3 grid((p.cols + BN - 1) / BN, (p.rows + BM - 1) / BM);
        k_product_f32<T, P, decltype(act)::value><<<grid, 256, 0, ctx->stream>>>(p);
        PLX_LAUNCH_CHECK("k_product_f32");
        return PLX_OK;
      });
    };
    return p.f.param_dtype == PLX_F32 ? go(float{}) : go(t);
  });
}

}  // namespace plx
