// Products of 16-bit rows and weights on the tensor cores.
//
// Bound by the products (large calls) or by reading the weights (few rows). A
// block makes tiles of 128 x BN sums: one thread has tensor copies fill a ring of
// stages of 64 values of k, one issues the products on them, eight warps finish
// the tile before (bias, activation, residual, rounding) out of the other half of
// TMEM meanwhile. Blocks stay and take every gridDim-th tile.
// Where tiles are few, a cluster of blocks shares one tile's k: each leaves its
// sums in shared memory, and all of them add and finish a part of the tile, in
// the order of the blocks.
// Few rows (at most 64) are the tile's second side, so that the first one's 128
// are units of the layer.
#include "cluster.cuh"
#include "dense.cuh"
#include "tensor.cuh"

namespace plx {
namespace {

constexpr uint32_t kTileA = 128, kTileK = 64;
constexpr int kFinishWarps = 8, kThreads = 64 + 32 * kFinishWarps;
constexpr uint32_t kSmem = 232448;  // a block can have

template <int BN>
struct Stages {
  static constexpr uint32_t a_bytes = kTileA * kTileK * 2, b_bytes = BN * kTileK * 2;
  static constexpr uint32_t bytes = a_bytes + b_bytes;
  static constexpr uint32_t most = (kSmem - 2048) / bytes;
  static constexpr uint32_t count = most < 12 ? most : 12;
  static constexpr uint32_t smem = count * bytes + 1024;  // to a multiple of 1,024
  static constexpr uint32_t columns = 2 * BN < 32 ? 32 : 2 * BN;
};

struct TensorProduct {
  CUtensorMap a, b;  // a has the tile's 128
  uint32_t rows, cols, depth;  // of the tiles' sides
  uint32_t tiles_a, tiles_b;
  uint32_t kind;
  bool a_k_major, b_k_major, swapped;  // swapped: a's side are the result's columns
  Finish f;
  int32_t* status;
  uint64_t timeout_ns;
};

// Waits, with a limit, unless another thread of the block has given up.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile uint32_t* gave_up,
                                     const TensorProduct& p) {
  if (mbar_try_wait(bar, parity)) return true;
  if (!*gave_up && mbar_wait_bounded(bar, parity, p.timeout_ns)) return true;
  *gave_up = 1;
  record_status(p.status, kStatusTimeout);
  return false;
}

template <int C>
__device__ __forceinline__ void activate(int act, float (&v)[C]) {
  auto all = [&](auto a) {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = act_value<decltype(a)::value>(v[i]);
  };
  using std::integral_constant;
  switch (act) {
    case PLX_ACT_SIGMOID: all(integral_constant<int, PLX_ACT_SIGMOID>{}); break;
    case PLX_ACT_TANH: all(integral_constant<int, PLX_ACT_TANH>{}); break;
    case PLX_ACT_RELU: all(integral_constant<int, PLX_ACT_RELU>{}); break;
    case PLX_ACT_SILU: all(integral_constant<int, PLX_ACT_SILU>{}); break;
    case PLX_ACT_GELU: all(integral_constant<int, PLX_ACT_GELU>{}); break;
    default: break;
  }
}
template <typename T>
__device__ __forceinline__ float bias_at(const Finish& f, uint32_t col) {
  return f.param_dtype == PLX_F32 ? __ldg((const float*)f.bias + col)
                                  : to_f32(((const T*)f.bias)[col]);
}

// One sum of the result.
template <typename T>
__device__ __forceinline__ void finish_one(const Finish& f, uint32_t row, uint32_t col,
                                           uint32_t cols, float z) {
  float v[1] = {f.bias ? z + bias_at<T>(f, col) : z};
  if (f.pre) f.pre[(uint64_t)row * cols + col] = v[0];
  activate(f.act, v);
  if (f.residual) v[0] += to_f32(((const T*)f.residual)[(int64_t)row * f.ldr + col]);
  ((T*)f.y)[(int64_t)row * f.ldy + col] = from_f32<T>(v[0]);
}

// A thread's C consecutive columns of a row of the result; `wide`: all there, in
// 16-byte pieces.
template <typename T, int C>
__device__ __forceinline__ void finish_row(const Finish& f, uint32_t row, uint32_t col,
                                           uint32_t cols, bool wide, float (&v)[C]) {
  if (f.bias) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (wide || col + i < cols) v[i] += bias_at<T>(f, col + i);
  }
  if (f.pre) {
    float* to = f.pre + (uint64_t)row * cols + col;
    if (wide) {
#pragma unroll
      for (int i = 0; i < C; i += 4)
        *reinterpret_cast<float4*>(to + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (col + i < cols) to[i] = v[i];
    }
  }
  activate(f.act, v);
  T* to = (T*)f.y + (int64_t)row * f.ldy + col;
  const T* res = (const T*)f.residual + (int64_t)row * f.ldr + col;
  if (wide) {
#pragma unroll
    for (int i = 0; i < C; i += 8) {
      Pack<T, 8> q;
      if (f.residual) {
        q = load_pack<T, 8>(res + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i + e] += to_f32(q.v[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) put_pair(q, e, pack2(v[i + e], v[i + e + 1]));
      *reinterpret_cast<Pack<T, 8>*>(to + i) = q;
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (col + i < cols) {
        if (f.residual) v[i] += to_f32(res[i]);
        to[i] = from_f32<T>(v[i]);
      }
  }
}

template <typename T, int BN, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
k_product_tensor(const __grid_constant__ TensorProduct p, bool wide) {
  using S = Stages<BN>;
  constexpr uint32_t C = BN < 32 ? 16 : 32;  // columns at a time
  extern __shared__ uint8_t smem_bytes[];
  uint8_t* ring = smem_bytes + (1024 - (smem_addr(smem_bytes) & 1023)) % 1024;
  __shared__ uint64_t full[S::count], empty[S::count], done[2], taken[2];
  __shared__ uint32_t tmem, gave_up;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t blocks = (p.depth + kTileK - 1) / kTileK;
  uint32_t k_first = 0, k_last = blocks, rank = 0, parts = 1;
  uint32_t tile0 = blockIdx.x, step = gridDim.x;
  const uint32_t tiles = p.tiles_a * p.tiles_b;
  if constexpr (SPLIT) {
    rank = cluster_rank();
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(parts));
    tile0 = blockIdx.x / parts;
    step = tiles;  // one tile
    const uint32_t each = (blocks + parts - 1) / parts;
    k_first = min(rank * each, blocks);
    k_last = min(k_first + each, blocks);
  }
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < S::count; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&done[h], 1);
      mbar_init(&taken[h], kFinishWarps);
    }
    mbar_init_fence();
    gave_up = 0;
  }
  if (warp == 1) tmem_alloc(&tmem, S::columns);
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t sums = *(volatile uint32_t*)&tmem;
  // Tiles in groups of eight along a's side, so that what is under way at one
  // time shares both operands.
  auto place = [&](uint32_t tile, uint32_t& ia, uint32_t& ib) {
    const uint32_t group = 8 * p.tiles_b, first = tile / group * 8;
    const uint32_t size = min(p.tiles_a - first, 8u), in = tile % group;
    ia = first + in % size;
    ib = in / size;
  };

  if (warp == 0 && lane == 0) {  // copies
    uint32_t it = 0;
    bool ok = true;
    for (uint32_t tile = tile0; ok && tile < tiles; tile += step) {
      uint32_t ia, ib;
      place(tile, ia, ib);
      for (uint32_t k = k_first; k < k_last; ++k, ++it) {
        const uint32_t s = it % S::count;
        if (it >= S::count && !(ok = wait(&empty[s], (it / S::count - 1) & 1, &gave_up, p))) break;
        uint8_t* a = ring + s * S::bytes;
        uint8_t* b = a + S::a_bytes;
        mbar_arrive_expect_tx(&full[s], S::bytes);
        if (p.a_k_major) {
          tensor_load(a, &p.a, (int)(k * kTileK), (int)(ia * kTileA), &full[s]);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < kTileA / 64; ++j)
            tensor_load(a + j * 8192, &p.a, (int)(ia * kTileA + j * 64), (int)(k * kTileK),
                        &full[s]);
        }
        if (p.b_k_major) {
          tensor_load(b, &p.b, (int)(k * kTileK), (int)(ib * BN), &full[s]);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < (BN + 63) / 64; ++j)
            tensor_load(b + j * 8192, &p.b, (int)(ib * BN + j * 64), (int)(k * kTileK), &full[s]);
        }
      }
    }
    if (!ok)  // what is still on its way
      for (uint32_t j = it > S::count ? it - S::count : 0; j < it; ++j)
        mbar_wait_bounded(&full[j % S::count], (j / S::count) & 1, p.timeout_ns);
  } else if (warp == 1 && lane == 0) {  // products
    uint32_t it = 0, turn = 0;
    bool ok = true;
    for (uint32_t tile = tile0; ok && tile < tiles; tile += step, ++turn) {
      const uint32_t half = turn & 1, to = sums + half * BN;
      if (turn >= 2 && !(ok = wait(&taken[half], (turn / 2 - 1) & 1, &gave_up, p))) break;
      tmem_fence_after();
      for (uint32_t k = k_first; k < k_last; ++k, ++it) {
        const uint32_t s = it % S::count;
        if (!(ok = wait(&full[s], (it / S::count) & 1, &gave_up, p))) break;
        tmem_fence_after();
        const uint8_t* at = ring + s * S::bytes;
        const uint64_t a = p.a_k_major ? operand_k_major(at) : operand_i_major(at, 8192);
        const uint64_t b = p.b_k_major ? operand_k_major(at + S::a_bytes)
                                       : operand_i_major(at + S::a_bytes, 8192);
        // 16 values of k further on: 32 bytes of a row, or sixteen rows
        const uint32_t da = p.a_k_major ? 2 : 128, db = p.b_k_major ? 2 : 128;
#pragma unroll
        for (uint32_t j = 0; j < kTileK / 16; ++j)
          tensor_product(to, a + j * da, b + j * db, p.kind, k > k_first || j > 0);
        products_arrive(&empty[s]);
      }
      if (ok) products_arrive(&done[half]);
    }
  } else if (warp >= 2) {  // finishing
    const uint32_t quarter = warp % 4, side = (warp - 2) / 4;  // lanes of TMEM; half of the columns
    uint32_t turn = 0;
    for (uint32_t tile = tile0; tile < tiles; tile += step, ++turn) {
      uint32_t ia, ib;
      place(tile, ia, ib);
      const uint32_t half = turn & 1;
      const uint32_t i = ia * kTileA + quarter * 32 + lane;  // on a's side
      const bool sound = __all_sync(~0u, wait(&done[half], (turn / 2) & 1, &gave_up, p));
      tmem_fence_after();
      if (!sound && !SPLIT) break;
#pragma unroll 1
      for (uint32_t c = BN < 32 ? 0 : side * (BN / 2); c < (BN < 32 ? BN : (side + 1) * (BN / 2));
           c += C) {
        float v[C];
        if (BN < 32 && side) break;
        if constexpr (C == 32) tmem_load32(sums + half * BN + (quarter << 21) + c, v);
        else tmem_load16(sums + half * BN + (quarter << 21) + c, v);
        const uint32_t j0 = ib * BN + c;
        if constexpr (SPLIT) {
          const bool any = k_last > k_first;
          float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
          for (uint32_t e = 0; e < C; ++e) {
            const uint32_t at = p.swapped ? (c + e) * kTileA + quarter * 32 + lane
                                          : (quarter * 32 + lane) * (BN + 1) + c + e;
            mine[at] = any ? v[e] : 0.0f;
          }
        } else if (p.swapped) {
          if (i < p.rows)
#pragma unroll
            for (uint32_t e = 0; e < C; ++e)
              if (j0 + e < p.cols) finish_one<T>(p.f, j0 + e, i, p.rows, v[e]);
        } else if (i < p.rows && j0 < p.cols) {
          finish_row<T, C>(p.f, i, j0, p.cols, wide && j0 + C <= p.cols, v);
        }
      }
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&taken[half]);
    }
  }
  __syncwarp();
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  __syncwarp();
  if (warp == 1) tmem_free(sums, S::columns);
  if constexpr (SPLIT) {
    cluster_barrier();  // every block's sums are there
    uint32_t ia, ib;
    place(tile0, ia, ib);
    const uint32_t inner = p.swapped ? kTileA : BN, outer = p.swapped ? BN : kTileA;
    const uint32_t pitch = p.swapped ? kTileA : BN + 1;
    const float* mine = reinterpret_cast<const float*>(ring);
    // every parts-th row of the result's is this block's
    for (uint32_t at = threadIdx.x; at < outer / parts * inner; at += kThreads) {
      const uint32_t o = at / inner * parts + rank, n = at % inner;
      const uint32_t row = p.swapped ? ib * BN + o : ia * kTileA + o;
      const uint32_t col = p.swapped ? ia * kTileA + n : ib * BN + n;
      const uint32_t rows = p.swapped ? p.cols : p.rows, cols = p.swapped ? p.rows : p.cols;
      if (row >= rows || col >= cols) continue;
      float z = 0.0f;
      for (uint32_t r = 0; r < parts; ++r) z += ld_peer(peer_smem(mine + o * pitch + n, r));
      finish_one<T>(p.f, row, col, cols, z);
    }
    cluster_barrier();  // nobody reads this block's any more
  }
}

template <typename T, int BN>
int launch(plx_ctx* ctx, TensorProduct& t, const Product& p, const Operand& a, const Operand& b,
           uint32_t parts, bool wide) {
  using S = Stages<BN>;
  constexpr bool bf16 = std::is_same_v<T, __nv_bfloat16>;
  t.tiles_a = (t.rows + kTileA - 1) / kTileA;
  t.tiles_b = (t.cols + BN - 1) / BN;
  t.kind = product_kind(bf16, !a.k_major, !b.k_major, BN);
  auto map = [&](CUtensorMap* m, const Operand& o, uint32_t count, uint32_t tile) {
    return tensor_map(m, bf16 ? PLX_BF16 : PLX_F16, o.p, o.k_major ? t.depth : count,
                      o.k_major ? count : t.depth, o.ld, 64, o.k_major ? tile : kTileK, true);
  };
  if (int rc = map(&t.a, a, t.rows, kTileA)) return rc;
  if (int rc = map(&t.b, b, t.cols, BN)) return rc;
  const uint64_t tiles = (uint64_t)t.tiles_a * t.tiles_b;
  if (tiles >= (1ull << 28))
    return set_error(PLX_ERR_CAPACITY, "%u x %u results are too many for one call", p.rows, p.cols);
  if (parts > 1) {
    constexpr auto kernel = k_product_tensor<T, BN, true>;
    constexpr uint32_t sums = (BN + 1) * kTileA * 4;
    constexpr uint32_t smem = S::smem < sums + 1024 ? sums + 1024 : S::smem;
    PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * parts));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    PLX_TRY_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const TensorProduct)t, wide));
  } else {
    constexpr auto kernel = k_product_tensor<T, BN, false>;
    PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, S::smem));
    const unsigned grid = (unsigned)std::min<uint64_t>(tiles, ctx->num_sms);
    kernel<<<grid, kThreads, S::smem, ctx->stream>>>(t, wide);
    PLX_LAUNCH_CHECK("k_product_tensor");
  }
  return PLX_OK;
}

}  // namespace

int product_tensor(plx_ctx* ctx, int dtype, const Product& p) {
  TensorProduct t = {};
  t.depth = p.depth;
  t.f = p.f;
  t.status = ctx->d_status;
  t.timeout_ns = ctx->timeout_ns;
  Operand a = p.a, b = p.b;
  t.rows = p.rows;
  t.cols = p.cols;
  t.swapped = p.rows <= 64 && p.cols > p.rows && a.k_major;
  if (t.swapped) {
    std::swap(a, b);
    std::swap(t.rows, t.cols);
  }
  t.a_k_major = a.k_major;
  t.b_k_major = b.k_major;
  const bool wide = p.f.ldy % 8 == 0 && aligned16(p.f.y) &&
                    (!p.f.residual || (p.f.ldr % 8 == 0 && aligned16(p.f.residual))) &&
                    (!p.f.pre || (p.cols % 4 == 0 && aligned16(p.f.pre)));
  // What the tiles of a width take: rounds of blocks, each with its share of k.
  const uint32_t sms = (uint32_t)ctx->num_sms, ks = (p.depth + kTileK - 1) / kTileK;
  uint32_t bn = 0, parts = 1;
  double best = 0;
  for (uint32_t width : {256u, 128u, 64u, 32u, 16u}) {
    if (width < 64 && !b.k_major) break;
    if (width > (b.k_major ? 16u : 64u) && width / 2 >= t.cols) continue;
    const uint64_t tiles =
        (uint64_t)((t.rows + kTileA - 1) / kTileA) * ((t.cols + width - 1) / width);
    for (uint32_t s = 1; s <= 8; s *= 2) {
      if (s > 1 && (tiles * s > sms || s > ks)) break;
      const double rounds = (double)((tiles * s + sms - 1) / sms);
      const double took = rounds * ((width + 64.0) * ((ks + s - 1) / s) + (s > 1 ? 800 : 400));
      if (bn == 0 || took < best) {
        best = took;
        bn = width;
        parts = s;
      }
    }
  }
  auto go = [&](auto v) -> int {
    using T = decltype(v);
    switch (bn) {
      case 256: return launch<T, 256>(ctx, t, p, a, b, parts, wide);
      case 128: return launch<T, 128>(ctx, t, p, a, b, parts, wide);
      case 64: return launch<T, 64>(ctx, t, p, a, b, parts, wide);
      case 32: return launch<T, 32>(ctx, t, p, a, b, parts, wide);
      default: return launch<T, 16>(ctx, t, p, a, b, parts, wide);
    }
  };
  return dtype == PLX_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

}  // namespace plx
