// Products of rows and weights on the tensor cores. 32-bit values come as three
// planes of 16 bits each (dense.cu); a stage has all three of both operands, and the
// six products of planes that matter are made of it, the small ones first. The tensor
// cores cut sums off, they do not round them: a stage's sums are therefore taken to
// registers and added there, which is as exact as multiply-adds in 32 bits (all in
// TMEM were off by 1e-5 after 1,000 values of k). 16-bit values' sums stay there for up
// to 16,384 (float16) or 131,072 (bfloat16) values of k: a step of 16 of them costs 3.4 x
// 2^-24 of the sum so far where terms have one sign (measured), so that it comes out a
// fifth of the type's half step too small then; longer sums (LONG) leave TMEM as often
// (weights' gradients of 131,072 rows of 4,096 x 1,024 f16 902 -> 970 us).
//
// Bound by the products (large calls) or by reading the weights (few rows). A
// block makes tiles of 128 x BN sums: one thread has tensor copies fill a ring of
// stages of 64 values of k, one issues the products on them, eight warps finish
// the tile before (bias, activation, residual, rounding) out of the other half of
// TMEM meanwhile. Blocks stay and take every gridDim-th tile.
// PAIR: two blocks make a tile of 256 x 256 together, each with half of both
// operands, so that what a block reads is two thirds of what it reads for 128 x 256
// (all blocks together read as fast as L2 gives).
// SPLIT: where tiles are few, a cluster of blocks shares one tile's k: each sends
// its sums to the blocks' shared memory, and each block adds and finishes the rows
// of the tile that are its own, in the order of the blocks.
// Few rows (at most 64) are the tile's second side, so that the first one's 128
// are units of the layer.
// Measured, 16,384 x 4,096 x 4,096 bf16 with bias, GELU and residual: 431 us for some
// milliseconds, 500 (1.1 PFLOP/s) for seconds on end under the power cap, 456 of them
// without bias, activation and residual, where the library's product takes 400. Results
// stored from registers, 16 bytes a lane, and biases read one by one took 24 us a tile
// to finish, now 11, beside 29 of products. What is left is the tiles' operands out of
// L2: 454 ns for 64 values of k where the tensor cores need 280 at full clock. 1,501 x
// 1,001 x 777 f32 34 us (library 73), its weights' gradient on wide tiles shared by two
// blocks 29 (64), on tiles of 64 columns 45; 8 rows against 4,096 x 4,096 weights 13 us, of
// which 5 are memory's, the rest start, joining and finish.
#include <algorithm>

#include "cluster.cuh"
#include "dense.cuh"
#include "tensor.cuh"

namespace plx {
namespace {

constexpr uint32_t kTileA = 128, kTileK = 64;
constexpr int kFinishWarps = 8, kThreads = 64 + 32 * kFinishWarps;
constexpr uint32_t kSmem = 232448;  // a block can have

enum Mode { ONE, SPLIT, PAIR };

template <typename T, int BN, Mode MODE, bool LONG>
struct Stages {
  static constexpr uint32_t planes = sizeof(T) == 4 ? 3 : 1;
  // Sums leave TMEM after so many stages, for registers that add them up.
  static constexpr bool by_stage = sizeof(T) == 4 || LONG;
  static constexpr uint32_t period =
      sizeof(T) == 4 ? 1 : std::is_same_v<T, __half> ? 256 : 2048;
  static constexpr uint32_t b_rows = MODE == PAIR ? BN / 2 : BN;  // a block's
  static constexpr uint32_t a_bytes = kTileA * kTileK * 2, b_bytes = b_rows * kTileK * 2;
  static constexpr uint32_t bytes = planes * (a_bytes + b_bytes);
  // Sums that the blocks of a cluster are sent, of a tile in all; in the ring's place
  // where all blocks are done with that first (by_stage: sums are in registers).
  static constexpr uint32_t sent = MODE == SPLIT ? (BN + 4) * kTileA * 4 : 0;
  static constexpr uint32_t sums = by_stage ? 0 : sent;
  // pieces of results (32 rows of 128 bytes) on their way out, of each warp
  static constexpr uint32_t pieces =
      MODE == SPLIT || BN < 128 ? 0 : MODE == PAIR || sizeof(T) == 2 ? 2 : 1;

  static constexpr uint32_t out = pieces * kFinishWarps * 4096;
  static constexpr uint32_t most = (kSmem - 2048 - sums - out) / bytes;
  static constexpr uint32_t count = most < 12 ? most : 12;
  static_assert(count >= 2, "copies beside products");
  static_assert(!by_stage || count * bytes >= sent, "room for sums");
  static constexpr uint32_t smem = count * bytes + out + sums + 1024;  // to a multiple of 1,024
  static constexpr uint32_t columns = 2 * BN < 32 ? 32 : 2 * BN;
};

struct TensorProduct {
  CUtensorMap a[3], b[3];  // a has the tile's 128; planes of 32-bit values
  CUtensorMap y, residual, pre;  // where results go by tensor copies
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

template <typename T, int C>
__device__ __forceinline__ void activate(int act, float (&v)[C]) {
  auto all = [&](auto a) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      v[i] = sizeof(T) == 2 ? act_value16<decltype(a)::value>(v[i])
                            : act_value<decltype(a)::value>(v[i]);
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
  if (std::is_same_v<T, __half> && f.factor) z *= *f.factor;
  float v[1] = {f.bias ? z + bias_at<T>(f, col) : z};
  if (f.pre) f.pre[(uint64_t)row * cols + col] = v[0];
  activate<T>(f.act, v);
  if (f.residual) v[0] += to_f32(((const T*)f.residual)[(int64_t)row * f.ldr + col]);
  ((T*)f.y)[(int64_t)row * f.ldy + col] = from_f32<T>(v[0]);
}

// Applies the factor to C consecutive columns and adds their bias; `wide`: all there, in
// 16-byte pieces.
template <typename T, int C>
__device__ __forceinline__ void add_bias(const Finish& f, uint32_t col, uint32_t cols, bool wide,
                                         float (&v)[C]) {
  if (std::is_same_v<T, __half> && f.factor) {
    const float by = *f.factor;
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] *= by;
  }
  if (!f.bias) return;
  if (!wide) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (col + i < cols) v[i] += bias_at<T>(f, col + i);
  } else if (f.param_dtype == PLX_F32) {
    Pack<float, 4> q[C / 4];
#pragma unroll
    for (int i = 0; i < C / 4; ++i) q[i] = load_pack<float, 4>((const float*)f.bias + col + i * 4);
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += q[i / 4].v[i % 4];
  } else {
    constexpr int N = C < 8 ? C : 8;
    Pack<T, N> q[C / N];
#pragma unroll
    for (int i = 0; i < C / N; ++i) q[i] = load_pack<T, N>((const T*)f.bias + col + i * N);
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += to_f32(q[i / N].v[i % N]);
  }
}

// A thread's C consecutive columns of a row of the result; `wide`: all there, in
// 16-byte pieces.
template <typename T, int C>
__device__ __forceinline__ void finish_row(const Finish& f, uint32_t row, uint32_t col,
                                           uint32_t cols, bool wide, float (&v)[C]) {
  add_bias<T, C>(f, col, cols, wide, v);
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
  activate<T>(f.act, v);
  T* to = (T*)f.y + (int64_t)row * f.ldy + col;
  const T* res = (const T*)f.residual + (int64_t)row * f.ldr + col;
  if (wide) {
    constexpr int N = C < 8 ? C : 8;
#pragma unroll
    for (int i = 0; i < C; i += N) {
      Pack<T, N> q;
      if (f.residual) {
        q = load_pack<T, N>(res + i);
#pragma unroll
        for (int e = 0; e < N; ++e) v[i + e] += to_f32(q.v[e]);
      }
#pragma unroll
      for (int e = 0; e < N; e += 2) put_pair(q, e, pack2(v[i + e], v[i + e + 1]));
      *reinterpret_cast<Pack<T, N>*>(to + i) = q;
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

template <typename T, int BN, Mode MODE, bool LONG>
__global__ void __launch_bounds__(kThreads, 1)
k_product_tensor(const __grid_constant__ TensorProduct p, bool wide) {
  using S = Stages<T, BN, MODE, LONG>;
  constexpr bool TWO = MODE == PAIR;
  constexpr uint32_t C = BN <= 32 ? 16 : 32;  // columns at a time, at most half of a tile's
  static_assert(BN == 16 || BN % (2 * C) == 0, "halves of a tile");
  constexpr uint32_t kHigh = TWO ? 2 * kTileA : kTileA;  // of a tile
  extern __shared__ __align__(128) uint8_t product_bytes[];
  uint8_t* ring = product_bytes + (1024 - (smem_addr(product_bytes) & 1023)) % 1024;
  uint8_t* out = ring + S::count * S::bytes;
  float* sent = reinterpret_cast<float*>(S::by_stage ? ring : out + S::out);
  constexpr int kPieces = S::pieces ? S::pieces : 1;
  __shared__ uint64_t arrived[kFinishWarps][kPieces];  // the residual's piece is there
  __shared__ uint64_t full[S::count], empty[S::count], done[2], taken[2];
  __shared__ uint32_t tmem, gave_up;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t blocks = (p.depth + kTileK - 1) / kTileK;
  uint32_t k_first = 0, k_last = blocks, rank = 0, parts = 1;
  uint32_t tile0 = blockIdx.x, step = gridDim.x;
  const uint32_t tiles = p.tiles_a * p.tiles_b;
  if constexpr (MODE == SPLIT) {
    rank = cluster_rank();
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(parts));
    tile0 = blockIdx.x / parts;
    step = tiles;  // one tile
    const uint32_t each = (blocks + parts - 1) / parts;
    k_first = min(rank * each, blocks);
    k_last = min(k_first + each, blocks);
  } else if constexpr (TWO) {
    rank = cluster_rank();
    tile0 = blockIdx.x / 2;
    step = gridDim.x / 2;
  }
  // Tiles in groups of eight along a's side, so that what is under way at one
  // time shares both operands.
  auto place = [&](uint32_t tile, uint32_t& ia, uint32_t& ib) {
    const uint32_t group = 8 * p.tiles_b, first = tile / group * 8;
    const uint32_t size = min(p.tiles_a - first, 8u), in = tile % group;
    ia = first + in % size;
    ib = in / size;
  };
  // Starts the copies of a stage.
  auto load_stage = [&](uint32_t s, uint32_t ia, uint32_t ib, uint32_t k) {
    const int a0 = (int)(ia * kHigh + (TWO ? rank * kTileA : 0));
    const int b0 = (int)(ib * BN + (TWO ? rank * S::b_rows : 0)), k0 = (int)(k * kTileK);
    // a pair's first block counts the bytes of both
    const uint32_t bar = TWO ? peer_smem(&full[s], 0) : 0;
    if (!TWO || rank == 0) mbar_arrive_expect_tx(&full[s], TWO ? 2 * S::bytes : S::bytes);
    auto load = [&](uint8_t* to, const CUtensorMap* map, int x, int y) {
      if constexpr (TWO) tensor_load_pair(to, map, x, y, bar);
      else tensor_load(to, map, x, y, &full[s]);
    };
#pragma unroll
    for (uint32_t q = 0; q < S::planes; ++q) {
      uint8_t* a = ring + s * S::bytes + q * S::a_bytes;
      uint8_t* b = ring + s * S::bytes + S::planes * S::a_bytes + q * S::b_bytes;
      if (p.a_k_major) {
        load(a, &p.a[q], k0, a0);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < kTileA / 64; ++j) load(a + j * 8192, &p.a[q], a0 + j * 64, k0);
      }
      if (p.b_k_major) {
        load(b, &p.b[q], k0, b0);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < (S::b_rows + 63) / 64; ++j)
          load(b + j * 8192, &p.b[q], b0 + j * 64, k0);
      }
    }
  };
  uint32_t early = 0;  // stages of the first tile that are under way before all else is ready
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < S::count; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int h = 0; h < 2; ++h) {
      mbar_init(&done[h], 1);
      mbar_init(&taken[h], TWO ? 2 * kFinishWarps : kFinishWarps);
    }
    for (int w = 0; w < kFinishWarps; ++w)
      for (int i = 0; i < kPieces; ++i) mbar_init(&arrived[w][i], 1);
    mbar_init_fence();
    gave_up = 0;
    if constexpr (!TWO) {  // (a pair's barriers are not this block's alone)
      uint32_t ia, ib;
      place(tile0, ia, ib);
      for (; early < S::count && k_first + early < k_last; ++early)
        load_stage(early, ia, ib, k_first + early);
    }
  }
  if (warp == 1) tmem_alloc<TWO>(&tmem, S::columns);
  tmem_fence_before();
  __syncthreads();
  // The others' barriers are there; SPLIT: and their memory, by the time that sums are
  // sent (by_stage: once they have made their sums).
  if constexpr (TWO) cluster_barrier();
  if constexpr (MODE == SPLIT && !S::by_stage) cluster_arrive();
  auto others_ready = [&] {
    if constexpr (S::by_stage) cluster_arrive();
    cluster_wait();
  };
  tmem_fence_after();
  const uint32_t sums = *(volatile uint32_t*)&tmem;

  if (warp == 0 && lane == 0) {  // copies
    uint32_t it = 0;
    bool ok = true;
    for (uint32_t tile = tile0; ok && tile < tiles; tile += step) {
      uint32_t ia, ib;
      place(tile, ia, ib);
      for (uint32_t k = k_first; k < k_last; ++k, ++it) {
        if (it < early) continue;
        const uint32_t s = it % S::count;
        if (it >= S::count && !(ok = wait(&empty[s], (it / S::count - 1) & 1, &gave_up, p))) break;
        load_stage(s, ia, ib, k);
      }
    }
    if (!ok && (!TWO || rank == 0))  // what is still on its way
      for (uint32_t j = it > S::count ? it - S::count : 0; j < it; ++j)
        mbar_wait_bounded(&full[j % S::count], (j / S::count) & 1, p.timeout_ns);
  } else if (warp == 1 && lane == 0 && (!TWO || rank == 0)) {  // products
    uint32_t it = 0, turn = 0;
    bool ok = true;
    // TMEM's other half, once its sums have been taken
    auto next_half = [&] {
      if (turn >= 2) ok = wait(&taken[turn & 1], (turn / 2 - 1) & 1, &gave_up, p);
      tmem_fence_after();
      return sums + (turn & 1) * BN;
    };
    for (uint32_t tile = tile0; ok && tile < tiles; tile += step) {
      uint32_t to = 0;
      if constexpr (!S::by_stage) {
        to = next_half();
        if (!ok) break;
      }
      for (uint32_t k = k_first; k < k_last; ++k, ++it) {
        const uint32_t in = S::by_stage ? (k - k_first) % S::period : k - k_first;
        if constexpr (S::by_stage) {
          if (in == 0) to = next_half();
          if (!ok) break;
        }
        const uint32_t s = it % S::count;
        if (!(ok = wait(&full[s], (it / S::count) & 1, &gave_up, p))) break;
        tmem_fence_after();
        const uint8_t* at = ring + s * S::bytes;
        // 16 values of k further on: 32 bytes of a row, or sixteen rows
        const uint32_t da = p.a_k_major ? 2 : 128, db = p.b_k_major ? 2 : 128;
        // of the planes, the smallest products first
        constexpr uint32_t kProducts = S::planes == 3 ? 6 : 1;
        constexpr uint8_t plane_a[6] = {1, 0, 2, 0, 1, 0}, plane_b[6] = {1, 2, 0, 1, 0, 0};
#pragma unroll
        for (uint32_t q = 6 - kProducts; q < 6; ++q) {
          const uint8_t* at_a = at + plane_a[q] * S::a_bytes;
          const uint8_t* at_b = at + S::planes * S::a_bytes + plane_b[q] * S::b_bytes;
          const uint64_t a = p.a_k_major ? operand_k_major(at_a) : operand_i_major(at_a, 8192);
          const uint64_t b = p.b_k_major ? operand_k_major(at_b) : operand_i_major(at_b, 8192);
#pragma unroll
          for (uint32_t j = 0; j < kTileK / 16; ++j)
            tensor_product<TWO>(to, a + j * da, b + j * db, p.kind,
                                in > 0 || q > 6 - kProducts || j > 0);
        }
        products_arrive<TWO>(&empty[s]);
        if constexpr (S::by_stage) {
          if (in + 1 == S::period || k + 1 == k_last) products_arrive<TWO>(&done[turn++ & 1]);
        }
      }
      if constexpr (!S::by_stage) {
        if (ok) products_arrive<TWO>(&done[turn++ & 1]);
      }
    }
  } else if (warp >= 2) {  // finishing
    const uint32_t quarter = warp % 4, side = (warp - 2) / 4;  // lanes of TMEM; half of the columns
    uint32_t turn = 0, arrivals = 0;  // the parities of `arrived`
    // What the sums of a tile have come to, of this thread's columns.
    constexpr uint32_t kMine = BN < 32 ? BN : BN / 2;
    float acc[S::by_stage ? kMine : 1];
    auto let_go = [&](uint32_t half) {
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (TWO) mbar_arrive_peer(peer_smem(&taken[half], 0));
        else mbar_arrive(&taken[half]);
      }
    };
    for (uint32_t tile = tile0; tile < tiles; tile += step) {
      uint32_t ia, ib;
      place(tile, ia, ib);
      const uint32_t half = turn & 1;
      // on a's side
      const uint32_t i = ia * kHigh + (TWO ? rank * kTileA : 0) + quarter * 32 + lane;
      // Pieces of 32 rows of 128 bytes go out through shared memory, by tensor copies or
      // (rows that are no multiples of 16 bytes) row by row. The residual's are on
      // their way in before the sums are done.
      constexpr uint32_t kWide = 128 / sizeof(T), kChunks = S::pieces ? BN / 2 / kWide : 0;
      constexpr uint32_t kHalves = kWide / 32;
      const uint32_t row0 = i - lane, col0 = ib * BN + side * (BN / 2);
      constexpr bool staged = S::pieces > 0;
      constexpr uint32_t kFirst = kChunks < kPieces ? kChunks : kPieces;  // under way at once
      auto piece = [&](uint32_t c) { return out + ((warp - 2) * kPieces + c % kPieces) * 4096; };
      auto there = [&](uint32_t c) { return row0 < p.rows && col0 + c * kWide < p.cols; };
      auto fetch = [&](uint32_t c) {  // by one lane, which has stored what was there
        if (!there(c)) return;
        uint64_t* bar = &arrived[warp - 2][c % kPieces];
        mbar_arrive_expect_tx(bar, 4096);
        tensor_load(piece(c), &p.residual, (int)(col0 + c * kWide), (int)row0, bar);
      };
      const bool fetched = staged && wide && p.f.residual;
      if constexpr (staged) {
        if (fetched && lane == 0) {
          bulk_wait_read<0>();
          for (uint32_t c = 0; c < kFirst; ++c) fetch(c);
        }
      }
      const uint32_t column = sums + (quarter << 21) + (BN < 32 ? 0 : side * (BN / 2));
      bool sound = true;
      if constexpr (S::by_stage) {
#pragma unroll
        for (uint32_t e = 0; e < kMine; ++e) acc[e] = 0.0f;
        for (uint32_t k = k_first; sound && k < k_last; k += S::period, ++turn) {
          sound = __all_sync(~0u, wait(&done[turn & 1], (turn / 2) & 1, &gave_up, p));
          tmem_fence_after();
          if (!sound) break;
#pragma unroll
          for (uint32_t c = 0; c < kMine; c += C) {
            float v[C];
            if constexpr (C == 32) tmem_load32(column + (turn & 1) * BN + c, v);
            else tmem_load16(column + (turn & 1) * BN + c, v);
#pragma unroll
            for (uint32_t e = 0; e < C; ++e) acc[c + e] += v[e];
          }
          let_go(turn & 1);
        }
      } else {
        sound = __all_sync(~0u, wait(&done[half], (turn / 2) & 1, &gave_up, p));
        tmem_fence_after();
      }
      // C of this thread's sums, from column c of its own.
      auto take = [&](uint32_t c, float (&v)[C]) {
        if constexpr (S::by_stage) {
#pragma unroll
          for (uint32_t e = 0; e < C; ++e) v[e] = acc[c + e];
        } else if constexpr (C == 32) {
          tmem_load32(column + half * BN + c, v);
        } else {
          tmem_load16(column + half * BN + c, v);
        }
      };
      constexpr int kUnroll = S::by_stage ? 8 : 1;  // registers have no addresses
      if constexpr (MODE == SPLIT) others_ready();
      if (!sound && MODE != SPLIT) {
        if constexpr (staged)
          if (fetched && lane == 0)  // what is still on its way
            for (uint32_t c = 0; c < kFirst; ++c)
              if (there(c))
                mbar_wait_bounded(&arrived[warp - 2][c], arrivals >> c & 1, p.timeout_ns);
        break;
      }
      if constexpr (staged) {
        // of this lane's row, the 16-byte chunk k of a piece; and value `col` of a row
        auto chunk = [&](uint8_t* of, uint32_t k) {
          return of + lane * 128 + ((k ^ (lane & 7)) << 4);
        };
        auto value = [&](auto* of, uint32_t row, uint32_t col) {
          using Q = std::remove_pointer_t<decltype(of)>;
          const uint32_t byte = col * sizeof(Q);
          return reinterpret_cast<Q*>(reinterpret_cast<uint8_t*>(of) + row * 128 +
                                      (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15));
        };
        // Sends a piece out: columns from j0 of rows from row0 of an array.
        auto send = [&](const CUtensorMap* map, auto* array, int64_t ld, uint32_t j0, uint8_t* of) {
          using Q = std::remove_pointer_t<decltype(array)>;
          if (wide) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tensor_store(map, (int)j0, (int)row0, of);
              bulk_commit();
            }
          } else {
            __syncwarp();
            const uint32_t rows = min(32u, p.rows - row0);
#pragma unroll
            for (uint32_t col = lane; col < 128 / sizeof(Q); col += 32) {
              if (j0 + col >= p.cols) continue;
              Q* to = array + (int64_t)row0 * ld + j0 + col;
#pragma unroll 8
              for (uint32_t r = 0; r < rows; ++r, to += ld)
                *to = *value(reinterpret_cast<Q*>(of), r, col);
            }
            __syncwarp();
          }
        };
#pragma unroll kUnroll
        for (uint32_t c = 0; c < kChunks; ++c) {
          if (!there(c)) continue;
          uint8_t* at = piece(c);
          const uint32_t j1 = col0 + c * kWide;
          if (fetched) {
            wait(&arrived[warp - 2][c % kPieces], arrivals >> (c % kPieces) & 1, &gave_up, p);
            arrivals ^= 1u << (c % kPieces);
          } else if (p.f.residual) {
            const T* res = (const T*)p.f.residual;
            const uint32_t rows = min(32u, p.rows - row0);
#pragma unroll
            for (uint32_t col = lane; col < kWide; col += 32) {
              if (j1 + col >= p.cols) continue;
              const T* from = res + (int64_t)row0 * p.f.ldr + j1 + col;
#pragma unroll 8
              for (uint32_t r = 0; r < rows; ++r, from += p.f.ldr)
                *value(reinterpret_cast<T*>(at), r, col) = *from;
            }
            __syncwarp();
          } else if (wide) {
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
          }
#pragma unroll (S::by_stage ? 2 : 1)
          for (uint32_t h = 0; h < kHalves; ++h) {
            float v[32];
            take(c * kWide + h * 32, v);
            const uint32_t j0 = j1 + h * 32;
            add_bias<T, 32>(p.f, j0, p.cols, wide && j0 + 32 <= p.cols, v);
            if (p.f.pre) {
              // the other piece takes it out, or the same one before the result (of as
              // many columns)
              if (!p.f.residual && (kPieces == 2 || sizeof(T) == 4)) {
                uint8_t* z = piece(c + 1);
                if (wide) {
                  if (lane == 0) bulk_wait_read<0>();
                  __syncwarp();
                }
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k)
                  *reinterpret_cast<float4*>(chunk(z, k)) =
                      make_float4(v[k * 4], v[k * 4 + 1], v[k * 4 + 2], v[k * 4 + 3]);
                if (j0 < p.cols) send(&p.pre, p.f.pre, (int64_t)p.cols, j0, z);
                if (kPieces == 1 && wide) {
                  if (lane == 0) bulk_wait_read<0>();
                  __syncwarp();
                }
              } else if (i < p.rows) {
                float* to = p.f.pre + (uint64_t)i * p.cols + j0;
                if (wide && j0 + 32 <= p.cols) {
#pragma unroll
                  for (uint32_t k = 0; k < 32; k += 4)
                    *reinterpret_cast<float4*>(to + k) =
                        make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                } else {
#pragma unroll
                  for (uint32_t k = 0; k < 32; ++k)
                    if (j0 + k < p.cols) to[k] = v[k];
                }
              }
            }
            activate<T>(p.f.act, v);
            constexpr uint32_t N = 16 / sizeof(T);
#pragma unroll
            for (uint32_t k = 0; k < 32 / N; ++k) {
              auto* q = reinterpret_cast<Pack<T, N>*>(chunk(at, h * 4 + k));
              Pack<T, N> o;
              if (p.f.residual) {
                o = *q;
#pragma unroll
                for (int e = 0; e < N; ++e) v[k * N + e] += to_f32(o.v[e]);
              }
#pragma unroll
              for (int e = 0; e < N; e += 2) put_pair(o, e, pack2(v[k * N + e], v[k * N + e + 1]));
              *q = o;
            }
          }
          send(&p.y, (T*)p.f.y, p.f.ldy, j1, at);
          if (fetched && lane == 0 && c + kPieces < kChunks) {
            bulk_wait_read<0>();
            fetch(c + kPieces);
          }
        }
      }
      if constexpr (!staged)
#pragma unroll kUnroll
      for (uint32_t mine = 0; mine < kMine; mine += C) {
        float v[C];
        if (BN < 32 && side) break;
        const uint32_t c = mine + (BN < 32 ? 0 : side * (BN / 2));
        take(mine, v);
        const uint32_t j0 = ib * BN + c;
        if constexpr (MODE == SPLIT) {
          if (k_last <= k_first)
#pragma unroll
            for (uint32_t e = 0; e < C; ++e) v[e] = 0.0f;
          // to the block that the row is of: [block that sends][row of its own][column]
          const uint32_t row = quarter * 32 + lane;
          if (p.swapped) {
            const uint32_t own = BN / parts;
#pragma unroll
            for (uint32_t e = 0; e < C; ++e)
              st_peer(peer_smem(sent + (rank * own + (c + e) % own) * kTileA + row, (c + e) / own),
                      v[e]);
          } else {
            const uint32_t own = kTileA / parts;
            const uint32_t to =
                peer_smem(sent + (rank * own + row % own) * (BN + 4) + c, row / own);
#pragma unroll
            for (uint32_t e = 0; e < C; e += 4)
              st_peer(to + e * 4, make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]));
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
      if constexpr (!S::by_stage) {
        let_go(half);
        ++turn;
      }
    }
    if (S::pieces && lane == 0) bulk_wait_all<0>();
  }
  __syncwarp();
  if constexpr (MODE == SPLIT)
    if (warp < 2) others_ready();
  tmem_fence_before();
  __syncthreads();
  if constexpr (MODE != ONE) cluster_barrier();  // SPLIT: every block's sums are there
  tmem_fence_after();
  __syncwarp();
  if (warp == 1) tmem_free<TWO>(sums, S::columns);
  if constexpr (MODE == SPLIT) {
    uint32_t ia, ib;
    place(tile0, ia, ib);
    const uint32_t inner = p.swapped ? kTileA : BN, own = (p.swapped ? BN : kTileA) / parts;
    const uint32_t pitch = p.swapped ? kTileA : BN + 4;
    const uint32_t rows = p.swapped ? p.cols : p.rows, cols = p.swapped ? p.rows : p.cols;
    for (uint32_t at = threadIdx.x; at < own * inner / 4; at += kThreads) {
      const uint32_t o = at / (inner / 4), n = at % (inner / 4) * 4;
      const uint32_t row = (p.swapped ? ib * BN : ia * kTileA) + rank * own + o;
      const uint32_t col = (p.swapped ? ia * kTileA : ib * BN) + n;
      if (row >= rows || col >= cols) continue;
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (uint32_t r = 0; r < parts; ++r) {
        const float4 z = *reinterpret_cast<const float4*>(sent + (r * own + o) * pitch + n);
        v[0] += z.x;
        v[1] += z.y;
        v[2] += z.z;
        v[3] += z.w;
      }
      finish_row<T, 4>(p.f, row, col, cols, wide && col + 4 <= cols, v);
    }
  }
}

template <typename T, int BN, Mode MODE, bool LONG = false>
int launch(plx_ctx* ctx, TensorProduct& t, const Product& p, const Operand& a, const Operand& b,
           uint32_t parts, bool wide) {
  using S = Stages<T, BN, MODE, LONG>;
  constexpr bool bf16 = !std::is_same_v<T, __half>;  // what is multiplied
  constexpr uint32_t high = MODE == PAIR ? 2 * kTileA : kTileA;
  t.tiles_a = (t.rows + high - 1) / high;
  t.tiles_b = (t.cols + BN - 1) / BN;
  t.kind = product_kind(bf16, !a.k_major, !b.k_major, high, BN);
  auto maps = [&](CUtensorMap (&m)[3], const Operand& o, uint32_t count, uint32_t tile) {
    for (int plane = 0; plane < (int)S::planes; ++plane)
      if (int rc = tensor_map(&m[plane], bf16 ? PLX_BF16 : PLX_F16,
                              (const char*)o.p + plane * o.plane, o.k_major ? t.depth : count,
                              o.k_major ? count : t.depth, o.ld, 64,
                              o.k_major ? tile : kTileK, true))
        return rc;
    return PLX_OK;
  };
  if (int rc = maps(t.a, a, t.rows, kTileA)) return rc;
  if (int rc = maps(t.b, b, t.cols, S::b_rows)) return rc;
  if (S::pieces && wide) {
    const int dtype = sizeof(T) == 4 ? PLX_F32 : bf16 ? PLX_BF16 : PLX_F16;
    auto map = [&](CUtensorMap* m, int of, const void* q, int64_t ld) {
      return tensor_map(m, of, q, t.cols, t.rows, ld, of == PLX_F32 ? 32 : 64, 32, true);
    };
    if (int rc = map(&t.y, dtype, p.f.y, p.f.ldy)) return rc;
    if (p.f.residual)
      if (int rc = map(&t.residual, dtype, p.f.residual, p.f.ldr)) return rc;
    if (p.f.pre)
      if (int rc = map(&t.pre, PLX_F32, p.f.pre, t.cols)) return rc;
  }
  const uint64_t tiles = (uint64_t)t.tiles_a * t.tiles_b;
  if (tiles >= (1ull << 28))
    return set_error(PLX_ERR_CAPACITY, "%u x %u results are too many for one call", p.rows, p.cols);
  constexpr auto kernel = k_product_tensor<T, BN, MODE, LONG>;
  PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, S::smem));
  cudaLaunchConfig_t cfg = {};
  const uint32_t sms = (uint32_t)ctx->num_sms;
  cfg.gridDim = dim3((unsigned)(MODE == SPLIT  ? tiles * parts
                                : MODE == PAIR ? 2 * std::min<uint64_t>(tiles, sms / 2)
                                               : std::min<uint64_t>(tiles, sms)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::smem;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = MODE == SPLIT ? parts : 2;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = MODE == ONE ? 0 : 1;
  PLX_TRY_CUDA(cudaLaunchKernelEx(&cfg, kernel, (const TensorProduct)t, wide));
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
  const int per = 16 / (int)dtype_bytes(dtype);
  const bool wide = p.f.ldy % per == 0 && aligned16(p.f.y) &&
                    (!p.f.residual || (p.f.ldr % per == 0 && aligned16(p.f.residual))) &&
                    (!p.f.pre || (p.cols % 4 == 0 && aligned16(p.f.pre))) && aligned16(p.f.bias);
  // What the tiles of a width take: rounds of blocks, each with its share of k (a unit is
  // the products of 64 values of k by one column). A block waits for its products or
  // for its operands, of 128 + width rows; starting and finishing a tile takes 500
  // units, sending and joining a shared one's sums another 500, of wide tiles of 32-bit
  // values more. Blocks of a cluster are neighbours, so that 33 clusters of 4 and 15 of 8
  // have room at once; one more waits for a whole round (256 x 1,024 x 1,024 f32 on 16
  // clusters of 8: 23 us; on tiles of 64 columns 15).
  const bool f32 = dtype == PLX_F32;
  const uint32_t sms = (uint32_t)ctx->num_sms, ks = (p.depth + kTileK - 1) / kTileK;
  // by products; by their operands out of shared memory; by copies into it. (The factors,
  // and with them the 500, 1,000 and 1,300 + 150 s below, are fitted to measured calls:
  // six products of planes cost six times one, their operands' three planes three to six
  // times one.)
  auto step_of = [&](uint32_t width, uint32_t b_rows) {
    const double read = 128 + b_rows;
    return std::max({(f32 ? 6.3 : 1.05) * width, (f32 ? 3.45 : 0.575) * read,
                     (f32 ? 2.7 : 0.9) * read});
  };
  uint32_t bn = 0, parts = 1;
  bool pair = false;
  double best = 0;
  for (uint32_t width : {256u, 128u, 64u, 32u, 16u}) {
    if (width < 64 && !b.k_major) break;
    if (width > 128 && f32) continue;
    if (width > (b.k_major ? 16u : 64u) && width / 2 >= t.cols) continue;
    const uint64_t tiles =
        (uint64_t)((t.rows + kTileA - 1) / kTileA) * ((t.cols + width - 1) / width);
    for (uint32_t s = 1; s <= 8; s *= 2) {
      const uint32_t room = s < 4 ? sms : s == 4 ? sms * 8 / 9 : sms * 4 / 5;
      if (s > 1 && (tiles * s > room || s > ks || width > 128)) break;
      const double rounds = (double)((tiles * s + sms - 1) / sms);
      const double took =
          rounds * (step_of(width, width) * ((ks + s - 1) / s) +
                    (s == 1 ? 500 : f32 && width == 128 ? 1300 + 150 * s : 1000));
      if (bn == 0 || took < best) {
        best = took;
        bn = width;
        parts = s;
      }
    }
  }
  if (t.rows > kTileA && t.cols > 64) {
    const uint32_t width = f32 ? 128 : 256;
    const uint64_t tiles =
        (uint64_t)((t.rows + 2 * kTileA - 1) / (2 * kTileA)) * ((t.cols + width - 1) / width);
    const double rounds = (double)((tiles + sms / 2 - 1) / (sms / 2));
    pair = rounds * (step_of(width, width / 2) * ks + 500) < best;
  }
  auto go = [&](auto v) -> int {
    using T = decltype(v);
    constexpr int WIDEST = sizeof(T) == 4 ? 128 : 256;  // stages of 32-bit values are long
    const bool split = parts > 1;
    if constexpr (sizeof(T) == 2) {
      // sums too long for TMEM
      if ((pair ? ks : (ks + parts - 1) / parts) > Stages<T, 128, ONE, true>::period) {
        if (pair) return launch<T, 256, PAIR, true>(ctx, t, p, a, b, 1, wide);
        if (bn == 256) return launch<T, 256, ONE, true>(ctx, t, p, a, b, 1, wide);
        if (bn == 128)
          return (split ? launch<T, 128, SPLIT, true> : launch<T, 128, ONE, true>)(ctx, t, p, a, b,
                                                                                  parts, wide);
        return (split ? launch<T, 64, SPLIT, true> : launch<T, 64, ONE, true>)(ctx, t, p, a, b,
                                                                              parts, wide);
      }
    }
    if (pair) return launch<T, WIDEST, PAIR>(ctx, t, p, a, b, 1, wide);
    switch (bn) {
      case 256: return launch<T, WIDEST, ONE>(ctx, t, p, a, b, parts, wide);
      case 128:
        return (split ? launch<T, 128, SPLIT> : launch<T, 128, ONE>)(ctx, t, p, a, b, parts,
                                                                     wide);
      case 64:
        return (split ? launch<T, 64, SPLIT> : launch<T, 64, ONE>)(ctx, t, p, a, b, parts, wide);
      case 32:
        return (split ? launch<T, 32, SPLIT> : launch<T, 32, ONE>)(ctx, t, p, a, b, parts, wide);
      default:
        return (split ? launch<T, 16, SPLIT> : launch<T, 16, ONE>)(ctx, t, p, a, b, parts, wide);
    }
  };
  return with_dtype(dtype, go);
}

}  // namespace plx
