// One pass over a row of logits (log_probs.cu, distill.cu): the running maximum
// m, s = sum 2^((x-m)c) and t = sum 2^((x-m)c) (x-m) of a thread's share, joined
// over a block and over the blocks of a cluster.
//
// A row may start anywhere: its 16-byte pieces are read whole, the elements
// before the first and after the last piece one by one. "Unit" below is such a
// piece or single element; units are disjoint and ordered by their first index.
#pragma once

#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "rows.cuh"

namespace plx {

namespace cg = cooperative_groups;

// ---- sixteen bytes of a row ----------------------------------------------
template <typename T>
struct Piece;
template <>
struct Piece<float> {
  static constexpr int V = 4;
  // Value pair k of the piece.
  static __device__ __forceinline__ F2 pair(const uint4& q, int k) {
    return k == 0 ? pack2(__uint_as_float(q.x), __uint_as_float(q.y))
                  : pack2(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  template <int N>
  static __device__ __forceinline__ float most(const uint4* q) {
    float m = __uint_as_float(q[0].x);
#pragma unroll
    for (int u = 0; u < N; ++u)
      m = max_nan(max_nan(max_nan(m, __uint_as_float(q[u].x)), __uint_as_float(q[u].y)),
                  max_nan(__uint_as_float(q[u].z), __uint_as_float(q[u].w)));
    return m;
  }
  static __device__ __forceinline__ void put(uint4& q, int k, float a, float b) {
    (&q.x)[2 * k] = __float_as_uint(a);
    (&q.x)[2 * k + 1] = __float_as_uint(b);
  }
};
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ F2 pair(const uint4& q, int k) {
    const uint32_t w = (&q.x)[k];
    return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) {
    return *reinterpret_cast<__nv_bfloat162*>(&w);
  }
  template <int N>
  static __device__ __forceinline__ float most(const uint4* q) {
    __nv_bfloat162 m = two(q[0].x);
#pragma unroll
    for (int u = 0; u < N; ++u)
      m = __hmax2_nan(__hmax2_nan(__hmax2_nan(m, two(q[u].x)), two(q[u].y)),
                      __hmax2_nan(two(q[u].z), two(q[u].w)));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void put(uint4& q, int k, float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    (&q.x)[k] = *reinterpret_cast<uint32_t*>(&v);
  }
};
template <>
struct Piece<__half> {
  static constexpr int V = 8;
  static __device__ __forceinline__ __half2 two(uint32_t w) {
    return *reinterpret_cast<__half2*>(&w);
  }
  static __device__ __forceinline__ F2 pair(const uint4& q, int k) {
    const float2 f = __half22float2(two((&q.x)[k]));
    return pack2(f.x, f.y);
  }
  template <int N>
  static __device__ __forceinline__ float most(const uint4* q) {
    __half2 m = two(q[0].x);
#pragma unroll
    for (int u = 0; u < N; ++u)
      m = __hmax2_nan(__hmax2_nan(__hmax2_nan(m, two(q[u].x)), two(q[u].y)),
                      __hmax2_nan(two(q[u].z), two(q[u].w)));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void put(uint4& q, int k, float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    (&q.x)[k] = *reinterpret_cast<uint32_t*>(&v);
  }
};

// What the threads of a block saw: each thread's pieces in up to kSlots runs of
// 2^shift, and of every run the upper half of its maximum's bits.
constexpr uint32_t kSlots = 8;
template <int THREADS>
struct Slots {
  uint16_t most[kSlots * THREADS];  // run s of thread i at s * THREADS + i
};

// ---- a contiguous share of a row -----------------------------------------
// Elements [start, start + count): `head` single ones, `pieces` whole pieces,
// `tail` single ones. Thread i of a block has head element i, pieces i, i + T,
// ... and tail element i.
template <typename T>
struct Share {
  const T* p;
  uint32_t start, count, head, pieces, tail;

  // Part `part` of a row of n, each part (but the last) part_length() long.
  __device__ __forceinline__ Share(const T* row, uint32_t n, uint32_t part, uint32_t each) {
    constexpr uint32_t V = Piece<T>::V;
    start = (uint32_t)min((uint64_t)n, (uint64_t)each * part);
    count = min(each, n - start);
    p = row + start;
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T);
    head = min(count, (V - off) % V);
    pieces = (count - head) / V;
    tail = count - head - pieces * V;
  }
  __device__ __forceinline__ uint32_t piece_at(uint32_t i) const {
    return head + i * Piece<T>::V;  // within the share
  }
  __device__ __forceinline__ uint32_t tail_at() const { return count - tail; }
  // Runs of 2^shift of a thread's pieces, kSlots at most.
  __device__ __forceinline__ uint32_t slot_shift(uint32_t threads) const {
    const uint32_t times = (pieces + threads * 4 * kSlots - 1) / (threads * 4 * kSlots);
    return times <= 1 ? 2 : 34 - __clz(times - 1);
  }
  // Calls f(true) if pieces of `out`, the same place in another row, are whole
  // 16-byte ones too, else f(false); as types, so that loops are made for each.
  template <typename F>
  __device__ __forceinline__ void with_whole(const T* out, F f) const {
    if ((reinterpret_cast<uintptr_t>(out + head) & 15u) == 0) f(std::true_type{});
    else f(std::false_type{});
  }
  template <bool WHOLE>
  __device__ __forceinline__ void put_piece(T* out, uint32_t i, const uint4& o, int on = 0) const {
    if (WHOLE) {
      (reinterpret_cast<uint4*>(out + head) + i)[on] = o;
    } else {
      T* to = out + piece_at(i + on);
      const T* e = reinterpret_cast<const T*>(&o);
#pragma unroll
      for (int k = 0; k < Piece<T>::V; ++k) to[k] = e[k];
    }
  }
  // Piece i, and one a constant further on: as pointer and constant, which a
  // load takes without arithmetic.
  __device__ __forceinline__ uint4 piece(uint32_t i, int on = 0) const {
    return (reinterpret_cast<const uint4*>(p + head) + i)[on];
  }
};

// Values a part: whole pieces, so that every part starts at the row's alignment.
inline uint32_t part_length(uint32_t n, uint32_t parts, uint32_t v) {
  return (uint32_t)((((uint64_t)n + parts - 1) / parts + v - 1) / v * v);
}

// The row a block works on: one a cluster (a block alone is its own).
__device__ __forceinline__ uint32_t cluster_row() {
  uint32_t r;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}

struct Sums {
  float m, s, t;
};

// Low bits of a value of type T that say nothing once it is 32 bits wide.
template <typename T>
constexpr int kSpareBits =
    std::is_same_v<T, __nv_bfloat16> ? 16 : std::is_same_v<T, __half> ? 13 : 0;

// A number that orders values: larger for larger ones, NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o == 0xffffffffu ? 0x7fffffffu : (o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

// In place of a difference of -inf (a masked value): 2^ of it is 0, and 0 times
// it is 0, not NaN.
constexpr float kFloor = -3.4028234664e38f;

// Moves s and t from maximum a to maximum b >= a (a = -inf: both are 0).
template <bool ENT>
__device__ __forceinline__ void rebase(Sums& v, float b, float c) {
  if (v.m != -INFINITY) {
    const float d = v.m - b, f = exp2_approx(d * c);
    v.s *= f;
    if (ENT) v.t = fmaf(v.s, fmaxf(d, kFloor), v.t * f);
  }
  v.m = b;
}

// A thread's share of a row. RUNS: also the maxima of its runs of pieces, into
// `slots`. KEEP: the first `kept` pieces stay in `keep` (shared memory), piece i
// at keep[i], where the thread that scanned them can read them again.
template <typename T, bool ENT, bool RUNS, bool KEEP, int THREADS>
__device__ __forceinline__ Sums scan_share(const Share<T>& sh, float c, Slots<THREADS>* slots,
                                           uint4* keep = nullptr, uint32_t kept = 0) {
  constexpr int V = Piece<T>::V, U = 4;
  Sums v{-INFINITY, 0.0f, 0.0f};
  const uint32_t tid = threadIdx.x;
  uint32_t half = tid;  // first piece of the second group of copies
  if (KEEP) {  // all of them in flight at once, in two groups
    const uint32_t rounds = (kept + THREADS - 1) / THREADS;
    half = tid + (rounds + 1) / 2 * THREADS;
    uint32_t i = tid;
    for (; i < min(kept, half); i += THREADS) copy_async<16>(keep + i, sh.p + sh.piece_at(i));
    copy_commit();
    for (; i < kept; i += THREADS) copy_async<16>(keep + i, sh.p + sh.piece_at(i));
    copy_commit();
  }
  auto single = [&](uint32_t at) {
    const float x = to_f32(sh.p[at]);
    if (!(x <= v.m) && v.m == v.m) rebase<ENT>(v, x, c);
    if (v.m == -INFINITY) return;
    const float d = x - v.m, e = exp2_approx(d * c);
    v.s += e;
    if (ENT) v.t = fmaf(e, fmaxf(d, kFloor), v.t);
  };
  if (tid < sh.head) single(tid);
  if (tid < sh.tail) single(sh.tail_at() + tid);
  const F2 c2 = pack2(c, c);
  const uint32_t run = RUNS ? (1u << sh.slot_shift(THREADS)) - 1 : 0;
  uint32_t nth = 0;  // of this thread's pieces
  uint16_t* slot = RUNS ? slots->most + tid : nullptr;
  float run_most = -INFINITY;
  auto batch = [&](const uint4* q, auto count_c) {
    constexpr int count = decltype(count_c)::value;
    const float b = Piece<T>::template most<count>(q);
    if (RUNS) {  // batches of four start at a multiple of four: whole in one run
      run_most = max_nan(run_most, b);
      *slot = (uint16_t)(__float_as_uint(run_most) >> 16);
      nth += count;
      if ((nth & run) == 0) {
        slot += THREADS;
        run_most = -INFINITY;
      }
    }
    if (!(b <= v.m) && v.m == v.m) rebase<ENT>(v, b, c);
    const float base = v.m == -INFINITY ? 0.0f : v.m;
    const F2 minus = pack2(-base, -base);
    F2 s2 = pack2(0.0f, 0.0f), t2 = s2;
#pragma unroll
    for (int u = 0; u < count; ++u) {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        const F2 d = add2(Piece<T>::pair(q[u], k), minus), a = mul2(d, c2);
        const F2 e = pack2(exp2_approx(a.x), exp2_approx(a.y));
        s2 = add2(s2, e);
        if (ENT) t2 = fma2(e, pack2(fmaxf(d.x, kFloor), fmaxf(d.y, kFloor)), t2);
      }
    }
    v.s += s2.x + s2.y;
    if (ENT) v.t += t2.x + t2.y;
  };
  uint32_t i = tid;
  auto go = [&](uint32_t end, auto get) {
    if (RUNS) {
      // The next batch is on its way while one is worked on. (Without runs
      // there are registers for half as many threads more, which does more.)
      uint4 q[U], next[U];
      if (i + (U - 1) * THREADS < end)
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = get(i, u * THREADS);
      for (; i + (U - 1) * THREADS < end; i += U * THREADS) {
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = next[u];
        if (i + (2 * U - 1) * THREADS < end)
#pragma unroll
          for (int u = 0; u < U; ++u) next[u] = get(i, (U + u) * THREADS);
        batch(q, std::integral_constant<int, U>{});
      }
    } else {
      for (; i + (U - 1) * THREADS < end; i += U * THREADS) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = get(i, u * THREADS);
        batch(q, std::integral_constant<int, U>{});
      }
    }
    if (i >= end) return;
    uint4 q[U];  // the rest, loaded together
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (i + u * THREADS < end) q[u] = get(i, u * THREADS);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (i + u * THREADS < end) batch(q + u, std::integral_constant<int, 1>{});
    i += (end - i + THREADS - 1) / THREADS * THREADS;
  };
  if (KEEP) {  // a thread reads what it copied itself: no barrier
    auto get = [&](uint32_t k, int on) { return (keep + k)[on]; };
    copy_wait<1>();
    go(min(kept, half), get);
    copy_wait<0>();
    go(kept, get);
  }
  go(sh.pieces, [&](uint32_t k, int on) { return sh.piece(k, on); });
  return v;
}

// Sums of the lanes `from` to 2 from - 1 apart, ..., 1 apart: the same in all.
template <bool ENT>
__device__ __forceinline__ Sums join_lanes(Sums v, float c, int from) {
  float m = v.m;
  for (int d = from; d; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (v.m != -INFINITY) rebase<ENT>(v, m, c);
  for (int d = from; d; d >>= 1) {
    v.s += __shfl_xor_sync(0xffffffffu, v.s, d);
    if (ENT) v.t += __shfl_xor_sync(0xffffffffu, v.t, d);
  }
  v.m = m;
  return v;
}

// The block's sums from those of its first WARPS warps' threads, the same in
// every thread, in a fixed order. One barrier: `all` is used once a launch.
template <bool ENT, int WARPS>
__device__ __forceinline__ Sums join_block(Sums v, float c, Sums* all) {
  static_assert(WARPS <= 32, "one lane a warp");
  constexpr int HALF = WARPS > 16 ? 16 : WARPS > 8 ? 8 : WARPS > 4 ? 4 : WARPS > 2 ? 2 : 1;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp < WARPS) {
    v = join_lanes<ENT>(v, c, 16);
    if (lane == 0) all[warp] = v;
  }
  __syncthreads();
  const uint32_t k = lane & (2 * HALF - 1);
  return join_lanes<ENT>(k < WARPS ? all[k] : Sums{-INFINITY, 0.0f, 0.0f}, c, HALF);
}

// The row's sums from its cluster's blocks', in rank order: `mine` of each, in
// shared memory that a cluster barrier has made visible.
template <bool ENT>
__device__ __forceinline__ Sums join_parts(cg::cluster_group& cl, Sums* mine, float c) {
  const uint32_t parts = cl.num_blocks();
  float m = -INFINITY;
  for (uint32_t k = 0; k < parts; ++k) m = max_nan(m, cl.map_shared_rank(mine, k)->m);
  Sums r{m, 0.0f, 0.0f};
  for (uint32_t k = 0; k < parts; ++k) {
    Sums o = *cl.map_shared_rank(mine, k);
    if (o.m == -INFINITY) continue;
    rebase<ENT>(o, m, c);
    r.s += o.s;
    r.t += o.t;
  }
  return r;
}

// Blocks a row is split over, 8 at most (the largest portable cluster): more
// than one where the rows alone would leave SMs without two blocks and a part
// keeps 4,096 values (less is not worth the barrier).
inline uint32_t row_parts(uint64_t rows, uint32_t n) {
  uint32_t parts = 1;
  while (parts < 8 && rows * parts * 2 <= 2 * 148 && n / (parts * 2) >= 4096) parts *= 2;
  return parts;
}

inline int check_logits(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                        const void* logits, int64_t ld, float scale, const char* what) {
  PLX_CHECK_ARG(ctx, "ctx is required");
  PLX_CHECK_ARG(valid_dtype(dtype), "dtype %d is none of PLX_F32, PLX_BF16, PLX_F16", dtype);
  PLX_CHECK_ARG(n > 0 && n < (1u << 31), "n = %u is out of range", n);
  if (rows >= (1ull << 31))
    return set_error(PLX_ERR_CAPACITY, "%llu rows: fewer than 2^31 are supported",
                     (unsigned long long)rows);
  PLX_CHECK_ARG(scale > 0.0f && scale < INFINITY, "%s = %g has to be positive and finite", what,
                scale);
  PLX_CHECK_ARG(rows == 0 || logits, "logits is required");
  PLX_CHECK_ARG(rows <= 1 || ld >= (int64_t)n, "the logits' row stride %lld is less than n",
                (long long)ld);
  return check_aligned(dtype_bytes(dtype), {logits});
}

// Threads that go over a row (part) of n values: 256, or fewer where each would
// have less than 64 values, since joining them costs about as much as scanning
// 64. Measured on 8,192 rows of 4,096 bf16: 64 threads 18.9 us, 128 20.6, 256
// 33.1; on 2,047 of 20,011: 23.5, 23.6, 25.2 (with gradient 58, 52, 40); on
// 4,096 of 65,536: 101, 93, 89.
// Where `blocks` leave SMs with two blocks at most, latency counts, and 16 are
// enough.
inline uint32_t row_threads(uint64_t blocks, uint32_t n) {
  const uint32_t each = blocks <= 2 * 148 ? 16 : 64;
  return n < each * 128 ? 64 : n < each * 256 ? 128 : 256;
}

// Launches one row a cluster of `parts` blocks (no cluster for one).
template <typename... Params, typename... Args>
cudaError_t launch_rows(void (*kernel)(Params...), uint64_t rows, uint32_t parts, uint32_t threads,
                        size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace plx
