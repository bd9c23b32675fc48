// One pass over a row of logits (log_probs.cu, distill.cu): the running maximum
// m, s = sum 2^((x-m)c) and t = sum 2^((x-m)c) (x-m) of a thread's share, joined
// over a block and over the blocks of a cluster.
//
// A row may start anywhere: its 16-byte pieces are read whole, the elements
// before the first and after the last piece one by one. "Unit" below is such a
// piece or single element; units are disjoint and ordered by their first index.
#pragma once

#include <cooperative_groups.h>

#include "rows.cuh"

namespace plx {

namespace cg = cooperative_groups;

// ---- two 32-bit values at once -------------------------------------------
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(F2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

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
  static __device__ __forceinline__ float most(const uint4& q) {
    return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)),
                   max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
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
  static __device__ __forceinline__ float most(const uint4& q) {
    const __nv_bfloat162 m =
        __hmax2_nan(__hmax2_nan(two(q.x), two(q.y)), __hmax2_nan(two(q.z), two(q.w)));
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
  static __device__ __forceinline__ float most(const uint4& q) {
    const __half2 m =
        __hmax2_nan(__hmax2_nan(two(q.x), two(q.y)), __hmax2_nan(two(q.z), two(q.w)));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void put(uint4& q, int k, float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    (&q.x)[k] = *reinterpret_cast<uint32_t*>(&v);
  }
};

// ---- a contiguous share of a row -----------------------------------------
// Elements [start, start + count): `head` single ones, `pieces` whole pieces,
// `tail` single ones. Thread i of a block has head element i, pieces i, i + T,
// ... and tail element i.
template <typename T>
struct Share {
  const T* p;
  uint32_t start, count, head, pieces, tail;

  __device__ __forceinline__ Share(const T* row, uint32_t n, uint32_t part, uint32_t parts) {
    constexpr uint32_t V = Piece<T>::V;
    // Whole pieces a part, so that every part starts at the row's alignment.
    const uint32_t each = ((n + parts - 1) / parts + V - 1) / V * V;
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
  __device__ __forceinline__ uint4 piece(uint32_t i) const {
    return *reinterpret_cast<const uint4*>(p + piece_at(i));
  }
};

struct Sums {
  float m, s, t;
};

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

// A thread's share of a row. POS: also the first index (within the row) of the
// first of its units that attains m.
template <typename T, bool ENT, bool POS, int THREADS>
__device__ __forceinline__ Sums scan_share(const Share<T>& sh, float c, uint32_t& pos) {
  constexpr int V = Piece<T>::V, U = 4;
  Sums v{-INFINITY, 0.0f, 0.0f};
  pos = 0xffffffffu;
  const uint32_t tid = threadIdx.x;
  auto single = [&](uint32_t at) {
    const float x = to_f32(sh.p[at]);
    if (POS && pos == 0xffffffffu) pos = sh.start + at;
    if (!(x <= v.m) && v.m == v.m) {
      if (POS) pos = sh.start + at;
      rebase<ENT>(v, x, c);
    }
    if (v.m == -INFINITY) return;
    const float d = x - v.m, e = exp2_approx(d * c);
    v.s += e;
    if (ENT) v.t = fmaf(e, fmaxf(d, kFloor), v.t);
  };
  if (tid < sh.head) single(tid);
  if (POS && pos == 0xffffffffu && tid < sh.pieces) pos = sh.start + sh.piece_at(tid);
  const F2 c2 = pack2(c, c);
  auto batch = [&](const uint4* q, int count, uint32_t first) {
    float most[U];
#pragma unroll
    for (int u = 0; u < count; ++u) most[u] = Piece<T>::most(q[u]);
    float b = most[0];
#pragma unroll
    for (int u = 1; u < count; ++u) b = max_nan(b, most[u]);
    if (!(b <= v.m) && v.m == v.m) {  // seldom after the first batches
      if (POS) {
        int at = count - 1;
#pragma unroll
        for (int u = count - 2; u >= 0; --u)
          if (most[u] == b || (b != b && most[u] != most[u])) at = u;
        pos = sh.start + sh.piece_at(first + at * THREADS);
      }
      rebase<ENT>(v, b, c);
    }
    const float base = v.m == -INFINITY ? 0.0f : v.m;
    const F2 minus = pack2(-base, -base);
    F2 s2 = pack2(0.0f, 0.0f), t2 = s2;
#pragma unroll
    for (int u = 0; u < count; ++u) {
#pragma unroll
      for (int k = 0; k < V / 2; ++k) {
        const F2 d = add2(Piece<T>::pair(q[u], k), minus);
        float a0, a1;
        unpack2(mul2(d, c2), a0, a1);
        const F2 e = pack2(exp2_approx(a0), exp2_approx(a1));
        s2 = add2(s2, e);
        if (ENT) {
          float d0, d1;
          unpack2(d, d0, d1);
          t2 = fma2(e, pack2(fmaxf(d0, kFloor), fmaxf(d1, kFloor)), t2);
        }
      }
    }
    float a, b2;
    unpack2(s2, a, b2);
    v.s += a + b2;
    if (ENT) {
      unpack2(t2, a, b2);
      v.t += a + b2;
    }
  };
  uint32_t i = tid;
  for (; i + (U - 1) * THREADS < sh.pieces; i += U * THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = sh.piece(i + u * THREADS);
    batch(q, U, i);
  }
  for (; i < sh.pieces; i += THREADS) {
    const uint4 q = sh.piece(i);
    batch(&q, 1, i);
  }
  if (tid < sh.tail) single(sh.tail_at() + tid);
  return v;
}

// The block's sums from its threads', the same in every thread.
template <bool ENT, int WARPS>
__device__ __forceinline__ Sums join_block(Sums v, float c, float* red) {
  const float m = block_max<WARPS>(v.m, red);
  if (v.m != -INFINITY) rebase<ENT>(v, m, c);
  Sums r{m, block_sum<WARPS>(v.s, red), 0.0f};
  if (ENT) r.t = block_sum<WARPS>(v.t, red);
  return r;
}

// The row's sums from its cluster's blocks', in rank order. `mine` is shared
// memory; the caller ends with a cluster barrier before any block exits.
template <bool ENT>
__device__ __forceinline__ Sums join_cluster(cg::cluster_group& cl, Sums* mine, Sums v, float c) {
  if (threadIdx.x == 0) *mine = v;
  cl.sync();
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

// Blocks a row is split over. One each while the rows alone give every SM two
// blocks; with fewer rows as many as fill the device, at least `least` values
// each (less is not worth the barrier), 8 at most (the largest portable cluster).
inline uint32_t row_parts(uint64_t rows, uint32_t n, uint32_t least) {
  uint32_t parts = 1;
  while (parts < 8 && rows * parts * 2 <= 2 * 148 && n / (parts * 2) >= least) parts *= 2;
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
  return PLX_OK;
}

// Launches one row a cluster of `parts` blocks (no cluster for one).
template <typename... Params, typename... Args>
cudaError_t launch_rows(void (*kernel)(Params...), uint64_t rows, uint32_t parts, uint32_t threads,
                        cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(threads);
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
