// What a row of output units answers: log probabilities of given outputs,
// entropy, best alternatives; and their gradient. With M the row's largest
// logit and d_i = scale (x_i - M):
//   s = sum exp d_i; lse = scale M + log s; logp_i = d_i - log s;
//   entropy = log s - (sum exp(d_i) d_i) / s
// M is subtracted before scaling, which is exact near M, so large common
// offsets cost no accuracy. All sums are in 32 bits.
//
// Bound by memory: the forward pass reads a row once (running maximum and
// sums, logits.cuh) and finds the alternatives from what the threads saw: of
// the threads' own maxima the `top` best are a threshold, only the threads at
// or above it can hold an alternative, and only those look at their share
// again (out of L2, a few kilobytes a row).
#include "logits.cuh"

namespace plx {
namespace {

// A number that orders values: larger for larger ones, NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);
  return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o == 0xffffffffu ? 0x7fffffffu : (o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
// With its index: the lower one first among equals. 0 is no element.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t i) {
  return (uint64_t)order_of(v) << 32 | (0xffffffffu - i);
}

constexpr uint32_t kCandidates = 1024;

template <int THREADS>
struct TopShared {
  uint64_t red[THREADS / 32];
  uint64_t keys[kCandidates];
  uint64_t best[PLX_TOP_MAX];
  uint32_t count;
};

// The block's `top` best elements into sh.best, best first, 0 where there are
// fewer. m, pos: the thread's maximum and the first unit that attains it.
template <typename T, int THREADS>
__device__ void block_top(const Share<T>& share, float m, uint32_t pos, uint32_t top,
                          TopShared<THREADS>& sh) {
  const uint32_t tid = threadIdx.x;
  const uint32_t mine = pos == 0xffffffffu ? 0u : order_of(m);
  // The largest value that at least `top` threads' maxima reach.
  uint64_t lo = 1, hi = 1ull << 32;
  uint32_t at_lo = (uint32_t)__syncthreads_count(mine >= 1u), above = 0;
  if (at_lo > top)
    while (hi - lo > 1) {
      const uint64_t mid = (lo + hi) / 2;
      const uint32_t n = (uint32_t)__syncthreads_count(mine >= mid);
      if (n >= top) {
        lo = mid;
        at_lo = n;
        if (n == top) break;
      } else {
        hi = mid;
        above = n;
      }
    }
  // Among equals at the threshold the units that come first are enough.
  uint32_t last = 0xfffffffeu;
  auto narrow = [&] {
    uint32_t a = 0, b = share.start + share.count - 1;
    while (a < b) {
      const uint32_t mid = a + (b - a) / 2;
      if ((uint32_t)__syncthreads_count(mine == lo && pos <= mid) >= top - above) b = mid;
      else a = mid + 1;
    }
    last = a;
  };
  bool narrowed = at_lo <= top;
  if (at_lo > top + 32) {
    narrow();
    narrowed = true;
  }
  // Calls f(value, index) for every element of this thread that can count.
  auto candidates = [&](auto f) {
    if (mine < lo || (mine == lo && pos > last)) return;
    auto unit = [&](uint32_t first, uint32_t n) {
      for (uint32_t k = 0; k < n; ++k) {
        const float x = to_f32(share.p[first + k]);
        const uint32_t o = order_of(x);
        if (o > lo || (o == lo && share.start + first <= last)) f(x, share.start + first + k);
      }
    };
    constexpr int V = Piece<T>::V;
    if (tid < share.head) unit(tid, 1);
    for (uint32_t i = tid; i < share.pieces; i += THREADS) {
      const uint4 q = share.piece(i);
      const float most = Piece<T>::most(q);
      if (order_of(most) >= lo) unit(share.piece_at(i), V);
    }
    if (tid < share.tail) unit(share.tail_at() + tid, 1);
  };
  for (;;) {
    if (tid == 0) sh.count = 0;
    __syncthreads();
    candidates([&](float x, uint32_t i) {
      const uint32_t k = atomicAdd(&sh.count, 1u);
      if (k < kCandidates) sh.keys[k] = rank_key(x, i);
    });
    __syncthreads();
    if (sh.count <= kCandidates || narrowed) break;
    narrow();
    narrowed = true;
  }
  for (uint32_t k = tid; k < top; k += THREADS) sh.best[k] = 0;
  const uint32_t count = sh.count;
  __syncthreads();
  if (count <= kCandidates) {  // each candidate's place is the number of better ones
    for (uint32_t i = tid; i < count; i += THREADS) {
      const uint64_t key = sh.keys[i];
      uint32_t place = 0;
      for (uint32_t j = 0; j < count; ++j) place += sh.keys[j] > key;
      if (place < top) sh.best[place] = key;
    }
  } else {  // a few threads hold very many: one alternative at a time
    uint64_t below = ~0ull;
    for (uint32_t k = 0; k < top; ++k) {
      uint64_t best = 0;
      candidates([&](float x, uint32_t i) {
        const uint64_t key = rank_key(x, i);
        if (key < below && key > best) best = key;
      });
#pragma unroll
      for (int d = 16; d; d >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, d));
      __syncthreads();
      if ((tid & 31) == 0) sh.red[tid >> 5] = best;
      __syncthreads();
      best = sh.red[0];
#pragma unroll
      for (int w = 1; w < THREADS / 32; ++w) best = max(best, sh.red[w]);
      if (tid == 0) sh.best[k] = best;
      below = best;
    }
  }
  __syncthreads();
}

template <typename T, bool ENT, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS)
k_log_probs(uint32_t n, const T* __restrict__ x, int64_t ld, const int32_t* __restrict__ target,
            float scale, uint32_t top, float* __restrict__ logp, float* __restrict__ lse,
            float* __restrict__ entropy, int32_t* __restrict__ top_ids,
            float* __restrict__ top_logp, int32_t* __restrict__ status) {
  constexpr int WARPS = THREADS / 32;
  __shared__ float red[WARPS];
  __shared__ Sums mine;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t parts = cl.num_blocks(), part = cl.block_rank();
  const int64_t r = blockIdx.x / parts;
  const T* xr = x + r * ld;
  const Share<T> share(xr, n, part, parts);
  const float c = scale * kLog2e;
  uint32_t pos;
  const Sums own = scan_share<T, ENT, TOP, THREADS>(share, c, pos);
  Sums v = join_block<ENT, WARPS>(own, c, red);
  __shared__ TopShared<TOP ? THREADS : 32> sh;
  if constexpr (TOP) block_top<T, THREADS>(share, own.m, pos, top, sh);
  if (parts > 1) v = join_cluster<ENT>(cl, &mine, v, c);
  if (part == 0) {
    const bool none = v.m == -INFINITY;  // every output masked
    const float ls = logf(v.s);
    auto log_p = [&](float at) { return none ? -INFINITY : scale * (at - v.m) - ls; };
    if (threadIdx.x == 0) {
      lse[r] = none ? -INFINITY : fmaf(scale, v.m, ls);
      if (ENT) entropy[r] = none ? 0.0f : ls - scale * (v.t / v.s);
      if (logp) {
        const int32_t at = target[r];
        const bool out = at < -1 || at >= (int64_t)n;
        if (out) record_status(status, kStatusBadOutput);
        logp[r] = out || at < 0 ? 0.0f : log_p(to_f32(xr[at]));
      }
    }
    if constexpr (TOP) {
      auto put = [&](uint32_t place, uint64_t key) {
        top_ids[r * top + place] = (int32_t)(0xffffffffu - (uint32_t)key);
        top_logp[r * top + place] = log_p(value_of((uint32_t)(key >> 32)));
      };
      if (parts == 1) {
        for (uint32_t k = threadIdx.x; k < top; k += THREADS) put(k, sh.best[k]);
      } else {  // the blocks' lists side by side, each key's place as above
        for (uint32_t i = threadIdx.x; i < parts * top; i += THREADS)
          sh.keys[i] = cl.map_shared_rank(&sh.best[0], i / top)[i % top];
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < parts * top; i += THREADS) {
          const uint64_t key = sh.keys[i];
          uint32_t place = 0;
          for (uint32_t j = 0; j < parts * top; ++j) place += sh.keys[j] > key;
          if (key && place < top) put(place, key);
        }
      }
    }
  }
  if (parts > 1) cl.sync();  // no block leaves while another reads its memory
}

constexpr int kBwdThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kBwdThreads)
k_log_probs_bwd(uint32_t n, uint32_t parts, const T* x, int64_t ld,
                const int32_t* __restrict__ target, float scale, const float* __restrict__ lse,
                const float* __restrict__ entropy, const float* __restrict__ grad_logp,
                const float* __restrict__ grad_entropy, T* dx, int64_t ldd) {
  constexpr int V = Piece<T>::V;
  const int64_t r = blockIdx.x / parts;
  const Share<T> sh(x + r * ld, n, blockIdx.x % parts, parts);
  T* out = dx + r * ldd + sh.start;
  const float z = lse[r];
  const int32_t at = target ? target[r] : -1;
  const float g = grad_logp && at >= 0 && at < (int64_t)n ? grad_logp[r] : 0.0f;
  const float gh = grad_entropy ? grad_entropy[r] : 0.0f;
  const float h = grad_entropy ? entropy[r] : 0.0f;
  auto one = [&](float v, uint32_t i) {
    const float l = fmaf(v, scale, -z);
    const float p = z == -INFINITY ? 0.0f : exp2_approx(l * kLog2e);
    float d = p == 0.0f ? 0.0f : -p * fmaf(gh, l + h, g);
    if (sh.start + i == (uint32_t)at) d += g;
    return d * scale;
  };
  auto single = [&](uint32_t i) { out[i] = from_f32<T>(one(to_f32(sh.p[i]), i)); };
  if (threadIdx.x < sh.head) single(threadIdx.x);
  if (threadIdx.x < sh.tail) single(sh.tail_at() + threadIdx.x);
  const bool whole = (reinterpret_cast<uintptr_t>(out + sh.head) & 15u) == 0;
  for (uint32_t i = threadIdx.x; i < sh.pieces; i += kBwdThreads) {
    const uint4 q = sh.piece(i);
    const uint32_t first = sh.piece_at(i);
    uint4 o;
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      float a, b;
      unpack2(Piece<T>::pair(q, k), a, b);
      Piece<T>::put(o, k, one(a, first + 2 * k), one(b, first + 2 * k + 1));
    }
    if (whole) {
      *reinterpret_cast<uint4*>(out + first) = o;
    } else {
      const T* e = reinterpret_cast<const T*>(&o);
#pragma unroll
      for (int k = 0; k < V; ++k) out[first + k] = e[k];
    }
  }
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" int plx_log_probs(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                             const void* logits, int64_t ld, const int32_t* target, float scale,
                             uint32_t top, float* logp, float* lse, float* entropy,
                             int32_t* top_ids, float* top_logp) {
  if (int rc = check_logits(ctx, rows, n, dtype, logits, ld, scale, "scale")) return rc;
  PLX_CHECK_ARG(top <= n, "top = %u exceeds the %u outputs of a row", top, n);
  if (top > PLX_TOP_MAX)
    return set_error(PLX_ERR_CAPACITY, "top = %u: at most %d are supported", top, PLX_TOP_MAX);
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(lse, "lse is required");
  PLX_CHECK_ARG(!target == !logp, "target and logp go together");
  PLX_CHECK_ARG(!top || (top_ids && top_logp), "top_ids and top_logp are required");
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel, uint32_t threads) {
      PLX_TRY_CUDA(launch_rows(kernel, rows, row_parts(rows, n, 4096), threads, ctx->stream, n,
                               (const T*)logits, rows == 1 ? (int64_t)0 : ld, target, scale, top,
                               logp, lse, entropy, top_ids, top_logp, ctx->d_status));
      return PLX_OK;
    };
    // Blocks of 512 keep enough reads in flight; rows too short for one batch
    // of pieces each take blocks of 128.
    auto pick = [&](auto ent, auto best) {
      constexpr bool E = decltype(ent)::value, B = decltype(best)::value;
      return n < 128 * 4 * Piece<T>::V ? go(k_log_probs<T, E, B, 128>, 128)
                                       : go(k_log_probs<T, E, B, 512>, 512);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (entropy) return top ? pick(Yes{}, Yes{}) : pick(Yes{}, No{});
    return top ? pick(No{}, Yes{}) : pick(No{}, No{});
  });
}

extern "C" int plx_log_probs_backward(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                                      const void* logits, int64_t ld, const int32_t* target,
                                      float scale, const float* lse, const float* entropy,
                                      const float* grad_logp, const float* grad_entropy,
                                      void* dlogits, int64_t ldd) {
  if (int rc = check_logits(ctx, rows, n, dtype, logits, ld, scale, "scale")) return rc;
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(grad_logp || grad_entropy, "grad_logp or grad_entropy is required");
  PLX_CHECK_ARG(!grad_logp || target, "grad_logp needs target");
  PLX_CHECK_ARG(!grad_entropy || entropy, "grad_entropy needs entropy");
  PLX_CHECK_ARG(lse && dlogits, "lse and dlogits are required");
  PLX_CHECK_ARG(rows == 1 || ldd >= (int64_t)n, "the gradient's row stride is less than n");
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  if (rows == 1) ld = ldd = 0;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    // Four pieces a thread, as far as the grid's size allows.
    const uint64_t each = kBwdThreads * 4 * Piece<T>::V;
    const uint32_t parts = (uint32_t)std::max<uint64_t>(
        1, std::min<uint64_t>((n + each - 1) / each, ((1ull << 31) - 1) / rows));
    k_log_probs_bwd<T><<<(unsigned)(rows * parts), kBwdThreads, 0, ctx->stream>>>(
        n, parts, (const T*)logits, ld, target, scale, lse, entropy, grad_logp, grad_entropy,
        (T*)dlogits, ldd);
    PLX_LAUNCH_CHECK("k_log_probs_bwd");
    return PLX_OK;
  });
}
