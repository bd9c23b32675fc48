// What a row of output units answers: log probabilities of given outputs,
// entropy, best alternatives; and their gradient. With M the row's largest
// logit and d_i = scale (x_i - M):
//   s = sum exp d_i; lse = scale M + log s; logp_i = d_i - log s;
//   entropy = log s - (sum exp(d_i) d_i) / s
// M is subtracted before scaling, which is exact near M, so large common
// offsets cost no accuracy. All sums are in 32 bits.
//
// The gradient needs log p_i = scale x_i - lse, and lse in 32 bits is off by up
// to |lse| 2^-24, which every p_i takes over: 2^-20 for |lse| up to 32, as much
// as a dozen other roundings; a thousandth around 30,000; and in a row of the
// type's lowest values log s is gone altogether and every p_i comes out as 1.
// So rows above 32 (and those of lse -inf or NaN) take M and log s from the row
// itself: one block reads it, and once more to write its gradient. 4,096 rows
// of 65,536 bf16: 164 us for ordinary rows, 239 if all are far from zero; one
// row of 131,072 f32 2.3 and 24 (one block instead of 32).
//
// Bound by memory: the forward pass reads a row once (running maximum and
// sums, logits.cuh) and finds the alternatives from what the threads saw: of
// the threads' own maxima the `top` best are a threshold, only threads at or
// above it can hold an alternative, and of those only the runs of pieces whose
// maximum reaches it are looked at again (a few kilobytes a row, out of L2).
// For 16-bit logits the arithmetic is close behind: six instructions a value,
// one of them of the special-function unit. Measured, 4,096 rows of 65,536
// bf16: 86 us, 6.2 TB/s; with entropy 89; and 8 alternatives 101, 5.3 TB/s; 64
// 129. 2,048 rows of 65,536 f32: 86, 87, 93, 114. The gradient (read and written
// once) of 1,024 rows of 131,072 bf16: 84 us, 6.4 TB/s.
#include "logits.cuh"

namespace plx {
namespace {

// A value's order with its index: the lower one first among equals. 0 is no
// element.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t i) {
  return (uint64_t)order_of(v) << 32 | (0xffffffffu - i);
}

constexpr uint32_t kCandidates = 1024;
constexpr uint32_t kSpare = 32;  // threads more than asked for that may reach the threshold

template <int THREADS>
struct TopShared {
  uint64_t keys[kCandidates];
  uint64_t best[PLX_TOP_MAX];  // best first, 0 where there are fewer
  uint64_t red[THREADS / 32];
  uint32_t most[THREADS];      // each thread's maximum, as a number that orders
  Slots<THREADS> slots;
  uint16_t runs[(PLX_TOP_MAX + kSpare) * kSlots];  // that can hold an alternative
  uint32_t listed, count, threshold, reached;
};

// A value that at least `top` threads' maxima reach, and (in `reached`) by how
// many: a few more than `top`, unless many are equal to it; then it is the
// largest such value. At least `top` elements are at or above it, so no element
// below it counts, and no other thread's. By one warp; most[i] is of thread
// lane + 32 i.
template <int K>
__device__ __forceinline__ uint32_t find_threshold(uint32_t top, const uint32_t (&most)[K],
                                                   uint32_t& reached) {
  static_assert(PLX_TOP_MAX <= 64 && K >= 2, "two of each lane are enough");
  uint32_t a = 0, b = 0;  // the lane's two best
#pragma unroll
  for (int i = 0; i < K; ++i) {
    b = max(b, min(a, most[i]));
    a = max(a, most[i]);
  }
  auto reach = [&](uint32_t v) {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < K; ++i) n += most[i] >= v;
    return __reduce_add_sync(0xffffffffu, n);
  };
  uint32_t lo = 1;
  reached = reach(1);
  if (reached <= top) return lo;
  // 32 (64) maxima reach the least of the lanes' best (second best) ones. No
  // more than one reaches the largest.
  uint32_t hi = __reduce_max_sync(0xffffffffu, a);
  const uint32_t least = __reduce_min_sync(0xffffffffu, top <= 32 ? a : b);
  if (least > 1) reached = reach(lo = least);
  if (const uint32_t n = reach(hi); n >= top) {
    reached = n;
    return hi;
  }
  while (hi - lo > 1 && reached > top + kSpare / 4) {
    const uint32_t mid = lo + (hi - lo) / 2, n = reach(mid);
    if (n >= top) {
      lo = mid;
      reached = n;
    } else {
      hi = mid;
    }
  }
  return lo;
}

// Places of `count` different keys (0 is none) by the number of better ones; put(place, key)
// for the places below `top`. By `threads` threads, of which this is the me-th.
template <typename F>
__device__ __forceinline__ void place_keys(const uint64_t* keys, uint32_t count, uint32_t top,
                                           uint32_t me, uint32_t threads, F put) {
  for (uint32_t i = me; i < count; i += threads) {
    const uint64_t key = keys[i];
    uint32_t place = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < count; ++j) place += keys[j] > key;
    if (key && place < top) put(place, key);
  }
}

// A share's `top` best elements into sh.best, from what scan_share left in
// sh.slots and sh.most (after a barrier).
template <typename T, int THREADS>
__device__ __forceinline__ void share_top(const Share<T>& share, uint32_t top,
                                          TopShared<THREADS>& sh) {
  constexpr int K = THREADS / 32, SPARE = kSpareBits<T>;
  constexpr uint32_t V = Piece<T>::V;
  const uint32_t tid = threadIdx.x;
  if (tid < 32) {
    uint32_t most[K], reached;
#pragma unroll
    for (int i = 0; i < K; ++i) most[i] = sh.most[tid + 32 * i] >> SPARE;
    const uint32_t threshold = find_threshold<K>(top, most, reached);
    if (tid == 0) {
      sh.threshold = threshold;
      sh.reached = reached;
      sh.listed = sh.count = 0;
    }
  }
  for (uint32_t k = tid; k < top; k += THREADS) sh.best[k] = 0;
  __syncthreads();
  const uint32_t threshold = sh.threshold;
  // Values that very many threads reach at best (a row of few distinct values):
  // those above are taken first, then ties from the row's start.
  const bool ties = sh.reached > top + kSpare;
  const uint32_t bar = ties ? threshold : threshold - 1;  // elements above it
  auto order = [](float v) { return order_of(v) >> SPARE; };
  const uint32_t shift = share.slot_shift(THREADS);
  if (sh.most[tid] >> SPARE > bar) {
    const uint32_t pieces = share.pieces > tid ? (share.pieces - tid - 1) / THREADS + 1 : 0;
#pragma unroll
    for (uint32_t s = 0; s < kSlots; ++s) {
      if (s << shift >= pieces) break;
      const uint32_t h = sh.slots.most[s * THREADS + tid];
      if ((h & 0x8000u ? ~h & 0xffffu : h | 0x8000u) >= bar << SPARE >> 16)
        sh.runs[atomicAdd(&sh.listed, 1u)] = (uint16_t)(s * THREADS + tid);
    }
  }
  __syncthreads();
  auto elements = [&](const uint4& q, uint32_t first, auto f) {
#pragma unroll
    for (uint32_t e = 0; e < V / 2; ++e) {
      const F2 v = Piece<T>::pair(q, e);
      f(v.x, first + 2 * e);
      f(v.y, first + 2 * e + 1);
    }
  };
  // Calls f(value, index) for every element above the bar: of the pieces of
  // the listed runs, spread over the block, and of the single elements.
  auto candidates = [&](auto f) {
    auto element = [&](float x, uint32_t i) {
      if (order(x) > bar) f(x, share.start + i);
    };
    if (tid < share.head) element(to_f32(share.p[tid]), tid);
    if (tid < share.tail) element(to_f32(share.p[share.tail_at() + tid]), share.tail_at() + tid);
    const uint32_t pieces = sh.listed << shift;
    for (uint32_t k = tid; k < pieces; k += THREADS) {
      const uint32_t run = sh.runs[k >> shift];
      const uint64_t i = run % THREADS +
                         (uint64_t)((run / THREADS << shift) + (k & ((1u << shift) - 1))) * THREADS;
      if (i >= share.pieces) continue;
      const uint4 q = share.piece((uint32_t)i);
      if (order(Piece<T>::template most<1>(&q)) > bar)
        elements(q, share.piece_at((uint32_t)i), element);
    }
  };
  auto keep = [&](float x, uint32_t i) {
    const uint32_t k = atomicAdd(&sh.count, 1u);
    if (k < kCandidates) sh.keys[k] = rank_key(x, i);
  };
  candidates(keep);
  __syncthreads();
  if (ties) {
    // If fewer than `top` are above, the list holds every one of them and has
    // room for a step of ties (64 units, at most 512 values) more than it
    // takes to fill up.
    const uint32_t units = share.head + share.pieces + share.tail;
    uint32_t have = sh.count;
    for (uint32_t u = 0; u < units && have < top; u += 64) {
      __syncthreads();
      const uint32_t k = u + tid, i = k - share.head;  // of the pieces
      auto element = [&](float x, uint32_t at) {
        if (order(x) == threshold) keep(x, share.start + at);
      };
      if (tid < 64 && k < units) {
        if (k < share.head) {
          element(to_f32(share.p[k]), k);
        } else if (i >= share.pieces) {
          const uint32_t at = share.tail_at() + (i - share.pieces);
          element(to_f32(share.p[at]), at);
        } else {
          elements(share.piece(i), share.piece_at(i), element);
        }
      }
      __syncthreads();
      have = sh.count;
    }
  }
  const uint32_t count = sh.count;
  if (count <= kCandidates) {
    place_keys(sh.keys, count, top, tid, THREADS,
               [&](uint32_t place, uint64_t key) { sh.best[place] = key; });
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
      for (int w = 1; w < K; ++w) best = max(best, sh.red[w]);
      if (tid == 0) sh.best[k] = best;
      below = best;
    }
  }
  __syncthreads();
}

// A block has a row, or a cluster of blocks a part each.
template <typename T, bool ENT, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, (TOP ? 1024 : 1536) / THREADS)
k_log_probs(uint32_t n, uint32_t each, const T* __restrict__ x, int64_t ld,
            const int32_t* __restrict__ target, float scale, uint32_t top,
            float* __restrict__ logp, float* __restrict__ lse, float* __restrict__ entropy,
            int32_t* __restrict__ top_ids, float* __restrict__ top_logp,
            int32_t* __restrict__ status) {
  constexpr int WARPS = THREADS / 32;
  __shared__ Sums all[WARPS], mine;
  __shared__ std::conditional_t<TOP, TopShared<THREADS>, char> sh;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t parts = cl.num_blocks(), part = cl.block_rank();
  const int64_t r = cluster_row();
  const T* xr = x + r * ld;
  const Share<T> share(xr, n, part, each);
  const float c = scale * kLog2e;
  // The target's logit is two dependent loads away: both are on their way early.
  const bool first = part == 0 && threadIdx.x == 0;
  int32_t at = first && logp ? target[r] : -1;
  Slots<THREADS>* slots = nullptr;
  if constexpr (TOP) slots = &sh.slots;
  Sums v = scan_share<T, ENT, TOP, false, THREADS>(share, c, slots);
  if (at < -1 || at >= (int64_t)n) {
    record_status(status, kStatusBadOutput);
    at = -1;
  }
  const float x_at = at < 0 ? 0.0f : to_f32(xr[at]);
  if constexpr (TOP) {
    const uint32_t tid = threadIdx.x;
    const bool any = tid < share.head || tid < share.pieces || tid < share.tail;
    sh.most[tid] = any ? order_of(v.m) : 0u;
  }
  v = join_block<ENT, WARPS>(v, c, all);
  if constexpr (TOP) share_top<T, THREADS>(share, top, sh);
  if (parts > 1) {
    if (threadIdx.x == 0) mine = v;
    cl.sync();
    v = join_parts<ENT>(cl, &mine, c);
  }
  if (part == 0) {
    const bool none = v.m == -INFINITY;  // every output masked
    const float ls = logf(v.s);
    auto log_p = [&](float y) { return none ? -INFINITY : scale * (y - v.m) - ls; };
    if (first) {
      lse[r] = none ? -INFINITY : fmaf(scale, v.m, ls);
      if (ENT) entropy[r] = none ? 0.0f : ls - scale * (v.t / v.s);
      if (logp) logp[r] = at < 0 ? 0.0f : log_p(x_at);
    }
    if constexpr (TOP) {
      auto put = [&](uint32_t place, uint64_t key) {
        top_ids[r * top + place] = (int32_t)(0xffffffffu - (uint32_t)key);
        top_logp[r * top + place] = log_p(value_of((uint32_t)(key >> 32)));
      };
      if (parts == 1) {
        for (uint32_t k = threadIdx.x; k < top; k += THREADS) put(k, sh.best[k]);
      } else {  // the blocks' lists side by side
        for (uint32_t i = threadIdx.x; i < parts * top; i += THREADS)
          sh.keys[i] = cl.map_shared_rank(&sh.best[0], i / top)[i % top];
        __syncthreads();
        place_keys(sh.keys, parts * top, top, threadIdx.x, THREADS, put);
      }
    }
  }
  if (parts > 1) cl.sync();  // no block leaves while another reads its memory
}

// Rows of which |lse| is above this have their sum made anew.
constexpr float kLseExact = 32.0f;

// dx = p (A l + B) (+ the target's own term), with l = log p, A = -scale h',
// B = -scale (h' H + g'); h', g': gradients of entropy H and of logp. l is
// scale x - lse, or scale (x - m) - ls where that would lose too much.
template <typename T, bool ENT, int THREADS>
__global__ void __launch_bounds__(THREADS)
k_log_probs_bwd(uint32_t n, uint32_t parts, uint32_t each, const T* x, int64_t ld,
                const int32_t* __restrict__ target, float scale, const float* __restrict__ lse,
                const float* __restrict__ entropy, const float* __restrict__ grad_logp,
                const float* __restrict__ grad_entropy, T* dx, int64_t ldd) {
  constexpr int V = Piece<T>::V, U = 4;
  const int64_t r = parts == 1 ? blockIdx.x : blockIdx.x / parts;
  const uint32_t part = blockIdx.x - (uint32_t)r * parts;
  const T* xr = x + r * ld;
  const int32_t at = grad_logp ? target[r] : -1;
  const bool has = at >= 0 && at < (int64_t)n;
  const float z = lse[r], g = has ? grad_logp[r] : 0.0f;
  const float gh = ENT ? grad_entropy[r] : 0.0f;
  const float A = -scale * gh, B = -scale * fmaf(gh, ENT ? entropy[r] : 0.0f, g);
  const F2 s2 = pack2(scale, scale), e2 = pack2(kLog2e, kLog2e);
  const F2 A2 = pack2(A, A), B2 = pack2(B, B);
  // A share's gradient: `first` holds the thread's first U pieces already
  // (FROM_LSE), or each is loaded where it is needed.
  auto write = [&](auto from_lse, const Share<T>& sh, const uint4 (&first)[U], float m, float ls) {
    constexpr bool FROM_LSE = decltype(from_lse)::value;
    T* out = dx + r * ldd + sh.start;
    // Where the target is within this share; no index where it is not.
    const uint32_t hot = has && (uint32_t)at - sh.start < sh.count ? (uint32_t)at - sh.start : ~0u;
    const F2 m2 = pack2(-m, -m), z2 = pack2(-ls, -ls);
    // Gradients of two values. l is kept off -inf (p is 0 long before): 0 times it would be NaN.
    auto two = [&](F2 v, float& a, float& b) {
      F2 l = fma2(FROM_LSE ? v : add2(v, m2), s2, z2);
      if (ENT) {
        unpack2(l, a, b);
        l = pack2(max_nan(a, -1000.0f), max_nan(b, -1000.0f));
      }
      unpack2(mul2(l, e2), a, b);
      const F2 p = pack2(exp2_approx(a), exp2_approx(b));
      unpack2(mul2(p, ENT ? fma2(A2, l, B2) : B2), a, b);
    };
    auto single = [&](uint32_t i) {
      const float v = to_f32(sh.p[i]);
      float a, b;
      two(pack2(v, v), a, b);
      out[i] = from_f32<T>(a);
    };
    // The target's own term is added by the thread that has written it.
    uint32_t owner = hot - sh.head;
    if (hot < sh.head) owner = hot;
    else if (hot >= sh.tail_at()) owner = hot - sh.tail_at();
    else owner = owner / V % THREADS;
    const bool mine = hot != ~0u && threadIdx.x == owner;
    const float x_hot = mine ? to_f32(sh.p[hot]) : 0.0f;
    if (threadIdx.x < sh.head) single(threadIdx.x);
    if (threadIdx.x < sh.tail) single(sh.tail_at() + threadIdx.x);
    sh.with_whole(out, [&](auto whole) {
      auto piece = [&](uint32_t i, const uint4& q, int on = 0) {
        uint4 o;
#pragma unroll
        for (int k = 0; k < V / 2; ++k) {
          float a, b;
          two(Piece<T>::pair(q, k), a, b);
          Piece<T>::put(o, k, a, b);
        }
        sh.template put_piece<decltype(whole)::value>(out, i, o, on);
      };
      uint32_t i = threadIdx.x;
      if (FROM_LSE) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i + u * THREADS < sh.pieces) piece(i, first[u], u * THREADS);
        i += U * THREADS;
      }
      for (; i + (U - 1) * THREADS < sh.pieces; i += U * THREADS) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = sh.piece(i, u * THREADS);
#pragma unroll
        for (int u = 0; u < U; ++u) piece(i, q[u], u * THREADS);
      }
      for (; i < sh.pieces; i += THREADS) piece(i, sh.piece(i));
    });
    if (mine) {
      float a, b;
      two(pack2(x_hot, x_hot), a, b);
      out[hot] = from_f32<T>(fmaf(g, scale, a));
    }
  };
  const Share<T> own(xr, n, part, each);
  uint4 first[U];  // on their way while lse is
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (threadIdx.x + u * THREADS < own.pieces) first[u] = own.piece(threadIdx.x, u * THREADS);
  if (fabsf(z) <= kLseExact) {
    write(std::true_type{}, own, first, 0.0f, z);
    return;
  }
  // The whole row is the first block's: others may not write while it is read.
  if (part != 0) return;
  __shared__ Sums all[THREADS / 32];
  const float c = scale * kLog2e;
  const Share<T> row(xr, n, 0, n);
  const Sums v = join_block<false, THREADS / 32>(
      scan_share<T, false, false, false, THREADS>(row, c, nullptr), c, all);
  const bool none = v.m == -INFINITY;  // masked whole: p = 0
  write(std::false_type{}, row, first, none ? 0.0f : v.m, none ? INFINITY : logf(v.s));
}

int check_scores(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, const void* logits,
                 int64_t ld, float scale) {
  if (int rc = check_logits(ctx, rows, n, dtype, logits, ld, scale, "scale")) return rc;
  PLX_CHECK_ARG(scale * kLog2e < INFINITY, "scale = %g is too large", scale);
  return PLX_OK;
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" int plx_log_probs(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                             const void* logits, int64_t ld, const int32_t* target, float scale,
                             uint32_t top, float* logp, float* lse, float* entropy,
                             int32_t* top_ids, float* top_logp) {
  if (int rc = check_scores(ctx, rows, n, dtype, logits, ld, scale)) return rc;
  PLX_CHECK_ARG(top <= n, "top = %u exceeds the %u outputs of a row", top, n);
  if (top > PLX_TOP_MAX)
    return set_error(PLX_ERR_CAPACITY, "top = %u: at most %d are supported", top, PLX_TOP_MAX);
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(lse, "lse is required");
  PLX_CHECK_ARG(!target == !logp, "target and logp go together");
  PLX_CHECK_ARG(!top || (top_ids && top_logp), "top_ids and top_logp are required");
  if (int rc = check_aligned(4, {target, logp, lse, entropy, top_ids, top_logp})) return rc;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const uint32_t parts = row_parts(rows, n);
    auto go = [&](auto kernel, uint32_t threads) {
      PLX_TRY_CUDA(launch_rows(kernel, rows, parts, threads, (size_t)0, ctx->stream, n,
                               part_length(n, parts, Piece<T>::V), (const T*)logits,
                               rows == 1 ? (int64_t)0 : ld, target, scale, top, logp, lse, entropy,
                               top_ids, top_logp, ctx->d_status));
      return PLX_OK;
    };
    auto pick = [&](auto ent, auto best) {
      constexpr bool E = decltype(ent)::value, B = decltype(best)::value;
      // With alternatives 128 threads at most (4,096 rows of 65,536 bf16, 8
      // alternatives: 101 us, with 256 threads 109), but twice as many as
      // alternatives, or their maxima say too little; four times for long rows
      // (64 alternatives of 65,536: 128 threads 143 us, 256 129; of 20,011 the
      // other way, 43 and 48).
      uint32_t threads = row_threads(rows * parts, n / parts);
      if (B && rows * parts > 2 * 148) threads = std::min(threads, 128u);
      if (B && top > 16)
        threads = std::max(threads, top > 32 && n / parts >= 32768 ? 256u : 128u);
      switch (threads) {
        case 64: return go(k_log_probs<T, E, B, 64>, 64);
        case 128: return go(k_log_probs<T, E, B, 128>, 128);
        default: return go(k_log_probs<T, E, B, 256>, 256);
      }
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
  if (int rc = check_scores(ctx, rows, n, dtype, logits, ld, scale)) return rc;
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(grad_logp || grad_entropy, "grad_logp or grad_entropy is required");
  PLX_CHECK_ARG(!grad_logp || target, "grad_logp needs target");
  PLX_CHECK_ARG(!grad_entropy || entropy, "grad_entropy needs entropy");
  PLX_CHECK_ARG(lse && dlogits, "lse and dlogits are required");
  PLX_CHECK_ARG(rows == 1 || ldd >= (int64_t)n, "the gradient's row stride is less than n");
  if (int rc = check_aligned(dtype_bytes(dtype), {dlogits})) return rc;
  if (int rc = check_aligned(4, {target, lse, entropy, grad_logp, grad_entropy})) return rc;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  if (rows == 1) ld = ldd = 0;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto ent, auto threads_c) {
      constexpr int THREADS = decltype(threads_c)::value;
      // Sixteen pieces a thread hide what a block costs; down to four where
      // that would leave SMs without eight blocks. As far as the grid's size
      // allows. (1,500 rows of 32,003 f16, before the first pieces were loaded
      // ahead: 37 us; always four: 43; now 34.)
      uint64_t each = THREADS * 16 * Piece<T>::V;
      while (each > THREADS * 4 * Piece<T>::V && rows * ((n + each - 1) / each) < 148 * 8)
        each /= 2;
      const uint32_t parts = (uint32_t)std::max<uint64_t>(
          1, std::min<uint64_t>((n + each - 1) / each, ((1ull << 31) - 1) / rows));
      k_log_probs_bwd<T, decltype(ent)::value, THREADS>
          <<<(unsigned)(rows * parts), THREADS, 0, ctx->stream>>>(
              n, parts, part_length(n, parts, Piece<T>::V), (const T*)logits, ld, target, scale,
              lse, entropy, grad_logp, grad_entropy, (T*)dlogits, ldd);
    };
    // Rows too short for eight pieces a thread get fewer threads.
    auto pick = [&](auto ent) {
      if (n >= 256 * 8 * Piece<T>::V) go(ent, std::integral_constant<int, 256>{});
      else if (n >= 128 * 8 * Piece<T>::V) go(ent, std::integral_constant<int, 128>{});
      else go(ent, std::integral_constant<int, 64>{});
    };
    if (grad_entropy) pick(std::true_type{});
    else pick(std::false_type{});
    PLX_LAUNCH_CHECK("k_log_probs_bwd");
    return PLX_OK;
  });
}
