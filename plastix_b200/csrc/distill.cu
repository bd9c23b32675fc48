// Distillation from a teacher's top outputs: per row, with p = softmax(x/tau)
// and the teacher's entries (id_j, q_j), Q = sum q_j,
//   loss = w tau^2 sum_j q_j (log q_j - log p_{id_j})
//   dx_i = w tau (Q p_i - sum_{j: id_j = i} q_j)
//
// Bound by memory: logits read once, gradient written once. The gradient needs
// the row's sum first, so the row is gone over twice: for maximum and sum
// (logits.cuh) and for the gradient. In between it stays in shared memory, up
// to kKeepBytes a block, a long row spread over the blocks of a cluster; what
// does not fit is read again out of L2. A warp of its own takes care of the
// teacher's entries meanwhile; the outputs they name are put right at the end.
// Measured, 4,096 rows of 65,536 bf16: loss 84 us, 6.4 TB/s; with gradient 191
// us, 5.6 TB/s (special functions and issue slots are more than half busy);
// second read out of L2 alone 244. 2,048 rows of 65,536 f32: 80, 202.
#include "logits.cuh"

namespace plx {
namespace {

// Of a row in a block's shared memory: three blocks an SM fit, so that one's
// loads run beside another's stores (110 KB and two blocks: 220 us, 54 KB: 242).
constexpr uint32_t kKeepBytes = 72 * 1024;

// THREADS threads go over the row; one more warp takes care of the teacher.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS + 32, 1536 / (THREADS < 256 ? THREADS + 32 : THREADS))
k_distill(uint32_t n, uint32_t each, const T* x, int64_t ld, uint32_t k,
          const int32_t* __restrict__ ids, const float* __restrict__ values, int kind, float tau,
          float inv_tau, const float* __restrict__ weight, float* __restrict__ loss, T* dx,
          int64_t ldd, uint32_t keep_pieces, int32_t* __restrict__ status) {
  constexpr int WARPS = THREADS / 32, V = Piece<T>::V, E = PLX_DISTILL_MAX_K / 32;
  extern __shared__ uint4 keep[];
  __shared__ Sums all[WARPS], mine;
  __shared__ int32_t sid[PLX_DISTILL_MAX_K];
  __shared__ float sq[PLX_DISTILL_MAX_K], qsum_of;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t parts = cl.num_blocks(), part = cl.block_rank();
  const int64_t r = cluster_row();
  const T* xr = x + r * ld;
  const Share<T> share(xr, n, part, each);
  T* out = dx ? dx + r * ldd + share.start : nullptr;
  const bool teacher = threadIdx.x >= THREADS;
  const uint32_t lane = threadIdx.x & 31;
  auto clear = [&] {  // the row does not count, whatever it holds
    if (part == 0 && threadIdx.x == 0) loss[r] = 0.0f;
    if (!out || teacher) return;
    if (threadIdx.x < share.head) out[threadIdx.x] = from_f32<T>(0.0f);
    share.with_whole(out, [&](auto whole) {
      for (uint32_t i = threadIdx.x; i < share.pieces; i += THREADS)
        share.template put_piece<decltype(whole)::value>(out, i, make_uint4(0, 0, 0, 0));
    });
    if (threadIdx.x < share.tail) out[share.tail_at() + threadIdx.x] = from_f32<T>(0.0f);
  };
  const float w = weight ? weight[r] : 1.0f;
  if (w == 0.0f) {  // so says every block of the row's cluster
    clear();
    return;
  }

  const float c = inv_tau * kLog2e;
  const uint32_t kept = out ? min(share.pieces, keep_pieces) : 0;
  Sums v{-INFINITY, 0.0f, 0.0f};
  // The teacher's row, E entries a lane: of an output named twice the first
  // entry has the sum, `all_q`, and is the one that writes.
  int32_t id[E];
  float lq[E], q[E], all_q[E], x_at[E], qsum = 0.0f;
  if (!teacher) {
    v = scan_share<T, false, false, true, THREADS>(share, c, nullptr, keep, kept);
  } else {
    float most = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t j = lane + 32 * e;
      id[e] = j < k ? ids[r * k + j] : -1;
      lq[e] = j < k ? values[r * k + j] : -INFINITY;
      if (id[e] < -1 || id[e] >= (int64_t)n) {
        record_status(status, kStatusBadOutput);
        id[e] = -1;
      }
      if (id[e] < 0) lq[e] = -INFINITY;
      x_at[e] = id[e] < 0 ? 0.0f : to_f32(xr[id[e]]);  // before a gradient takes its place
      most = max_nan(most, lq[e]);
    }
    if (kind == PLX_TEACHER_LOGITS) {
      most = warp_max(most);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (most != -INFINITY) lq[e] = (lq[e] - most) * inv_tau;
        sum += expf(lq[e]);
      }
      sum = warp_sum(sum);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (kind == PLX_TEACHER_LOGITS && most != -INFINITY) lq[e] -= logf(sum);
      q[e] = lq[e] == -INFINITY ? 0.0f : expf(lq[e]);
      qsum += q[e];
      sid[lane + 32 * e] = id[e];
      sq[lane + 32 * e] = q[e];
    }
    qsum = warp_sum(qsum);
    if (lane == 0) qsum_of = qsum;
    __syncwarp();
    if (out) {
      // Mostly no output is named twice, which 32 entries tell at once.
      const uint32_t same = __match_any_sync(0xffffffffu, id[0]);
      const bool search =
          k > 32 || __any_sync(0xffffffffu, id[0] >= 0 && (same & (same - 1)) != 0);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        all_q[e] = q[e];
        if (search) {
          all_q[e] = 0.0f;
          bool first = true;
          for (uint32_t j = 0; j < k; ++j)
            if (sid[j] == id[e]) {
              all_q[e] += sq[j];
              first = first && j >= lane + 32 * e;
            }
          if (!first) id[e] = -1;  // not written here
        }
        if ((uint32_t)id[e] - share.start >= share.count) id[e] = -1;
      }
    }
  }
  v = join_block<false, WARPS>(v, c, all);
  if (parts > 1) {
    if (threadIdx.x == 0) mine = v;
    cl.sync();
    v = join_parts<false>(cl, &mine, c);
    cl.barrier_arrive();  // done with the others' memory; waited for before leaving
  }
  qsum = qsum_of;
  if (qsum == 0.0f) {
    clear();
    if (parts > 1) cl.barrier_wait();
    return;
  }
  const bool none = v.m == -INFINITY;  // the student masks every output
  const float a = w * tau, f = none ? 0.0f : a * qsum / v.s;
  float fixed[E];  // the gradients at the teacher's outputs
  if (teacher) {
    const float ls = logf(v.s);
    float term = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float logp = none ? -INFINITY : (x_at[e] - v.m) * inv_tau - ls;
      if (q[e] != 0.0f) term += q[e] * (lq[e] - logp);
      fixed[e] = a * (qsum * expf(logp) - all_q[e]);
    }
    term = warp_sum(term);
    if (part == 0 && lane == 0) loss[r] = w * tau * tau * term;
  } else if (out) {
    const float m = none ? INFINITY : v.m;  // 2^-inf = 0
    auto single = [&](uint32_t i) {
      out[i] = from_f32<T>(f * exp2_approx((to_f32(share.p[i]) - m) * c));
    };
    if (threadIdx.x < share.head) single(threadIdx.x);
    if (threadIdx.x < share.tail) single(share.tail_at() + threadIdx.x);
    const F2 minus = pack2(-m, -m), c2 = pack2(c, c), f2 = pack2(f, f);
    share.with_whole(out, [&](auto whole) {
      auto piece = [&](uint32_t i, const uint4& p, int on = 0) {
        uint4 o;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const F2 d = mul2(add2(Piece<T>::pair(p, e), minus), c2);
          const F2 g = mul2(pack2(exp2_approx(d.x), exp2_approx(d.y)), f2);
          Piece<T>::put(o, e, g.x, g.y);
        }
        share.template put_piece<decltype(whole)::value>(out, i, o, on);
      };
      uint32_t i = threadIdx.x;
      for (; i < kept; i += THREADS) piece(i, keep[i]);
      for (; i + 3 * THREADS < share.pieces; i += 4 * THREADS) {
        uint4 q4[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) q4[u] = share.piece(i, u * THREADS);
#pragma unroll
        for (int u = 0; u < 4; ++u) piece(i, q4[u], u * THREADS);
      }
      for (; i < share.pieces; i += THREADS) piece(i, share.piece(i));
    });
  }
  if (out) {
    __syncthreads();
    if (teacher)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (id[e] >= 0) out[(uint32_t)id[e] - share.start] = from_f32<T>(fixed[e]);
  }
  if (parts > 1) cl.barrier_wait();
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" int plx_distill(plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype, const void* logits,
                           int64_t ld, uint32_t k, const int32_t* teacher_ids,
                           const float* teacher_values, int teacher_kind, float temperature,
                           const float* row_weight, float* loss, void* dlogits, int64_t ldd) {
  if (int rc = check_logits(ctx, rows, n, dtype, logits, ld, temperature, "temperature"))
    return rc;
  PLX_CHECK_ARG(1.0f / temperature * kLog2e < INFINITY, "temperature = %g is too small", temperature);
  PLX_CHECK_ARG(teacher_kind == PLX_TEACHER_LOGITS || teacher_kind == PLX_TEACHER_LOG_PROBS,
                "teacher_kind %d is neither PLX_TEACHER_LOGITS nor PLX_TEACHER_LOG_PROBS",
                teacher_kind);
  PLX_CHECK_ARG(k > 0, "k has to be positive");
  if (k > PLX_DISTILL_MAX_K)
    return set_error(PLX_ERR_CAPACITY, "k = %u: at most %d entries a row are supported", k,
                     PLX_DISTILL_MAX_K);
  if (rows == 0) return PLX_OK;
  PLX_CHECK_ARG(teacher_ids && teacher_values && loss,
                "teacher_ids, teacher_values and loss are required");
  PLX_CHECK_ARG(!dlogits || rows == 1 || ldd >= (int64_t)n,
                "the gradient's row stride is less than n");
  if (int rc = check_aligned(dtype_bytes(dtype), {dlogits})) return rc;
  if (int rc = check_aligned(4, {teacher_ids, teacher_values, row_weight, loss})) return rc;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  if (rows == 1) ld = ldd = 0;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr uint32_t V = Piece<T>::V;
    // A row that has to stay is split until half of a part fits: what is read
    // again of 444 parts at once is then still in L2.
    uint32_t parts = row_parts(rows, n);
    if (dlogits)
      while (parts < 8 && (uint64_t)n * sizeof(T) > (uint64_t)parts * 2 * kKeepBytes &&
             rows * parts < (1ull << 30))
        parts *= 2;
    auto go = [&](auto threads_c) {
      constexpr int THREADS = decltype(threads_c)::value;
      constexpr auto kernel = k_distill<T, THREADS>;
      uint32_t pieces = 0;
      if (dlogits) {
        pieces = std::min<uint32_t>((n + parts - 1) / parts / V + 1, kKeepBytes / 16);
        if (pieces * 16 > 47 * 1024) PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, kKeepBytes));
      }
      PLX_TRY_CUDA(launch_rows(kernel, rows, parts, THREADS + 32, (size_t)pieces * 16, ctx->stream,
                               n, part_length(n, parts, V), (const T*)logits, ld, k, teacher_ids,
                               teacher_values, teacher_kind, temperature, 1.0f / temperature,
                               row_weight, loss, (T*)dlogits, ldd, pieces, ctx->d_status));
      return PLX_OK;
    };
    // Where three blocks an SM have all the shared memory they are the largest
    // (4,096 rows of 65,536 bf16: 512 threads 191 us, 256 205; 480, for 40
    // registers each and not 32, 220: the last of a row's rounds is mostly idle).
    const bool large = dlogits && (uint64_t)n * sizeof(T) > (uint64_t)parts * 48 * 1024;
    switch (large ? 512 : row_threads(rows * parts, n / parts)) {
      case 512: return go(std::integral_constant<int, 512>{});
      case 256: return go(std::integral_constant<int, 256>{});
      case 128: return go(std::integral_constant<int, 128>{});
      default: return go(std::integral_constant<int, 64>{});
    }
  });
}
