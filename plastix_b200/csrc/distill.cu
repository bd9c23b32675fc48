// Distillation from a teacher's top outputs: per row, with p = softmax(x/tau)
// and the teacher's entries (id_j, q_j), Q = sum q_j,
//   loss = w tau^2 sum_j q_j (log q_j - log p_{id_j})
//   dx_i = w tau (Q p_i - sum_{j: id_j = i} q_j)
//
// Bound by memory: logits read once, gradient written once. The gradient needs
// the row's sum first, so the row is gone over twice: once for maximum and sum
// (logits.cuh), once, out of L2, for the gradient. The few outputs the teacher
// lists are put right after that.
#include "logits.cuh"

namespace plx {
namespace {

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
k_distill(uint32_t n, const T* x, int64_t ld, uint32_t k, const int32_t* __restrict__ ids,
          const float* __restrict__ values, int kind, float tau, float inv_tau,
          const float* __restrict__ weight, float* __restrict__ loss, T* dx, int64_t ldd,
          int32_t* __restrict__ status) {
  constexpr int WARPS = THREADS / 32, V = Piece<T>::V;
  static_assert(THREADS >= PLX_DISTILL_MAX_K, "one thread an entry");
  __shared__ float red[WARPS];
  __shared__ int32_t sid[PLX_DISTILL_MAX_K];
  __shared__ float sq[PLX_DISTILL_MAX_K];
  __shared__ Sums mine;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t parts = cl.num_blocks(), part = cl.block_rank();
  const int64_t r = blockIdx.x / parts;
  const T* xr = x + r * ld;
  const Share<T> share(xr, n, part, parts);
  T* out = dx ? dx + r * ldd + share.start : nullptr;
  const bool whole = (reinterpret_cast<uintptr_t>(out + share.head) & 15u) == 0;
  auto store = [&](uint32_t i, const uint4& o) {
    const uint32_t first = share.piece_at(i);
    if (whole) {
      *reinterpret_cast<uint4*>(out + first) = o;
    } else {
      const T* e = reinterpret_cast<const T*>(&o);
#pragma unroll
      for (int j = 0; j < V; ++j) out[first + j] = e[j];
    }
  };

  // The teacher's row: one thread an entry.
  const uint32_t j = threadIdx.x;
  int32_t id = j < k ? ids[r * k + j] : -1;
  if (id < -1 || id >= (int64_t)n) {
    record_status(status, kStatusBadOutput);
    id = -1;
  }
  float lq = id < 0 ? -INFINITY : values[r * k + j];
  const float x_at = id < 0 ? 0.0f : to_f32(xr[id]);  // before any gradient takes its place
  if (kind == PLX_TEACHER_LOGITS) {
    const float most = block_max<WARPS>(lq, red);
    if (most != -INFINITY) lq = (lq - most) * inv_tau;
    const float sum = block_sum<WARPS>(expf(lq), red);
    if (most != -INFINITY) lq -= logf(sum);
  }
  const float q = id < 0 || lq == -INFINITY ? 0.0f : expf(lq);
  if (j < k) {
    sid[j] = id;
    sq[j] = q;
  }
  const float qsum = block_sum<WARPS>(q, red);
  const float w = weight ? weight[r] : 1.0f;
  if (w == 0.0f || qsum == 0.0f) {  // the row does not count, whatever it holds
    if (part == 0 && threadIdx.x == 0) loss[r] = 0.0f;
    if (out) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      if (threadIdx.x < share.head) out[threadIdx.x] = from_f32<T>(0.0f);
      for (uint32_t i = threadIdx.x; i < share.pieces; i += THREADS) store(i, zero);
      if (threadIdx.x < share.tail) out[share.tail_at() + threadIdx.x] = from_f32<T>(0.0f);
    }
    return;  // every block of the row's cluster does
  }

  const float c = inv_tau * kLog2e;
  uint32_t pos;
  Sums v = join_block<false, WARPS>(scan_share<T, false, false, THREADS>(share, c, pos), c, red);
  if (parts > 1) {
    v = join_cluster<false>(cl, &mine, v, c);
    cl.barrier_arrive();  // done with the others' memory; waited for before leaving
  }
  const bool none = v.m == -INFINITY;  // the student masks every output
  const float ls = logf(v.s);
  const float logp = none ? -INFINITY : (x_at - v.m) * inv_tau - ls;
  if (part == 0) {
    const float term = block_sum<WARPS>(q != 0.0f ? q * (lq - logp) : 0.0f, red);
    if (threadIdx.x == 0) loss[r] = w * tau * tau * term;
  }
  if (out) {
    const float a = w * tau, f = none ? 0.0f : a * qsum / v.s;
    const float m = none ? INFINITY : v.m;  // 2^-inf = 0
    auto single = [&](uint32_t i) {
      out[i] = from_f32<T>(f * exp2_approx((to_f32(share.p[i]) - m) * c));
    };
    if (threadIdx.x < share.head) single(threadIdx.x);
    const F2 minus = pack2(-m, -m), c2 = pack2(c, c), f2 = pack2(f, f);
    for (uint32_t i = threadIdx.x; i < share.pieces; i += THREADS) {
      const uint4 p = share.piece(i);
      uint4 o;
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        float a0, a1;
        unpack2(mul2(add2(Piece<T>::pair(p, e), minus), c2), a0, a1);
        unpack2(mul2(pack2(exp2_approx(a0), exp2_approx(a1)), f2), a0, a1);
        Piece<T>::put(o, e, a0, a1);
      }
      store(i, o);
    }
    if (threadIdx.x < share.tail) single(share.tail_at() + threadIdx.x);
    __syncthreads();
    // An output named twice is written by its first entry.
    if (id >= 0 && (uint32_t)id - share.start < share.count) {
      float both = 0.0f;
      bool first = true;
      for (uint32_t i = 0; i < k; ++i)
        if (sid[i] == id) {
          both += sq[i];
          if (i < j) first = false;
        }
      if (first) out[(uint32_t)id - share.start] = from_f32<T>(a * (qsum * expf(logp) - both));
    }
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
  PLX_CHECK_ARG(1.0f / temperature < INFINITY, "temperature = %g is too small", temperature);
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
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  if (rows == 1) ld = ldd = 0;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto kernel, uint32_t threads) {
      PLX_TRY_CUDA(launch_rows(kernel, rows, row_parts(rows, n, 4096), threads, ctx->stream, n,
                               (const T*)logits, ld, k, teacher_ids, teacher_values, teacher_kind,
                               temperature, 1.0f / temperature, row_weight, loss, (T*)dlogits, ldd,
                               ctx->d_status));
      return PLX_OK;
    };
    return n < 128 * 4 * Piece<T>::V ? go(k_distill<T, 128>, 128) : go(k_distill<T, 512>, 512);
  });
}
