// Gated linear recurrence of units over the steps of streams, and its gradients.
//   h_t = a_t h_{t-1} + c_t x_t,   a = gate or sigmoid(gate),   c = 1 or 1 - a
//   g_t = dh_t + a_{t+1} g_{t+1};  dx = c g;  da = g h_{t-1}  or  g (h_{t-1} - x)
// Units are independent; steps are folded as pairs (A, H): a run of steps takes
// what it is given, h, to A h + H, and two runs join to (A1 A2, A2 H1 + H2).
//
// Bound by memory: a tile of steps x units is read once, its values stay in
// registers between the fold of its runs and the second walk that writes its
// results. A warp has the steps of one run, a lane one or two units; the block's
// runs are joined through shared memory, tiles of one stream through scratch: a
// tile leaves its pair, looks back over up to 16 tiles before it to the nearest
// one that already has its end value, and folds from there on in the order of
// the steps, which gives the bits that the tile in between gives itself: the
// result does not depend on who was first. Tiles are handed out in the order of
// the steps, so those waited for are under way.
#include <type_traits>

#include "norm.cuh"

namespace plx {
namespace {

// Runs of a tile, forwards and backwards, which has more values in registers: two
// blocks an SM either way.
__host__ __device__ constexpr int warps_of(bool back) { return back ? 12 : 16; }
constexpr int kRun = 8;      // steps of a run
__host__ __device__ constexpr uint32_t tile_steps(bool back) { return warps_of(back) * kRun; }
constexpr uint32_t kLook = 32;  // tiles that one looks back over

// How rows are cut: `parts` parts of `part_rows` rows (the last may be shorter),
// each of `chunks` tiles of `chunk_rows` rows (a multiple of the runs' length
// but for the last). No stream crosses a part's end.
struct Cut {
  uint32_t parts, part_rows, chunks, chunk_rows;
};

Cut cut_rows(uint32_t streams, uint64_t rows, bool ragged, bool back) {
  Cut c;
  const uint64_t steps = ragged ? rows : rows / streams;
  const uint32_t tile = tile_steps(back);
  if (steps <= tile && !ragged) {  // whole streams in a tile
    c.chunk_rows = c.part_rows = (uint32_t)(tile / steps * steps);
    c.chunks = 1;
  } else {
    c.part_rows = (uint32_t)steps;
    c.chunks = (uint32_t)((steps + tile - 1) / tile);
    c.chunk_rows = tile;
  }
  c.parts = (uint32_t)((rows + c.part_rows - 1) / c.part_rows);
  return c;
}

struct Scratch {  // at the head of the scratch; the flags of the tiles follow
  uint32_t ticket, gave_up, pad[62];
};
constexpr uint32_t kPair = 1, kEnd = 2;  // a tile has left its pair, its end value

struct Args {
  uint64_t rows;
  uint32_t n, streams, steps;  // steps of a stream; 0 with offsets
  Cut cut;
  uint32_t tiles;              // across the units
  const int32_t* offsets;
  const void *x, *gate, *h, *dh;
  int64_t ldx, ldg, ldh, lddh;
  const float *state, *dfinal;
  void *out, *out2;            // h; or dx and dgate
  int64_t ldo, ldo2;
  float* state_out;            // final; or dstate
  Scratch* scratch;
  uint32_t* flags;
  float2* pairs;
  float* ends;
  int32_t* status;
  uint64_t timeout_ns;
};

__device__ __forceinline__ uint32_t ld_acquire(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void st_release(uint32_t* p, uint32_t v) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// One or two units at once.
template <int V>
using Units = std::conditional_t<V == 2, F2, float>;
__device__ __forceinline__ float addw(float a, float b) { return __fadd_rn(a, b); }
__device__ __forceinline__ float mulw(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ float fmaw(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ F2 addw(F2 a, F2 b) { return add2(a, b); }
__device__ __forceinline__ F2 mulw(F2 a, F2 b) { return mul2(a, b); }
__device__ __forceinline__ F2 fmaw(F2 a, F2 b, F2 c) { return fma2(a, b, c); }
template <typename W>
__device__ __forceinline__ W all(float v) {
  if constexpr (std::is_same_v<W, F2>) return pack2(v, v);
  else return v;
}
template <typename F>
__device__ __forceinline__ float each(float v, F f) { return f(v); }
template <typename F>
__device__ __forceinline__ F2 each(F2 v, F f) { return pack2(f(v.x), f(v.y)); }
template <typename T, int V>
__device__ __forceinline__ Units<V> wide(const Pack<T, V>& q) {
  if constexpr (V == 2) return pair_of(q, 0);
  else return to_f32(q.v[0]);
}
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> narrow(Units<V> v) {
  Pack<T, V> q;
  if constexpr (V == 2) put_pair(q, 0, v);
  else q.v[0] = from_f32<T>(v);
  return q;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}

// a and 1 - a of a gate, neither by a difference that cancels: with e = exp(-gate),
// 1 / (1 + e) and e / (1 + e). The quotient gets one Newton step: what a is off by, a
// long memory raises to its length. e is at most 2^126 (a gate of -infinity leaves
// 2^-126 of h).
template <typename W>
__device__ __forceinline__ W exp_minus(W g) {
  return each(mulw(g, all<W>(-kLog2e)), [](float t) { return exp2_approx(min_nan(t, 126.0f)); });
}
template <bool SIGMOID, typename W>
__device__ __forceinline__ void gate_value(W g, W& a, W& keep) {
  if constexpr (SIGMOID) {
    const W e = exp_minus(g);
    const W d = addw(e, all<W>(1.0f)), minus = each(d, [](float t) { return -t; });
    const W r = each(d, rcp_approx);
    a = fmaw(r, fmaw(minus, r, all<W>(1.0f)), r);
    keep = mulw(e, a);
  } else {
    a = g;
    keep = each(g, [](float t) { return __fsub_rn(1.0f, t); });
  }
}

// The stream of a row, and whether it begins or ends there.
struct Place {
  uint32_t stream;
  bool valid, first, last;
};
__device__ __forceinline__ Place place_of(const Args& p, uint64_t row) {
  Place q;
  if (!p.offsets) {
    q.stream = (uint32_t)(row / p.steps);
    const uint32_t at = (uint32_t)(row - (uint64_t)q.stream * p.steps);
    q.valid = true;
    q.first = at == 0;
    q.last = at + 1 == p.steps;
    return q;
  }
  // the last stream that begins at or before the row (empty ones come before it)
  uint32_t lo = 0, hi = p.streams;  // offsets[lo] <= row where any is
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if ((int64_t)__ldg(p.offsets + mid) <= (int64_t)row) lo = mid;
    else hi = mid;
  }
  const int64_t begin = __ldg(p.offsets + lo), end = __ldg(p.offsets + lo + 1);
  q.stream = lo;
  q.valid = begin <= (int64_t)row && (int64_t)row < end;
  q.first = q.valid && begin == (int64_t)row;
  q.last = q.valid && end == (int64_t)row + 1;
  return q;
}

// A step's values as both walks use them: forwards a and b (h = a h + b), where a
// stream begins with its state in b; backwards a, dh and what g is multiplied by.
template <typename T, int V, bool SIGMOID, bool MIX, bool BACK>
struct Step {
  using W = Units<V>;
  using P = Pack<T, V>;
  W a, b;     // b: forwards
  P dh;       // backwards
  W slope;    // dgate = g slope
  P gate;     // with a, 1 - a
  __device__ __forceinline__ void forward(P gate, P x) {
    W k;
    gate_value<SIGMOID>(wide<T, V>(gate), a, k);
    b = wide<T, V>(x);
    if (MIX) b = mulw(b, k);
  }
  __device__ __forceinline__ void backward(P gate_, P d, W before, P x) {
    gate = gate_;
    W k;
    gate_value<SIGMOID>(wide<T, V>(gate), a, k);
    dh = d;
    slope = before;
    if (MIX) slope = addw(slope, each(wide<T, V>(x), [](float t) { return -t; }));
    if (SIGMOID) slope = mulw(slope, mulw(a, k));
  }
  __device__ __forceinline__ W dx(W g) const {
    if (!MIX) return g;
    if (SIGMOID) return mulw(g, mulw(exp_minus(wide<T, V>(gate)), a));
    return mulw(g, each(a, [](float t) { return __fsub_rn(1.0f, t); }));
  }
};

template <int V>
__device__ __forceinline__ Units<V> load_units(const float* p, bool in) {
  if constexpr (V == 2) return in ? pack2(p[0], p[1]) : pack2(0.0f, 0.0f);
  else return in ? p[0] : 0.0f;
}
template <int V>
__device__ __forceinline__ void store_units(float* p, Units<V> v) {
  if constexpr (V == 2) {
    p[0] = v.x;
    p[1] = v.y;
  } else {
    p[0] = v;
  }
}

template <typename T, int V, bool SIGMOID, bool MIX, bool BACK>
__global__ void __launch_bounds__(warps_of(BACK) * 32, 2)
k_recurrence(const __grid_constant__ Args p) {
  constexpr int kWarps = warps_of(BACK);
  using W = Units<V>;
  using P = Pack<T, V>;
  struct alignas(8 * V) Pair {
    W a, h;
  };
  __shared__ Pair runs[kWarps][32], look[kLook][32];
  __shared__ W look_end[32];
  __shared__ uint32_t run_shut[kWarps], ticket, near;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const W zero = all<W>(0.0f);

  if (p.offsets) {  // offsets that no rows have; streams without steps hand their state on
    for (uint32_t s = blockIdx.x; s < p.streams; s += gridDim.x) {
      const int64_t begin = p.offsets[s], end = p.offsets[s + 1];
      if (threadIdx.x == 0 && (begin < 0 || begin > end || (uint64_t)end > p.rows))
        record_status(p.status, kStatusBadOffsets);
      const float* given = BACK ? p.dfinal : p.state;
      if (begin == end && p.state_out)
        for (uint32_t i = threadIdx.x; i < p.n; i += kWarps * 32)
          p.state_out[(uint64_t)s * p.n + i] = given ? given[(uint64_t)s * p.n + i] : 0.0f;
    }
  }

  // Tiles in the order of the steps (backwards: from the last), those of all
  // parts beside each other.
  uint32_t id = blockIdx.x;
  const bool chained = p.cut.chunks > 1;
  if (chained) {
    if (threadIdx.x == 0) ticket = atomicAdd(&p.scratch->ticket, 1u);
    __syncthreads();
    id = ticket;
  }
  const uint32_t across = id % p.tiles, rest = id / p.tiles;
  const uint32_t part = rest % p.cut.parts, turn = rest / p.cut.parts;
  const uint32_t chunk = BACK ? p.cut.chunks - 1 - turn : turn;
  const uint64_t part_end = min((uint64_t)(part + 1) * p.cut.part_rows, p.rows);
  const uint64_t row0 = (uint64_t)part * p.cut.part_rows + (uint64_t)chunk * p.cut.chunk_rows;
  const uint64_t row1 = min(row0 + p.cut.chunk_rows, part_end);
  const uint32_t unit = (across * 32 + lane) * V;
  const bool in = unit < p.n;  // V divides n
  // This warp's run, in the order that it is walked.
  const uint32_t run = BACK ? kWarps - 1 - warp : warp;
  const uint64_t at = row0 + run * kRun;
  const int len = at < row1 ? (int)min((uint64_t)kRun, row1 - at) : 0;

  P qg[kRun], q1[kRun], q2[BACK ? kRun : 1], q3[BACK && MIX ? kRun : 1];
  P nothing;
#pragma unroll
  for (int e = 0; e < V; ++e) nothing.v[e] = from_f32<T>(0.0f);
  auto load = [&](P(&q)[kRun], const void* array, int64_t ld) {
    const T* from = (const T*)array + (int64_t)at * ld + unit;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      q[i] = nothing;
      if (in && i < len) q[i] = load_pack<T, V>(from + i * ld);
    }
  };
  load(qg, p.gate, p.ldg);
  load(q1, BACK ? p.dh : p.x, BACK ? p.lddh : p.ldx);
  if constexpr (BACK && MIX) load(q3, p.x, p.ldx);
  // Where streams begin and end in the run: a row to a lane.
  Place mine = {0, false, false, false};
  if ((int)lane < len) mine = place_of(p, at + lane);
  const uint32_t valid = __ballot_sync(~0u, mine.valid);
  const uint32_t first = __ballot_sync(~0u, mine.first), last = __ballot_sync(~0u, mine.last);
  auto state_at = [&](const float* states, int i) {
    const uint32_t s = __shfl_sync(~0u, mine.stream, i);
    return states ? load_units<V>(states + (uint64_t)s * p.n + unit, in) : zero;
  };
  if constexpr (BACK) {
    const T* from = (const T*)p.h + ((int64_t)at - 1) * p.ldh + unit;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      q2[i] = nothing;
      if (in && (valid >> i & 1) && !(first >> i & 1)) q2[i] = load_pack<T, V>(from + i * p.ldh);
    }
  }

  // ---- the run's pair. `stop`: rows at which what was before does not count.
  const uint32_t stop = BACK ? last : first;
  Step<T, V, SIGMOID, MIX, BACK> steps[kRun];
  W A = all<W>(1.0f), H = zero;
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = BACK ? kRun - 1 - k : k;
    if (i >= len) continue;
    auto& st = steps[i];
    if constexpr (BACK) {
      W before = wide<T, V>(q2[i]);
      if (first >> i & 1) before = state_at(p.state, i);
      st.backward(qg[i], q1[i], before, q3[MIX ? i : 0]);
      if (stop >> i & 1) {  // the same for the whole warp
        H = state_at(p.dfinal, i);
        A = zero;
      }
      H = mulw(st.a, addw(wide<T, V>(st.dh), H));
      A = mulw(A, st.a);
    } else {
      st.forward(qg[i], q1[i]);
      if (stop >> i & 1) {
        st.b = fmaw(st.a, state_at(p.state, i), st.b);
        H = st.b;
        A = zero;
      } else {
        H = fmaw(st.a, H, st.b);
        A = mulw(A, st.a);
      }
    }
  }
  runs[warp][lane] = {A, H};
  if (lane == 0) run_shut[warp] = stop;
  __syncthreads();

  // ---- what the tile is given, and what it leaves
  W carry = zero;
  if (chained) {
    const uint32_t step = p.cut.parts * p.tiles;  // between tiles of a part
    Pair* pairs = reinterpret_cast<Pair*>(p.pairs);
    W* ends = reinterpret_cast<W*>(p.ends);
    W ta = all<W>(1.0f), th = zero;
    bool shut = turn == 0;
    auto leave = [&](bool end) {
      if (end) ends[(uint64_t)id * 32 + lane] = th;
      else pairs[(uint64_t)id * 32 + lane] = {ta, th};
      __threadfence();
      __syncwarp();
      if (lane == 0) st_release(p.flags + id, end ? kEnd : kPair);
    };
    if (warp == 0) {
      for (int w = 0; w < kWarps; ++w) {
        const Pair v = runs[w][lane];
        const bool s = run_shut[w] != 0;
        shut |= s;
        th = s ? v.h : fmaw(v.a, th, v.h);
        ta = s ? zero : mulw(ta, v.a);
      }
      leave(shut);
    } else if (warp == 1 && turn > 0) {
      // The nearest tile before that has its end value, all in between their pairs.
      const bool there = lane < turn;
      const uint32_t* flag = p.flags + id - (lane + 1) * (there ? step : 0);
      const uint64_t t0 = global_timer_ns();
      uint32_t found = kLook;
      for (uint32_t spin = 1;; ++spin) {
        const uint32_t v = there ? ld_acquire(flag) : kPair;
        const uint32_t ended = __ballot_sync(~0u, v == kEnd);
        const uint32_t waiting = __ballot_sync(~0u, v == 0);
        if (ended) {
          found = __ffs(ended) - 1;
          if (!(waiting & ((1u << found) - 1))) break;
        }
        if ((spin & 63u) == 0) {
          bool stop_now = *(volatile uint32_t*)&p.scratch->gave_up != 0;
          if (global_timer_ns() - t0 > p.timeout_ns) {
            record_status(p.status, kStatusTimeout);
            *(volatile uint32_t*)&p.scratch->gave_up = 1;
            stop_now = true;
          }
          if (__any_sync(~0u, stop_now)) {
            found = kLook;
            break;
          }
        }
      }
      __threadfence();
      if (lane == 0) near = found;
    }
    __syncthreads();
    if (turn > 0 && near < kLook) {
      const uint32_t count = near;
      for (uint32_t j = warp; j <= count; j += kWarps) {
        const uint64_t from = (uint64_t)(id - (j + 1) * step) * 32 + lane;
        if (j == count) {
          if constexpr (V == 2) look_end[lane] = __ldcg(reinterpret_cast<const float2*>(ends + from));
          else look_end[lane] = __ldcg(ends + from);
        } else if constexpr (V == 2) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(pairs + from));
          look[j][lane] = {pack2(v.x, v.y), pack2(v.z, v.w)};
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(pairs + from));
          look[j][lane] = {v.x, v.y};
        }
      }
      __syncthreads();
      carry = look_end[lane];
      for (int j = (int)count - 1; j >= 0; --j) {
        const Pair v = look[j][lane];
        carry = fmaw(v.a, carry, v.h);
      }
    }
    if (warp == 0 && !shut) {
      th = fmaw(ta, carry, th);
      leave(true);
    }
  }
  for (uint32_t w = 0; w < warp; ++w) {
    const Pair v = runs[w][lane];
    carry = run_shut[w] ? v.h : fmaw(v.a, carry, v.h);
  }

  // ---- the run once more, from what it is given
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = BACK ? kRun - 1 - k : k;
    if (i >= len) continue;
    const auto& st = steps[i];
    const int64_t row = (int64_t)(at + i);
    const bool write = in && (valid >> i & 1);
    if constexpr (BACK) {
      if (stop >> i & 1) carry = state_at(p.dfinal, i);
      const W g = addw(wide<T, V>(st.dh), carry);
      carry = mulw(st.a, g);
      if (write) {
        *reinterpret_cast<P*>((T*)p.out + row * p.ldo + unit) = narrow<T, V>(st.dx(g));
        *reinterpret_cast<P*>((T*)p.out2 + row * p.ldo2 + unit) = narrow<T, V>(mulw(g, st.slope));
      }
    } else {
      carry = stop >> i & 1 ? st.b : fmaw(st.a, carry, st.b);
      if (write) *reinterpret_cast<P*>((T*)p.out + row * p.ldo + unit) = narrow<T, V>(carry);
    }
    if (p.state_out && ((BACK ? first : last) >> i & 1)) {
      const uint32_t s = __shfl_sync(~0u, mine.stream, i);
      if (in) store_units<V>(p.state_out + (uint64_t)s * p.n + unit, carry);
    }
  }
}

__global__ void k_copy_state(uint64_t count, const float* from, float* to) {
  const uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < count) to[i] = from ? from[i] : 0.0f;
}

int check_recurrence(const plx_ctx* ctx, uint32_t streams, uint64_t rows, uint32_t n, int dtype,
                     const int32_t* offsets, int gate_kind, const void* scratch,
                     size_t scratch_bytes) {
  PLX_CHECK_ARG(ctx, "ctx is required");
  PLX_CHECK_ARG(valid_dtype(dtype), "dtype %d is none of PLX_F32, PLX_BF16, PLX_F16", dtype);
  PLX_CHECK_ARG(gate_kind == PLX_GATE_DECAY || gate_kind == PLX_GATE_SIGMOID,
                "gate_kind %d is neither PLX_GATE_DECAY nor PLX_GATE_SIGMOID", gate_kind);
  PLX_CHECK_ARG(n > 0 && n < (1u << 31), "n = %u is out of range", n);
  PLX_CHECK_ARG(streams < (1u << 31), "%u streams: fewer than 2^31 are supported", streams);
  if (rows >= (1ull << 31))
    return set_error(PLX_ERR_CAPACITY, "%llu rows: fewer than 2^31 are supported",
                     (unsigned long long)rows);
  PLX_CHECK_ARG(streams > 0 || rows == 0, "%llu rows of no stream", (unsigned long long)rows);
  PLX_CHECK_ARG(offsets || streams == 0 || rows % streams == 0,
                "%llu rows are not the same number of steps for each of %u streams",
                (unsigned long long)rows, streams);
  const size_t need = plx_recurrence_scratch_bytes(streams, rows, n, offsets != nullptr);
  PLX_CHECK_ARG(need == 0 || (scratch && scratch_bytes >= need),
                "%zu bytes of scratch are needed, got %zu", need,
                scratch ? scratch_bytes : (size_t)0);
  PLX_CHECK_ARG(aligned16(scratch), "scratch has to be 16-byte aligned");
  return check_aligned(4, {offsets});
}

template <bool BACK>
int launch(plx_ctx* ctx, Args a, int dtype, int gate_kind, bool mix, void* scratch) {
  if (a.streams == 0) return PLX_OK;
  DeviceGuard guard(ctx->device);
  PLX_TRY_CUDA(guard.err);
  if (a.rows == 0) {
    const float* from = BACK ? a.dfinal : a.state;
    const uint64_t count = (uint64_t)a.streams * a.n;
    if (a.state_out && a.state_out != from)
      k_copy_state<<<(unsigned)((count + 255) / 256), 256, 0, ctx->stream>>>(count, from,
                                                                            a.state_out);
    PLX_LAUNCH_CHECK("k_copy_state");
    return PLX_OK;
  }
  if (a.rows == 1) a.ldx = a.ldg = a.ldh = a.lddh = a.ldo = a.ldo2 = a.n;
  a.steps = a.offsets ? 0 : (uint32_t)(a.rows / a.streams);
  a.cut = cut_rows(a.streams, a.rows, a.offsets != nullptr, BACK);
  a.status = ctx->d_status;
  a.timeout_ns = ctx->timeout_ns;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    uint64_t odd = a.n;
    for (int64_t ld : {a.ldx, a.ldg, a.ldh, a.lddh, a.ldo, a.ldo2}) odd |= (uint64_t)ld;
    odd *= sizeof(T);
    for (const void* q : {a.x, a.gate, a.h, a.dh, (const void*)a.out, (const void*)a.out2})
      odd |= reinterpret_cast<uintptr_t>(q);
    auto go = [&](auto v_c, auto sigmoid_c, auto mix_c) -> int {
      constexpr int V = decltype(v_c)::value;
      a.tiles = (a.n + 32 * V - 1) / (32 * V);
      const uint64_t blocks = (uint64_t)a.tiles * a.cut.parts * a.cut.chunks;
      if (blocks >= (1ull << 31))
        return set_error(PLX_ERR_CAPACITY, "%llu rows of %u units are too many for one call",
                         (unsigned long long)a.rows, a.n);
      if (a.cut.chunks > 1) {
        char* at = (char*)scratch;
        a.scratch = (Scratch*)at;
        a.flags = (uint32_t*)(at + sizeof(Scratch));
        const uint64_t head = sizeof(Scratch) + (blocks * 4 + 255) / 256 * 256;
        a.pairs = (float2*)(at + head);
        a.ends = (float*)(at + head + blocks * 32 * V * 8);
        PLX_TRY_CUDA(cudaMemsetAsync(at, 0, head, ctx->stream));
      }
      k_recurrence<T, V, decltype(sigmoid_c)::value, decltype(mix_c)::value, BACK>
          <<<(unsigned)blocks, warps_of(BACK) * 32, 0, ctx->stream>>>(a);
      PLX_LAUNCH_CHECK("k_recurrence");
      return PLX_OK;
    };
    using std::integral_constant;
    auto kinds = [&](auto v) {
      using Yes = std::true_type;
      using No = std::false_type;
      if (gate_kind == PLX_GATE_SIGMOID) return mix ? go(v, Yes{}, Yes{}) : go(v, Yes{}, No{});
      return mix ? go(v, No{}, Yes{}) : go(v, No{}, No{});
    };
    return odd % (2 * sizeof(T)) == 0 ? kinds(integral_constant<int, 2>{})
                                      : kinds(integral_constant<int, 1>{});
  });
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" size_t plx_recurrence_scratch_bytes(uint32_t n_streams, uint64_t rows, uint32_t n,
                                               int ragged) {
  if (n_streams == 0 || rows == 0 || n == 0) return 0;
  const Cut c = cut_rows(n_streams, rows, ragged != 0, true);  // the shorter tiles
  if (c.chunks == 1) return 0;
  const uint64_t blocks = (uint64_t)c.parts * c.chunks * ((n + 31) / 32);
  return sizeof(Scratch) + (blocks * 4 + 255) / 256 * 256 + blocks * 32 * 12;
}

extern "C" int plx_recurrence(plx_ctx* ctx, uint32_t n_streams, uint64_t rows, uint32_t n,
                              int dtype, const int32_t* offsets, const void* x, int64_t ldx,
                              const void* gate, int64_t ldg, int gate_kind, int mix,
                              const float* state, void* h, int64_t ldh, float* final_state,
                              void* scratch, size_t scratch_bytes) {
  if (int rc = check_recurrence(ctx, n_streams, rows, n, dtype, offsets, gate_kind, scratch,
                                scratch_bytes))
    return rc;
  if (rows) PLX_CHECK_ARG(x && gate && h, "x, gate and h are required");
  PLX_CHECK_ARG(rows <= 1 || (ldx >= (int64_t)n && ldg >= (int64_t)n && ldh >= (int64_t)n),
                "a row stride is less than n");
  if (int rc = check_aligned(dtype_bytes(dtype), {x, gate, h})) return rc;
  if (int rc = check_aligned(4, {state, final_state})) return rc;
  Args a = {};
  a.rows = rows;
  a.n = n;
  a.streams = n_streams;
  a.offsets = offsets;
  a.x = x;
  a.ldx = ldx;
  a.gate = gate;
  a.ldg = ldg;
  a.state = state;
  a.out = h;
  a.ldo = ldh;
  a.state_out = final_state;
  return launch<false>(ctx, a, dtype, gate_kind, mix != 0, scratch);
}

extern "C" int plx_recurrence_backward(plx_ctx* ctx, uint32_t n_streams, uint64_t rows, uint32_t n,
                                       int dtype, const int32_t* offsets, const void* dh,
                                       int64_t lddh, const void* x, int64_t ldx, const void* gate,
                                       int64_t ldg, int gate_kind, int mix, const void* h,
                                       int64_t ldh, const float* state, const float* dfinal,
                                       void* dx, int64_t lddx, void* dgate, int64_t lddg,
                                       float* dstate, void* scratch, size_t scratch_bytes) {
  if (int rc = check_recurrence(ctx, n_streams, rows, n, dtype, offsets, gate_kind, scratch,
                                scratch_bytes))
    return rc;
  if (rows) {
    PLX_CHECK_ARG(dh && gate && h && dx && dgate, "dh, gate, h, dx and dgate are required");
    PLX_CHECK_ARG(x || !mix, "x is required where it is mixed in by 1 - a");
  }
  PLX_CHECK_ARG(rows <= 1 || (lddh >= (int64_t)n && ldg >= (int64_t)n && ldh >= (int64_t)n &&
                              lddx >= (int64_t)n && lddg >= (int64_t)n &&
                              (!mix || ldx >= (int64_t)n)),
                "a row stride is less than n");
  if (int rc = check_aligned(dtype_bytes(dtype), {dh, x, gate, h, dx, dgate})) return rc;
  if (int rc = check_aligned(4, {state, dfinal, dstate})) return rc;
  Args a = {};
  a.rows = rows;
  a.n = n;
  a.streams = n_streams;
  a.offsets = offsets;
  a.x = mix ? x : nullptr;
  a.ldx = mix ? ldx : 0;
  a.gate = gate;
  a.ldg = ldg;
  a.h = h;
  a.ldh = ldh;
  a.dh = dh;
  a.lddh = lddh;
  a.state = state;
  a.dfinal = dfinal;
  a.out = dx;
  a.ldo = lddx;
  a.out2 = dgate;
  a.ldo2 = lddg;
  a.state_out = dstate;
  return launch<true>(ctx, a, dtype, gate_kind, mix != 0, scratch);
}
