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

constexpr int kWarps = 16;   // runs of a tile
constexpr int kRun = 8;      // steps of a run
constexpr uint32_t kTileSteps = kWarps * kRun;

// How rows are cut: `parts` parts of `part_rows` rows (the last may be shorter),
// each of `chunks` tiles of `chunk_rows` rows (a multiple of the runs' length
// but for the last). No stream crosses a part's end.
struct Cut {
  uint32_t parts, part_rows, chunks, chunk_rows;
};

Cut cut_rows(uint32_t streams, uint64_t rows, bool ragged) {
  Cut c;
  const uint64_t steps = ragged ? rows : rows / streams;
  if (steps <= kTileSteps && !ragged) {  // whole streams in a tile
    c.chunk_rows = c.part_rows = (uint32_t)(kTileSteps / steps * steps);
    c.chunks = 1;
  } else {
    c.part_rows = (uint32_t)steps;
    c.chunks = (uint32_t)((steps + kTileSteps - 1) / kTileSteps);
    c.chunk_rows = kTileSteps;
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

// Waits until a tile's flag is at least `least`; 0 once somebody has given up.
__device__ __forceinline__ uint32_t wait_flag(const uint32_t* flag, uint32_t least, Scratch* s,
                                              int32_t* status, uint64_t timeout_ns) {
  uint32_t v = ld_acquire(flag);
  if (v >= least) return v;
  const uint64_t t0 = global_timer_ns();
  for (uint32_t spin = 1;; ++spin) {
    v = ld_acquire(flag);
    if (v >= least) return v;
    if ((spin & 63u) == 0) {
      if (*(volatile uint32_t*)&s->gave_up) return 0;
      if (global_timer_ns() - t0 > timeout_ns) {
        record_status(status, kStatusTimeout);
        *(volatile uint32_t*)&s->gave_up = 1;
        return 0;
      }
    }
  }
}

// a and 1 - a of a gate, neither by a difference that cancels. The quotient gets
// one Newton step: what a is off by, a long memory raises to its length.
template <bool SIGMOID>
__device__ __forceinline__ void gate_value(float g, float& a, float& keep) {
  if constexpr (SIGMOID) {
    const float e = exp2_approx(-fabsf(g) * kLog2e), d = 1.0f + e;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    r = fmaf(r, fmaf(-d, r, 1.0f), r);
    const float er = e * r;
    a = g < 0.0f ? er : r;
    keep = g < 0.0f ? r : er;
  } else {
    a = g;
    keep = 1.0f - g;
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

template <typename T, int V, bool SIGMOID, bool MIX, bool BACK>
__global__ void __launch_bounds__(kWarps * 32, 2) k_recurrence(const __grid_constant__ Args p) {
  constexpr uint32_t C = 32 * V;
  __shared__ float run_a[kWarps][C], run_h[kWarps][C];
  __shared__ float look_a[kWarps][C], look_h[kWarps][C];
  __shared__ uint32_t run_shut[kWarps], look_kind[kWarps], ticket;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

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
  const uint32_t unit = across * C + lane * V;
  const bool in = unit < p.n;  // V divides n
  // This warp's run, in the order that it is walked.
  const uint32_t run = BACK ? kWarps - 1 - warp : warp;
  const uint64_t at = row0 + run * kRun;
  const int len = at < row1 ? (int)min((uint64_t)kRun, row1 - at) : 0;

  using P = Pack<T, V>;
  P qg[kRun], q1[kRun], q2[kRun], q3[kRun];  // gate; x or dh; backwards h before and x
  const T zero = from_f32<T>(0.0f);
  auto load = [&](P(&q)[kRun], const void* array, int64_t ld, int64_t first) {
    const T* from = (const T*)array + first * ld + unit;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) q[i].v[e] = zero;
      if (in && i < len) q[i] = load_pack<T, V>(from + i * ld);
    }
  };
  load(qg, p.gate, p.ldg, (int64_t)at);
  load(q1, BACK ? p.dh : p.x, BACK ? p.lddh : p.ldx, (int64_t)at);
  if (BACK && MIX) load(q3, p.x, p.ldx, (int64_t)at);
  // Where streams begin and end in the run: a row to a lane.
  Place mine = {0, false, false, false};
  if ((int)lane < len) mine = place_of(p, at + lane);
  const uint32_t valid = __ballot_sync(~0u, mine.valid);
  const uint32_t first = __ballot_sync(~0u, mine.first), last = __ballot_sync(~0u, mine.last);
  auto state_at = [&](const float* states, int i, float (&v)[V]) {
    const uint32_t s = __shfl_sync(~0u, mine.stream, i);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = states && in ? states[(uint64_t)s * p.n + unit + e] : 0.0f;
  };
  if constexpr (BACK) {
    const T* from = (const T*)p.h + ((int64_t)at - 1) * p.ldh + unit;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) q2[i].v[e] = zero;
      if (in && (valid >> i & 1) && !(first >> i & 1)) q2[i] = load_pack<T, V>(from + i * p.ldh);
    }
  }

  // ---- the run's pair. `stop`: rows at which what was before does not count.
  const uint32_t stop = BACK ? last : first;
  float A[V], H[V], extra[kRun][V];  // what a stream's state adds where it begins
#pragma unroll
  for (int e = 0; e < V; ++e) {
    A[e] = 1.0f;
    H[e] = 0.0f;
  }
  // One step: forwards h = a h + b; backwards g = dh + c, c' = a g (h is c).
  auto forward = [&](int i, int e, float before) {
    float a, keep;
    gate_value<SIGMOID>(to_f32(qg[i].v[e]), a, keep);
    float b = to_f32(q1[i].v[e]);
    if (MIX) b *= keep;
    return fmaf(a, before, b);
  };
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = BACK ? kRun - 1 - k : k;
#pragma unroll
    for (int e = 0; e < V; ++e) extra[i][e] = 0.0f;
    if (i >= len) continue;
    if (stop >> i & 1) {  // the same for the whole warp
      state_at(BACK ? p.dfinal : p.state, i, extra[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        H[e] = extra[i][e];
        A[e] = 0.0f;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float a, keep;
      gate_value<SIGMOID>(to_f32(qg[i].v[e]), a, keep);
      if constexpr (BACK) H[e] = a * (to_f32(q1[i].v[e]) + H[e]);
      else H[e] = forward(i, e, H[e]);
      A[e] *= a;
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    run_a[warp][lane * V + e] = A[e];
    run_h[warp][lane * V + e] = H[e];
  }
  if (lane == 0) run_shut[warp] = stop;
  __syncthreads();

  // ---- what the tile is given, and what it leaves
  float carry[V];
#pragma unroll
  for (int e = 0; e < V; ++e) carry[e] = 0.0f;
  if (chained) {
    float ta[V], th[V];
    bool shut = false;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      ta[e] = 1.0f;
      th[e] = 0.0f;
    }
    for (int w = 0; w < kWarps; ++w) {
      const bool s = run_shut[w] != 0;
      shut |= s;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float a = run_a[w][lane * V + e], h = run_h[w][lane * V + e];
        th[e] = s ? h : fmaf(a, th[e], h);
        ta[e] = s ? 0.0f : ta[e] * a;
      }
    }
    const uint32_t step = p.cut.parts * p.tiles;  // between tiles of a part
    const uint64_t slot = (uint64_t)id * C + lane * V;
    auto leave = [&](bool end, const float (&h)[V]) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (end) p.ends[slot + e] = h[e];
        else p.pairs[slot + e] = make_float2(ta[e], h[e]);
      }
      __threadfence();
      __syncwarp();
      if (lane == 0) st_release(p.flags + id, end ? kEnd : kPair);
    };
    const bool ready = shut || turn == 0;
    if (warp == 0) leave(ready, th);
    if (turn > 0) {
      uint32_t kind = kEnd;
      if (warp < turn) {
        const uint32_t from = id - (warp + 1) * step;
        // the furthest one is waited for until it has its end value
        kind = wait_flag(p.flags + from, warp == kWarps - 1 ? kEnd : kPair, p.scratch, p.status,
                         p.timeout_ns);
        kind = __reduce_min_sync(~0u, kind);  // what every lane has seen
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint64_t s = (uint64_t)from * C + lane * V + e;
          float2 v = make_float2(0.0f, 0.0f);
          if (kind == kPair) v = __ldcg(p.pairs + s);
          else if (kind == kEnd) v.y = __ldcg(p.ends + s);
          look_a[warp][lane * V + e] = v.x;
          look_h[warp][lane * V + e] = v.y;
        }
      }
      if (lane == 0) look_kind[warp] = kind;
      __syncthreads();
      int near = 0;
      while (near < kWarps - 1 && look_kind[near] == kPair) ++near;
#pragma unroll
      for (int e = 0; e < V; ++e) carry[e] = look_h[near][lane * V + e];
      for (int w = near - 1; w >= 0; --w)
#pragma unroll
        for (int e = 0; e < V; ++e)
          carry[e] = fmaf(look_a[w][lane * V + e], carry[e], look_h[w][lane * V + e]);
      if (warp == 0 && !ready) {
#pragma unroll
        for (int e = 0; e < V; ++e) th[e] = fmaf(ta[e], carry[e], th[e]);
        leave(true, th);
      }
    }
  }
  for (uint32_t w = 0; w < warp; ++w) {
    const bool s = run_shut[w] != 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = run_a[w][lane * V + e], h = run_h[w][lane * V + e];
      carry[e] = s ? h : fmaf(a, carry[e], h);
    }
  }

  // ---- the run once more, from what it is given
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = BACK ? kRun - 1 - k : k;
    if (i >= len) continue;
    if (stop >> i & 1)
#pragma unroll
      for (int e = 0; e < V; ++e) carry[e] = extra[i][e];
    float before[V];
    if constexpr (BACK) {
      if (first >> i & 1) {
        state_at(p.state, i, before);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) before[e] = to_f32(q2[i].v[e]);
      }
    }
    P o1, o2;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (BACK) {
        float a, keep;
        gate_value<SIGMOID>(to_f32(qg[i].v[e]), a, keep);
        const float g = to_f32(q1[i].v[e]) + carry[e];
        carry[e] = a * g;
        float da = g * (MIX ? before[e] - to_f32(q3[i].v[e]) : before[e]);
        if (SIGMOID) da *= a * keep;
        o1.v[e] = from_f32<T>(MIX ? g * keep : g);
        o2.v[e] = from_f32<T>(da);
      } else {
        carry[e] = forward(i, e, carry[e]);
        o1.v[e] = from_f32<T>(carry[e]);
      }
    }
    const int64_t row = (int64_t)(at + i);
    if (in && (valid >> i & 1)) {
      *reinterpret_cast<P*>((T*)p.out + row * p.ldo + unit) = o1;
      if (BACK) *reinterpret_cast<P*>((T*)p.out2 + row * p.ldo2 + unit) = o2;
    }
    if (p.state_out && ((BACK ? first : last) >> i & 1)) {
      const uint32_t s = __shfl_sync(~0u, mine.stream, i);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (in) p.state_out[(uint64_t)s * p.n + unit + e] = carry[e];
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
  a.cut = cut_rows(a.streams, a.rows, a.offsets != nullptr);
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
          <<<(unsigned)blocks, kWarps * 32, 0, ctx->stream>>>(a);
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
  const Cut c = cut_rows(n_streams, rows, ragged != 0);
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
