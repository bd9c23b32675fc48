// Gated linear recurrence of units over the steps of streams, and its gradients.
//   h_t = a_t h_{t-1} + c_t x_t,   a = gate or sigmoid(gate),   c = 1 or 1 - a
//   g_t = dh_t + a_{t+1} g_{t+1};  dx = c g;  da = g h_{t-1}  or  g (h_{t-1} - x)
// Units are independent; steps are folded as pairs (A, H): a run of steps takes
// what it is given, h, to A h + H, and two runs join to (A1 A2, A2 H1 + H2).
//
// Bound by memory. Long streams are walked by a block each (64 units), tile after
// tile of 64 steps, the next tiles on their way into shared memory: a warp has a run
// of eight steps, whose pairs are joined behind one barrier a tile. Where that leaves
// SMs idle (few streams of few units) or streams have lengths that only the device
// knows, rows are cut into parts: a first kernel leaves every part's pair, the
// second folds those before its own and walks again with results. Reading twice
// costs less than parts that wait for one another: tiles that look back over the
// ones before them took 205 us for 65,536 steps of 512 units. Short streams are taken
// in tiles that hold them whole: values stay in registers between the two walks.
// Everything is folded in an order that the arguments set.
// Decays may be of any size, and their product A leaves 32 bits where no h does (200
// steps of 1.5 before the first x; 1e20, 1e20, 0). Where A h + H is not finite, the run
// is walked step by step from h instead; where a part's is not, the block before it
// goes on through it. Units and streams whose pairs are finite keep the same bits. (A
// product below 2^-149 counts as 0: it would leave less than that of h. Sigmoids are at
// most 1; behind an infinite x their h may be NaN.)
// Measured: 8 streams of 2,048 steps of 4,096 units bf16, sigmoid gates, mixed,
// forwards and backwards 225 us, 5.4 TB/s (205 without the Newton step in a, whose
// error a long memory shows; 477 with a lane's own copies in place of tensor copies);
// 65,536 steps of 512 units 72 us, 2.8 TB/s of what has to be read (4.7 of what is);
// 37 ragged streams of 20,017 steps of 501 units f32 (no multiple of 16 bytes), both
// ways, 127 us, 2.5 TB/s (3.4 of what is read); 121 without the steps that decays above
// 1 may need. In the sigmoids' kernels those steps took 88 to 106 us forwards without
// ever being reached (registers), so that only decays have them.
#include <type_traits>

#include "norm.cuh"
#include "tensor.cuh"

namespace plx {
namespace {

// Runs of a tile, forwards and backwards, which has more values in registers: two
// blocks an SM either way.
__host__ __device__ constexpr int warps_of(bool back) { return back ? 12 : 16; }
constexpr int kRun = 8;      // steps of a run, and of a stage of a walk
__host__ __device__ constexpr uint32_t tile_steps(bool back) { return warps_of(back) * kRun; }

struct Args {
  uint64_t rows;
  uint32_t n, streams, steps;  // steps of a stream; 0 with offsets
  uint32_t tiles;              // across the units
  uint32_t tile_rows;          // of short streams: whole ones
  uint32_t groups, group_rows, parts, part_rows;  // of long ones: no stream crosses a group's end
  const int32_t* offsets;
  const void *x, *gate, *h, *dh;
  int64_t ldx, ldg, ldh, lddh;
  const float *state, *dfinal;
  void *out, *out2;            // h; or dx and dgate
  int64_t ldo, ldo2;
  bool clear;                  // rows of no stream become zero (with offsets)
  float* state_out;            // final; or dstate
  float2* pairs;               // of the parts, [group][part][unit]
  uint32_t* shut;              // parts in which a stream begins (ends), [group][part]
  int32_t* status;
  uint64_t timeout_ns;
};

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
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }
__device__ __forceinline__ bool finite(F2 v) { return finite(v.x) && finite(v.y); }
// Of each unit the first value where that is finite, else the second.
__device__ __forceinline__ float finite_or(float v, float w) { return finite(v) ? v : w; }
__device__ __forceinline__ F2 finite_or(F2 v, F2 w) {
  return pack2(finite_or(v.x, w.x), finite_or(v.y, w.y));
}
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

// The larger of each value and -87 (NaN stays NaN): e^87 is a 32-bit number.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> at_least_minus_87(Pack<T, V> q) {
  if constexpr (sizeof(T) == 2 && V == 2) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    T2 v = *reinterpret_cast<T2*>(&q);
    if constexpr (std::is_same_v<T, __half>) v = __hmax2_nan(v, __floats2half2_rn(-87.0f, -87.0f));
    else v = __hmax2_nan(v, __floats2bfloat162_rn(-87.0f, -87.0f));
    return *reinterpret_cast<Pack<T, V>*>(&v);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) q.v[e] = from_f32<T>(max_nan(to_f32(q.v[e]), -87.0f));
    return q;
  }
}

// a and 1 - a of a gate, neither by a difference that cancels: with e = exp(-gate),
// 1 / (1 + e) and e / (1 + e). Gates below -87 count as -87 (which leaves e^-87 of
// h). The quotient gets one step of Newton's method (r + r (1 - d r)): what a is off by,
// a long memory raises to its length.
template <bool SIGMOID, typename T, int V>
__device__ __forceinline__ void gate_value(Pack<T, V> gate, Units<V>& a, Units<V>& keep) {
  using W = Units<V>;
  if constexpr (SIGMOID) {
    const W g = wide<T, V>(at_least_minus_87(gate));
    const W e = each(mulw(g, all<W>(-kLog2e)), exp2_approx);
    const W d = addw(e, all<W>(1.0f)), r = each(d, rcp_approx);
    a = fmaw(r, fmaw(each(d, [](float t) { return -t; }), r, all<W>(1.0f)), r);
    keep = mulw(e, a);
  } else {
    a = wide<T, V>(gate);
    keep = addw(all<W>(1.0f), each(a, [](float t) { return -t; }));
  }
}

// The stream of a row, its rows, and whether it begins or ends there.
struct Place {
  uint32_t stream;
  bool valid, first, last;
  int64_t begin, end;
};
__device__ __forceinline__ Place place_of(const Args& p, uint64_t row) {
  Place q;
  if (!p.offsets) {
    q.stream = (uint32_t)row / p.steps;  // rows < 2^31
    q.begin = (int64_t)q.stream * p.steps;
    q.end = q.begin + p.steps;
  } else {
    // the last stream that begins at or before the row (empty ones come before it)
    uint32_t lo = 0, hi = p.streams;
    while (hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if ((int64_t)__ldg(p.offsets + mid) <= (int64_t)row) lo = mid;
      else hi = mid;
    }
    q.stream = lo;
    q.begin = __ldg(p.offsets + lo);
    q.end = __ldg(p.offsets + lo + 1);
  }
  q.valid = q.begin <= (int64_t)row && (int64_t)row < q.end;
  q.first = q.valid && q.begin == (int64_t)row;
  q.last = q.valid && q.end == (int64_t)row + 1;
  return q;
}

// A step's values as both walks use them: forwards a and b (h = a h + b), where a
// stream begins in a tile of several with its state in b; backwards a, dh and what g
// is multiplied by.
template <typename T, int V, bool SIGMOID, bool MIX, bool BACK>
struct Step {
  using W = Units<V>;
  using P = Pack<T, V>;
  W a, b;     // b: forwards
  P dh;       // backwards
  W slope;    // dgate = g slope
  W keep;     // dx = g keep
  __device__ __forceinline__ void forward(P gate, P x) {
    gate_value<SIGMOID>(gate, a, keep);
    b = wide<T, V>(x);
    if (MIX) b = mulw(b, keep);
  }
  __device__ __forceinline__ void backward(P gate, P d, W before, P x) {
    gate_value<SIGMOID>(gate, a, keep);
    dh = d;
    slope = before;
    if (MIX) slope = addw(slope, each(wide<T, V>(x), [](float t) { return -t; }));
    if (SIGMOID) slope = mulw(slope, mulw(a, keep));
  }
  __device__ __forceinline__ W dx(W g) const { return MIX ? mulw(g, keep) : g; }
  // What the step hands on of what it is given.
  __device__ __forceinline__ W on(W given) const {
    return BACK ? mulw(a, addw(wide<T, V>(dh), given)) : fmaw(a, given, b);
  }
};

// A lane's units of an array: V of them, GAP apart; those there are.
template <int V, int GAP>
struct Lane {
  uint32_t unit;
  bool in[V];
  __device__ __forceinline__ Lane(uint32_t tile, uint32_t n)
      : unit(tile * 32 * V + (threadIdx.x & 31) * (GAP == 1 ? V : 1)) {
#pragma unroll
    for (int e = 0; e < V; ++e) in[e] = unit + e * GAP < n;  // GAP 1: V divides n
  }
  __device__ __forceinline__ Units<V> load(const float* p) const {
    if constexpr (V == 2) return pack2(in[0] ? p[0] : 0.0f, in[1] ? p[GAP] : 0.0f);
    else return in[0] ? p[0] : 0.0f;
  }
  __device__ __forceinline__ void store(float* p, Units<V> v) const {
    if constexpr (V == 2) {
      if (in[0]) p[0] = v.x;
      if (in[1]) p[GAP] = v.y;
    } else {
      if (in[0]) p[0] = v;
    }
  }
  template <typename T>
  __device__ __forceinline__ Pack<T, V> load_rows(const T* p) const {
    Pack<T, V> q;
#pragma unroll
    for (int e = 0; e < V; ++e) q.v[e] = from_f32<T>(0.0f);
    if constexpr (GAP == 1) {
      if (in[0]) q = load_pack<T, V>(p);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (in[e]) q.v[e] = p[e * GAP];
    }
    return q;
  }
  template <typename T>
  __device__ __forceinline__ void store_rows(T* p, Pack<T, V> q) const {
    if constexpr (GAP == 1) {
      if (in[0]) *reinterpret_cast<Pack<T, V>*>(p) = q;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (in[e]) p[e * GAP] = q.v[e];
    }
  }
};

// Short streams, whole ones in a tile.
template <typename T, int V, bool SIGMOID, bool MIX, bool BACK>
__global__ void __launch_bounds__(warps_of(BACK) * 32, 2)
k_recurrence_tile(const __grid_constant__ Args p) {
  constexpr int kWarps = warps_of(BACK);
  using W = Units<V>;
  using P = Pack<T, V>;
  struct alignas(8 * V) Pair {
    W a, h;
  };
  __shared__ Pair runs[kWarps][32];
  __shared__ W handed[SIGMOID ? 1 : 32];
  __shared__ uint32_t run_shut[kWarps];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const W zero = all<W>(0.0f);
  const uint64_t row0 = (uint64_t)(blockIdx.x / p.tiles) * p.tile_rows;
  const uint64_t row1 = min(row0 + p.tile_rows, p.rows);
  const Lane<V, 1> mine(blockIdx.x % p.tiles, p.n);
  const uint32_t unit = mine.unit;
  // This warp's run, in the order that it is walked.
  const uint32_t run = BACK ? blockDim.x / 32 - 1 - warp : warp;
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
      if (i < len) q[i] = mine.load_rows(from + i * ld);
    }
  };
  load(qg, p.gate, p.ldg);
  load(q1, BACK ? p.dh : p.x, BACK ? p.lddh : p.ldx);
  if constexpr (BACK && MIX) load(q3, p.x, p.ldx);
  // Where streams begin and end in the run: a row to a lane.
  uint32_t stream = 0, place = 0;
  if ((int)lane < len) {
    stream = (uint32_t)(at + lane) / p.steps;
    place = (uint32_t)(at + lane) - stream * p.steps;
  }
  const uint32_t first = __ballot_sync(~0u, (int)lane < len && place == 0);
  const uint32_t last = __ballot_sync(~0u, (int)lane < len && place + 1 == p.steps);
  auto state_at = [&](const float* states, int i) {
    const uint32_t s = __shfl_sync(~0u, stream, i);
    return states ? mine.load(states + (uint64_t)s * p.n + unit) : zero;
  };
  // what streams are given where their walk begins
  W given[kRun];
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    given[i] = zero;
    if ((BACK ? last : first) >> i & 1) given[i] = state_at(BACK ? p.dfinal : p.state, i);
  }
  if constexpr (BACK) {
    const T* from = (const T*)p.h + ((int64_t)at - 1) * p.ldh + unit;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      q2[i] = nothing;
      if (i < len && !(first >> i & 1)) q2[i] = mine.load_rows(from + i * p.ldh);
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
        H = given[i];
        A = zero;
      }
      H = mulw(st.a, addw(wide<T, V>(st.dh), H));
      A = mulw(A, st.a);
    } else {
      st.forward(qg[i], q1[i]);
      if (stop >> i & 1) {
        st.b = fmaw(st.a, given[i], st.b);
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
  W carry = zero;
  for (uint32_t w = 0; w < warp; ++w) {
    const Pair v = runs[w][lane];
    carry = run_shut[w] ? v.h : fmaw(v.a, carry, v.h);
  }
  if (!SIGMOID && __syncthreads_or(!finite(carry))) {  // run after run
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) {
      if (w == warp) {
        carry = w ? handed[lane] : zero;
        W end = H;
        if (!stop) {
          end = carry;
#pragma unroll
          for (int k = 0; k < kRun; ++k) {
            const int i = BACK ? kRun - 1 - k : k;
            if (i < len) end = steps[i].on(end);
          }
          end = finite_or(fmaw(A, carry, H), end);
        }
        handed[lane] = end;
      }
      __syncthreads();
    }
  }

  // ---- the run once more, from what it is given
#pragma unroll
  for (int k = 0; k < kRun; ++k) {
    const int i = BACK ? kRun - 1 - k : k;
    if (i >= len) continue;
    const auto& st = steps[i];
    const int64_t row = (int64_t)(at + i);
    if constexpr (BACK) {
      if (stop >> i & 1) carry = state_at(p.dfinal, i);
      const W g = addw(wide<T, V>(st.dh), carry);
      carry = mulw(st.a, g);
      mine.store_rows((T*)p.out + row * p.ldo + unit, narrow<T, V>(st.dx(g)));
      mine.store_rows((T*)p.out2 + row * p.ldo2 + unit, narrow<T, V>(mulw(g, st.slope)));
    } else {
      carry = stop >> i & 1 ? st.b : fmaw(st.a, carry, st.b);
      mine.store_rows((T*)p.out + row * p.ldo + unit, narrow<T, V>(carry));
    }
    if (p.state_out && ((BACK ? first : last) >> i & 1)) {
      const uint32_t s = __shfl_sync(~0u, stream, i);
      mine.store(p.state_out + (uint64_t)s * p.n + unit, carry);
    }
  }
}

// Stages of a walk under way: tiles of every array that it reads.
constexpr int kWalkWarps = 8, kWalkUnits = 64;
constexpr uint32_t kWalkSteps = kWalkWarps * kRun;  // of a tile
template <typename T, int ARRAYS, bool TENSOR>
struct WalkRing {
  static constexpr int row = kWalkUnits * sizeof(T);
  static constexpr int run = kRun * row;
  static constexpr int array = kWalkWarps * run;
  static constexpr int stage = ARRAYS * array;
  static constexpr int stages = stage <= 16 * 1024 ? 4 : stage <= 32 * 1024 ? 3 : 2;
  static constexpr int bytes = TENSOR ? stages * stage : 0;
};

struct Maps {
  CUtensorMap of[4];  // gate; x or dh; h; x
};

// A part of a long stream (or of ragged ones behind each other), tile after tile.
// LEAVE: the part's pair, else its results. TENSOR: one thread has a tile's arrays
// copied by tensor copies (rows whose start and stride are multiples of 16 bytes) and
// a lane has two units side by side; else every lane reads its own, of two units 32
// apart (through shared memory by four-byte copies took a quarter longer).
template <typename T, bool SIGMOID, bool MIX, bool BACK, bool LEAVE, bool TENSOR>
__global__ void __launch_bounds__(kWalkWarps * 32, BACK && !LEAVE ? 2 : 3)
k_recurrence_walk(const __grid_constant__ Args p, const __grid_constant__ Maps maps) {
  constexpr int V = 2, GAP = TENSOR ? 1 : 32;
  constexpr bool SAFE = !SIGMOID && !LEAVE;  // pairs may not be finite
  using W = Units<V>;
  using P = Pack<T, V>;
  constexpr int ARRAYS = LEAVE || !BACK ? 2 : MIX ? 4 : 3;
  using R = WalkRing<T, ARRAYS, TENSOR>;
  constexpr int S = R::stages;
  struct alignas(8 * V) Pair {
    W a, h;
  };
  extern __shared__ __align__(128) uint8_t walk_bytes[];
  __shared__ uint64_t full[S];
  __shared__ uint32_t gave_up;
  __shared__ Pair runs[2][kWalkWarps][32];
  __shared__ W handed[SAFE ? 32 : 1];
  __shared__ uint32_t run_shut[2][kWalkWarps];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const W zero = all<W>(0.0f);

  // offsets that no rows have; streams without steps hand their state on
  if (p.offsets && !LEAVE) {
    for (uint32_t s = blockIdx.x; s < p.streams; s += gridDim.x) {
      const int64_t begin = p.offsets[s], end = p.offsets[s + 1];
      if (threadIdx.x == 0 && (begin < 0 || begin > end || (uint64_t)end > p.rows))
        record_status(p.status, kStatusBadOffsets);
      const float* given = BACK ? p.dfinal : p.state;
      if (begin == end && p.state_out)
        for (uint32_t i = threadIdx.x; i < p.n; i += kWalkWarps * 32)
          p.state_out[(uint64_t)s * p.n + i] = given ? given[(uint64_t)s * p.n + i] : 0.0f;
    }
  }
  // rows before the first stream and behind the last one
  if (p.clear && !LEAVE) {
    const int64_t rows = (int64_t)p.rows;
    const int64_t first = min(max((int64_t)p.offsets[0], (int64_t)0), rows);
    const int64_t last = min(max((int64_t)p.offsets[p.streams], first), rows);
    for (int64_t k = blockIdx.x; k < first + rows - last; k += gridDim.x) {
      const int64_t row = k < first ? k : last + k - first;
      for (uint32_t i = threadIdx.x; i < p.n; i += kWalkWarps * 32) {
        ((T*)p.out)[row * p.ldo + i] = from_f32<T>(0.0f);
        if constexpr (BACK) ((T*)p.out2)[row * p.ldo2 + i] = from_f32<T>(0.0f);
      }
    }
  }
  const uint32_t across = blockIdx.x % p.tiles, rest = blockIdx.x / p.tiles;
  const uint32_t group = rest / p.parts, part = rest % p.parts;
  const Lane<V, GAP> own(across, p.n);
  const uint32_t unit = own.unit;
  const int64_t g0 = (int64_t)group * p.group_rows, g1 = min(g0 + p.group_rows, (int64_t)p.rows);
  int64_t row0 = min(g0 + (int64_t)part * p.part_rows, g1);
  int64_t row1 = min(row0 + p.part_rows, g1);
  int tiles = (int)((row1 - row0 + kWalkSteps - 1) / kWalkSteps);
  // Steps are walked in the direction `dir`, and so are tiles for results. For a
  // part's pair they are taken the other way round: what is read last is what the
  // next kernel reads first, out of L2.
  constexpr int dir = BACK ? -1 : 1;
  constexpr bool FROM_END = BACK != LEAVE;
  constexpr int tile_dir = FROM_END ? -1 : 1;
  // This warp's run of the first tile.
  int64_t at = row0 + (FROM_END ? (int64_t)(tiles - 1) * kWalkSteps : 0) +
               (BACK ? kWalkWarps - 1 - warp : warp) * kRun;

  const T* from[4] = {(const T*)p.gate, (const T*)(BACK ? p.dh : p.x), (const T*)p.h,
                      (const T*)p.x};
  const int64_t ld[4] = {p.ldg, BACK ? p.lddh : p.ldx, p.ldh, p.ldx};
  // of this warp's run in a tile in the ring, this lane's values
  const char* ring = reinterpret_cast<const char*>(walk_bytes) + lane * V * sizeof(T) +
                     (BACK ? kWalkWarps - 1 - warp : warp) * R::run;
  int fetched = 0;
  auto fetch = [&](uint32_t stage) {
    if constexpr (TENSOR) {  // by one thread
      if (fetched < tiles) {
        const int64_t tile = FROM_END ? tiles - 1 - fetched : fetched;
        const int y = (int)(row0 + tile * kWalkSteps);
        mbar_arrive_expect_tx(&full[stage], R::stage);
#pragma unroll
        for (int k = 0; k < ARRAYS; ++k)
          tensor_load(walk_bytes + stage * R::stage + k * R::array, &maps.of[k],
                      (int)(across * 32 * V), y - (k == 2 ? 1 : 0), &full[stage]);
      }
      ++fetched;
    }
  };
  if constexpr (TENSOR) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < S; ++s) mbar_init(&full[s], 1);
      mbar_init_fence();
      gave_up = 0;
      for (int s = 0; s < S; ++s) fetch(s);
    }
    __syncthreads();
  }

  W A = all<W>(1.0f), given = zero;  // forwards h; backwards what a step hands to the one before
  bool shut = false;
  // What the part that is walked as the j-th hands on of what it is given.
  auto part_hands = [&](uint32_t j, W h) {
    const uint32_t q = group * p.parts + (BACK ? p.parts - 1 - j : j);
    const bool s = p.shut[q] != 0;
    const Pair v =
        reinterpret_cast<const Pair*>(p.pairs)[((uint64_t)q * p.tiles + across) * 32 + lane];
    return s ? v.h : fmaw(v.a, h, v.h);
  };
  const uint32_t before = BACK ? p.parts - 1 - part : part;  // parts walked before this one
  int next_part = 0x7fffffff;  // the tile at which a part begins that is this block's as well
  if constexpr (!LEAVE) {
    if (SAFE ? p.parts > 1 : before > 0) {
      // what the parts walked before leave
      if (warp == 0) {
#pragma unroll 8
        for (uint32_t j = 0; j < before; ++j) given = part_hands(j, given);
        if constexpr (SAFE) {
          // a part that is not given a finite value is left to the block before it
          uint32_t more = 0;
          if (__any_sync(~0u, !finite(given))) {
            more = ~0u;
          } else if (before + 1 < p.parts) {
            W h = part_hands(before, given);
            while (__any_sync(~0u, !finite(h)) && before + ++more + 1 < p.parts)
              h = part_hands(before + more, h);
          }
          if (lane == 0) run_shut[0][0] = more;
        }
        runs[0][0][lane].h = given;
      }
      __syncthreads();
      given = runs[0][0][lane].h;
      const uint32_t more = SAFE ? run_shut[0][0] : 0;
      __syncthreads();
      if (more == ~0u) {
        if constexpr (TENSOR) {
          if (threadIdx.x == 0)  // what is on its way
            for (int s = 0; s < min(S, tiles); ++s)
              mbar_wait_bounded(&full[s], 0, p.timeout_ns);
        }
        return;
      }
      if (more) {  // parts begin at whole tiles of one another
        next_part = tiles;
        if (BACK) row0 -= (int64_t)more * p.part_rows;
        else row1 = min(row1 + (int64_t)more * p.part_rows, g1);
        tiles = (int)((row1 - row0 + kWalkSteps - 1) / kWalkSteps);
        if constexpr (TENSOR) {
          if (threadIdx.x == 0 && next_part < S) {
            fetched = next_part;
            for (int s = next_part; s < S; ++s) fetch(s);
          }
        }
      }
    }
  }
  P nothing;
#pragma unroll
  for (int e = 0; e < V; ++e) nothing.v[e] = from_f32<T>(0.0f);
  // rows in which no stream begins or ends, and all are some stream's
  int64_t clear0 = 0, clear1 = 0;
  uint32_t stage = 0, half = 0, parity = 0;
  bool tainted = false;  // what is given may not be finite
  for (int tile = 0; tile < tiles; ++tile, at += tile_dir * (int)kWalkSteps, half ^= 1) {
    const int len = (int)max((int64_t)0, min((int64_t)kRun, row1 - at));
    if constexpr (SAFE) {
      if (tile == next_part) {  // units that the pairs do for go on from those
        W h = zero;
        const uint32_t done = BACK ? p.parts - 1 - (uint32_t)((at - g0) / p.part_rows)
                                   : (uint32_t)((at - g0) / p.part_rows);
        for (uint32_t j = 0; j < done; ++j) h = part_hands(j, h);
        given = finite_or(h, given);
        tainted = true;
        next_part += (int)(p.part_rows / kWalkSteps);
      }
    }
    P q[4][kRun];
    if constexpr (TENSOR) {
      if (!mbar_try_wait(&full[stage], parity) &&
          (*(volatile uint32_t*)&gave_up ||
           !mbar_wait_bounded(&full[stage], parity, p.timeout_ns))) {
        *(volatile uint32_t*)&gave_up = 1;
        record_status(p.status, kStatusTimeout);
      }
      const char* to = ring + stage * R::stage;
#pragma unroll
      for (int k = 0; k < ARRAYS; ++k)
#pragma unroll
        for (int i = 0; i < kRun; ++i)
          q[k][i] = *reinterpret_cast<const P*>(to + k * R::array + i * R::row);
    } else {
#pragma unroll
      for (int k = 0; k < ARRAYS; ++k)
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
          q[k][i] = nothing;
          const int64_t r = at + i - (k == 2 ? 1 : 0);
          if (i < len && r >= 0) q[k][i] = own.load_rows(from[k] + r * ld[k] + unit);
        }
    }
    uint32_t valid = 0xff, first = 0, last = 0;
    Place mine = {0, false, false, false};
    if (len && !(clear0 <= at && at + len <= clear1)) {
      if ((int)lane < len) mine = place_of(p, (uint64_t)(at + lane));
      valid = __ballot_sync(~0u, mine.valid);
      first = __ballot_sync(~0u, mine.first);
      last = __ballot_sync(~0u, mine.last);
      // the stream that the row nearest to the next tile is in goes on
      clear0 = __shfl_sync(~0u, mine.begin, FROM_END ? 0 : len - 1) + 1;
      clear1 = __shfl_sync(~0u, mine.end, FROM_END ? 0 : len - 1) - 1;
    }
    const uint32_t stop = BACK ? last : first;  // rows at which what was before does not count
    auto state_at = [&](const float* states, int i) {
      const uint32_t s = __shfl_sync(~0u, mine.stream, i);
      return states ? own.load(states + (uint64_t)s * p.n + unit) : zero;
    };

    // ---- the run's pair
    Step<T, V, SIGMOID, MIX, BACK> st[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      if constexpr (BACK && LEAVE) {
        W k;
        gate_value<SIGMOID>(q[0][i], st[i].a, k);
        st[i].dh = q[1][i];
      } else if constexpr (BACK) {
        W before = wide<T, V>(q[2][i]);
        if (first >> i & 1) before = state_at(p.state, i);
        st[i].backward(q[0][i], q[1][i], before, q[MIX ? 3 : 2][i]);
      } else {
        st[i].forward(q[0][i], q[1][i]);
      }
    }
    W a = all<W>(1.0f), h = zero;
    if (len == kRun && !stop && (SIGMOID || valid == 0xff)) {
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        const int i = BACK ? kRun - 1 - k : k;
        h = st[i].on(h);
        a = mulw(a, st[i].a);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        const int i = BACK ? kRun - 1 - k : k;
        if (i >= len) continue;
        if (!SIGMOID && !(valid >> i & 1)) continue;  // rows of no stream hand on what they get
        if (stop >> i & 1) {  // the same for the whole warp
          h = state_at(BACK ? p.dfinal : p.state, i);
          a = zero;
        }
        h = st[i].on(h);
        a = mulw(a, st[i].a);
      }
    }
    runs[half][warp][lane] = {a, h};
    if (lane == 0) run_shut[half][warp] = stop;
    // the half is written again after the next tile's barrier; a stage has been read
    // (any: a stream's border, or what may not be folded)
    const bool any =
        __syncthreads_or(stop != 0 || (SAFE && (tainted || !finite(fmaw(a, zero, h)))));
    if constexpr (TENSOR) {
      if (threadIdx.x == 0) fetch(stage);
    }
    parity ^= stage == S - 1;
    stage = stage == S - 1 ? 0 : stage + 1;
    if constexpr (LEAVE) {
      if (warp == 0 && !shut) {  // before a stream's start nothing counts
        W ta = all<W>(1.0f), th = zero;
        bool cut = false;
        for (uint32_t w = 0; w < kWalkWarps; ++w) {
          const Pair v = runs[half][w][lane];
          const bool s = any && run_shut[half][w] != 0;
          th = s ? v.h : fmaw(v.a, th, v.h);
          ta = s ? zero : mulw(ta, v.a);
          cut |= s;
        }
        given = fmaw(A, th, given);
        A = mulw(A, ta);
        shut = cut;
      }
    }
    W carry = given;
    if (!LEAVE && !any) {
#pragma unroll
      for (uint32_t w = 0; w < kWalkWarps; ++w) {
        const Pair v = runs[half][w][lane];
        if (w == warp) carry = given;
        given = fmaw(v.a, given, v.h);
      }
    } else if (!LEAVE) {
      const W was = given;
      bool fine = finite(was);
      for (uint32_t w = 0; w < kWalkWarps; ++w) {
        const Pair v = runs[half][w][lane];
        if (w == warp) carry = given;
        given = run_shut[half][w] ? v.h : fmaw(v.a, given, v.h);
        if (SAFE) fine &= finite(given);
      }
      if (SAFE) tainted = __any_sync(~0u, !fine);
      if (SAFE && tainted) {  // so say all warps: run after run
        for (uint32_t w = 0; w < kWalkWarps; ++w) {
          if (w == warp) {
            carry = w ? handed[lane] : was;
            const Pair v = runs[half][warp][lane];
            W end = v.h;
            if (!run_shut[half][warp]) {
              end = carry;
#pragma unroll
              for (int k = 0; k < kRun; ++k) {
                const int i = BACK ? kRun - 1 - k : k;
                if (i < len && (valid >> i & 1)) end = st[i].on(end);
              }
              end = finite_or(fmaw(v.a, carry, v.h), end);
            }
            handed[lane] = end;
          }
          __syncthreads();
        }
        given = handed[lane];
      }
    }
    if constexpr (!LEAVE) {
      // ---- the run once more, from what it is given
      T *o1 = (T*)p.out + at * p.ldo + unit, *o2 = (T*)p.out2 + at * p.ldo2 + unit;
      if (BACK) {
        o1 += (kRun - 1) * p.ldo;
        o2 += (kRun - 1) * p.ldo2;
      }
      auto results = [&](int i) {
        if constexpr (BACK) {
          const W g = addw(wide<T, V>(st[i].dh), carry);
          carry = mulw(st[i].a, g);
          own.store_rows(o1, narrow<T, V>(st[i].dx(g)));
          own.store_rows(o2, narrow<T, V>(mulw(g, st[i].slope)));
        } else {
          carry = fmaw(st[i].a, carry, st[i].b);
          own.store_rows(o1, narrow<T, V>(carry));
        }
      };
      if (len == kRun && valid == 0xff && !first && !last) {
        if (own.in[0])
#pragma unroll
          for (int k = 0; k < kRun; ++k) {
            results(BACK ? kRun - 1 - k : k);
            o1 += dir * p.ldo;
            if (BACK) o2 += dir * p.ldo2;
          }
      } else {
#pragma unroll
        for (int k = 0; k < kRun; ++k) {
          const int i = BACK ? kRun - 1 - k : k;
          if (i < len) {
            if (stop >> i & 1) carry = state_at(BACK ? p.dfinal : p.state, i);
            if (valid >> i & 1) results(i);
            if (p.state_out && ((BACK ? first : last) >> i & 1)) {
              const uint32_t s = __shfl_sync(~0u, mine.stream, i);
              own.store(p.state_out + (uint64_t)s * p.n + unit, carry);
            }
          }
          o1 += dir * p.ldo;
          if (BACK) o2 += dir * p.ldo2;
        }
      }
    }
  }
  if constexpr (TENSOR) {
    if (threadIdx.x == 0 && *(volatile uint32_t*)&gave_up)  // what is still on its way
      for (int j = max(0, min(fetched, tiles) - S); j < min(fetched, tiles); ++j)
        mbar_wait_bounded(&full[j % S], (j / S) & 1, p.timeout_ns);
  }
  if constexpr (LEAVE) {
    if (warp == 0) {
      const uint32_t q = group * p.parts + part;
      reinterpret_cast<Pair*>(p.pairs)[((uint64_t)q * p.tiles + across) * 32 + lane] = {A, given};
      if (across == 0 && lane == 0) p.shut[q] = shut;
    }
  }
}

__global__ void __launch_bounds__(256)
k_copy_state(uint64_t count, const float* from, float* to) {
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256ull)
    to[i] = from ? from[i] : 0.0f;
}

// Offsets of streams without any rows: all 0.
__global__ void __launch_bounds__(256)
k_check_offsets(uint32_t count, const int32_t* offsets, int32_t* status) {
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256)
    if (offsets[i] != 0) record_status(status, kStatusBadOffsets);
}

// How a call is cut, and what it needs of scratch.
struct Plan {
  bool short_streams, states_apart;
  uint32_t tiles, tile_rows, groups, group_rows, parts, part_rows;
  uint64_t pair_bytes, shut_bytes;
};

// Blocks of a walk for results that the 148 SMs of a B200 hold at a time (as many parts
// as that, so that none waits for a second round). The number is fixed: scratch is asked
// for without a context, and the order of the sums goes by it.
uint32_t walks_at_once(int dtype, bool mix, bool back, bool tensor) {
  if (!tensor) return 148u * (back ? 2 : 3);
  return 148u * (dtype == PLX_F32 && back && mix ? 1 : back || dtype == PLX_F32 ? 2 : 3);
}

// Short streams go in tiles, 16-bit ones that tensor copies take only where they are few.
// Measured, in tiles and in walks, forwards and backwards: 1,024 streams of 16 steps of
// 4,096 units bf16 203 and 468 us, 167 and 214; 4,096 of 4 steps of 2,048 units 107 and
// 240, 129 and 144; 256 of 64 steps of 1,000 units f32 46 and 88, 82 and 96; of 96 steps
// (in two tiles of a walk) 70 and 129, 75 and 112; 256 of 80 steps of 501 units bf16
// without tensor copies 44 and 82, 42 and 75. A step of 256 streams of 2,048 units takes
// 5 us in tiles.
Plan plan_of(uint32_t streams, uint64_t rows, uint32_t n, int dtype, bool ragged, bool mix,
             int units, bool back, bool tensor) {
  Plan c = {};
  const uint32_t steps = ragged ? (uint32_t)rows : (uint32_t)(rows / streams);
  const uint32_t most = walks_at_once(dtype, mix, back, tensor);
  c.tiles = (n + kWalkUnits - 1) / kWalkUnits;
  const uint64_t share = rows * c.tiles / most;  // rows of a block, in one round of them
  // Streams of up to 512 steps: as many whole ones a walk as make a round of blocks.
  const bool half = tensor && dtype != PLX_F32;
  const uint32_t brief = half ? 32 : tile_steps(true);
  const bool several = !ragged && tensor && (half || steps > brief) && steps <= 512 &&
                       share >= kWalkSteps;
  c.short_streams = !ragged && !several && steps <= brief;
  if (c.short_streams) {
    c.tiles = (n + 32 * units - 1) / (32 * units);
    // whole streams, as many as a block takes or as leave two blocks an SM
    const uint64_t spread = rows * c.tiles / (2 * 148);
    c.tile_rows = (uint32_t)std::min<uint64_t>(tile_steps(back), std::max<uint64_t>(spread, kRun));
    c.tile_rows = std::max(c.tile_rows / steps, 1u) * steps;
    c.states_apart = back;
    return c;
  }
  c.parts = 1;
  c.group_rows = c.part_rows = steps;
  if (several) {
    c.group_rows = c.part_rows =
        std::max((uint32_t)std::min<uint64_t>(share, 1024) / steps, 1u) * steps;
    c.groups = (uint32_t)((rows + c.group_rows - 1) / c.group_rows);
  } else {
    c.groups = ragged ? 1 : streams;
    const uint64_t walks = (uint64_t)c.groups * c.tiles;
    if (walks < most / 2)
      c.parts = std::max(1u, std::min((uint32_t)(most / walks), steps / kWalkSteps));
    c.part_rows = (steps + c.parts - 1) / c.parts;
    c.part_rows = (c.part_rows + kWalkSteps - 1) / kWalkSteps * kWalkSteps;
    c.parts = (steps + c.part_rows - 1) / c.part_rows;
  }
  // a stream may begin and end in one tile, or in two parts
  c.states_apart = ragged || several || c.parts > 1 || steps <= kWalkSteps;
  if (c.parts > 1) {
    c.pair_bytes = (uint64_t)c.groups * c.parts * c.tiles * kWalkUnits * 8;
    c.shut_bytes = ((uint64_t)c.groups * c.parts * 4 + 255) / 256 * 256;
  }
  return c;
}

uint64_t state_bytes(uint32_t streams, uint32_t n) {
  return ((uint64_t)streams * n * 4 + 255) / 256 * 256;
}

int check_recurrence(const plx_ctx* ctx, uint32_t streams, uint64_t rows, uint32_t n, int dtype,
                     const int32_t* offsets, int gate_kind, int mix, bool back, const void* scratch,
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
  const size_t need =
      plx_recurrence_scratch_bytes(streams, rows, n, dtype, offsets != nullptr, mix, back);
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
  const float* given = BACK ? a.dfinal : a.state;
  const uint64_t count = (uint64_t)a.streams * a.n;
  float* state_out = a.state_out;
  auto copy_state = [&](const float* from) {
    k_copy_state<<<(unsigned)std::min<uint64_t>((count + 255) / 256, 1 << 16), 256, 0,
                   ctx->stream>>>(count, from, state_out);
    PLX_LAUNCH_CHECK("k_copy_state");
    return PLX_OK;
  };
  if (a.rows == 0) {
    if (a.offsets) {
      k_check_offsets<<<std::min((a.streams + 256) / 256, 1024u), 256, 0, ctx->stream>>>(
          a.streams + 1, a.offsets, ctx->d_status);
      PLX_LAUNCH_CHECK("k_check_offsets");
    }
    return state_out && state_out != given ? copy_state(given) : PLX_OK;
  }
  if (a.rows == 1) a.ldx = a.ldg = a.ldh = a.lddh = a.ldo = a.ldo2 = a.n;
  a.steps = a.offsets ? 0 : (uint32_t)(a.rows / a.streams);
  a.status = ctx->d_status;
  a.timeout_ns = ctx->timeout_ns;
  bool copied = false;
  const int rc = with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    uint64_t odd = a.n;
    for (int64_t ld : {a.ldx, a.ldg, a.ldh, a.lddh, a.ldo, a.ldo2}) odd |= (uint64_t)ld;
    odd *= sizeof(T);
    for (const void* q : {a.x, a.gate, a.h, a.dh, (const void*)a.out, (const void*)a.out2})
      odd |= reinterpret_cast<uintptr_t>(q);
    auto go = [&](auto v_c, auto sigmoid_c, auto mix_c) -> int {
      constexpr int V = decltype(v_c)::value;
      constexpr bool SIGMOID = decltype(sigmoid_c)::value, MIX = decltype(mix_c)::value;
      // units side by side and 16-byte rows: whole tiles of long streams at a time
      bool tensor = V == 2;
      for (int64_t ld : {a.ldx, a.ldg, a.ldh, a.lddh}) tensor &= ld * sizeof(T) % 16 == 0;
      for (const void* q : {a.x, a.gate, a.h, a.dh}) tensor &= aligned16(q);
      const Plan c =
          plan_of(a.streams, a.rows, a.n, dtype, a.offsets != nullptr, MIX, V, BACK, tensor);
      a.tiles = c.tiles;
      a.tile_rows = c.tile_rows;
      a.groups = c.groups;
      a.group_rows = c.group_rows;
      a.parts = c.parts;
      a.part_rows = c.part_rows;
      const uint64_t blocks =
          c.short_streams ? (a.rows + c.tile_rows - 1) / c.tile_rows * c.tiles
                          : (uint64_t)c.groups * c.parts * c.tiles;
      if (blocks >= (1ull << 31))
        return set_error(PLX_ERR_CAPACITY, "%llu rows of %u units are too many for one call",
                         (unsigned long long)a.rows, a.n);
      char* at = (char*)scratch;
      if (c.states_apart) {
        // What is given is read by other warps than those that write the result:
        // where both are one array, the result goes to scratch first.
        copied = state_out && state_out == given;
        if (copied) a.state_out = (float*)at;
        at += state_bytes(a.streams, a.n);
      }
      if (c.short_streams) {
        k_recurrence_tile<T, V, SIGMOID, MIX, BACK>
            <<<(unsigned)blocks, (c.tile_rows + kRun - 1) / kRun * 32, 0, ctx->stream>>>(a);
        PLX_LAUNCH_CHECK("k_recurrence_tile");
        return PLX_OK;
      }
      if (c.parts > 1) {
        a.shut = (uint32_t*)at;
        a.pairs = (float2*)(at + c.shut_bytes);
      }
      auto walk = [&](auto tensor_c) -> int {
        constexpr bool TENSOR = decltype(tensor_c)::value;
        constexpr int ARRAYS = BACK ? (MIX ? 4 : 3) : 2;
        Maps maps = {};
        if constexpr (TENSOR) {
          const void* of[4] = {a.gate, BACK ? a.dh : a.x, a.h, a.x};
          const int64_t ld[4] = {a.ldg, BACK ? a.lddh : a.ldx, a.ldh, a.ldx};
          for (int k = 0; k < ARRAYS; ++k)
            if (int rc = tensor_map(&maps.of[k], dtype, of[k], a.n, a.rows, ld[k], kWalkUnits,
                                    kWalkSteps, false))
              return rc;
        }
        if (c.parts > 1) {
          constexpr auto leave = k_recurrence_walk<T, SIGMOID, MIX, BACK, true, TENSOR>;
          using R = WalkRing<T, 2, TENSOR>;
          PLX_TRY_CUDA(allow_shared<leave>(ctx->device, R::bytes));
          leave<<<(unsigned)blocks, kWalkWarps * 32, R::bytes, ctx->stream>>>(a, maps);
          PLX_LAUNCH_CHECK("k_recurrence_walk");
        }
        constexpr auto kernel = k_recurrence_walk<T, SIGMOID, MIX, BACK, false, TENSOR>;
        using R = WalkRing<T, ARRAYS, TENSOR>;
        PLX_TRY_CUDA(allow_shared<kernel>(ctx->device, R::bytes));
        kernel<<<(unsigned)blocks, kWalkWarps * 32, R::bytes, ctx->stream>>>(a, maps);
        PLX_LAUNCH_CHECK("k_recurrence_walk");
        return PLX_OK;
      };
      return tensor ? walk(std::true_type{}) : walk(std::false_type{});
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
  if (rc != PLX_OK) return rc;
  return copied ? copy_state(a.state_out) : PLX_OK;
}

}  // namespace
}  // namespace plx

using namespace plx;

extern "C" size_t plx_recurrence_scratch_bytes(uint32_t n_streams, uint64_t rows, uint32_t n,
                                               int dtype, int ragged, int mix, int backward) {
  if (n_streams == 0 || rows == 0 || n == 0 || rows >= (1ull << 31) || !valid_dtype(dtype))
    return 0;
  uint64_t most = 0;  // whatever the arrays' alignment
  for (bool tensor : {false, true}) {
    const Plan c =
        plan_of(n_streams, rows, n, dtype, ragged != 0, mix != 0, 1, backward != 0, tensor);
    most = std::max(most, (c.states_apart ? state_bytes(n_streams, n) : 0) + c.pair_bytes +
                              c.shut_bytes);
  }
  return most;
}

static int forward(plx_ctx* ctx, bool clear, uint32_t n_streams, uint64_t rows, uint32_t n,
                   int dtype, const int32_t* offsets, const void* x, int64_t ldx,
                   const void* gate, int64_t ldg, int gate_kind, int mix, const float* state,
                   void* h, int64_t ldh, float* final_state, void* scratch,
                   size_t scratch_bytes) {
  if (int rc = check_recurrence(ctx, n_streams, rows, n, dtype, offsets, gate_kind, mix, false,
                                scratch, scratch_bytes))
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
  a.clear = clear && offsets;
  a.state_out = final_state;
  return launch<false>(ctx, a, dtype, gate_kind, mix != 0, scratch);
}

extern "C" int plx_recurrence(plx_ctx* ctx, uint32_t n_streams, uint64_t rows, uint32_t n,
                              int dtype, const int32_t* offsets, const void* x, int64_t ldx,
                              const void* gate, int64_t ldg, int gate_kind, int mix,
                              const float* state, void* h, int64_t ldh, float* final_state,
                              void* scratch, size_t scratch_bytes) {
  return forward(ctx, false, n_streams, rows, n, dtype, offsets, x, ldx, gate, ldg, gate_kind,
                 mix, state, h, ldh, final_state, scratch, scratch_bytes);
}

extern "C" int plx_recurrence_new(plx_ctx* ctx, uint32_t n_streams, uint64_t rows, uint32_t n,
                                  int dtype, const int32_t* offsets, const void* x, int64_t ldx,
                                  const void* gate, int64_t ldg, int gate_kind, int mix,
                                  const float* state, void* h, int64_t ldh, float* final_state,
                                  void* scratch, size_t scratch_bytes) {
  return forward(ctx, true, n_streams, rows, n, dtype, offsets, x, ldx, gate, ldg, gate_kind,
                 mix, state, h, ldh, final_state, scratch, scratch_bytes);
}

extern "C" int plx_recurrence_backward(plx_ctx* ctx, uint32_t n_streams, uint64_t rows, uint32_t n,
                                       int dtype, const int32_t* offsets, const void* dh,
                                       int64_t lddh, const void* x, int64_t ldx, const void* gate,
                                       int64_t ldg, int gate_kind, int mix, const void* h,
                                       int64_t ldh, const float* state, const float* dfinal,
                                       void* dx, int64_t lddx, void* dgate, int64_t lddg,
                                       float* dstate, void* scratch, size_t scratch_bytes) {
  if (int rc = check_recurrence(ctx, n_streams, rows, n, dtype, offsets, gate_kind, mix, true,
                                scratch, scratch_bytes))
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
  a.clear = offsets != nullptr;
  a.ldo2 = lddg;
  a.state_out = dstate;
  return launch<true>(ctx, a, dtype, gate_kind, mix != 0, scratch);
}
