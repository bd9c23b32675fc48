// Shared by block_norm.cu (forward) and block_norm_backward.cu.
#pragma once

#include "norm.cuh"

namespace plx {

struct BlockNorm {
  uint32_t rows, n;
  float inv_n, scale, eps;
  int gate;
  bool layer, post, sigmoid, param_f32;
  const void *x, *o, *gate_values;
  int64_t ldx, ldo, ldg;
  const void *post_weight, *post_bias, *pre_weight, *pre_bias;
  // forward
  void *r, *u;
  int64_t ldr, ldu;
  float4* stats_out;
  // backward
  const void *dr, *du;
  int64_t lddr, lddu;
  const float4* stats;  // mean and rstd of o, of r
  void *dx, *d_o, *dgate;
  int64_t lddx, lddo, lddg;
  float* partial;  // column sums
};

int check_block_norm(const plx_ctx* ctx, uint64_t rows, uint32_t n, int dtype,
                     const plx_block_norm_params* p);
BlockNorm block_norm_of(uint64_t rows, uint32_t n, const plx_block_norm_params* p);

// Pieces of a row, STEP values apart; 0 past its end.
template <int STEP, int NV, int V, typename T>
__device__ __forceinline__ void load_row(const T* from, int left, Pack<T, V> (&q)[NV]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j * STEP < left) {
      q[j] = load_pack<T, V>(from + j * STEP);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) q[j].v[e] = from_f32<T>(0.0f);
    }
  }
}

// A thread's columns of the rows that TPR threads share: NV pieces of V consecutive
// values, STEP apart, taken as pairs. A group is a piece, or where pieces are single
// values two of them.
template <typename T, int V, int NV, int TPR>
struct Columns {
  static constexpr int STEP = TPR * V;
  static constexpr int HV = V == 1 ? 1 : V / 2, G = V == 1 ? NV / 2 : NV;  // pairs, groups
  static constexpr int GSTEP = V == 1 ? 2 * STEP : STEP;
  static constexpr int H = G * HV, E = NV * V;
  static_assert(E % 2 == 0, "columns in pairs");
  using P = Pack<T, V>;
  uint32_t c0;
  int left;  // values from the first column to the row's end
  __device__ __forceinline__ Columns(uint32_t n, uint32_t first)
      : c0(first), left((int)n - (int)first) {}
  __device__ __forceinline__ bool in(int group) const { return group * GSTEP < left; }
  // whether the second value of a pair is in the row as well
  __device__ __forceinline__ bool both(int group) const {
    return V > 1 || group * GSTEP + STEP < left;
  }
  // Pairs of a group out of its pieces (`piece(j)`).
  template <typename F>
  static __device__ __forceinline__ void get(F piece, int group, F2 (&v)[HV]) {
    if constexpr (V == 1) {
      v[0] = pack2(to_f32(piece(2 * group).v[0]), to_f32(piece(2 * group + 1).v[0]));
    } else {
      const P q = piece(group);
#pragma unroll
      for (int e = 0; e < HV; ++e) v[e] = pair_of(q, 2 * e);
    }
  }
  // `row`: at this thread's first column
  __device__ __forceinline__ void put(T* row, int group, const F2 (&v)[HV]) const {
    T* to = row + group * GSTEP;
    if constexpr (V == 1) {
      to[0] = from_f32<T>(v[0].x);
      if (both(group)) to[STEP] = from_f32<T>(v[0].y);
    } else {
      P q;
#pragma unroll
      for (int e = 0; e < HV; ++e) put_pair(q, 2 * e, v[e]);
      *reinterpret_cast<P*>(to) = q;
    }
  }
  // A parameter of every column; `none` where it is not given or past the row's end.
  template <typename Q>
  __device__ __forceinline__ void param_of(const Q* w, F2 (&v)[H], float none) const {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if constexpr (V == 1) {
        const Q* at = w + c0 + g * GSTEP;
        v[g] = pack2(w && in(g) ? to_f32(at[0]) : none,
                     w && in(g) && both(g) ? to_f32(at[STEP]) : none);
      } else if (w && in(g)) {
        const Pack<Q, V> q = load_pack<Q, V>(w + c0 + g * GSTEP);
#pragma unroll
        for (int e = 0; e < HV; ++e) v[g * HV + e] = pair_of(q, 2 * e);
      } else {
#pragma unroll
        for (int e = 0; e < HV; ++e) v[g * HV + e] = pack2(none, none);
      }
    }
  }
  __device__ __forceinline__ void param(const void* w, bool f32, F2 (&v)[H], float none) const {
    if (f32) param_of((const float*)w, v, none);
    else param_of((const T*)w, v, none);
  }
};

// Rows of K arrays under way at once, in shared memory; a thread reads what it copied
// itself, so that no barrier is needed. Pieces of less than four bytes go to registers.
// S stages: 512 threads an SM (in one block or more) share 160 to 192 KB.
template <typename T, int V, int NV, int TPR, int K, int S>
struct BlockRing {
  static constexpr int piece = V * sizeof(T);
  static constexpr bool used = piece >= 4;
  static constexpr int threads = TPR == 32 ? 256 : TPR;
  static constexpr int array_bytes = NV * threads * piece;
  static constexpr int stage_bytes = K * array_bytes;
  static constexpr int stages = S;
  static constexpr int bytes = used ? stages * stage_bytes : 0;
  using C = Columns<T, V, NV, TPR>;
  using P = Pack<T, V>;
  char* ring;
  const T* from[K];  // this thread's first column of the row fetched next; NULL: not given
  int64_t step[K];   // to the next one
  P held[used ? 1 : K][used ? 1 : NV];
  __device__ __forceinline__ P* slot(uint32_t stage, int array, int j) const {
    return reinterpret_cast<P*>(ring + stage * stage_bytes + array * array_bytes) + j * threads +
           threadIdx.x;
  }
  // Columns past the row's end, and arrays that are not given, are 0.
  __device__ __forceinline__ void clear(const C& c) {
    P zero;
#pragma unroll
    for (int e = 0; e < V; ++e) zero.v[e] = from_f32<T>(0.0f);
    if constexpr (used)
      for (int s = 0; s < stages; ++s)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (!from[k] || j * C::STEP >= c.left) *slot(s, k, j) = zero;
  }
  // Starts the copies of the next row (`there`: it is one), or reads it.
  __device__ __forceinline__ void fetch(const C& c, bool there, uint32_t stage) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if constexpr (used) {
        if (there && from[k])
#pragma unroll
          for (int j = 0; j < NV; ++j)
            if (j * C::STEP < c.left) copy_async<piece>(slot(stage, k, j), from[k] + j * C::STEP);
      } else {
        if (there && from[k]) load_row<C::STEP>(from[k], c.left, held[k]);
        else
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) held[k][j].v[e] = from_f32<T>(0.0f);
      }
      from[k] = from[k] ? from[k] + step[k] : nullptr;
    }
  }
  // Pairs of a group of an array of the row under way.
  __device__ __forceinline__ void get(uint32_t stage, int array, int group, F2 (&v)[C::HV]) const {
    C::get([&](int j) {
      if constexpr (used) return *slot(stage, array, j);
      else return held[array][j];
    }, group, v);
  }
};

// The values of a row, made from what is read (rows that no registers hold).
template <typename T, typename P>
struct RowOf {
  const BlockNorm& a;
  int64_t row;
  float m1, s1, m2, s2;
  __device__ __forceinline__ RowOf(const BlockNorm& b, int64_t r) : a(b), row(r) {}
  __device__ __forceinline__ float affine(float h, const void* w, const void* b, uint32_t i) const {
    if (w) h *= to_f32(((const P*)w)[i]);
    if (b) h += to_f32(((const P*)b)[i]);
    return h;
  }
  __device__ __forceinline__ float o(uint32_t i) const {
    return to_f32(((const T*)a.o)[row * a.ldo + i]);
  }
  __device__ __forceinline__ float h1(uint32_t i) const { return a.post ? (o(i) - m1) * s1 : o(i); }
  __device__ __forceinline__ float p(uint32_t i) const {
    return a.post ? affine(h1(i), a.post_weight, a.post_bias, i) : o(i);
  }
  // The gate and its derivative.
  __device__ __forceinline__ float gate(uint32_t i, float& slope) const {
    slope = 1.0f;
    if (a.gate == PLX_BLOCK_GATE_NONE) return 1.0f;
    const float g = a.gate == PLX_BLOCK_GATE_UNITS
                        ? to_f32(((const P*)a.gate_values)[i])
                        : to_f32(((const T*)a.gate_values)[row * a.ldg + i]);
    if (!a.sigmoid) return g;
    const Sigmoid s = sigmoid(g);
    slope = s.a * s.keep;
    return s.a;
  }
  __device__ __forceinline__ float r(uint32_t i) const {
    float slope;
    const float g = gate(i, slope);
    return fmaf(g, p(i), a.scale * to_f32(((const T*)a.x)[row * a.ldx + i]));
  }
};

// Values that can be read together in every array of a call.
template <typename T, typename P>
uint32_t block_piece(const BlockNorm& a, std::initializer_list<const void*> rows,
                     std::initializer_list<int64_t> strides) {
  uint64_t at = 0, ld = 0, w = 0;
  for (const void* p : rows) at |= reinterpret_cast<uintptr_t>(p);
  for (int64_t s : strides) ld |= (uint64_t)s;
  const uint64_t g = reinterpret_cast<uintptr_t>(a.gate_values);
  if (a.gate == PLX_BLOCK_GATE_VALUES) {
    at |= g;
    ld |= (uint64_t)a.ldg;
  } else {
    w |= g;
  }
  for (const void* p : {a.post_weight, a.post_bias, a.pre_weight, a.pre_bias})
    w |= reinterpret_cast<uintptr_t>(p);
  return piece_values(a.n, sizeof(T), {(const void*)at}, {(int64_t)ld}, (const void*)w, nullptr,
                      sizeof(P));
}

}  // namespace plx
