// Kernels of the selective state space scan (selscan.cuh has the formulas and the split).
#pragma once

#include <cfloat>

#include "pairs.cuh"
#include "selscan.cuh"

namespace fdwt {
namespace {

// ------------------------------------------------------------------------------ arithmetic
template <typename A> struct alignas(4 * sizeof(A)) Four {
  A v[4];
};

template <typename A> __device__ __forceinline__ Two<A> low(const Four<A>& q) {
  return two(q.v[0], q.v[1]);
}
template <typename A> __device__ __forceinline__ Two<A> high(const Four<A>& q) {
  return two(q.v[2], q.v[3]);
}

// e^-|v| of two values: the product with log2 e is rounded, so what it lost corrects the result.
__device__ __forceinline__ Two<float> neg_exp(float v, float w) {
  constexpr float kHigh = 1.442695021629333f, kLow = 1.92596299e-8f;  // log2 e in two parts
  const Two<float> a = two(fminf(fabsf(v), 128.0f), fminf(fabsf(w), 128.0f));
  const Two<float> t = mul(a, both(-kHigh));
  const Two<float> lost = fma(a, both(kLow), fma(a, both(kHigh), t));
  const Two<float> e = exp_2(t);
  return fma(e, mul(lost, both(-static_cast<float>(kLn2))), e);
}
// log(1 + e^v) = max(v, 0) + log(1 + e^-|v|) of 4 values, to the last bits where it is small too
// (steps are often 1e-3), and with SLOPE its slope 1 / (1 + e^-v).  log(1 + e) = 2 atanh(s),
// s = e / (2 + e) <= 1/3: the odd series of atanh, its coefficients fitted for s^2 up to 1/9 (8e-9
// off).  Against expf and log1pf of the library: 11 instructions in place of 35, 2 to 4 roundings
// off as they are.
template <bool SLOPE>
__device__ __forceinline__ void softplus(const float* v, float* d, float* slope) {
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const Two<float> e = neg_exp(v[j], v[j + 1]);
    const Two<float> n = add(e, both(2.0f));
    const Two<float> s = mul(e, two(reciprocal(first(n)), reciprocal(second(n))));
    const Two<float> z = mul(s, s);
    Two<float> q = fma(both(0.2817465662956238f), z, both(0.2796141803264618f));
    q = fma(q, z, both(0.40024852752685547f));
    q = fma(q, z, both(0.6666631698608398f));
    q = fma(q, z, both(2.0f));
    // (max, and not (v + |v|) / 2, which is NaN for -inf and infinite above half the largest float; sums
    // that the compiler does not join with the product, so that other steps keep their last bits)
    const Two<float> rest = mul(s, q);
    const Two<float> r = two(__fadd_rn(max_nan(v[j], 0.0f), first(rest)),
                             __fadd_rn(max_nan(v[j + 1], 0.0f), second(rest)));
    if (SLOPE) {
      const Two<float> o = add(e, both(1.0f));
      const Two<float> w = two(reciprocal(first(o)), reciprocal(second(o))), ew = mul(e, w);
      slope[j] = v[j] < 0.0f ? first(ew) : first(w);
      slope[j + 1] = v[j + 1] < 0.0f ? second(ew) : second(w);
    }
    d[j] = first(r), d[j + 1] = second(r);
  }
}
template <bool SLOPE>
__device__ __forceinline__ void softplus(const double* v, double* d, double* slope) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const double e = exp(-fabs(v[j])), x = v[j];
    if (SLOPE) slope[j] = x < 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e);
    d[j] = (x < 0.0 ? 0.0 : x) + log1p(e);
  }
}
__device__ __forceinline__ float softplus(float v) {
  const float x[4] = {v, v, v, v};
  float d[4];
  softplus<false>(x, d, nullptr);  // (one of the pairs is all that is kept)
  return d[0];
}
__device__ __forceinline__ double softplus(double v) {
  return (v < 0.0 ? 0.0 : v) + log1p(exp(-fabs(v)));
}
// 1 / (1 + e^-v) of 4 values to a few roundings (NaN gives a number: a product with v follows), or,
// where the result is rounded to 16 bits (FAST), by the plain fast functions.
template <bool FAST> __device__ __forceinline__ void sigmoid_at(const float* v, float* g) {
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    if constexpr (FAST) {
      g[j] = __fdividef(1.0f, 1.0f + __expf(-v[j]));
      g[j + 1] = __fdividef(1.0f, 1.0f + __expf(-v[j + 1]));
    } else {
      const Two<float> e = neg_exp(v[j], v[j + 1]), o = add(e, both(1.0f));
      const Two<float> w = two(reciprocal(first(o)), reciprocal(second(o))), ew = mul(e, w);
      g[j] = v[j] < 0.0f ? first(ew) : first(w);
      g[j + 1] = v[j + 1] < 0.0f ? second(ew) : second(w);
    }
  }
}
template <bool FAST> __device__ __forceinline__ void sigmoid_at(const double* v, double* g) {
#pragma unroll
  for (int j = 0; j < 4; ++j) g[j] = 1.0 / (1.0 + exp(-v[j]));
}

// Added to the exponent of every decay.  The hardware's 2^x is 1.8e-8 to 2.7e-8 too small in the mean
// for -1/2 < x < -2^-8 (measured over 2^20 values for each power of two; 3e-8 to 4e-8 root mean square),
// and a state is a product of hundreds of decays: this takes half of the mean back or more (2^lift = 1 +
// 1.4e-8) at no cost, a product becoming a product and sum.  Nearer to zero, where the mean is -0.5e-8 to
// -0.8e-8, it becomes one of the same size and the other sign.  4 x 4096 x 2048 against 64 bits: last
// states 5e-7 off without, 2.8e-7 with; dL/da 1.7e-6 and 0.75e-6.  2^lift itself comes out as 1, so that a
// step of zero keeps the state as it is.
template <typename A> __device__ __forceinline__ A lift() { return sizeof(A) == 4 ? A(2e-8) : A(0); }
template <typename A> __device__ __forceinline__ Two<A> lift2() { return two(lift<A>(), lift<A>()); }

// A channel's rates times log2 e.  -inf (forgets everything) becomes the lowest finite value, so
// that a step of zero, as padding has, keeps the state.
__device__ __forceinline__ float rate(float a) {
  const float r = a * static_cast<float>(kLog2e);
  return r < -FLT_MAX ? -FLT_MAX : r;
}
__device__ __forceinline__ double rate(double a) {
  const double r = a * kLog2e;
  return r < -DBL_MAX ? -DBL_MAX : r;
}

// Four states carried over a segment: 2^(sum r) s + e, with the segment's sum of steps, the rates and the
// states that it forms from zero; whether a 2^(sum r) leaves the type's range (rates above or steps below
// zero, long segments).
template <typename A>
__device__ __forceinline__ bool carry(A* s, A sum, const A* r, const Four<A>& e) {
  bool grows = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const A q = sum * r[j];
    grows |= q > A(sizeof(A) == 4 ? 126 : 1022);
    s[j] = fma(exp_2(q), s[j], e.v[j]);
  }
  return grows;
}
// The same in two halves where it does: a state of zero stays zero, as it does token by token.
template <typename A>
__device__ __forceinline__ void carry_growing(A* s, A sum, const A* r, const Four<A>& e) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const A q = sum * r[j], half = exp_2(A(0.5) * q);
    s[j] = s[j] == A(0) && q > A(0) ? e.v[j] : fma(half * s[j], half, e.v[j]);
  }
}

// Sums of V values each over L lanes `STRIDE` apart (powers of two): with each step a lane hands
// over half of its values.  Afterwards v[0 .. max(V / L, 1)) are the sums of the values from
// index * V / L on, index being the lane's place among the L (where L > V, lanes in runs of L / V
// hold the same sum).
template <int V, int L, int STRIDE, typename A> __device__ __forceinline__ void fold(A* v, int lane) {
  if constexpr (L > 1) {
    constexpr int o = L / 2 * STRIDE;
    if constexpr (V > 1) {
      const bool upper = lane & o;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const A keep = upper ? v[V / 2 + i] : v[i], send = upper ? v[i] : v[V / 2 + i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
      }
      fold<V / 2, L / 2, STRIDE>(v, lane);
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
      fold<1, L / 2, STRIDE>(v, lane);
    }
  }
}

// The same with values in another order in every lane, so that no lane has to choose: where place
// p among L lanes holds its M values in the order 0 ^ p, 1 ^ p, ..., (bits of p from the top of the
// order down, as many as both have), each step keeps the first half of the registers and hands over
// the second.  v holds V runs of M values; afterwards register 0 of each run, or the first M / L, is
// a sum over the first log2 M bits of the lanes; fold takes the others.
template <int V, int M, int L, int STRIDE, typename A> __device__ __forceinline__ void fold_swapped(A* v) {
  if constexpr (M > 1 && L > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < M / 2; ++j)
        v[i * (M / 2) + j] = v[i * M + j] + __shfl_xor_sync(0xffffffffu, v[i * M + M / 2 + j], STRIDE);
    fold_swapped<V, M / 2, L / 2, 2 * STRIDE>(v);
  }
}
// The order of the M values of a lane at place p among L: register j holds value j ^ order.  Bit i
// of p decides about bit log2 M - 1 - i of the value.
template <int M, int L> __device__ __forceinline__ int order_at(int p) {
  if constexpr (M <= 1 || L <= 1) return 0;
  else return (p & 1) * (M / 2) | order_at<M / 2, L / 2>(p >> 1);
}
template <typename A> __device__ __forceinline__ Four<A> reorder(Four<A> q, int order) {
  if (order & 2) q = {q.v[2], q.v[3], q.v[0], q.v[1]};
  if (order & 1) q = {q.v[1], q.v[0], q.v[3], q.v[2]};
  return q;
}

__device__ __forceinline__ int64_t valid_tokens(const ScanArgs& p, int64_t b) {
  if (p.lengths == nullptr) return p.length;
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : (n < p.length ? n : p.length);
}

// What a block works on.
struct Place {
  int64_t b, t0, t1, count;  // sequence, its segment's tokens, the valid ones among them (an end)
  int64_t d0;                // first channel
  int group, segment, tile, width;  // width: channels of the tile
};
// `segments` of the sequence have a block, those from `first` on.
template <int CT>
__device__ __forceinline__ Place place_of(const ScanArgs& p, int segments, int first) {
  Place w;
  const int64_t tiles = p.tile_count;
  const int64_t id = blockIdx.x;
  w.tile = static_cast<int>(id % tiles + p.tile0);
  w.segment = static_cast<int>(id / tiles % segments) + first;
  w.b = id / tiles / segments;
  w.group = static_cast<int>(w.tile / p.tiles);
  const int64_t within = (w.tile % p.tiles) * CT;
  w.d0 = w.group * p.per + within;
  w.width = static_cast<int>(p.per - within < CT ? p.per - within : CT);
  w.t0 = w.segment * p.seg_len;
  w.t1 = w.t0 + p.seg_len < p.length ? w.t0 + p.seg_len : p.length;
  w.count = valid_tokens(p, w.b);
  if (w.count > w.t1) w.count = w.t1;
  return w;
}

// 4 neighbouring elements of a row, the first `have` of which exist (4 or none where the rows begin
// on their boundary); the others are zero.  16-bit elements stay packed until they are used: taken
// apart at once, each load would be waited for where it is issued.
template <typename T> struct Quad {
  using Raw = Four<T>;
  static __device__ __forceinline__ Raw some(const T* q, int have) {
    Raw r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = j < have ? q[j] : T(0);
    return r;
  }
  static __device__ __forceinline__ void values(const Raw& r, T* x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = r.v[j];
  }
};
template <typename T> struct Quad16 {
  using Raw = uint2;
  static __device__ __forceinline__ Raw some(const T* q, int have) {
    const unsigned short* u = reinterpret_cast<const unsigned short*>(q);
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < have ? u[j] : 0;
    return make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
  }
  static __device__ __forceinline__ void values(const Raw& r, float* x) {
    Half2<T>::split(r.x, x);
    Half2<T>::split(r.y, x + 2);
  }
};
template <> struct Quad<__half> : Quad16<__half> {};
template <> struct Quad<__nv_bfloat16> : Quad16<__nv_bfloat16> {};
template <typename T> using Raw4 = typename Quad<T>::Raw;
template <typename T> __device__ __forceinline__ Raw4<T> load4(const T* q, int have, bool vec) {
  if (vec) {
    Raw4<T> r = {};
    if (have >= 4) r = *reinterpret_cast<const Raw4<T>*>(q);
    return r;
  }
  return Quad<T>::some(q, have);
}
template <typename T, typename A>
__device__ __forceinline__ void store4(T* q, const A* x, int have, bool vec) {
  if (vec && have >= 4) {
    Group<T, 4>::store(q, x);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < have) q[j] = from_acc<T>(x[j]);
  }
}
template <typename A> __device__ __forceinline__ Four<A> params4(const void* q, int64_t at, int have) {
  Four<A> r = {A(0), A(0), A(0), A(0)};
  if (q != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < have) r.v[j] = static_cast<const A*>(q)[at + j];
  }
  return r;
}

// The threads of a block that stages TT tokens of CT channels: each takes 4 neighbouring channels
// (always the same) of IT tokens, ROWS apart.
template <int CT, int TT> struct Items {
  static constexpr int COLS = CT / 4, ROWS = 128 / COLS, IT = (TT + ROWS - 1) / ROWS;
};

// A thread's share of b (and c) of TT tokens: 4 states a load, on the way to shared memory.
template <typename T, int TT, int LN, int ARRAYS> struct States {
  using A = typename AccOf<T>::type;
  static constexpr int ALL = TT * LN * ARRAYS, IT = (ALL + 127) / 128;
  // loads that lie whole rows of tokens apart in one array share a pointer
  static constexpr int EACH = ARRAYS == 2 && TT * LN < 128 ? IT : (TT * LN + 127) / 128;
  static constexpr int PTRS = (IT + EACH - 1) / EACH;
  Raw4<T> raw[IT];
  const T* at[PTRS];
  int64_t stride[PTRS];
  __device__ __forceinline__ void start(const ScanArgs& p, const Place& w, const void* b,
                                        const int64_t* bs, const void* c, const int64_t* cs,
                                        int64_t t) {
#pragma unroll
    for (int i = 0; i < PTRS; ++i) {
      const int e = threadIdx.x + i * EACH * 128;
      const bool second = ARRAYS == 2 && e >= TT * LN;
      const int64_t* s = second ? cs : bs;
      stride[i] = s[1];
      at[i] = static_cast<const T*>(second ? c : b) + w.b * s[0] + w.group * s[2] +
              (t + e / LN % TT) * s[1] + e % LN * 4;
    }
  }
  // `left` tokens from the step's first on are valid; the next step is `step` tokens on.
  __device__ __forceinline__ void fetch(const ScanArgs& p, int left, int step) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int e = threadIdx.x + i * 128;
      if (ALL % 128 != 0 && e >= ALL) break;
      const int k = i / EACH;
      raw[i] = load4(at[k] + (i % EACH) * (128 / LN) * stride[k],
                     e / LN % TT < left ? p.states - e % LN * 4 : 0, p.vec_states);
    }
#pragma unroll
    for (int i = 0; i < PTRS; ++i) at[i] += step * stride[i];
  }
  __device__ __forceinline__ void store(Four<A>* out) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int e = threadIdx.x + i * 128;
      if (ALL % 128 != 0 && e >= ALL) break;
      Four<A> q;
      Quad<T>::values(raw[i], q.v);
      out[e] = q;
    }
  }
  // [ARRAYS TT][COPIES][LN], copy k in the order of lanes at place k
  template <int COPIES> __device__ __forceinline__ void store_orders(Four<A>* out) const {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int e = threadIdx.x + i * 128;
      if (ALL % 128 != 0 && e >= ALL) break;
      Four<A> q;
      Quad<T>::values(raw[i], q.v);
#pragma unroll
      for (int k = 0; k < COPIES; ++k)
        out[(e / LN * COPIES + k) * LN + e % LN] = reorder(q, order_at<4, COPIES>(k));
    }
  }
};

// Step and taken-in input of a token and channel.
template <typename A> struct alignas(2 * sizeof(A)) Step {
  A delta, u;
};
// ------------------------------------------------------------------------------ forward
// MAIN: outputs and last states.  STATES: a segment's end state from zero, and its sum of delta.
// REVERSE: the same back in time for the gradients, r = e^(delta a) (c dp + r).
//
// The next tokens' rows are loaded before the current ones' states are worked out, so that the
// loads' latency passes behind the exponentials.
enum ScanMode { MAIN, STATES, REVERSE };
template <typename A> constexpr int scan_fwd_tokens() { return sizeof(A) == 8 ? 8 : 16; }

template <typename T, int LN, int NC, int MODE>
__global__ void __launch_bounds__(128, sizeof(T) == 8 ? 1 : 4)
scan_fwd_kernel(const __grid_constant__ ScanArgs p) {
  using A = typename AccOf<T>::type;
  constexpr int LD = 32 / LN, CT = 4 * LD * NC, TT = scan_fwd_tokens<A>();
  constexpr int PAD = CT + 8;
  using I = Items<CT, TT>;
  __shared__ Step<A> slots[TT * CT];
  __shared__ Four<A> states[(MODE == MAIN ? 2 : 1) * TT * LN];  // b (REVERSE: c), then c
  __shared__ __align__(4 * sizeof(A)) A sums[MODE == MAIN ? TT * PAD : 1];
  // (no state is needed after the last segment, nor back in time before the first)
  const Place w = place_of<CT>(p, MODE == MAIN ? p.segments : p.segments - 1, MODE == REVERSE);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nl = lane % LN, dl = lane / LN;
  // The thread's channels of the tile: cl + (k ^ swap), in an order by its lane (fold_swapped).
  const int cl = (warp * LD + dl) * NC, swap = order_at<NC, LN>(nl);
  constexpr int KEPT = NC < LN ? NC : LN, OTHERS = LN / KEPT;  // lanes that share out channels, tokens
  static_assert(KEPT == NC || LN == 1);
  const A* rates = static_cast<const A*>(p.a);

  Two<A> ra[NC][2], h[NC][2];
  A total[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = cl + (k ^ swap);
    A r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = nl * 4 + j;
      r[j] = c < w.width && n < p.states ? rate(rates[(w.d0 + c) * p.states + n]) : A(0);
    }
    ra[k][0] = two(r[0], r[1]);
    ra[k][1] = two(r[2], r[3]);
    A s[4] = {A(0), A(0), A(0), A(0)};
    if (MODE == MAIN && c < w.width) {
      const int64_t d = w.d0 + c;
      auto initial = [&] {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[j] = p.initial != nullptr && nl * 4 + j < p.states
                     ? static_cast<const A*>(p.initial)[(w.b * p.dim + d) * p.states + nl * 4 + j]
                     : A(0);
      };
      auto segment = [&](int g, auto by) {
        const int64_t row = (w.b * p.segments + g) * p.dim + d;
        return by(s, static_cast<const A*>(p.seg_sum)[row], r,
                  static_cast<const Four<A>*>(p.seg_state)[row * LN + nl]);
      };
      // the segments before this one
      initial();
      bool grows = false;
#pragma unroll 4
      for (int g = 0; g < w.segment; ++g) grows |= segment(g, carry<A>);
      if (grows) {
        initial();
        for (int g = 0; g < w.segment; ++g) segment(g, carry_growing<A>);
      }
    }
    h[k][0] = two(s[0], s[1]);
    h[k][1] = two(s[2], s[3]);
    total[k] = A(0);
  }

  // the thread's items
  const int col = threadIdx.x % I::COLS * 4, row0 = threadIdx.x / I::COLS;
  const int have = w.width - col;
  const T* px = static_cast<const T*>(MODE == REVERSE ? p.dy : p.x) +
                w.b * (MODE == REVERSE ? p.dys[0] : p.xs[0]) + w.d0 + col;
  const int64_t xs = MODE == REVERSE ? p.dys[1] : p.xs[1];
  const T* pd = static_cast<const T*>(p.dt) + w.b * p.dts[0] + w.d0 + col;
  const T* pg = static_cast<const T*>(p.gate) + w.b * p.gs[0] + w.d0 + col;
  T* py = static_cast<T*>(p.y) + (w.b * p.length + w.t0 + row0) * p.dim + w.d0 + col;
  const Four<A> bias = params4<A>(p.dt_bias, w.d0 + col, have);
  const Four<A> skip = params4<A>(MODE == MAIN ? p.skip : nullptr, w.d0 + col, have);
  const bool gated = MODE != STATES && p.gate != nullptr;
  Raw4<T> xr[I::IT], dr[I::IT], zr[I::IT];
  States<T, TT, LN, MODE == MAIN ? 2 : 1> bc;
  const int64_t steps = w.count > w.t0 ? (w.count - w.t0 + TT - 1) / TT : 0;
  auto begin = [&](int64_t i) { return w.t0 + (MODE == REVERSE ? steps - 1 - i : i) * TT; };
  {  // from here on the pointers are those of the thread's first token of the step
    const int64_t t = begin(0) + row0;
    px += t * xs;
    pd += t * p.dts[1];
    pg += t * p.gs[1];
    bc.start(p, w, MODE == REVERSE ? p.c : p.b, MODE == REVERSE ? p.cs : p.bs, p.c, p.cs, begin(0));
  }
  auto on = [&](const T*& q, int64_t stride) { q += MODE == REVERSE ? -TT * stride : TT * stride; };
  auto rows = [&](const T* q, int64_t stride, Raw4<T>* raw, int left) {
#pragma unroll
    for (int i = 0; i < I::IT; ++i)
      raw[i] = load4(q + i * (I::ROWS * stride), i * I::ROWS < left ? have : 0, p.vec);
  };
  // tokens from the thread's first one to the end of the valid ones and of the step
  auto left_at = [&](int64_t t) {
    return static_cast<int>((w.count - t < TT ? w.count - t : TT) - row0);
  };
  auto fetch = [&](int64_t t) {
    const int left = left_at(t);
    rows(px, xs, xr, left);
    rows(pd, p.dts[1], dr, left);
    on(px, xs);
    on(pd, p.dts[1]);
    if (gated) {
      rows(pg, p.gs[1], zr, left);
      on(pg, p.gs[1]);
    }
    bc.fetch(p, static_cast<int>(w.count - t < TT ? w.count - t : TT), MODE == REVERSE ? -TT : TT);
  };

  Four<A>* kept = static_cast<Four<A>*>(p.check) +
                  ((w.b * ((p.length + 7) / 8) + w.t0 / 8) * p.dim + w.d0 + cl) * LN + nl;
  if (steps > 0) fetch(begin(0));
  for (int64_t i = 0; i < steps; ++i) {
    const int64_t t = begin(i);
    const int left = left_at(t);
    Raw4<T> xc[I::IT], zc[I::IT];
#pragma unroll
    for (int q = 0; q < I::IT; ++q) {
      const int row = row0 + q * I::ROWS;
      if (I::ROWS * I::IT > TT && row >= TT) break;
      A x[4], delta[4];
      Quad<T>::values(xr[q], x);
      Quad<T>::values(dr[q], delta);
#pragma unroll
      for (int j = 0; j < 4; ++j) delta[j] += bias.v[j];
      if (p.softplus) softplus<false>(delta, delta, nullptr);
      if (q * I::ROWS >= left) {  // (x and the rest are zero there)
#pragma unroll
        for (int j = 0; j < 4; ++j) delta[j] = A(0);
      }
      if (MODE == REVERSE && gated) {
        A z[4], g[4];
        Quad<T>::values(zr[q], z);
        sigmoid_at<false>(z, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] *= z[j] * g[j];
      }
      Step<A> out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = {delta[j], MODE == REVERSE ? x[j] : delta[j] * x[j]};
      Four<A>* to = reinterpret_cast<Four<A>*>(slots + row * CT + col);
      to[0] = {out[0].delta, out[0].u, out[1].delta, out[1].u};
      to[1] = {out[2].delta, out[2].u, out[3].delta, out[3].u};
      xc[q] = xr[q], zc[q] = zr[q];
    }
    bc.store(states);
    if (i + 1 < steps) fetch(begin(i + 1));
    __syncthreads();
#pragma unroll(MODE == MAIN ? TT / 8 : 1)
    for (int s = 0; s < TT; s += 8) {
      if (MODE == MAIN && p.check != nullptr && s < left + row0) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
          if (cl + (k ^ swap) < w.width)
            kept[(k ^ swap) * LN] = {first(h[k][0]), second(h[k][0]), first(h[k][1]),
                                     second(h[k][1])};
        kept += p.dim * LN;
      }
      A y[8 * NC];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int row = MODE == REVERSE ? TT - 1 - s - u : s + u;
        const Four<A> bq = states[row * LN + nl];
        Four<A> cq;
        if constexpr (MODE == MAIN) cq = states[(TT + row) * LN + nl];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const Step<A> st = slots[row * CT + cl + (k ^ swap)];
          const Two<A> d2 = two(st.delta, st.delta), u2 = two(st.u, st.u);
          const Two<A> e0 = exp_2(fma(d2, ra[k][0], lift2<A>())), e1 = exp_2(fma(d2, ra[k][1], lift2<A>()));
          if constexpr (MODE == REVERSE) {
            h[k][0] = mul(e0, fma(u2, low(bq), h[k][0]));
            h[k][1] = mul(e1, fma(u2, high(bq), h[k][1]));
          } else {
            h[k][0] = fma(e0, h[k][0], mul(u2, low(bq)));
            h[k][1] = fma(e1, h[k][1], mul(u2, high(bq)));
          }
          if constexpr (MODE == MAIN) {
            const Two<A> s2 = fma(h[k][1], high(cq), mul(h[k][0], low(cq)));
            y[u * NC + k] = first(s2) + second(s2);
          } else {
            total[k] += st.delta;
          }
        }
      }
      if constexpr (MODE == MAIN) {
        fold_swapped<8, NC, LN, 1>(y);
        fold<8, OTHERS, KEPT>(y, lane);
        constexpr int OWN = 8 >= OTHERS ? 8 / OTHERS : 1, SAME = OTHERS > 8 ? OTHERS / 8 : 1;
#pragma unroll
        for (int o = 0; o < OWN; ++o)
          sums[(s + nl / KEPT / SAME * OWN + o) * PAD + cl + (LN == 1 ? 0 : swap)] = y[o];
      }
    }
    __syncthreads();
    if constexpr (MODE == MAIN) {
#pragma unroll
      for (int q = 0; q < I::IT; ++q) {
        const int row = row0 + q * I::ROWS;
        if (q * I::ROWS >= left) break;
        const Four<A> f = *reinterpret_cast<const Four<A>*>(sums + row * PAD + col);
        A y[4] = {f.v[0], f.v[1], f.v[2], f.v[3]};
        if (p.skip != nullptr) {
          A x[4];
          Quad<T>::values(xc[q], x);
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] += skip.v[j] * x[j];
        }
        if (gated) {
          A z[4], g[4];
          Quad<T>::values(zc[q], z);
          sigmoid_at<sizeof(T) == 2>(z, g);
#pragma unroll
          for (int j = 0; j < 4; ++j) y[j] *= z[j] * g[j];
        }
        store4(py + q * (I::ROWS * p.dim), y, have, p.vec);
      }
      py += TT * p.dim;
    }
  }

  if constexpr (MODE == MAIN) {
    const A none[4] = {A(0), A(0), A(0), A(0)};
    T* rest = static_cast<T*>(p.y) + w.b * p.length * p.dim + w.d0 + col;
    for (int64_t t = (w.count > w.t0 ? w.count : w.t0) + row0; t < w.t1; t += I::ROWS)
      store4(rest + t * p.dim, none, have, p.vec);
    if (w.segment != p.segments - 1 || p.final_state == nullptr) return;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const A s[4] = {first(h[k][0]), second(h[k][0]), first(h[k][1]), second(h[k][1])};
      const int c = cl + (k ^ swap);
      A* to = static_cast<A*>(p.final_state) + (w.b * p.dim + w.d0 + c) * p.states;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c < w.width && nl * 4 + j < p.states) to[nl * 4 + j] = s[j];
    }
  } else {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = cl + (k ^ swap);
      if (c >= w.width) continue;
      const int64_t row = (w.b * p.segments + w.segment) * p.dim + w.d0 + c;
      static_cast<Four<A>*>(p.seg_state)[row * LN + nl] = {first(h[k][0]), second(h[k][0]),
                                                           first(h[k][1]), second(h[k][1])};
      if (nl == 0) static_cast<A*>(p.seg_sum)[row] = total[k];
    }
  }
}

// ------------------------------------------------------------------------------ backward
// A block walks its segment back in time, 8 tokens at a time, in two halves.  From the state that
// the forward pass kept before the 8 a thread forms the states and decays of a half's 4 tokens
// again (for the later half after passing over the earlier one) and keeps them in registers, then
// goes back over them.  One channel a thread and 8 tokens at once (no passing over, one channel's
// registers) was slower (4 x 4096 x 2048 with gradients: 4.7 ms against 3.1 ms then), as were 3
// blocks an SM with spills (1.65 ms against 1.51 ms then): the kernel is bound by its instructions
// (340 a token and channel of 16 states) at the 8 warps an SM that 255 registers leave.  What moved
// out of registers (sums of da, dt_bias, skip) and loads a step ahead gained 7 %, the slopes and
// openings in shared memory lost 2 %.
template <typename T, int LN, int NC>
__global__ void __launch_bounds__(128)
scan_bwd_kernel(const __grid_constant__ ScanArgs p) {
  using A = typename AccOf<T>::type;
  constexpr int LD = 32 / LN, CT = 4 * LD * NC, NP = 4 * LN, TT = kScanCheck, SUB = TT / 2;
  constexpr int PAD = CT + 8;
  constexpr int COPIES = LD < 4 ? LD : 4;  // orders of 4 states
  using I = Items<CT, TT>;
  extern __shared__ __align__(32) unsigned char smem_raw[];
  Four<A>* states = reinterpret_cast<Four<A>*>(smem_raw);  // b, then c: [TT][COPIES][LN]
  Step<A>* slots = reinterpret_cast<Step<A>*>(states + 2 * TT * COPIES * LN);  // [TT][CT]
  A* dps = reinterpret_cast<A*>(slots + TT * CT);                     // [TT][CT]
  A* joined = dps + TT * CT;                                          // [4 warps][TT][2][NP]
  A* sums = joined + 4 * TT * 2 * NP;                                 // [3][TT][PAD]: g b, p, a k
  Four<A>* params = reinterpret_cast<Four<A>*>(sums + 3 * TT * PAD);  // the threads' dt_bias and skip
  Four<A>* da = params + 256 + threadIdx.x;                           // theirs: [NC][128]

  const Place w = place_of<CT>(p, p.segments, 0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nl = lane % LN, dl = lane / LN;
  // The thread's channels of the tile and its 4 states: cl + (k ^ swap) and 4 nl + (j ^ order), by
  // its lane (fold_swapped); b and c stand in shared memory in every order.
  const int cl = (warp * LD + dl) * NC, swap = order_at<NC, LN>(nl), order = order_at<4, LD>(dl);
  constexpr int KEPT = NC < LN ? NC : LN, OTHERS = LN / KEPT;  // lanes that share out channels, tokens
  static_assert(KEPT == NC || LN == 1);
  const Four<A>* my_b = states + dl % COPIES * LN + nl;
  const Four<A>* my_c = my_b + TT * COPIES * LN;
  const Two<A> none = two(A(0), A(0));
  Two<A> ra[NC][2], r[NC][2];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const bool in = cl + (k ^ swap) < w.width;
    const int64_t d = w.d0 + cl + (k ^ swap);
    A q[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = nl * 4 + (j ^ order);
      q[j] = in && n < p.states ? rate(static_cast<const A*>(p.a)[d * p.states + n]) : A(0);
    }
    auto behind = [&] {  // the gradients of the last states
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = nl * 4 + (j ^ order);
        s[j] = in && n < p.states && p.d_final != nullptr
                   ? static_cast<const A*>(p.d_final)[(w.b * p.dim + d) * p.states + n]
                   : A(0);
      }
    };
    behind();
    if (in) {
      auto segment = [&](int g, auto by) {
        const int64_t row = (w.b * p.segments + g) * p.dim + d;
        return by(s, static_cast<const A*>(p.seg_sum)[row], q,
                  reorder(static_cast<const Four<A>*>(p.seg_state)[row * LN + nl], order));
      };
      // the segments after this one
      bool grows = false;
#pragma unroll 4
      for (int g = p.segments - 1; g > w.segment; --g) grows |= segment(g, carry<A>);
      if (grows) {
        behind();
        for (int g = p.segments - 1; g > w.segment; --g) segment(g, carry_growing<A>);
      }
    }
    ra[k][0] = two(q[0], q[1]), ra[k][1] = two(q[2], q[3]);
    r[k][0] = two(s[0], s[1]), r[k][1] = two(s[2], s[3]);
    da[k * 128] = {A(0), A(0), A(0), A(0)};
  }

  const int col = threadIdx.x % I::COLS * 4, row0 = threadIdx.x / I::COLS;
  const int have = w.width - col;
  const int64_t d0 = w.d0 + col;
  const int64_t steps = w.count > w.t0 ? (w.count - w.t0 + TT - 1) / TT : 0;
  const int64_t last = w.t0 + (steps - 1) * TT;  // the first token of the first step back in time
  // pointers of the thread's first token of a step
  const int64_t mine = last + row0;
  const T* px = static_cast<const T*>(p.x) + w.b * p.xs[0] + d0 + mine * p.xs[1];
  const T* pd = static_cast<const T*>(p.dt) + w.b * p.dts[0] + d0 + mine * p.dts[1];
  const T* pg = static_cast<const T*>(p.gate) + w.b * p.gs[0] + d0 + mine * p.gs[1];
  const T* pq = static_cast<const T*>(p.dy) + w.b * p.dys[0] + d0 + mine * p.dys[1];
  const int64_t to = w.b * p.length * p.dim + d0;
  T *ox = static_cast<T*>(p.dx) + to, *od = static_cast<T*>(p.ddt) + to,
    *og = static_cast<T*>(p.dgate) + to;
  // (the thread's own: in registers they would be eight that most of the step has no use for)
  params[threadIdx.x] = params4<A>(p.dt_bias, d0, have);
  params[128 + threadIdx.x] = params4<A>(p.skip, d0, have);
  const bool gated = p.gate != nullptr;
  Raw4<T> xr[I::IT], dr[I::IT], zr[I::IT], qr[I::IT];
  States<T, TT, LN, 2> bc;
  A dskip[4] = {A(0), A(0), A(0), A(0)}, dbias[4] = {A(0), A(0), A(0), A(0)};
  auto rows = [&](const T*& q, int64_t stride, Raw4<T>* raw, int left) {
#pragma unroll
    for (int i = 0; i < I::IT; ++i)
      raw[i] = load4(q + i * (I::ROWS * stride), i * I::ROWS < left ? have : 0, p.vec);
    q -= TT * stride;
  };
  // tokens from the thread's first one to the end of the valid ones and of the step
  auto left_at = [&](int64_t t) {
    return static_cast<int>((w.count - t < TT ? w.count - t : TT) - row0);
  };
  bc.start(p, w, p.b, p.bs, p.c, p.cs, last);
  auto fetch = [&](int64_t t) {
    const int left = left_at(t);
    rows(px, p.xs[1], xr, left);
    rows(pd, p.dts[1], dr, left);
    rows(pq, p.dys[1], qr, left);
    if (gated) rows(pg, p.gs[1], zr, left);
    bc.fetch(p, static_cast<int>(w.count - t < TT ? w.count - t : TT), -TT);
  };

  A* part_bc =
      static_cast<A*>(p.part_bc) + ((w.tile - p.tile0) * p.batch + w.b) * p.length * 2 * NP;
  {  // what lies after the valid tokens
    const A zero[4] = {A(0), A(0), A(0), A(0)};
    for (int64_t t = (w.count > w.t0 ? w.count : w.t0) + row0; t < w.t1; t += I::ROWS) {
      store4(ox + t * p.dim, zero, have, p.vec);
      store4(od + t * p.dim, zero, have, p.vec);
      if (gated) store4(og + t * p.dim, zero, have, p.vec);
    }
  }
  // of the step: the states kept before it, and the thread's results
  const Four<A>* kept = static_cast<const Four<A>*>(p.check) +
                        ((w.b * ((p.length + 7) / 8) + last / 8) * p.dim + w.d0 + cl) * LN + nl;
  int64_t result = mine * p.dim;
  part_bc += last * 2 * NP;
  Four<A> start[NC];
  auto fetch_start = [&] {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      start[k] = {A(0), A(0), A(0), A(0)};
      if (cl + (k ^ swap) < w.width) start[k] = kept[(k ^ swap) * LN];
    }
    kept -= p.dim * LN;
  };
  if (steps > 0) {
    fetch(last);
    fetch_start();
  }
  for (int64_t i = steps - 1; i >= 0; --i) {
    const int64_t t = w.t0 + i * TT;
    const int left = left_at(t);
    // kept for the results: x, the step's slope, dy silu'(gate)
    A xk[I::IT][4], slope[I::IT][4], opening[I::IT][4];
#pragma unroll
    for (int q = 0; q < I::IT; ++q) {
      const int row = row0 + q * I::ROWS;
      if (I::ROWS * I::IT > TT && row >= TT) break;
      const Four<A> bias = params[threadIdx.x];
      Four<A> dp;
      A delta[4];
      Quad<T>::values(xr[q], xk[q]);
      Quad<T>::values(dr[q], delta);
      Quad<T>::values(qr[q], dp.v);
#pragma unroll
      for (int j = 0; j < 4; ++j) delta[j] += bias.v[j], slope[q][j] = A(1);
      if (p.softplus) softplus<true>(delta, delta, slope[q]);
      if (q * I::ROWS >= left) {  // (x and dy are zero there)
#pragma unroll
        for (int j = 0; j < 4; ++j) delta[j] = A(0);
      }
      if (gated) {
        A z[4], g[4];
        Quad<T>::values(zr[q], z);
        sigmoid_at<false>(z, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          opening[q][j] = dp.v[j] * (g[j] * (A(1) + z[j] * (A(1) - g[j])));
          dp.v[j] *= z[j] * g[j];
        }
      }
      Step<A> out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = {delta[j], delta[j] * xk[q][j]};
      Four<A>* st = reinterpret_cast<Four<A>*>(slots + row * CT + col);
      st[0] = {out[0].delta, out[0].u, out[1].delta, out[1].u};
      st[1] = {out[2].delta, out[2].u, out[3].delta, out[3].u};
      *reinterpret_cast<Four<A>*>(dps + row * CT + col) = dp;
    }
    bc.template store_orders<COPIES>(states);
    if (i > 0) fetch(t - TT);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NC; ++k) start[k] = reorder(start[k], order);
    Two<A> dat[NC][2];
#pragma unroll
    for (int k = 0; k < NC; ++k) dat[k][0] = dat[k][1] = none;
#pragma unroll
    for (int half = 1; half >= 0; --half) {
      Two<A> h[SUB + 1][NC][2], e[SUB][NC][2];
#pragma unroll
      for (int k = 0; k < NC; ++k) h[0][k][0] = low(start[k]), h[0][k][1] = high(start[k]);
      if (half) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          const Four<A> bq = my_b[u * COPIES * LN];
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            const Step<A> st = slots[u * CT + cl + (k ^ swap)];
            const Two<A> d2 = two(st.delta, st.delta), u2 = two(st.u, st.u);
            h[0][k][0] = fma(exp_2(fma(d2, ra[k][0], lift2<A>())), h[0][k][0], mul(u2, low(bq)));
            h[0][k][1] = fma(exp_2(fma(d2, ra[k][1], lift2<A>())), h[0][k][1], mul(u2, high(bq)));
          }
        }
      }
      const int base = half * SUB;
      Four<A> bq[SUB];
      Step<A> st[SUB][NC];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        bq[u] = my_b[(base + u) * COPIES * LN];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          st[u][k] = slots[(base + u) * CT + cl + (k ^ swap)];
          const Two<A> d2 = two(st[u][k].delta, st[u][k].delta), u2 = two(st[u][k].u, st[u][k].u);
          e[u][k][0] = exp_2(fma(d2, ra[k][0], lift2<A>()));
          e[u][k][1] = exp_2(fma(d2, ra[k][1], lift2<A>()));
          h[u + 1][k][0] = fma(e[u][k][0], h[u][k][0], mul(u2, low(bq[u])));
          h[u + 1][k][1] = fma(e[u][k][1], h[u][k][1], mul(u2, high(bq[u])));
        }
      }
      // (from here on nothing needs these; the next step's are there when it does)
      if (half == 0 && i > 0) fetch_start();
      // sums over states and channels: each token's own first steps at once, so that few values live
      constexpr int LEFT = 4 / COPIES;  // states of each run (token, b or c) that a lane keeps
      A through[SUB], pre[SUB], by_rate[SUB], v[SUB * 2 * LEFT];
#pragma unroll
      for (int u = SUB - 1; u >= 0; --u) {
        const Four<A> cq = my_c[(base + u) * COPIES * LN];
        A dp[NC];
#pragma unroll
        for (int k = 0; k < NC; ++k) dp[k] = dps[(base + u) * CT + cl + (k ^ swap)];
        Two<A> db[2], dc[2];
        A over[3][NC];
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const Two<A> q2 = two(dp[k], dp[k]), d2 = two(st[u][k].delta, st[u][k].delta),
                       u2 = two(st[u][k].u, st[u][k].u);
          Two<A> g[2], kp[2];
          const Two<A> bb[2] = {low(bq[u]), high(bq[u])}, cc[2] = {low(cq), high(cq)};
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            g[m] = fma(cc[m], q2, r[k][m]);
            db[m] = k == 0 ? mul(u2, g[m]) : fma(u2, g[m], db[m]);
            dc[m] = k == 0 ? mul(q2, h[u + 1][k][m]) : fma(q2, h[u + 1][k][m], dc[m]);
            r[k][m] = mul(e[u][k][m], g[m]);
            kp[m] = mul(r[k][m], h[u][k][m]);
            dat[k][m] = fma(d2, kp[m], dat[k][m]);
          }
          const Two<A> tb = fma(g[1], bb[1], mul(g[0], bb[0]));
          const Two<A> tc = fma(h[u + 1][k][1], cc[1], mul(h[u + 1][k][0], cc[0]));
          const Two<A> ta = fma(ra[k][1], kp[1], mul(ra[k][0], kp[0]));
          over[0][k] = first(tb) + second(tb);
          over[1][k] = first(tc) + second(tc);
          over[2][k] = first(ta) + second(ta);
        }
        fold_swapped<3, NC, LN, 1>(&over[0][0]);
        through[u] = over[0][0], pre[u] = (&over[0][0])[1], by_rate[u] = (&over[0][0])[2];
        A runs[8] = {first(db[0]), second(db[0]), first(db[1]), second(db[1]),
                     first(dc[0]), second(dc[0]), first(dc[1]), second(dc[1])};
        fold_swapped<2, 4, LD, LN>(runs);
#pragma unroll
        for (int o = 0; o < 2 * LEFT; ++o) v[u * 2 * LEFT + o] = runs[o];
      }
      fold<SUB, OTHERS, KEPT>(through, lane);
      fold<SUB, OTHERS, KEPT>(pre, lane);
      fold<SUB, OTHERS, KEPT>(by_rate, lane);
      constexpr int OWN = SUB >= OTHERS ? SUB / OTHERS : 1, SAME = OTHERS > SUB ? OTHERS / SUB : 1;
#pragma unroll
      for (int o = 0; o < OWN; ++o) {
        A* q = sums + (base + nl / KEPT / SAME * OWN + o) * PAD + cl + (LN == 1 ? 0 : swap);
        q[0] = through[o];
        q[TT * PAD] = pre[o];
        q[2 * TT * PAD] = by_rate[o];
      }
      constexpr int FAR = LD / COPIES;           // lanes that share out the runs
      fold<SUB * 2, FAR, LN * COPIES>(v, lane);  // (FAR > 1 only where LEFT is 1)
      constexpr int RUNS = SUB * 2 / FAR;
#pragma unroll
      for (int o = 0; o < RUNS; ++o) {
        const int run = dl / COPIES * RUNS + o;
        A* q = joined + ((warp * TT + base) * 2 + run) * NP + nl * 4;
#pragma unroll
        for (int j = 0; j < LEFT; ++j) q[j ^ order] = v[o * LEFT + j];
      }
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      Four<A> sum = da[k * 128];
      sum = {sum.v[0] + first(dat[k][0]), sum.v[1] + second(dat[k][0]),
             sum.v[2] + first(dat[k][1]), sum.v[3] + second(dat[k][1])};
      da[k * 128] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < I::IT; ++q) {
      const int row = row0 + q * I::ROWS;
      if (q * I::ROWS >= left) break;
      const Four<A> th = *reinterpret_cast<const Four<A>*>(sums + row * PAD + col);
      const Four<A> pr = *reinterpret_cast<const Four<A>*>(sums + (TT + row) * PAD + col);
      const Four<A> br = *reinterpret_cast<const Four<A>*>(sums + (2 * TT + row) * PAD + col);
      const Four<A> dp = *reinterpret_cast<const Four<A>*>(dps + row * CT + col);
      const Four<A>* st = reinterpret_cast<const Four<A>*>(slots + row * CT + col);
      const Four<A> s0 = st[0], s1 = st[1];
      const A delta[4] = {s0.v[0], s0.v[2], s1.v[0], s1.v[2]};
      const Four<A> skip = params[128 + threadIdx.x];
      A gx[4], gd[4], gg[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        gx[j] = delta[j] * th.v[j] + skip.v[j] * dp.v[j];
        gd[j] = (A(kLn2) * br.v[j] + xk[q][j] * th.v[j]) * slope[q][j];
        gg[j] = opening[q][j] * (pr.v[j] + skip.v[j] * xk[q][j]);
        dskip[j] += dp.v[j] * xk[q][j];
        dbias[j] += gd[j];
      }
      const int64_t at = result + q * (I::ROWS * p.dim);
      store4(ox + at, gx, have, p.vec);
      store4(od + at, gd, have, p.vec);
      if (gated) store4(og + at, gg, have, p.vec);
    }
    result -= TT * p.dim;
    // (tokens past the valid ones have no part: scan_bc_kernel leaves them out)
    for (int e = p.part_bc != nullptr ? threadIdx.x : TT * 2 * LN; e < TT * 2 * LN; e += 128) {
      if (e / (2 * LN) >= left + row0) continue;
      Four<A> s = reinterpret_cast<const Four<A>*>(joined)[e];
#pragma unroll
      for (int q = 1; q < 4; ++q) {
        const Four<A> f = reinterpret_cast<const Four<A>*>(joined)[q * TT * 2 * LN + e];
#pragma unroll
        for (int j = 0; j < 4; ++j) s.v[j] += f.v[j];
      }
      reinterpret_cast<Four<A>*>(part_bc)[e] = s;
    }
    part_bc -= TT * 2 * NP;
    __syncthreads();
  }

  const int64_t row = w.b * p.segments + w.segment;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = cl + (k ^ swap);
    if (c >= w.width) continue;
    const int64_t d = w.d0 + c;
    static_cast<Four<A>*>(p.part_a)[(row * p.dim + d) * LN + nl] = reorder(da[k * 128], order);
    if (w.segment == 0 && p.d_initial != nullptr) {
      const A s[4] = {first(r[k][0]), second(r[k][0]), first(r[k][1]), second(r[k][1])};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = nl * 4 + (j ^ order);
        if (n < p.states) static_cast<A*>(p.d_initial)[(w.b * p.dim + d) * p.states + n] = s[j];
      }
    }
  }
  // dskip and ddt_bias over the block's tokens, in the order of the threads' rows
  constexpr int ROWS = I::ROWS < TT ? I::ROWS : TT;
  A* shares = sums;  // [2][ROWS][CT]
  if (row0 < ROWS) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      shares[row0 * CT + col + j] = dskip[j];
      shares[(ROWS + row0) * CT + col + j] = dbias[j];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * CT; e += 128) {
    const int which = e / CT, c = e % CT;
    if (c >= w.width) continue;
    A s = A(0);
#pragma unroll
    for (int u = 0; u < ROWS; ++u) s += shares[(which * ROWS + u) * CT + c];
    static_cast<A*>(p.part_ch)[(row * 2 + which) * p.dim + w.d0 + c] = s;
  }
}
template <typename A> constexpr size_t scan_bwd_smem(int ln, int nc) {
  const size_t ct = 4 * (32 / ln) * nc, np = 4 * ln, tt = kScanCheck;
  const size_t copies = 32 / ln < 4 ? 32 / ln : 4;
  return sizeof(A) * (2 * tt * np * copies + 3 * tt * ct + 4 * tt * 2 * np + 3 * tt * (ct + 8) +
                      (2 + nc) * 4 * 128);
}

// ------------------------------------------------------------------------------ single tokens
// One token of every sequence: a pass over the states, read and written once.  A thread takes 4 states
// of a channel in SEQ sequences (at most LN), whose loads are in flight together and share the
// rates.  The LN lanes of a channel share out the sequences' steps and gates, and hand them round.
template <typename T, int LN, int SEQ, bool WHOLE>
__global__ void __launch_bounds__(128)
scan_step_kernel(const __grid_constant__ ScanArgs p, const int32_t* __restrict__ slots,
                 int64_t pool, typename AccOf<T>::type* state) {
  using A = typename AccOf<T>::type;
  static_assert(SEQ <= LN);
  constexpr int CW = 128 / LN;  // channels of a block
  const unsigned dim = static_cast<unsigned>(p.dim), blocks = (dim + CW - 1) / CW;
  const int64_t b0 = int64_t(blockIdx.x / blocks) * SEQ;
  const int lane = threadIdx.x & 31, nl = lane % LN, n0 = nl * 4;
  unsigned d = blockIdx.x % blocks * CW + threadIdx.x / LN;
  const bool in = d < dim;
  if (!in) d = dim - 1;  // the lanes of a warp stay together
  const unsigned group = p.groups == 1 ? 0 : d / static_cast<unsigned>(p.per);
  const int have = WHOLE ? 4 : p.states - n0;
  const bool whole = WHOLE || (p.vec && have > 0), vec = WHOLE || p.vec;
  const bool vec_states = WHOLE || p.vec_states;

  // the lane's own sequence of them
  constexpr int SAME = LN / SEQ;
  const int64_t own = b0 + nl / SAME;
  int own_slot = -1;
  if (own < p.batch) {
    const int64_t slot = slots == nullptr ? own : slots[own];
    if (slot >= 0 && slot < pool) own_slot = static_cast<int>(slot);
  }
  A x = A(0), dt = A(0), z = A(0);
  if (own_slot >= 0) {
    x = to_acc(static_cast<const T*>(p.x)[own * p.xs[0] + d]);
    dt = to_acc(static_cast<const T*>(p.dt)[own * p.dts[0] + d]);
    if (p.gate != nullptr) z = to_acc(static_cast<const T*>(p.gate)[own * p.gs[0] + d]);
  }
  const int64_t row = p.dim * p.states;
  A* first_state = state + (int64_t(d) * p.states + n0);
  A* ps[SEQ];
  Four<A> h[SEQ];
  Raw4<T> rb[SEQ], rc[SEQ];
  const T* pb = static_cast<const T*>(p.b) + b0 * p.bs[0] + group * p.bs[2] + n0;
  const T* pc = static_cast<const T*>(p.c) + b0 * p.cs[0] + group * p.cs[2] + n0;
#pragma unroll
  for (int i = 0; i < SEQ; ++i, pb += p.bs[0], pc += p.cs[0]) {
    const int slot = SEQ == 1 ? own_slot : __shfl_sync(0xffffffffu, own_slot, i * SAME, LN);
    ps[i] = nullptr;
    if (slot < 0) continue;
    ps[i] = first_state + slot * row;
    h[i] = {A(0), A(0), A(0), A(0)};
    if (whole) h[i] = *reinterpret_cast<const Four<A>*>(ps[i]);
    else if (!vec) h[i] = params4<A>(ps[i], 0, have);
    rb[i] = load4(pb, have, vec_states);
    rc[i] = load4(pc, have, vec_states);
  }
  Four<A> r = {A(0), A(0), A(0), A(0)};
  const A* pa = static_cast<const A*>(p.a) + int64_t(d) * p.states + n0;
  if (whole) r = *reinterpret_cast<const Four<A>*>(pa);
  else if (!vec) r = params4<A>(pa, 0, have);
#pragma unroll
  for (int j = 0; j < 4; ++j) r.v[j] = rate(r.v[j]);

  A delta = dt;
  if (p.dt_bias != nullptr) delta += static_cast<const A*>(p.dt_bias)[d];
  if (p.softplus) delta = softplus(delta);
  const A u = delta * x;
  A y[SEQ];
#pragma unroll
  for (int i = 0; i < SEQ; ++i) {
    const A di = SEQ == 1 ? delta : __shfl_sync(0xffffffffu, delta, i * SAME, LN);
    const A ui = SEQ == 1 ? u : __shfl_sync(0xffffffffu, u, i * SAME, LN);
    y[i] = A(0);
    if (ps[i] == nullptr) continue;
    A vb[4], vc[4];
    Quad<T>::values(rb[i], vb);
    Quad<T>::values(rc[i], vc);
    const Two<A> d2 = two(di, di), u2 = two(ui, ui);
    const Two<A> h0 = fma(exp_2(fma(d2, low(r), lift2<A>())), low(h[i]), mul(u2, two(vb[0], vb[1])));
    const Two<A> h1 = fma(exp_2(fma(d2, high(r), lift2<A>())), high(h[i]), mul(u2, two(vb[2], vb[3])));
    const Two<A> sum = fma(h1, two(vc[2], vc[3]), mul(h0, two(vc[0], vc[1])));
    y[i] = first(sum) + second(sum);
    h[i] = {first(h0), second(h0), first(h1), second(h1)};
    if (!in) continue;
    if (whole) {
      *reinterpret_cast<Four<A>*>(ps[i]) = h[i];
    } else if (!vec) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < have) ps[i][j] = h[i].v[j];
    }
  }
  fold<SEQ, LN, 1>(y, lane);
  if (!in || nl % SAME != 0 || own >= p.batch) return;
  A out = A(0);
  if (own_slot >= 0) {
    out = y[0];
    if (p.skip != nullptr) out += static_cast<const A*>(p.skip)[d] * x;
    if (p.gate != nullptr) {
      const A zs[4] = {z, z, z, z};
      A g[4];
      sigmoid_at<sizeof(T) == 2>(zs, g);
      out *= z * g[0];
    }
  }
  static_cast<T*>(p.y)[own * p.dim + d] = from_acc<T>(out);
}

// ------------------------------------------------------------------------------ launches
template <typename F> int with_lanes(int lanes, F fn) {
  switch (lanes) {
    case 1: return fn(std::integral_constant<int, 1>{});
    case 2: return fn(std::integral_constant<int, 2>{});
    case 4: return fn(std::integral_constant<int, 4>{});
    case 8: return fn(std::integral_constant<int, 8>{});
    case 16: return fn(std::integral_constant<int, 16>{});
    case 32: return fn(std::integral_constant<int, 32>{});
    default: return FDWT_ERR_INVALID;
  }
}
inline int scan_grid(const ScanArgs& p, int segments, unsigned* grid) {
  const int64_t blocks = p.tile_count * segments * p.batch;
  if (blocks > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  *grid = static_cast<unsigned>(blocks);
  return FDWT_OK;
}

template <typename T, int MODE> int scan_launch(const ScanArgs& p, int lanes, cudaStream_t stream) {
  return with_lanes(lanes, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    unsigned grid;
    int st = scan_grid(p, MODE == MAIN ? p.segments : p.segments - 1, &grid);
    if (st == FDWT_OK) st = pre_launch(stream);
    if (st != FDWT_OK) return st;
    scan_fwd_kernel<T, LN, scan_fwd_channels(LN), MODE><<<grid, 128, 0, stream>>>(p);
    return launch_status();
  });
}

}  // namespace

template <typename T> int scan_forward(const ScanArgs& p, int lanes, cudaStream_t stream) {
  return scan_launch<T, MAIN>(p, lanes, stream);
}
template <typename T>
int scan_states(const ScanArgs& p, int lanes, bool reverse, cudaStream_t stream) {
  return reverse ? scan_launch<T, REVERSE>(p, lanes, stream) : scan_launch<T, STATES>(p, lanes, stream);
}

template <typename T> int scan_backward(const ScanArgs& p, int lanes, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  return with_lanes(lanes, [&](auto ln) {
    constexpr int LN = decltype(ln)::value, NC = scan_bwd_channels(LN, sizeof(A) == 8);
    auto kernel = scan_bwd_kernel<T, LN, NC>;
    unsigned grid;
    int st = scan_grid(p, p.segments, &grid);
    if (st == FDWT_OK) st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
    if (st == FDWT_OK) st = pre_launch(stream);
    if (st != FDWT_OK) return st;
    kernel<<<grid, 128, scan_bwd_smem<A>(LN, NC), stream>>>(p);
    return launch_status();
  });
}

template <typename T> int64_t scan_resident(int lanes, bool backward) {
  using A = typename AccOf<T>::type;
  int blocks = 1;
  with_lanes(lanes, [&](auto ln) {
    constexpr int LN = decltype(ln)::value, NC = scan_bwd_channels(LN, sizeof(A) == 8);
    if (!backward)
      return occupancy(reinterpret_cast<const void*>(
                           scan_fwd_kernel<T, LN, scan_fwd_channels(LN), MAIN>), 128, 0, &blocks);
    const void* kernel = reinterpret_cast<const void*>(scan_bwd_kernel<T, LN, NC>);
    const int st = allow_max_dynamic_smem(kernel);
    return st != FDWT_OK ? st : occupancy(kernel, 128, scan_bwd_smem<A>(LN, NC), &blocks);
  });
  return int64_t(blocks < 1 ? 1 : blocks) * sm_count();
}

template <typename T>
int scan_step(const ScanArgs& p, int lanes, const int32_t* slots, int64_t pool, void* state,
              cudaStream_t stream) {
  return with_lanes(lanes, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    auto launch = [&](auto seq) {
      constexpr int SEQ = decltype(seq)::value;
      const int64_t grid = cdiv(p.batch, SEQ) * cdiv(p.dim, 128 / LN);
      if (grid > INT32_MAX) return static_cast<int>(FDWT_ERR_UNSUPPORTED);
      const int st = pre_launch(stream);
      if (st != FDWT_OK) return st;
      auto kernel = scan_step_kernel<T, LN, SEQ, false>;
      // (without the conditions that other sizes need: 240 x 2048 of 16 states 15.4 us, with them 17)
      if (p.vec && p.vec_states && p.states == 4 * LN) kernel = scan_step_kernel<T, LN, SEQ, true>;
      kernel<<<static_cast<unsigned>(grid), 128, 0, stream>>>(
          p, slots, pool, static_cast<typename AccOf<T>::type*>(state));
      return launch_status();
    };
    // several sequences a thread where there are blocks enough
    constexpr int MOST = LN < 4 ? LN : 4;
    if (p.batch * cdiv(p.dim, 128 / LN) >= int64_t(sm_count()) * 4 * MOST)
      return launch(std::integral_constant<int, MOST>{});
    return launch(std::integral_constant<int, 1>{});
  });
}

#define FDWT_SCAN_TYPE(T)                                                            \
  template int scan_forward<T>(const ScanArgs&, int, cudaStream_t);                  \
  template int scan_states<T>(const ScanArgs&, int, bool, cudaStream_t);             \
  template int scan_backward<T>(const ScanArgs&, int, cudaStream_t);                 \
  template int64_t scan_resident<T>(int, bool);                                      \
  template int scan_step<T>(const ScanArgs&, int, const int32_t*, int64_t, void*, cudaStream_t);

}  // namespace fdwt
