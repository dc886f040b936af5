// Kernels of the selective state space scan (selscan.cuh has the formulas and the split).
#pragma once

#include <cfloat>

#include "selscan.cuh"

namespace fdwt {
namespace {

// ------------------------------------------------------------------------------ arithmetic
// Two neighbouring states: packed instructions for 32 bits.
template <typename A> struct Two;
template <> struct Two<float> {
  unsigned long long v;
};
template <> struct Two<double> {
  double x, y;
};
template <typename A> struct alignas(4 * sizeof(A)) Four {
  A v[4];
};

__device__ __forceinline__ Two<float> two(float x, float y) {
  Two<float> r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ Two<double> two(double x, double y) { return {x, y}; }
__device__ __forceinline__ float first(Two<float> a) {
  float x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v));
  return x;
}
__device__ __forceinline__ float second(Two<float> a) {
  float x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v));
  return y;
}
__device__ __forceinline__ double first(Two<double> a) { return a.x; }
__device__ __forceinline__ double second(Two<double> a) { return a.y; }
__device__ __forceinline__ Two<float> mul(Two<float> a, Two<float> b) {
  Two<float> r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two<double> mul(Two<double> a, Two<double> b) {
  return {a.x * b.x, a.y * b.y};
}
__device__ __forceinline__ Two<float> add(Two<float> a, Two<float> b) {
  Two<float> r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two<double> add(Two<double> a, Two<double> b) {
  return {a.x + b.x, a.y + b.y};
}
__device__ __forceinline__ Two<float> fma(Two<float> a, Two<float> b, Two<float> c) {
  Two<float> r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two<double> fma(Two<double> a, Two<double> b, Two<double> c) {
  return {::fma(a.x, b.x, c.x), ::fma(a.y, b.y, c.y)};
}
template <typename A> __device__ __forceinline__ Two<A> low(const Four<A>& q) {
  return two(q.v[0], q.v[1]);
}
template <typename A> __device__ __forceinline__ Two<A> high(const Four<A>& q) {
  return two(q.v[2], q.v[3]);
}

// 2^x: rates are kept times log2 e.
__device__ __forceinline__ float exp_2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ double exp_2(double x) { return exp2(x); }
template <typename A> __device__ __forceinline__ Two<A> exp_2(Two<A> x) {
  return two(exp_2(first(x)), exp_2(second(x)));
}
constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

// log(1 + e^v), to the last bits where it is small too: steps are often 1e-3.
__device__ __forceinline__ float softplus(float v) {
  return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v)));
}
__device__ __forceinline__ double softplus(double v) {
  return fmax(v, 0.0) + log1p(exp(-fabs(v)));
}
// 1 / (1 + e^-v): of a few roundings' error for rows of 32 bits and where the result stays in 32
// bits (EXACT), by the fast exponential and division where it is rounded to 16.
template <typename T, bool EXACT, typename A> __device__ __forceinline__ A sigmoid_at(A v) {
  if constexpr (sizeof(T) == 8) return 1.0 / (1.0 + exp(-v));
  else if constexpr (sizeof(T) == 4 || EXACT) return 1.0f / (1.0f + expf(-v));
  else return __fdividef(1.0f, 1.0f + __expf(-v));
}

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

__device__ __forceinline__ int64_t valid_tokens(const ScanArgs& p, int64_t b) {
  if (p.lengths == nullptr) return p.length;
  const int64_t n = p.lengths[b];
  return n < 0 ? 0 : (n < p.length ? n : p.length);
}

// Slots of a token's channels are staged by threads of 8 neighbouring ones and read by lanes of
// neighbouring ones: the order within 8 goes by the place of the 8, so that both reach all banks.
__device__ __forceinline__ int slot_of(int c) { return c ^ ((c >> 3) & 7); }

// What a block works on.
struct Place {
  int64_t b, t0, t1, count;  // sequence, its segment's tokens, valid tokens of the sequence
  int64_t d0;                // first channel
  int group, segment, tile, width;  // width: channels of the tile
};
template <int CT> __device__ __forceinline__ Place place_of(const ScanArgs& p) {
  Place w;
  const int64_t tiles = p.tiles * p.groups;
  const int64_t id = blockIdx.x;
  w.tile = static_cast<int>(id % tiles);
  w.segment = static_cast<int>(id / tiles % p.segments);
  w.b = id / tiles / p.segments;
  w.group = static_cast<int>(w.tile / p.tiles);
  const int64_t within = (w.tile % p.tiles) * CT;
  w.d0 = w.group * p.per + within;
  w.width = static_cast<int>(p.per - within < CT ? p.per - within : CT);
  w.t0 = w.segment * p.seg_len;
  w.t1 = w.t0 + p.seg_len < p.length ? w.t0 + p.seg_len : p.length;
  w.count = valid_tokens(p, w.b);
  return w;
}

// Rows of b or c: TT tokens from t on, in 32 bits, zeros past the states and the valid tokens.
template <typename T, int TT, int NP, typename A>
__device__ __forceinline__ void stage_states(const ScanArgs& p, const Place& w, const void* src,
                                             const int64_t* stride, int64_t t, A* out) {
  const T* q = static_cast<const T*>(src) + w.b * stride[0] + w.group * stride[2];
  for (int e = threadIdx.x; e < TT * NP; e += 128) {
    const int n = e % NP;
    const int64_t at = t + e / NP;
    out[e] = n < p.states && at < w.count ? to_acc(q[at * stride[1] + n]) : A(0);
  }
}

// ------------------------------------------------------------------------------ forward
// MAIN: outputs and last states.  STATES: a segment's end state from zero, and its sum of delta.
// REVERSE: the same back in time for the gradients, r = e^(delta a) (c dp + r).
enum ScanMode { MAIN, STATES, REVERSE };
template <typename A> constexpr int scan_fwd_tokens() { return sizeof(A) == 8 ? 8 : 16; }

template <typename T, int LN, int NC, int MODE>
__global__ void __launch_bounds__(128)
scan_fwd_kernel(const __grid_constant__ ScanArgs p) {
  using A = typename AccOf<T>::type;
  constexpr int LD = 32 / LN, CT = 4 * LD * NC, NP = 4 * LN, TT = scan_fwd_tokens<A>();
  constexpr int V = 16 / sizeof(T) < CT ? 16 / sizeof(T) : CT;
  constexpr int PAD = CT + 8;
  __shared__ Four<A> slots[TT * CT];           // delta, delta, delta x, delta x
  __shared__ Four<A> into[TT * LN], out[MODE == MAIN ? TT * LN : 1];  // b and c
  __shared__ A sums[MODE == MAIN ? TT * PAD : 1];
  const Place w = place_of<CT>(p);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nl = lane % LN, dl = lane / LN;
  const int cl = (warp * LD + dl) * NC;  // the thread's first channel of the tile
  const A* rates = static_cast<const A*>(p.a);

  Two<A> ra[NC][2], h[NC][2];
  A total[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    A r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = nl * 4 + j;
      r[j] = cl + k < w.width && n < p.states ? rate(rates[(w.d0 + cl + k) * p.states + n]) : A(0);
    }
    ra[k][0] = two(r[0], r[1]);
    ra[k][1] = two(r[2], r[3]);
    A s[4] = {A(0), A(0), A(0), A(0)};
    if (MODE == MAIN && cl + k < w.width) {
      const int64_t d = w.d0 + cl + k;
      if (p.initial != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (nl * 4 + j < p.states)
            s[j] = static_cast<const A*>(p.initial)[(w.b * p.dim + d) * p.states + nl * 4 + j];
      }
      // the segments before this one
      for (int g = 0; g < w.segment; ++g) {
        const int64_t row = (w.b * p.segments + g) * p.dim + d;
        const A sum = static_cast<const A*>(p.seg_sum)[row];
        const Four<A> e = static_cast<const Four<A>*>(p.seg_state)[row * LN + nl];
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = exp_2(sum * r[j]) * s[j] + e.v[j];
      }
    }
    h[k][0] = two(s[0], s[1]);
    h[k][1] = two(s[2], s[3]);
    total[k] = A(0);
  }

  const T* px = static_cast<const T*>(MODE == REVERSE ? p.dy : p.x) +
                w.b * (MODE == REVERSE ? p.dys[0] : p.xs[0]) + w.d0;
  const int64_t xs = MODE == REVERSE ? p.dys[1] : p.xs[1];
  const T* pd = static_cast<const T*>(p.dt) + w.b * p.dts[0] + w.d0;
  const T* pg = static_cast<const T*>(p.gate) + w.b * p.gs[0] + w.d0;
  const A* bias = static_cast<const A*>(p.dt_bias) + w.d0;
  const A* skip = static_cast<const A*>(p.skip) + w.d0;
  T* py = static_cast<T*>(p.y) + w.b * p.length * p.dim + w.d0;

  // G neighbouring channels of a token
  auto stage = [&](auto g, int64_t t, int at, int c, bool in) {
    constexpr int G = decltype(g)::value;
    A dt[G], x[G];
    if (in) {
      Group<T, G>::values(Group<T, G>::load(pd + t * p.dts[1] + c), dt);
      Group<T, G>::values(Group<T, G>::load(px + t * xs + c), x);
      if (MODE == REVERSE && p.gate != nullptr) {
        A z[G];
        Group<T, G>::values(Group<T, G>::load(pg + t * p.gs[1] + c), z);
#pragma unroll
        for (int j = 0; j < G; ++j) x[j] *= z[j] * sigmoid_at<T, true>(z[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      A delta = A(0), u = A(0);
      if (in) {
        delta = dt[j];
        if (p.dt_bias != nullptr) delta += bias[c + j];
        if (p.softplus) delta = softplus(delta);
        u = MODE == REVERSE ? x[j] : delta * x[j];
      }
      slots[at * CT + slot_of(c + j)] = {delta, delta, u, u};
    }
  };
  auto finish = [&](auto g, int64_t t, int at, int c) {
    constexpr int G = decltype(g)::value;
    A y[G];
    if (t < w.count) {
      A x[G], z[G];
      Group<T, G>::values(Group<T, G>::load(px + t * xs + c), x);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        y[j] = sums[at * PAD + c + j];
        if (p.skip != nullptr) y[j] += skip[c + j] * x[j];
      }
      if (p.gate != nullptr) {
        Group<T, G>::values(Group<T, G>::load(pg + t * p.gs[1] + c), z);
#pragma unroll
        for (int j = 0; j < G; ++j) y[j] *= z[j] * sigmoid_at<T, false>(z[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < G; ++j) y[j] = A(0);
    }
    Group<T, G>::store(py + t * p.dim + c, y);
  };
  // every (token, channels) of the staged tokens, by threads
  auto each = [&](auto fn) {
    if (p.vec) {
      for (int e = threadIdx.x; e < TT * (CT / V); e += 128)
        fn(std::integral_constant<int, V>{}, e / (CT / V), e % (CT / V) * V);
    } else {
      for (int e = threadIdx.x; e < TT * CT; e += 128)
        fn(std::integral_constant<int, 1>{}, e / CT, e % CT);
    }
  };

  const int64_t steps = w.t1 > w.t0 ? (w.t1 - w.t0 + TT - 1) / TT : 0;
  for (int64_t i = 0; i < steps; ++i) {
    const int64_t t = w.t0 + (MODE == REVERSE ? steps - 1 - i : i) * TT;
    if (t < w.count) {
      each([&](auto g, int at, int c) {
        stage(g, t + at, at, c, t + at < w.count && c < w.width);
      });
      stage_states<T, TT, NP>(p, w, MODE == REVERSE ? p.c : p.b, MODE == REVERSE ? p.cs : p.bs, t,
                              &into[0].v[0]);
      if constexpr (MODE == MAIN) stage_states<T, TT, NP>(p, w, p.c, p.cs, t, &out[0].v[0]);
      __syncthreads();
#pragma unroll 1
      for (int s = 0; s < TT; s += 8) {
        if (MODE == MAIN && p.check != nullptr && t + s < p.length) {
          const int64_t row = (w.b * ((p.length + 7) / 8) + (t + s) / 8) * p.dim + w.d0 + cl;
#pragma unroll
          for (int k = 0; k < NC; ++k)
            if (cl + k < w.width)
              static_cast<Four<A>*>(p.check)[(row + k) * LN + nl] = {
                  first(h[k][0]), second(h[k][0]), first(h[k][1]), second(h[k][1])};
        }
        A y[8 * NC];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int row = MODE == REVERSE ? TT - 1 - s - u : s + u;
          const Four<A> bq = into[row * LN + nl];
          Four<A> cq;
          if constexpr (MODE == MAIN) cq = out[row * LN + nl];
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            const Four<A> q = slots[row * CT + slot_of(cl + k)];
            const Two<A> d2 = low(q), u2 = high(q);
            const Two<A> e0 = exp_2(mul(d2, ra[k][0])), e1 = exp_2(mul(d2, ra[k][1]));
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
              total[k] += first(d2);
            }
          }
        }
        if constexpr (MODE == MAIN) {
          fold<8 * NC, LN, 1>(y, lane);
          constexpr int OWN = 8 * NC / LN;
#pragma unroll
          for (int o = 0; o < OWN; ++o) {
            const int v = nl * OWN + o;
            sums[(s + v / NC) * PAD + cl + v % NC] = y[o];
          }
        }
      }
      __syncthreads();
    }
    if constexpr (MODE == MAIN) {
      each([&](auto g, int at, int c) {
        if (t + at < w.t1 && c < w.width) finish(g, t + at, at, c);
      });
    }
  }

  if constexpr (MODE == MAIN) {
    if (w.segment != p.segments - 1 || p.final_state == nullptr) return;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const A s[4] = {first(h[k][0]), second(h[k][0]), first(h[k][1]), second(h[k][1])};
      A* to = static_cast<A*>(p.final_state) + (w.b * p.dim + w.d0 + cl + k) * p.states;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (cl + k < w.width && nl * 4 + j < p.states) to[nl * 4 + j] = s[j];
    }
  } else {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      if (cl + k >= w.width) continue;
      const int64_t row = (w.b * p.segments + w.segment) * p.dim + w.d0 + cl + k;
      static_cast<Four<A>*>(p.seg_state)[row * LN + nl] = {first(h[k][0]), second(h[k][0]),
                                                           first(h[k][1]), second(h[k][1])};
      if (nl == 0) static_cast<A*>(p.seg_sum)[row] = total[k];
    }
  }
}

// ------------------------------------------------------------------------------ backward
// A block walks its segment back in time, 8 tokens at a time.  From the state that the forward pass
// kept before them a thread forms its states and decays of the 8 tokens again and keeps them in
// registers, then goes back over them.  It does so for KC channels one after the other: their
// shares of db and dc add up in registers, and cross the lanes once for all of them.
template <typename T, int LN, int KC>
__global__ void __launch_bounds__(128)
scan_bwd_kernel(const __grid_constant__ ScanArgs p) {
  using A = typename AccOf<T>::type;
  constexpr int LD = 32 / LN, CT = 4 * LD * KC, NP = 4 * LN, TT = kScanCheck;
  constexpr int V = 16 / sizeof(T) < CT ? 16 / sizeof(T) : CT;
  constexpr int PAD = CT + 8;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Four<A>* slots = reinterpret_cast<Four<A>*>(smem_raw);  // delta, delta, delta x, delta x
  Four<A>* mine = slots + TT * CT;                        // [3][KC][128]: rates, r, da
  Four<A>* into = mine + 3 * KC * 128;                    // b
  Four<A>* from = into + TT * LN;                         // c
  A* joined = reinterpret_cast<A*>(from + TT * LN);       // [4 warps][TT][2][NP]
  A* dps = joined + 4 * TT * 2 * NP;                      // [TT][CT]
  A* sums = dps + TT * CT;                                // [3][TT][PAD]: g b, p, a k
  A* params = sums + 3 * TT * PAD;                        // [2][TT][CT]: dskip, ddt_bias

  const Place w = place_of<CT>(p);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nl = lane % LN, dl = lane / LN;
  const int c0 = warp * LD * KC + dl;  // the thread's channels: c0, c0 + LD, ...
  for (int k = 0; k < KC; ++k) {
    const int c = c0 + k * LD;
    const bool in = c < w.width;
    const int64_t d = w.d0 + c;
    Four<A> r, s = {A(0), A(0), A(0), A(0)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = nl * 4 + j;
      const bool live = in && n < p.states;
      r.v[j] = live ? rate(static_cast<const A*>(p.a)[d * p.states + n]) : A(0);
      if (live && p.d_final != nullptr)
        s.v[j] = static_cast<const A*>(p.d_final)[(w.b * p.dim + d) * p.states + n];
    }
    if (in) {
      for (int g = p.segments - 1; g > w.segment; --g) {  // the segments after this one
        const int64_t row = (w.b * p.segments + g) * p.dim + d;
        const A sum = static_cast<const A*>(p.seg_sum)[row];
        const Four<A> e = static_cast<const Four<A>*>(p.seg_state)[row * LN + nl];
#pragma unroll
        for (int j = 0; j < 4; ++j) s.v[j] = exp_2(sum * r.v[j]) * s.v[j] + e.v[j];
      }
    }
    mine[(0 * KC + k) * 128 + threadIdx.x] = r;
    mine[(1 * KC + k) * 128 + threadIdx.x] = s;
    mine[(2 * KC + k) * 128 + threadIdx.x] = {A(0), A(0), A(0), A(0)};
  }
  for (int e = threadIdx.x; e < 2 * TT * CT; e += 128) params[e] = A(0);

  const T* px = static_cast<const T*>(p.x) + w.b * p.xs[0] + w.d0;
  const T* pd = static_cast<const T*>(p.dt) + w.b * p.dts[0] + w.d0;
  const T* pg = static_cast<const T*>(p.gate) + w.b * p.gs[0] + w.d0;
  const T* pq = static_cast<const T*>(p.dy) + w.b * p.dys[0] + w.d0;
  const A* bias = static_cast<const A*>(p.dt_bias) + w.d0;
  const A* skip = static_cast<const A*>(p.skip) + w.d0;
  const int64_t to = w.b * p.length * p.dim + w.d0;
  T *ox = static_cast<T*>(p.dx) + to, *od = static_cast<T*>(p.ddt) + to,
    *og = static_cast<T*>(p.dgate) + to;

  auto stage = [&](auto g, int64_t t, int at, int c, bool in) {
    constexpr int G = decltype(g)::value;
    A dt[G], x[G], dp[G];
    if (in) {
      Group<T, G>::values(Group<T, G>::load(pd + t * p.dts[1] + c), dt);
      Group<T, G>::values(Group<T, G>::load(px + t * p.xs[1] + c), x);
      Group<T, G>::values(Group<T, G>::load(pq + t * p.dys[1] + c), dp);
      if (p.gate != nullptr) {
        A z[G];
        Group<T, G>::values(Group<T, G>::load(pg + t * p.gs[1] + c), z);
#pragma unroll
        for (int j = 0; j < G; ++j) dp[j] *= z[j] * sigmoid_at<T, true>(z[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < G; ++j) {
      A delta = A(0), u = A(0), q = A(0);
      if (in) {
        delta = dt[j];
        if (p.dt_bias != nullptr) delta += bias[c + j];
        if (p.softplus) delta = softplus(delta);
        u = delta * x[j];
        q = dp[j];
      }
      slots[at * CT + slot_of(c + j)] = {delta, delta, u, u};
      dps[at * CT + c + j] = q;
    }
  };
  auto finish = [&](auto g, int64_t t, int at, int c) {
    constexpr int G = decltype(g)::value;
    A gx[G], gd[G], gg[G];
    if (t < w.count) {
      A dt[G], x[G], z[G], dy[G];
      Group<T, G>::values(Group<T, G>::load(px + t * p.xs[1] + c), x);
      Group<T, G>::values(Group<T, G>::load(pd + t * p.dts[1] + c), dt);
      if (p.gate != nullptr) {
        Group<T, G>::values(Group<T, G>::load(pg + t * p.gs[1] + c), z);
        Group<T, G>::values(Group<T, G>::load(pq + t * p.dys[1] + c), dy);
      }
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const A delta = slots[at * CT + slot_of(c + j)].v[0], dp = dps[at * CT + c + j];
        const A through = sums[at * PAD + c + j];
        const A sk = p.skip != nullptr ? skip[c + j] : A(0);
        const A pre = sums[(TT + at) * PAD + c + j] + sk * x[j];
        gx[j] = delta * through + sk * dp;
        gd[j] = A(kLn2) * sums[(2 * TT + at) * PAD + c + j] + x[j] * through;
        if (p.softplus) {
          const A v = p.dt_bias != nullptr ? dt[j] + bias[c + j] : dt[j];
          gd[j] *= sigmoid_at<T, true>(v);
        }
        if (p.gate != nullptr) {
          const A s = sigmoid_at<T, false>(z[j]);
          gg[j] = dy[j] * pre * s * (A(1) + z[j] * (A(1) - s));
        }
        params[at * CT + c + j] += dp * x[j];
        params[(TT + at) * CT + c + j] += gd[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < G; ++j) gx[j] = gd[j] = gg[j] = A(0);
    }
    Group<T, G>::store(ox + t * p.dim + c, gx);
    Group<T, G>::store(od + t * p.dim + c, gd);
    if (p.gate != nullptr) Group<T, G>::store(og + t * p.dim + c, gg);
  };
  auto each = [&](auto fn) {
    if (p.vec) {
      for (int e = threadIdx.x; e < TT * (CT / V); e += 128)
        fn(std::integral_constant<int, V>{}, e / (CT / V), e % (CT / V) * V);
    } else {
      for (int e = threadIdx.x; e < TT * CT; e += 128)
        fn(std::integral_constant<int, 1>{}, e / CT, e % CT);
    }
  };

  const int64_t steps = w.t1 > w.t0 ? (w.t1 - w.t0 + TT - 1) / TT : 0;
  A* part_bc = static_cast<A*>(p.part_bc) + (w.tile * p.batch + w.b) * p.length * 2 * NP;
  for (int64_t i = steps - 1; i >= 0; --i) {
    const int64_t t = w.t0 + i * TT;
    const bool any = t < w.count;
    if (any) {
      each([&](auto g, int at, int c) {
        stage(g, t + at, at, c, t + at < w.count && c < w.width);
      });
      stage_states<T, TT, NP>(p, w, p.b, p.bs, t, &into[0].v[0]);
      stage_states<T, TT, NP>(p, w, p.c, p.cs, t, &from[0].v[0]);
      __syncthreads();
      Two<A> db[TT][2], dc[TT][2];
      const Two<A> none = two(A(0), A(0));
#pragma unroll
      for (int u = 0; u < TT; ++u) db[u][0] = db[u][1] = dc[u][0] = dc[u][1] = none;
#pragma unroll 1
      for (int k = 0; k < KC; ++k) {
        const int c = c0 + k * LD;
        const Four<A> rq = mine[(0 * KC + k) * 128 + threadIdx.x];
        const Two<A> r0 = low(rq), r1 = high(rq);
        Two<A> h[TT + 1][2], e[TT][2];
        Four<A> start = {A(0), A(0), A(0), A(0)};
        if (c < w.width)
          start = static_cast<const Four<A>*>(
              p.check)[((w.b * ((p.length + 7) / 8) + t / 8) * p.dim + w.d0 + c) * LN + nl];
        h[0][0] = low(start);
        h[0][1] = high(start);
#pragma unroll
        for (int u = 0; u < TT; ++u) {
          const Four<A> q = slots[u * CT + slot_of(c)], bq = into[u * LN + nl];
          e[u][0] = exp_2(mul(low(q), r0));
          e[u][1] = exp_2(mul(low(q), r1));
          h[u + 1][0] = fma(e[u][0], h[u][0], mul(high(q), low(bq)));
          h[u + 1][1] = fma(e[u][1], h[u][1], mul(high(q), high(bq)));
        }
        const Four<A> sq = mine[(1 * KC + k) * 128 + threadIdx.x];
        Two<A> s0 = low(sq), s1 = high(sq), a0 = none, a1 = none;
        A through[TT], pre[TT], by_rate[TT];
#pragma unroll
        for (int u = TT - 1; u >= 0; --u) {
          const Four<A> q = slots[u * CT + slot_of(c)], bq = into[u * LN + nl],
                        cq = from[u * LN + nl];
          const A dp = dps[u * CT + c];
          const Two<A> dp2 = two(dp, dp);
          const Two<A> g0 = fma(low(cq), dp2, s0), g1 = fma(high(cq), dp2, s1);
          dc[u][0] = fma(dp2, h[u + 1][0], dc[u][0]);
          dc[u][1] = fma(dp2, h[u + 1][1], dc[u][1]);
          db[u][0] = fma(high(q), g0, db[u][0]);
          db[u][1] = fma(high(q), g1, db[u][1]);
          const Two<A> tb = fma(g1, high(bq), mul(g0, low(bq)));
          const Two<A> tc = fma(h[u + 1][1], high(cq), mul(h[u + 1][0], low(cq)));
          s0 = mul(e[u][0], g0);
          s1 = mul(e[u][1], g1);
          const Two<A> k0 = mul(s0, h[u][0]), k1 = mul(s1, h[u][1]);
          const Two<A> ta = fma(r1, k1, mul(r0, k0));
          a0 = fma(low(q), k0, a0);
          a1 = fma(low(q), k1, a1);
          through[u] = first(tb) + second(tb);
          pre[u] = first(tc) + second(tc);
          by_rate[u] = first(ta) + second(ta);
        }
        mine[(1 * KC + k) * 128 + threadIdx.x] = {first(s0), second(s0), first(s1), second(s1)};
        Four<A> da = mine[(2 * KC + k) * 128 + threadIdx.x];
        da.v[0] += first(a0), da.v[1] += second(a0), da.v[2] += first(a1), da.v[3] += second(a1);
        mine[(2 * KC + k) * 128 + threadIdx.x] = da;
        fold<TT, LN, 1>(through, lane);
        fold<TT, LN, 1>(pre, lane);
        fold<TT, LN, 1>(by_rate, lane);
        constexpr int OWN = TT >= LN ? TT / LN : 1;
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
          const int u = TT >= LN ? nl * OWN + o : nl / (LN / TT);
          sums[u * PAD + c] = through[o];
          sums[(TT + u) * PAD + c] = pre[o];
          sums[(2 * TT + u) * PAD + c] = by_rate[o];
        }
      }
      // over the warp's channels: value (token, b or c, state of the thread)
      A v[TT * 8];
#pragma unroll
      for (int u = 0; u < TT; ++u) {
        v[u * 8 + 0] = first(db[u][0]), v[u * 8 + 1] = second(db[u][0]);
        v[u * 8 + 2] = first(db[u][1]), v[u * 8 + 3] = second(db[u][1]);
        v[u * 8 + 4] = first(dc[u][0]), v[u * 8 + 5] = second(dc[u][0]);
        v[u * 8 + 6] = first(dc[u][1]), v[u * 8 + 7] = second(dc[u][1]);
      }
      fold<TT * 8, LD, LN>(v, lane);
      constexpr int OWN = TT * 8 / LD;
#pragma unroll
      for (int o = 0; o < OWN; ++o) {
        const int at = dl * OWN + o;
        joined[((warp * TT + at / 8) * 2 + at / 4 % 2) * NP + nl * 4 + at % 4] = v[o];
      }
      __syncthreads();
    }
    each([&](auto g, int at, int c) {
      if (t + at < w.t1 && c < w.width) finish(g, t + at, at, c);
    });
    for (int e = threadIdx.x; e < TT * 2 * NP; e += 128) {
      if (t + e / (2 * NP) >= w.t1) continue;
      A s = A(0);
      if (any) {
#pragma unroll
        for (int q = 0; q < 4; ++q) s += joined[q * TT * 2 * NP + e];
      }
      part_bc[t * 2 * NP + e] = s;
    }
    __syncthreads();
  }

  if (steps == 0) __syncthreads();
  const int64_t row = w.b * p.segments + w.segment;
  for (int k = 0; k < KC; ++k) {
    const int c = c0 + k * LD;
    if (c >= w.width) continue;
    const int64_t d = w.d0 + c;
    static_cast<Four<A>*>(p.part_a)[(row * p.dim + d) * LN + nl] =
        mine[(2 * KC + k) * 128 + threadIdx.x];
    if (w.segment == 0 && p.d_initial != nullptr) {
      const Four<A> s = mine[(1 * KC + k) * 128 + threadIdx.x];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (nl * 4 + j < p.states)
          static_cast<A*>(p.d_initial)[(w.b * p.dim + d) * p.states + nl * 4 + j] = s.v[j];
    }
  }
  for (int e = threadIdx.x; e < 2 * CT; e += 128) {
    const int which = e / CT, c = e % CT;
    if (c >= w.width) continue;
    A s = A(0);
#pragma unroll
    for (int u = 0; u < TT; ++u) s += params[(which * TT + u) * CT + c];
    static_cast<A*>(p.part_ch)[(row * 2 + which) * p.dim + w.d0 + c] = s;
  }
}
template <typename A> constexpr size_t scan_bwd_smem(int ln, int kc) {
  const int ct = 4 * (32 / ln) * kc, np = 4 * ln, tt = kScanCheck;
  return sizeof(A) * (4 * (size_t(tt) * ct + 3 * kc * 128 + 2 * tt * ln) + 4 * tt * 2 * np +
                      tt * ct + 3 * tt * (ct + 8) + 2 * tt * ct);
}

// ------------------------------------------------------------------------------ single tokens
// One token of every sequence: a pass over the states, read and written once.
template <typename T, int LN>
__global__ void __launch_bounds__(128)
scan_step_kernel(const __grid_constant__ ScanArgs p, const int32_t* __restrict__ slots,
                 int64_t pool, typename AccOf<T>::type* state) {
  using A = typename AccOf<T>::type;
  constexpr int CW = 128 / LN;  // channels of a block
  const int64_t blocks = (p.dim + CW - 1) / CW;
  const int64_t b = blockIdx.x / blocks;
  const int nl = threadIdx.x % LN;
  int64_t d = blockIdx.x % blocks * CW + threadIdx.x / LN;
  const bool in = d < p.dim;
  if (!in) d = p.dim - 1;  // the lanes of a warp stay together
  const int64_t slot = slots == nullptr ? b : slots[b];
  const bool live = slot >= 0 && slot < pool;
  A y = A(0), x = A(0);
  if (live) {
    x = to_acc(static_cast<const T*>(p.x)[b * p.xs[0] + d]);
    A delta = to_acc(static_cast<const T*>(p.dt)[b * p.dts[0] + d]);
    if (p.dt_bias != nullptr) delta += static_cast<const A*>(p.dt_bias)[d];
    if (p.softplus) delta = softplus(delta);
    const int64_t group = d / p.per;
    const T* pb = static_cast<const T*>(p.b) + b * p.bs[0] + group * p.bs[2];
    const T* pc = static_cast<const T*>(p.c) + b * p.cs[0] + group * p.cs[2];
    const A* pa = static_cast<const A*>(p.a) + d * p.states;
    A* ps = state + (slot * p.dim + d) * p.states;
    if (p.vec) {  // states in whole fours
      if (nl * 4 < p.states) {
        Four<A> h = reinterpret_cast<Four<A>*>(ps)[nl];
        const Four<A> r = reinterpret_cast<const Four<A>*>(pa)[nl];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h.v[j] = exp_2(delta * rate(r.v[j])) * h.v[j] + delta * x * A(to_acc(pb[nl * 4 + j]));
          y += h.v[j] * A(to_acc(pc[nl * 4 + j]));
        }
        if (in) reinterpret_cast<Four<A>*>(ps)[nl] = h;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = nl * 4 + j;
        if (n < p.states) {
          const A h = exp_2(delta * rate(pa[n])) * ps[n] + delta * x * A(to_acc(pb[n]));
          y += h * A(to_acc(pc[n]));
          if (in) ps[n] = h;
        }
      }
    }
  }
#pragma unroll
  for (int o = LN / 2; o > 0; o /= 2) y += __shfl_xor_sync(0xffffffffu, y, o);
  if (!in || nl != 0) return;
  if (live) {
    if (p.skip != nullptr) y += static_cast<const A*>(p.skip)[d] * x;
    if (p.gate != nullptr) {
      const A z = to_acc(static_cast<const T*>(p.gate)[b * p.gs[0] + d]);
      y *= z * sigmoid_at<T, false>(z);
    }
  }
  static_cast<T*>(p.y)[b * p.dim + d] = from_acc<T>(y);
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
inline int scan_grid(const ScanArgs& p, unsigned* grid) {
  const int64_t blocks = p.tiles * p.groups * p.segments * p.batch;
  if (blocks > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  *grid = static_cast<unsigned>(blocks);
  return FDWT_OK;
}

template <typename T, int MODE> int scan_launch(const ScanArgs& p, int lanes, cudaStream_t stream) {
  return with_lanes(lanes, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    unsigned grid;
    int st = scan_grid(p, &grid);
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

template <typename T> int scan_backward(const ScanArgs& p, int lanes, bool wide, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  return with_lanes(lanes, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    auto launch = [&](auto kc) {
      constexpr int KC = decltype(kc)::value;
      auto kernel = scan_bwd_kernel<T, LN, KC>;
      unsigned grid;
      int st = scan_grid(p, &grid);
      if (st == FDWT_OK) st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
      if (st == FDWT_OK) st = pre_launch(stream);
      if (st != FDWT_OK) return st;
      kernel<<<grid, 128, scan_bwd_smem<A>(LN, KC), stream>>>(p);
      return launch_status();
    };
    constexpr int narrow = scan_bwd_channels(LN, false), broad = scan_bwd_channels(LN, true);
    if constexpr (narrow != broad && sizeof(A) == 4) {
      if (wide) return launch(std::integral_constant<int, broad>{});
    }
    return launch(std::integral_constant<int, narrow>{});
  });
}

template <typename T>
int scan_step(const ScanArgs& p, int lanes, const int32_t* slots, int64_t pool, void* state,
              cudaStream_t stream) {
  return with_lanes(lanes, [&](auto ln) {
    constexpr int LN = decltype(ln)::value;
    const int64_t grid = p.batch * cdiv(p.dim, 128 / LN);
    if (grid > INT32_MAX) return static_cast<int>(FDWT_ERR_UNSUPPORTED);
    const int st = pre_launch(stream);
    if (st != FDWT_OK) return st;
    scan_step_kernel<T, LN><<<static_cast<unsigned>(grid), 128, 0, stream>>>(
        p, slots, pool, static_cast<typename AccOf<T>::type*>(state));
    return launch_status();
  });
}

#define FDWT_SCAN_TYPE(T)                                                            \
  template int scan_forward<T>(const ScanArgs&, int, cudaStream_t);                  \
  template int scan_states<T>(const ScanArgs&, int, bool, cudaStream_t);             \
  template int scan_backward<T>(const ScanArgs&, int, bool, cudaStream_t);           \
  template int scan_step<T>(const ScanArgs&, int, const int32_t*, int64_t, void*, cudaStream_t);

}  // namespace fdwt
