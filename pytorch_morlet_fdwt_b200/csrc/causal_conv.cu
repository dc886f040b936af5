// Short causal convolution of every channel with its own taps, over tokens: forward, gradients and
// the single-token form.
//
//   p_t = bias + sum_j w[j] x_{t-W+1+j},   y = p   or   y = p sigmoid(p)
//   dp = dy dy/dp,   dx_t = sum_j w[j] dp_{t+W-1-j},   dw[j] = sum_t dp_t x_{t-W+1+j},   db = sum_t dp_t
//
// Tokens before the first come from the state (the last W-1 inputs of what came before), zeros
// without one.  Bound by HBM (2 W + 4 operations an element forward): a thread takes V
// neighbouring channels (16 bytes, forward) and walks over a run of tokens with the last W inputs
// in registers, so that every input is read once (and W-1 of a run's neighbours, from L2) and the
// loads of several tokens are in flight.  Sums are 32 bits (64 for fp64) on pairs of channels (one
// packed instruction a pair); y and the gradients are rounded once.
//
// Measured, 4 taps with silu: 4 x 4096 x 2048 bf16 forward 33 us (4.1 TB/s), backward 62 us (3.2
// TB/s); fp32 52 us forward (5.2 TB/s).  In 16 bits it is latency that bounds them, not bytes: forward
// 143 registers, 12 warps an SM, 0.46 instructions issued a cycle and scheduler, DRAM 31 % busy, stalls on
// results of fixed latency 1.5 and on loads 1.1 warps an issue; backward 96 registers, 20 warps, 0.61,
// 32 %, and 82 instructions a token of two channels.  A thread of the backward pass takes 2 channels (4:
// 160 registers, 1.2 times the time; 1 in fp64).
#include "pairs.cuh"
#include "row_groups.cuh"

namespace fdwt {
namespace {

struct ConvCall {
  int64_t batch, length, dim, xs_b, xs_t, ds_b, ds_t;
  bool silu, param_f32;
  const void *x, *weight, *bias, *initial;
  const int32_t* lengths;
  cudaStream_t stream;
};

// V channels' values: pairs of them, or one.
template <typename A, int V> struct Channels {
  using E = std::conditional_t<V == 1, A, Two<A>>;
  static constexpr int M = V == 1 ? 1 : V / 2;
  E e[M];
  __device__ __forceinline__ void set(const A* x) {
    if constexpr (V == 1) {
      e[0] = x[0];
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m) e[m] = two(x[2 * m], x[2 * m + 1]);
    }
  }
  __device__ __forceinline__ void get(A* x) const {
    if constexpr (V == 1) {
      x[0] = e[0];
    } else {
#pragma unroll
      for (int m = 0; m < M; ++m) x[2 * m] = first(e[m]), x[2 * m + 1] = second(e[m]);
    }
  }
  __device__ __forceinline__ void clear() {
    A zero[V];
#pragma unroll
    for (int j = 0; j < V; ++j) zero[j] = A(0);
    set(zero);
  }
};

// 1 / (1 + e^-p): of a few roundings' error in 32 bits for rows of 32 bits, and by the fast
// exponential and reciprocal, on pairs, for 16-bit rows, whose rounding is 2^12 times theirs.
template <typename T, int V, typename A>
__device__ __forceinline__ Channels<A, V> sigmoid(const Channels<A, V>& p) {
  using E = typename Channels<A, V>::E;
  Channels<A, V> r;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int m = 0; m < Channels<A, V>::M; ++m)
      r.e[m] = reciprocal(add(exp_2(mul(p.e[m], splat<E>(-static_cast<float>(kLog2e)))),
                              splat<E>(1.0f)));
  } else {
    A v[V];
    p.get(v);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (sizeof(T) == 4) v[j] = 1.0f / (1.0f + expf(-v[j]));
      else v[j] = 1.0 / (1.0 + exp(-v[j]));
    }
    r.set(v);
  }
  return r;
}

// One parameter of the rows' type or of 32 bits.
template <typename T>
__device__ __forceinline__ typename AccOf<T>::type param(const void* p, bool f32, int64_t i) {
  using A = typename AccOf<T>::type;
  if (sizeof(T) == 2 && f32) return static_cast<A>(static_cast<const float*>(p)[i]);
  return to_acc(static_cast<const T*>(p)[i]);
}

// The taps of V channels, contiguous in memory (`whole`: on a boundary of V elements).
template <typename T, int V, int W, typename A>
__device__ __forceinline__ void load_taps(const void* weight, bool f32, bool whole, int64_t c,
                                          Channels<A, V> (&taps)[W]) {
  A w[W][V];
  if (whole && !(sizeof(T) == 2 && f32)) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      A x[V];
      Group<T, V>::values(Group<T, V>::load(static_cast<const T*>(weight) + c * W + i * V), x);
#pragma unroll
      for (int j = 0; j < V; ++j) w[(i * V + j) % W][(i * V + j) / W] = x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < W; ++i) w[i][j] = param<T>(weight, f32, (c + j) * W + i);
  }
#pragma unroll
  for (int i = 0; i < W; ++i) taps[i].set(w[i]);
}
template <typename T, int V, typename A>
__device__ __forceinline__ Channels<A, V> load_bias(const void* bias, bool f32, int64_t c) {
  A x[V];
#pragma unroll
  for (int j = 0; j < V; ++j) x[j] = bias == nullptr ? A(0) : param<T>(bias, f32, c + j);
  Channels<A, V> r;
  r.set(x);
  return r;
}

__device__ __forceinline__ int64_t tokens_of(const int32_t* lengths, int64_t b, int64_t length) {
  if (lengths == nullptr) return length;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : (n < length ? n : length);
}

// V inputs of token t (before the first: of the state; none past the `count` valid ones).
template <typename T, int V, typename A>
__device__ __forceinline__ void input_at(const T* x, int64_t xs_t, const T* before, int64_t dim,
                                         int width, int64_t t, int64_t count, A* v) {
  using G = Group<T, V>;
  if (t >= 0 && t < count) {
    G::values(G::load(x + t * xs_t), v);
  } else if (t < 0 && before != nullptr) {
    G::values(G::load(before + (t + width - 1) * dim), v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0;
  }
}

// Thread: V channels, `run` tokens.  Threads go over channels first, then runs, then sequences.
// The next U tokens are loaded before the current ones are worked out.
template <typename T, int V, int W>
__global__ void __launch_bounds__(128)
conv_fwd_kernel(const T* __restrict__ x, const void* __restrict__ weight,
                const void* __restrict__ bias, const T* __restrict__ initial,
                const int32_t* __restrict__ lengths, T* __restrict__ y,
                T* __restrict__ final_state, int64_t batch, int64_t length, int64_t dim,
                int64_t xs_b, int64_t xs_t, int run, bool silu, bool param_f32, bool whole) {
  using A = typename AccOf<T>::type;
  using G = Group<T, V>;
  // tokens whose loads are issued together (fp32 of odd widths, one element a load: 26 us with 4,
  // 24 us with 8 for 5 x 3001 x 1001)
  constexpr int U = V == 1 ? 8 : 4;
  const int64_t per = dim / V, runs = length > run ? (length + run - 1) / run : 1;
  const int64_t id = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t c = id % per * V, k = id / per % runs, b = id / per / runs;
  if (b >= batch) return;
  const int64_t count = tokens_of(lengths, b, length);
  x += b * xs_b + c;
  y += b * length * dim + c;
  const T* before = initial == nullptr ? nullptr : initial + b * (W - 1) * dim + c;
  if (final_state != nullptr && k == 0) {
    for (int i = 0; i < W - 1; ++i) {
      A v[V];
      input_at<T, V>(x, xs_t, before, dim, W, count - (W - 1) + i, count, v);
      G::store(final_state + (b * (W - 1) + i) * dim + c, v);
    }
  }
  const int64_t t0 = k * run, t1 = t0 + run < length ? t0 + run : length;
  const int valid = static_cast<int>((count < t1 ? count : t1) - t0);  // tokens of the run that count
  const int all = static_cast<int>(t1 - t0);
  x += t0 * xs_t;
  y += t0 * dim;
  typename G::Raw next[U];
  const T* px = x;
  auto fetch = [&](int t) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u < valid) next[u] = G::load(px + u * xs_t);
    px += U * xs_t;
  };
  fetch(0);
  using C = Channels<A, V>;
  C w[W];
  load_taps<T, V, W>(weight, param_f32, whole, c, w);
  const C at = load_bias<T, V, A>(bias, param_f32, c);
  C win[W - 1 + U];  // the inputs of tokens t - W + 1 ... t + U - 1
#pragma unroll
  for (int i = 0; i < W - 1; ++i) {
    A v[V];
    input_at<T, V>(x - t0 * xs_t, xs_t, before, dim, W, t0 - (W - 1) + i, count, v);
    win[i].set(v);
  }
  T* out = y;
  for (int t = 0; t < valid; t += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (past the end: not used)
      A v[V];
      G::values(next[u], v);
      win[W - 1 + u].set(v);
    }
    if (t + U < valid) fetch(t + U);
    auto token = [&](int u) {
      C p;
#pragma unroll
      for (int m = 0; m < C::M; ++m) {
        p.e[m] = fma(w[0].e[m], win[u].e[m], at.e[m]);
#pragma unroll
        for (int i = 1; i < W; ++i) p.e[m] = fma(w[i].e[m], win[u + i].e[m], p.e[m]);
      }
      if (silu) {
        const C g = sigmoid<T, V, A>(p);
#pragma unroll
        for (int m = 0; m < C::M; ++m) p.e[m] = mul(p.e[m], g.e[m]);
      }
      A v[V];
      p.get(v);
      G::store(out, v);
      out += dim;
    };
    if (t + U <= valid) {
#pragma unroll
      for (int u = 0; u < U; ++u) token(u);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t + u < valid) token(u);
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) win[i] = win[i + U];
  }
  A none[V];
#pragma unroll
  for (int j = 0; j < V; ++j) none[j] = A(0);
  for (int t = valid > 0 ? valid : 0; t < all; ++t) G::store(y + t * dim, none);
}

// Backward.  A block is 32 threads of channels by 4 runs of tokens; a thread walks its run and the
// W-1 tokens after it (whose dp its last inputs need), so dx is written once.  dw and db are summed
// in registers over the run, joined over the block's runs in shared memory and written as one
// partial row (dim x (W + 1)) a block row, added in a fixed order by conv_params_kernel.
constexpr int kBwdLanes = 32, kBwdRuns = 4;
template <typename T, int V, int W>
__global__ void __launch_bounds__(kBwdLanes* kBwdRuns)
conv_bwd_kernel(const T* __restrict__ x, const void* __restrict__ weight,
                const void* __restrict__ bias, const T* __restrict__ initial,
                const int32_t* __restrict__ lengths, const T* __restrict__ dy,
                const T* __restrict__ d_final, T* __restrict__ dx, T* __restrict__ d_initial,
                typename AccOf<T>::type* __restrict__ partial, int64_t length, int64_t dim,
                int64_t xs_b, int64_t xs_t, int64_t ds_b, int64_t ds_t, int run, int64_t rows,
                int64_t columns, bool silu, bool param_f32, bool whole) {
  using A = typename AccOf<T>::type;
  using G = Group<T, V>;
  __shared__ A joined[kBwdRuns][kBwdLanes * V + 1];
  const int64_t per = dim / V;
  const int64_t column = blockIdx.x % columns, part = blockIdx.x / columns;
  const int64_t cg = column * kBwdLanes + threadIdx.x;
  const int64_t b = part / rows, row = part % rows;
  const int64_t k = row * kBwdRuns + threadIdx.y;  // the thread's run
  const bool in = cg < per;
  const int64_t c = (in ? cg : per - 1) * V;
  const int64_t count = tokens_of(lengths, b, length);
  x += b * xs_b + c;
  dy += b * ds_b + c;
  const T* before = initial == nullptr ? nullptr : initial + b * (W - 1) * dim + c;
  using C = Channels<A, V>;
  C w[W], dw[W], db;
  load_taps<T, V, W>(weight, param_f32, whole, c, w);
  const C at = load_bias<T, V, A>(bias, param_f32, c);
#pragma unroll
  for (int i = 0; i < W; ++i) dw[i].clear();
  db.clear();
  const int64_t t0 = k * run;
  const bool first = k == 0;
  // relative to the run's first token: its tokens, and the valid ones of the sequence
  const int all = static_cast<int>(length - t0 < run ? length - t0 : run);
  const int valid = static_cast<int>(count - t0 < all + W - 1 ? count - t0 : all + W - 1);
  if (in && (all > 0 || first)) {
    C win[W], dp[W];  // inputs t-W+1 ... t and gradients of the sums p of the same tokens
    win[0].clear();
#pragma unroll
    for (int i = 0; i < W; ++i) dp[i].clear();
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
      A v[V];
      input_at<T, V>(x, xs_t, before, dim, W, t0 - (W - 1) + i, count, v);
      win[i + 1].set(v);
    }
    constexpr int U = 4;
    const int end = all + W - 1, begin = first && d_initial != nullptr ? -(W - 1) : 0;
    const T *px = x + t0 * xs_t, *pd = dy + t0 * ds_t;
    T* out = dx + (b * length + t0 - (W - 1)) * dim + c;  // of input t - W + 1
    typename G::Raw nx[U], nd[U];
    auto fetch = [&](int t) {
      if (t + U <= valid) {
#pragma unroll
        for (int u = 0; u < U; ++u) nx[u] = G::load(px + u * xs_t), nd[u] = G::load(pd + u * ds_t);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          nx[u] = nd[u] = typename G::Raw{};
          if (t + u < valid) nx[u] = G::load(px + u * xs_t), nd[u] = G::load(pd + u * ds_t);
        }
      }
      px += U * xs_t;
      pd += U * ds_t;
    };
    // Moves on by a token: its window, its dp (zero where it does not count) and its share of dw and
    // db (where it is the run's own); g: the gradient of input t - W + 1, all of whose dp are there.
    auto token = [&](const typename G::Raw& rx, const typename G::Raw& rd, bool counts, bool own,
                     A* g) {
#pragma unroll
      for (int i = 0; i < W - 1; ++i) win[i] = win[i + 1], dp[i] = dp[i + 1];
      A v[V], q[V];
      G::values(rx, v);
      win[W - 1].set(v);
      G::values(rd, q);
      if (silu) {
        C p;
#pragma unroll
        for (int m = 0; m < C::M; ++m) {
          p.e[m] = fma(w[0].e[m], win[0].e[m], at.e[m]);
#pragma unroll
          for (int i = 1; i < W; ++i) p.e[m] = fma(w[i].e[m], win[i].e[m], p.e[m]);
        }
        const C g = sigmoid<T, V, A>(p);
        C slope;
#pragma unroll
        for (int m = 0; m < C::M; ++m) {  // g (1 + p (1 - g))
          using E = typename C::E;
          const E rest = fma(g.e[m], splat<E>(-1.0f), splat<E>(1.0f));
          slope.e[m] = mul(g.e[m], fma(p.e[m], rest, splat<E>(1.0f)));
        }
        slope.get(v);
#pragma unroll
        for (int j = 0; j < V; ++j) q[j] *= v[j];
      }
      // (chosen, not multiplied by zero: what the window holds may be no number)
#pragma unroll
      for (int j = 0; j < V; ++j) q[j] = counts ? q[j] : A(0);
      dp[W - 1].set(q);
      C r;
#pragma unroll
      for (int m = 0; m < C::M; ++m) {
        r.e[m] = mul(w[W - 1].e[m], dp[0].e[m]);
#pragma unroll
        for (int i = 1; i < W; ++i) r.e[m] = fma(w[W - 1 - i].e[m], dp[i].e[m], r.e[m]);
      }
      if (own) {  // (the same for a warp's threads; and no product of zero with the window either)
#pragma unroll
        for (int m = 0; m < C::M; ++m) {
          db.e[m] = add(db.e[m], dp[W - 1].e[m]);
#pragma unroll
          for (int i = 0; i < W; ++i) dw[i].e[m] = fma(dp[W - 1].e[m], win[i].e[m], dw[i].e[m]);
        }
      }
      r.get(g);
    };
    // up to here the tokens' shares are all the run's own, and their inputs not in the state
    const int sure = valid < all ? valid : all;
    const int64_t last = count - t0;
    fetch(0);
    for (int s = 0; s < end; s += U) {
      typename G::Raw rx[U], rd[U];
#pragma unroll
      for (int u = 0; u < U; ++u) rx[u] = nx[u], rd[u] = nd[u];
      if (s + U < end) fetch(s + U);
      if (s >= W - 1 && s + U <= sure && dx != nullptr &&
          (d_final == nullptr || s + U - (W - 1) <= last - (W - 1))) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          A g[V];
          token(rx[u], rd[u], true, true, g);
          G::store(out, g);
          out += dim;
        }
        continue;
      }
#pragma unroll
      for (int u = 0; u < U; ++u, out += dim) {
        const int t = s + u, to = t - (W - 1);
        A g[V];
        token(rx[u], rd[u], t < valid, t < all && t < valid, g);
        if (to < begin || t >= end) continue;
        const int64_t behind = last - to;  // 1: the last valid token
        if (d_final != nullptr && behind >= 1 && behind <= W - 1) {
          A f[V];
          G::values(G::load(d_final + (b * (W - 1) + W - 1 - behind) * dim + c), f);
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] += f[j];
        }
        if (to < 0) G::store(d_initial + (b * (W - 1) + to + W - 1) * dim + c, g);
        else if (dx != nullptr) G::store(out, g);
      }
    }
  }
  if (partial == nullptr) return;
  // one tap (or the bias) after the other through shared memory
#pragma unroll
  for (int i = 0; i <= W; ++i) {
    if (i > 0) __syncthreads();
    A v[V];
    if (i < W) dw[i % W].get(v);
    else db.get(v);
#pragma unroll
    for (int j = 0; j < V; ++j) joined[threadIdx.y][threadIdx.x * V + j] = v[j];
    __syncthreads();
    for (int e = threadIdx.y * kBwdLanes + threadIdx.x; e < kBwdLanes * V;
         e += kBwdLanes * kBwdRuns) {
      const int64_t channel = column * kBwdLanes * V + e;
      if (channel >= dim) continue;
      A sum = joined[0][e];
#pragma unroll
      for (int r = 1; r < kBwdRuns; ++r) sum += joined[r][e];
      partial[(part * (W + 1) + i) * dim + channel] = sum;
    }
  }
}

// dw (dim, W) and db from the partial rows [parts][W + 1][dim], added in a fixed order.
template <typename T>
__global__ void __launch_bounds__(256)
conv_params_kernel(const typename AccOf<T>::type* __restrict__ partial, int64_t parts, int64_t dim,
                   int width, void* __restrict__ dw, void* __restrict__ db, bool param_f32) {
  using A = typename AccOf<T>::type;
  __shared__ A cells[8][33];
  const int64_t cols = (width + 1) * dim, c = int64_t(blockIdx.x) * 32 + threadIdx.x;
  A sum = A(0);
  if (c < cols) {
#pragma unroll 8
    for (int64_t p = threadIdx.y; p < parts; p += 8) sum += partial[p * cols + c];
  }
  cells[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y != 0 || c >= cols) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) sum += cells[k][threadIdx.x];
  const int64_t tap = c / dim, channel = c % dim;
  void* out = tap < width ? dw : db;
  if (out == nullptr) return;
  const int64_t i = tap < width ? channel * width + tap : channel;
  if (sizeof(T) == 2 && param_f32) static_cast<float*>(out)[i] = static_cast<float>(sum);
  else static_cast<T*>(out)[i] = from_acc<T>(sum);
}

// One token of every sequence: the window is the state's rows and x; the state moves on by one.
template <typename T, int V>
__global__ void __launch_bounds__(128)
conv_step_kernel(const T* __restrict__ x, const void* __restrict__ weight,
                 const void* __restrict__ bias, T* state, const int32_t* __restrict__ slots,
                 T* __restrict__ y, int64_t batch, int64_t dim, int64_t xs_b, int64_t pool,
                 int width, bool silu, bool param_f32) {
  using A = typename AccOf<T>::type;
  using G = Group<T, V>;
  // threads over channels, blocks over channels first, then sequences
  const unsigned per = static_cast<unsigned>(dim / V), blocks = (per + 127) / 128;
  const unsigned place = blockIdx.x % blocks * 128 + threadIdx.x;
  const int64_t c = int64_t(place) * V, b = blockIdx.x / blocks;
  if (place >= per) return;
  const int64_t slot = slots == nullptr ? b : slots[b];
  A p[V];
  if (slot < 0 || slot >= pool) {
#pragma unroll
    for (int j = 0; j < V; ++j) p[j] = A(0);
    G::store(y + b * dim + c, p);
    return;
  }
  T* rows = state + slot * (width - 1) * dim + c;
  typename G::Raw raw[8];
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < width - 1) raw[i] = G::load(rows + i * dim);
  const typename G::Raw now = G::load(x + b * xs_b + c);
#pragma unroll
  for (int j = 0; j < V; ++j) p[j] = bias == nullptr ? A(0) : param<T>(bias, param_f32, c + j);
  A v[V];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i < width) {
      if (i == width - 1) raw[i] = now;
      G::values(raw[i], v);
#pragma unroll
      for (int j = 0; j < V; ++j) p[j] += param<T>(weight, param_f32, (c + j) * width + i) * v[j];
      if (i > 0) G::store(rows + (i - 1) * dim, v);
    }
  }
  if (silu) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      Channels<A, 1> one;
      one.e[0] = p[j];
      p[j] *= sigmoid<T, 1, A>(one).e[0];
    }
  }
  G::store(y + b * dim + c, p);
}

// ------------------------------------------------------------------------------ launches
// Whether rows of these strides and pointers take groups of v elements.
template <typename T>
bool grouped(int v, int64_t dim, std::initializer_list<int64_t> strides, Pointers pointers) {
  uintptr_t bits = 0;
  for (const void* q : pointers) bits |= reinterpret_cast<uintptr_t>(q);
  if (dim % v != 0 || bits % (v * sizeof(T)) != 0) return false;
  for (int64_t s : strides)
    if (s % v != 0) return false;
  return true;
}

template <typename F> int with_width(int width, F fn) {
  switch (width) {
    case 2: return fn(std::integral_constant<int, 2>{});
    case 3: return fn(std::integral_constant<int, 3>{});
    case 4: return fn(std::integral_constant<int, 4>{});
    case 5: return fn(std::integral_constant<int, 5>{});
    case 6: return fn(std::integral_constant<int, 6>{});
    case 7: return fn(std::integral_constant<int, 7>{});
    case 8: return fn(std::integral_constant<int, 8>{});
    default: return FDWT_ERR_INVALID;
  }
}

template <typename T, int V> int conv_forward_v(const ConvCall& c, int width, void* y, void* fin) {
  // runs as long as leaves 512 threads for every multiprocessor, 8 to 64 tokens
  int run = 64;
  while (run > 8 && c.batch * cdiv(c.length, run) * (c.dim / V) < int64_t(sm_count()) * 512) run /= 2;
  const int64_t threads = c.batch * imax(1, cdiv(c.length, run)) * (c.dim / V);
  const int64_t grid = cdiv(threads, 128);
  if (grid > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  const int st = pre_launch(c.stream);
  if (st != FDWT_OK) return st;
  return with_width(width, [&](auto w) {
    conv_fwd_kernel<T, V, decltype(w)::value><<<static_cast<unsigned>(grid), 128, 0, c.stream>>>(
        static_cast<const T*>(c.x), c.weight, c.bias, static_cast<const T*>(c.initial), c.lengths,
        static_cast<T*>(y), static_cast<T*>(fin), c.batch, c.length, c.dim, c.xs_b, c.xs_t, run,
        c.silu, c.param_f32, grouped<T>(V, c.dim, {}, {c.weight}));
    return launch_status();
  });
}

// Tokens a thread of the backward pass, and rows of blocks a sequence.
struct BwdRuns {
  int run;
  int64_t rows;
};
inline BwdRuns bwd_runs(int64_t batch, int64_t length, int64_t dim, int v) {
  int run = 64;
  while (run > 8 && batch * cdiv(length, run) * cdiv(dim, v) < int64_t(sm_count()) * 512) run /= 2;
  return {run, imax(1, cdiv(length, int64_t(run) * kBwdRuns))};
}
template <typename T> constexpr int bwd_group = sizeof(T) == 8 ? 1 : 2;

template <typename T, int V>
int conv_backward_v(const ConvCall& c, int width, const void* dy, const void* d_final, void* dx,
                    void* dw, void* db, void* d_initial, void* ws) {
  using A = typename AccOf<T>::type;
  const BwdRuns r = bwd_runs(c.batch, c.length, c.dim, bwd_group<T>);
  A* partial = dw != nullptr || db != nullptr ? static_cast<A*>(ws) : nullptr;
  const int64_t parts = c.batch * r.rows;
  const int64_t columns = cdiv(c.dim / V, kBwdLanes);
  if (columns * parts > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  int st = pre_launch(c.stream);
  if (st != FDWT_OK) return st;
  st = with_width(width, [&](auto w) {
    conv_bwd_kernel<T, V, decltype(w)::value>
        <<<static_cast<unsigned>(columns * parts), dim3(kBwdLanes, kBwdRuns), 0, c.stream>>>(
            static_cast<const T*>(c.x), c.weight, c.bias, static_cast<const T*>(c.initial),
            c.lengths, static_cast<const T*>(dy), static_cast<const T*>(d_final),
            static_cast<T*>(dx), static_cast<T*>(d_initial), partial, c.length, c.dim, c.xs_b,
            c.xs_t, c.ds_b, c.ds_t, r.run, r.rows, columns, c.silu, c.param_f32,
            grouped<T>(V, c.dim, {}, {c.weight}));
    return launch_status();
  });
  if (st != FDWT_OK || partial == nullptr) return st;
  st = pre_launch(c.stream);
  if (st != FDWT_OK) return st;
  conv_params_kernel<T><<<static_cast<unsigned>(cdiv((width + 1) * c.dim, 32)), dim3(32, 8), 0,
                          c.stream>>>(partial, parts, c.dim, width, dw, db, c.param_f32);
  return launch_status();
}

template <typename F> int with_type(int dtype, F fn) {
  switch (dtype) {
    case FDWT_F32: return fn(float{});
    case FDWT_F64: return fn(double{});
    case FDWT_F16: return fn(__half{});
    default: return fn(__nv_bfloat16{});
  }
}

// The largest sizes: token and element counts that the kernels' grids and 64-bit offsets hold.
constexpr int64_t kMostTokens = int64_t(1) << 30;

bool conv_ok(const fdwt_conv1d_desc* d) {
  return d != nullptr && dtype_size(d->dtype) != 0 &&
         (d->param_dtype == d->dtype || (d->param_dtype == FDWT_F32 && d->dtype != FDWT_F64)) &&
         d->width >= 2 && d->width <= FDWT_MAX_CONV_WIDTH && d->batch >= 0 && d->length >= 0 &&
         d->dim >= 1 && d->batch < kMostTokens && d->length < kMostTokens && d->dim < kMostTokens;
}
ConvCall conv_call(const fdwt_conv1d_desc* d, const void* x, const void* weight, const void* bias,
                   const void* initial, const int32_t* lengths, void* stream) {
  return {d->batch, d->length, d->dim, d->x_stride[0], d->x_stride[1], d->dy_stride[0],
          d->dy_stride[1], d->silu != 0, d->param_dtype == FDWT_F32, x, weight, bias, initial,
          lengths, static_cast<cudaStream_t>(stream)};
}

}  // namespace
}  // namespace fdwt

using namespace fdwt;

extern "C" int fdwt_causal_conv1d_forward(const fdwt_conv1d_desc* desc, const void* x,
                                          const void* weight, const void* bias,
                                          const void* initial_state, const int32_t* lengths,
                                          void* y, void* final_state, void* stream) {
  FDWT_CHECK(conv_ok(desc));
  if (desc->batch == 0 || (desc->length == 0 && final_state == nullptr)) return FDWT_OK;
  FDWT_CHECK(weight != nullptr && (desc->length == 0 || (x != nullptr && y != nullptr)));
  const ConvCall c = conv_call(desc, x, weight, bias, initial_state, lengths, stream);
  return with_type(desc->dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = 16 / sizeof(T);
    if (grouped<T>(V, c.dim, {c.xs_b, c.xs_t}, {x, y, initial_state, final_state}))
      return conv_forward_v<T, V>(c, desc->width, y, final_state);
    return conv_forward_v<T, 1>(c, desc->width, y, final_state);
  });
}

extern "C" size_t fdwt_causal_conv1d_backward_workspace(const fdwt_conv1d_desc* desc) {
  if (!conv_ok(desc) || desc->batch == 0) return 0;
  const int v = desc->dtype == FDWT_F64 ? 1 : 2;
  const BwdRuns r = bwd_runs(desc->batch, desc->length, desc->dim, v);
  return size_t(desc->batch * r.rows) * (desc->width + 1) * desc->dim *
         (desc->dtype == FDWT_F64 ? 8 : 4);
}

extern "C" int fdwt_causal_conv1d_backward(const fdwt_conv1d_desc* desc, const void* x,
                                           const void* weight, const void* bias,
                                           const void* initial_state, const int32_t* lengths,
                                           const void* dy, const void* d_final_state, void* dx,
                                           void* dweight, void* dbias, void* d_initial_state,
                                           void* workspace, size_t workspace_bytes, void* stream) {
  FDWT_CHECK(conv_ok(desc));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (desc->batch == 0) {
    const size_t size = dtype_size(desc->param_dtype) * desc->dim;
    if (dweight != nullptr) FDWT_CUDA(cudaMemsetAsync(dweight, 0, size * desc->width, s));
    if (dbias != nullptr) FDWT_CUDA(cudaMemsetAsync(dbias, 0, size, s));
    return FDWT_OK;
  }
  FDWT_CHECK(weight != nullptr && (desc->length == 0 || (x != nullptr && dy != nullptr)));
  if ((dweight != nullptr || dbias != nullptr) &&
      (workspace == nullptr || workspace_bytes < fdwt_causal_conv1d_backward_workspace(desc)))
    return FDWT_ERR_WORKSPACE;
  const ConvCall c = conv_call(desc, x, weight, bias, initial_state, lengths, stream);
  return with_type(desc->dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int V = bwd_group<T>;
    if (grouped<T>(V, c.dim, {c.xs_b, c.xs_t, c.ds_b, c.ds_t},
                   {x, dy, dx, initial_state, d_final_state, d_initial_state}))
      return conv_backward_v<T, V>(c, desc->width, dy, d_final_state, dx, dweight, dbias,
                                   d_initial_state, workspace);
    return conv_backward_v<T, 1>(c, desc->width, dy, d_final_state, dx, dweight, dbias,
                                 d_initial_state, workspace);
  });
}

extern "C" int fdwt_causal_conv1d_step(const fdwt_conv1d_desc* desc, const void* x,
                                       const void* weight, const void* bias, void* state,
                                       int64_t state_slots, const int32_t* slots, void* y,
                                       void* stream) {
  FDWT_CHECK(conv_ok(desc) && desc->length == 1 && state_slots >= 0);
  FDWT_CHECK(slots != nullptr || state_slots >= desc->batch);
  if (desc->batch == 0) return FDWT_OK;
  FDWT_CHECK(x != nullptr && weight != nullptr && y != nullptr &&
             (state != nullptr || state_slots == 0));
  return with_type(desc->dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto v) {
      constexpr int V = decltype(v)::value;
      const int64_t grid = desc->batch * cdiv(desc->dim / V, 128);
      if (grid > INT32_MAX) return static_cast<int>(FDWT_ERR_UNSUPPORTED);
      const int st = pre_launch(static_cast<cudaStream_t>(stream));
      if (st != FDWT_OK) return st;
      conv_step_kernel<T, V><<<static_cast<unsigned>(grid), 128, 0,
                               static_cast<cudaStream_t>(stream)>>>(
          static_cast<const T*>(x), weight, bias, static_cast<T*>(state), slots,
          static_cast<T*>(y), desc->batch, desc->dim, desc->x_stride[0], state_slots, desc->width,
          desc->silu != 0, desc->param_dtype == FDWT_F32);
      return launch_status();
    };
    constexpr int V = sizeof(T) == 8 ? 2 : 4;
    if (grouped<T>(V, desc->dim, {desc->x_stride[0]}, {x, y, state}))
      return launch(std::integral_constant<int, V>{});
    return launch(std::integral_constant<int, 1>{});
  });
}
