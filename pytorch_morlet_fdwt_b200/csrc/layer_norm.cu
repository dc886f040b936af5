// Layer norm over the last axis: forward, and the gradients of its input, weight and bias.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   g = dy w, dx = r (g - mean g - h mean(g h)), dw = sum_rows dy h, db = sum_rows dy
//
// Both directions are bound by HBM (8 and 14 operations an element): each element is read once
// and kept in registers between the sums and the result.  The variance is the mean square of the
// centred values, a second pass over registers, since E x^2 - m^2 cancels for a large mean.
// Sums, statistics and the gradients' partial sums are 32 bits (64 for fp64 rows).
//
// Measured: 65536 x 2048 bf16 forward 96 us (5.6 TB/s), backward 165 us (4.9 TB/s); 65536 x 1024
// fp32 88 and 133 us (6.1 TB/s both); 40000 x 1001 fp32, whose rows start off 16-byte boundaries,
// 55 and 88 us (5.8 and 5.5 TB/s); 32768 x 1024 fp64 84 and 132 us (6.4 and 6.1 TB/s).  Rows too
// long for registers: 16384 x 12288 bf16 181 and 728 us (4.4 and 1.7 TB/s).
#include <initializer_list>
#include <type_traits>

#include "common.cuh"

namespace fdwt {
namespace {

// A group of V neighbouring elements, loaded and stored as a whole (16 bytes, two elements, or one),
// and its values in the type of the sums.
template <typename T, int V> struct Group {
  struct alignas(sizeof(T) * V) Raw {
    T v[V];
  };
  using A = typename AccOf<T>::type;
  static __device__ __forceinline__ Raw load(const T* p) {
    return *reinterpret_cast<const Raw*>(p);
  }
  static __device__ __forceinline__ void values(const Raw& r, A* x) {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = to_acc(r.v[j]);
  }
  static __device__ __forceinline__ void store(T* p, const A* x) {
    Raw r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = from_acc<T>(x[j]);
    *reinterpret_cast<Raw*>(p) = r;
  }
};
// 16-bit types in pairs: one conversion instruction a pair.
template <typename T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
  static __device__ __forceinline__ void split(uint32_t u, float* x) {
    x[0] = __uint_as_float(u << 16);
    x[1] = __uint_as_float(u & 0xffff0000u);
  }
  static __device__ __forceinline__ uint32_t join(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <> struct Half2<__half> {
  static __device__ __forceinline__ void split(uint32_t u, float* x) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    x[0] = f.x;
    x[1] = f.y;
  }
  static __device__ __forceinline__ uint32_t join(float a, float b) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <typename T> struct Group16 {
  using Raw = uint4;
  static __device__ __forceinline__ Raw load(const T* p) {
    return *reinterpret_cast<const uint4*>(p);
  }
  static __device__ __forceinline__ void values(const Raw& r, float* x) {
    Half2<T>::split(r.x, x);
    Half2<T>::split(r.y, x + 2);
    Half2<T>::split(r.z, x + 4);
    Half2<T>::split(r.w, x + 6);
  }
  static __device__ __forceinline__ void store(T* p, const float* x) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(Half2<T>::join(x[0], x[1]), Half2<T>::join(x[2], x[3]),
                   Half2<T>::join(x[4], x[5]), Half2<T>::join(x[6], x[7]));
  }
};
template <typename T> struct Group4 {
  using Raw = uint32_t;
  static __device__ __forceinline__ Raw load(const T* p) {
    return *reinterpret_cast<const uint32_t*>(p);
  }
  static __device__ __forceinline__ void values(const Raw& r, float* x) { Half2<T>::split(r, x); }
  static __device__ __forceinline__ void store(T* p, const float* x) {
    *reinterpret_cast<uint32_t*>(p) = Half2<T>::join(x[0], x[1]);
  }
};
template <> struct Group<__half, 2> : Group4<__half> {};
template <> struct Group<__nv_bfloat16, 2> : Group4<__nv_bfloat16> {};
template <> struct Group<__half, 8> : Group16<__half> {};
template <> struct Group<__nv_bfloat16, 8> : Group16<__nv_bfloat16> {};

// V parameters (weight or bias) as values: V elements of their own type, loaded 16 bytes (all of
// them, where they are fewer) at a time.  group_of() sees to their alignment.
template <typename P, int V, typename A>
__device__ __forceinline__ void load_params(const P* p, A* x) {
  if constexpr (sizeof(P) * V == 32) {
    float y[4];
    Group<float, 4>::values(Group<float, 4>::load(p), y);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = y[j];
    Group<float, 4>::values(Group<float, 4>::load(p + 4), y);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 + j] = y[j];
  } else {
    Group<P, V>::values(Group<P, V>::load(p), x);
  }
}

template <typename A> __device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of N values over the threads of a row: blockDim.x of them, either a power of two up to 32
// (lanes of one warp) or whole warps.  `slot` points at 32 N cells of shared memory; consecutive
// calls take different slots, so that one barrier a call is enough.
template <typename A, int N>
__device__ __forceinline__ void row_sum(A (&v)[N], A* slot) {
  if (blockDim.x < 32) {
    for (int o = blockDim.x / 2; o > 0; o >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if (blockDim.x == 32) return;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) slot[i * 32 + warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? slot[i * 32 + lane] : A(0));
}

// The same over NT threads, known when compiling (whole warps).
template <int NT, typename A, int N>
__device__ __forceinline__ void row_sum_of(A (&v)[N], A* slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
  if constexpr (NT > 32) {
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slot[i * 32 + (threadIdx.x >> 5)] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = slot[i * 32];
#pragma unroll
      for (int w = 1; w < NT / 32; ++w) v[i] += slot[i * 32 + w];
    }
  }
}

template <typename A> __device__ __forceinline__ A inv_sqrt(A v);
template <> __device__ __forceinline__ float inv_sqrt(float v) { return 1.0f / sqrtf(v); }
template <> __device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// ------------------------------------------------------------------------------ forward
// Threads a block may have when each keeps e elements.
constexpr int fwd_max_threads(int e) { return e <= 16 ? 1024 : (e <= 32 ? 512 : 256); }
// Blocks of that size a multiprocessor must hold: loads in flight count for more than registers
// (65536 x 2048 bf16: 106 us without, 96 us with).
constexpr int fwd_min_blocks(int e) { return e <= 8 ? 2 : (e <= 16 ? 1 : (e <= 32 ? 2 : 3)); }

// Single elements and pairs cost many instructions a byte, and with addresses and conditions worked
// out for every one of them the kernel is bound by those (85 % of issue slots, 40000 x 1001 fp32:
// 78 us, bf16: 86 us).  Their rows of more than 128 groups therefore take a number of threads
// known when compiling (NT, 32 to 512) and the 6 or 8 groups a thread that are enough: the offsets
// become constants and only the last two groups need a condition (54 and 50 us).
constexpr int fwd_row_threads(int nt) { return nt == 32 ? 128 : nt; }  // rows a block: 4 or 1
constexpr int fwd_threads(int e, int nt) { return nt ? fwd_row_threads(nt) : fwd_max_threads(e); }
constexpr int fwd_blocks(int e, int nt, int size) {
  return nt ? (e * size <= 32 ? 2048 : (e * size <= 64 ? 1024 : 512)) / fwd_row_threads(nt)
            : fwd_min_blocks(e);
}

// A row is held by blockDim.x threads, IT groups of V elements each (group i of thread t starts
// at (i * blockDim.x + t) * V: neighbouring lanes read neighbouring groups), blockDim.y rows a
// block (more than one only where a row has at most a warp).
template <typename T, typename P, int V, int IT, int NT>
__global__ void __launch_bounds__(fwd_threads(V * IT, NT),
                                  fwd_blocks(V * IT, NT, sizeof(typename AccOf<T>::type)))
layer_norm_fwd_kernel(const T* __restrict__ x, const P* __restrict__ weight,
                      const P* __restrict__ bias, T* __restrict__ y,
                      typename AccOf<T>::type* __restrict__ stats, int64_t rows, int dim,
                      typename AccOf<T>::type eps) {
  using A = typename AccOf<T>::type;
  using G = Group<T, V>;
  __shared__ A slots[2][32];
  int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool in = row < rows;
  if (!in) row = rows - 1;  // the lanes of a warp stay together
  const T* xr = x + row * dim + threadIdx.x * V;
  const int step = (NT ? NT : int(blockDim.x)) * V, left = dim - threadIdx.x * V;
  constexpr int SURE = NT ? IT - 2 : 0;  // groups that every thread has
  typename G::Raw raw[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i)
    if (i < SURE || i * step < left) raw[i] = G::load(xr + i * step);
  A v[IT * V];
  A sum[1] = {A(0)}, part[4] = {A(0), A(0), A(0), A(0)};
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    if (i < SURE || i * step < left) {
      G::values(raw[i], v + i * V);
#pragma unroll
      for (int j = 0; j < V; ++j) part[(i * V + j) % 4] += v[i * V + j];
    }
  }
  sum[0] = (part[0] + part[1]) + (part[2] + part[3]);
  if constexpr (NT) row_sum_of<NT>(sum, slots[0]);
  else row_sum(sum, slots[0]);
  const A mean = sum[0] / A(dim);
#pragma unroll
  for (int k = 0; k < 4; ++k) part[k] = A(0);
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    if (i < SURE || i * step < left) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        A& d = v[i * V + j];
        d -= mean;
        part[(i * V + j) % 4] += d * d;
      }
    }
  }
  sum[0] = (part[0] + part[1]) + (part[2] + part[3]);
  if constexpr (NT) row_sum_of<NT>(sum, slots[1]);
  else row_sum(sum, slots[1]);
  const A rstd = inv_sqrt(sum[0] / A(dim) + eps);
  if (!in) return;
  if (stats != nullptr && threadIdx.x == 0) {
    stats[2 * row] = mean;
    stats[2 * row + 1] = rstd;
  }
  T* yr = y + row * dim + threadIdx.x * V;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    if (i < SURE || i * step < left) {
      A p[V];
      A* d = v + i * V;
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] *= rstd;
      if (weight != nullptr) {
        load_params<P, V>(weight + threadIdx.x * V + i * step, p);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] *= p[j];
      }
      if (bias != nullptr) {
        load_params<P, V>(bias + threadIdx.x * V + i * step, p);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] += p[j];
      }
      G::store(yr + i * step, d);
    }
  }
}

// Rows too long for the registers of a block: three passes over the row (the second and third
// find it in L2).
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
layer_norm_fwd_long_kernel(const T* __restrict__ x, const P* __restrict__ weight,
                           const P* __restrict__ bias, T* __restrict__ y,
                           typename AccOf<T>::type* __restrict__ stats, int64_t dim,
                           typename AccOf<T>::type eps) {
  using A = typename AccOf<T>::type;
  __shared__ A slots[2][32];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * dim;
  A sum[1] = {A(0)};
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) sum[0] += to_acc(xr[c]);
  row_sum(sum, slots[0]);
  const A mean = sum[0] / A(dim);
  A sq[1] = {A(0)};
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
    const A d = to_acc(xr[c]) - mean;
    sq[0] += d * d;
  }
  row_sum(sq, slots[1]);
  const A rstd = inv_sqrt(sq[0] / A(dim) + eps);
  if (stats != nullptr && threadIdx.x == 0) {
    stats[2 * row] = mean;
    stats[2 * row + 1] = rstd;
  }
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
    A h = (to_acc(xr[c]) - mean) * rstd;
    if (weight != nullptr) h *= A(to_acc(weight[c]));
    if (bias != nullptr) h += A(to_acc(bias[c]));
    y[row * dim + c] = from_acc<T>(h);
  }
}

// ------------------------------------------------------------------------------ backward
// Persistent blocks walk the rows (block b takes the row groups b, b + gridDim.x, ...), each
// thread keeping its columns' sums of dy h and dy in registers; a block ends by adding its rows'
// sums in shared memory (blockDim.y > 1) and writing one (dw, db) partial row.  The partial rows
// are added in a fixed order by layer_norm_params_kernel: no atomics, the same bits every run.
// The next row's x and dy are loaded before the current row's sums are joined.
// Registers, E = V IT elements a thread: 2 E sums, E weights, 2 E values, and the next row's groups.
template <typename A> constexpr int bwd_max_threads(int e) {
  const int words = e * int(sizeof(A) / 4);
  return words <= 4 ? 1024 : (words <= 16 ? 512 : 256);
}

// Rows of single elements and pairs take NT threads and constant offsets as in the forward pass
// (40000 x 1001: fp32 113 -> 88 us, bf16 113 -> 70 us; 65536 x 491 fp16 118 -> 63 us).
constexpr int bwd_row_threads(int nt) { return nt == 32 ? 256 : nt; }  // rows a block: 8 or 1
template <typename A> constexpr int bwd_threads(int e, int nt) {
  return nt ? bwd_row_threads(nt) : bwd_max_threads<A>(e);
}

template <typename T, typename P, int V, int IT, int NT>
__global__ void __launch_bounds__(bwd_threads<typename AccOf<T>::type>(V * IT, NT))
layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                      const P* __restrict__ weight,
                      const typename AccOf<T>::type* __restrict__ stats, T* __restrict__ dx,
                      typename AccOf<T>::type* __restrict__ partial, int64_t rows, int dim) {
  using A = typename AccOf<T>::type;
  using G = Group<T, V>;
  __shared__ A slots[2][64];
  extern __shared__ __align__(16) unsigned char smem_raw[];
  A* joined = reinterpret_cast<A*>(smem_raw);  // [blockDim.y][2][dim], only blockDim.y > 1

  const int col = threadIdx.x * V, left = dim - col;
  const int step = (NT ? NT : int(blockDim.x)) * V;
  constexpr int SURE = NT ? IT - 2 / V : 0;  // groups that every thread has
  A dw[IT * V], db[IT * V], w[IT * V];
#pragma unroll
  for (int e = 0; e < IT * V; ++e) {
    dw[e] = db[e] = A(0);
    w[e] = A(1);
  }
  if (weight != nullptr) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (i < SURE || i * step < left) load_params<P, V>(weight + col + i * step, w + i * V);
  }
  const int64_t rows_step = int64_t(gridDim.x) * blockDim.y;
  // rows of the block's last round past the end are read as the last row and left out of the sums
  int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const int64_t rounds = (rows - int64_t(blockIdx.x) * blockDim.y + rows_step - 1) / rows_step;
  typename G::Raw nx[IT], ny[IT];
  A mean, rstd;
  auto fetch = [&](int64_t r) {
    if (r >= rows) r = rows - 1;
    const T* px = x + r * dim + col;
    const T* py = dy + r * dim + col;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i < SURE || i * step < left) {
        nx[i] = G::load(px + i * step);
        ny[i] = G::load(py + i * step);
      }
    }
    mean = stats[2 * r];
    rstd = stats[2 * r + 1];
  };
  fetch(row);
  const A inv = A(1) / A(dim);
  for (int64_t k = 0; k < rounds; ++k, row += rows_step) {
    const bool in = row < rows;
    const A m = mean, r = rstd;
    A h[IT * V], g[IT * V];
    A s[2] = {A(0), A(0)}, s1[2] = {A(0), A(0)};
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i < SURE || i * step < left) {
        A d[V];
        G::values(nx[i], h + i * V);
        G::values(ny[i], d);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int e = i * V + j;
          h[e] = (h[e] - m) * r;
          if (!in) d[j] = A(0);
          g[e] = d[j] * w[e];
          dw[e] += d[j] * h[e];
          db[e] += d[j];
          s[e % 2] += g[e];
          s1[e % 2] += g[e] * h[e];
        }
      }
    }
    if (k + 1 < rounds) fetch(row + rows_step);
    s[0] += s[1];
    s[1] = s1[0] + s1[1];
    if constexpr (NT) row_sum_of<NT>(s, slots[k & 1]);
    else row_sum(s, slots[k & 1]);
    const A mg = s[0] * inv, mgh = s[1] * inv;
    if (dx != nullptr && in) {
      T* out = dx + row * dim + col;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        if (i < SURE || i * step < left) {
          A d[V];
#pragma unroll
          for (int j = 0; j < V; ++j) d[j] = r * (g[i * V + j] - mg - h[i * V + j] * mgh);
          G::store(out + i * step, d);
        }
      }
    }
  }
  if (partial == nullptr) return;
  if (blockDim.y > 1) {  // join the block's rows in shared memory, a fixed order
    A* mine = joined + int64_t(threadIdx.y) * 2 * dim;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i < SURE || i * step < left) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          mine[col + i * step + j] = dw[i * V + j];
          mine[dim + col + i * step + j] = db[i * V + j];
        }
      }
    }
    __syncthreads();
    const int threads = blockDim.x * blockDim.y;
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < 2 * dim; c += threads) {
      A a = joined[c];
      for (int y = 1; y < blockDim.y; ++y) a += joined[int64_t(y) * 2 * dim + c];
      partial[int64_t(blockIdx.x) * 2 * dim + c] = a;
    }
    return;
  }
  A* out = partial + int64_t(blockIdx.x) * 2 * dim + col;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    if (i < SURE || i * step < left) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        out[i * step + j] = dw[i * V + j];
        out[dim + i * step + j] = db[i * V + j];
      }
    }
  }
}

// Rows too long for a block's registers: one block a row for dx, and dy h, dy summed over the
// rows by a grid over the columns (each row group of it writes a partial row).
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
layer_norm_bwd_long_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                           const P* __restrict__ weight,
                           const typename AccOf<T>::type* __restrict__ stats,
                           T* __restrict__ dx, int64_t dim) {
  using A = typename AccOf<T>::type;
  __shared__ A slots[64];
  const int64_t row = blockIdx.x;
  const A mean = stats[2 * row], rstd = stats[2 * row + 1];
  A s[2] = {A(0), A(0)};
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
    A g = to_acc(dy[row * dim + c]);
    if (weight != nullptr) g *= A(to_acc(weight[c]));
    s[0] += g;
    s[1] += g * (to_acc(x[row * dim + c]) - mean) * rstd;
  }
  row_sum(s, slots);
  const A mg = s[0] / A(dim), mgh = s[1] / A(dim);
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
    A g = to_acc(dy[row * dim + c]);
    if (weight != nullptr) g *= A(to_acc(weight[c]));
    const A h = (to_acc(x[row * dim + c]) - mean) * rstd;
    dx[row * dim + c] = from_acc<T>(rstd * (g - mg - h * mgh));
  }
}

template <typename T>
__global__ void __launch_bounds__(256)
layer_norm_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                          const typename AccOf<T>::type* __restrict__ stats,
                          typename AccOf<T>::type* __restrict__ partial, int64_t rows,
                          int64_t dim) {
  using A = typename AccOf<T>::type;
  const int64_t c = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (c >= dim) return;
  A dw = A(0), db = A(0);
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const A d = to_acc(dy[r * dim + c]);
    dw += d * (to_acc(x[r * dim + c]) - stats[2 * r]) * stats[2 * r + 1];
    db += d;
  }
  partial[int64_t(blockIdx.y) * 2 * dim + c] = dw;
  partial[int64_t(blockIdx.y) * 2 * dim + dim + c] = db;
}

// dw and db from the partial rows: 32 columns by 8 row lanes a block, joined in a fixed order.
template <typename A, typename P>
__global__ void __launch_bounds__(256)
layer_norm_params_kernel(const A* __restrict__ partial, int parts, int64_t dim,
                         P* __restrict__ dw, P* __restrict__ db) {
  __shared__ A cells[8][33];
  const int64_t c = int64_t(blockIdx.x) * 32 + threadIdx.x;  // over (dw, db): 2 * dim columns
  A sum = A(0);
  if (c < 2 * dim) {
#pragma unroll 8
    for (int p = threadIdx.y; p < parts; p += 8) sum += partial[int64_t(p) * 2 * dim + c];
  }
  cells[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y != 0 || c >= 2 * dim) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) sum += cells[k][threadIdx.x];
  if (c < dim) {
    if (dw != nullptr) dw[c] = from_acc<P>(sum);
  } else if (db != nullptr) {
    db[c - dim] = from_acc<P>(sum);
  }
}

// ------------------------------------------------------------------------------ launches
// Threads a row, groups a thread and rows a block for rows of `groups` groups.
struct Shape {
  int threads, items, rows;
  bool narrow = false;  // of narrow_shape: the kernels know the number of threads
};

// Lanes and groups of a row that one warp holds: with few elements a row several rows share a warp
// (no lanes idle), with many a lane takes more (no barrier, more loads in flight).
inline bool warp_shape(int64_t groups, int v, int most_items, Shape* s, int block) {
  int threads = 1, items = 1;
  while (threads * items < groups) {
    // 32 bytes a row and load keep the sectors whole; then items up to about 8 elements a lane,
    // then lanes, then items again
    if (threads < 4 || (threads < 32 && items * v >= 8)) threads *= 2;
    else if (items * v < 8) items *= 2;
    else items *= 2;
    if (items > most_items) return false;
  }
  *s = {threads, items, block / threads, false};
  return true;
}
// Rows of single elements or pairs, up to 512 threads of `most` groups: threads a power of two, 3/4
// of `most` or `most` groups a thread, of which the last quarter of `most` alone can be past the
// row's end.  The lower bound is what 32 threads need for that.
inline bool narrow_shape(int64_t groups, int most, int block, Shape* s) {
  if (groups <= 16 * most || groups > 512 * most) return false;
  int threads = 32;
  while (threads * most < groups) threads *= 2;
  *s = {threads, threads * (most * 3 / 4) >= groups ? most * 3 / 4 : most,
        threads == 32 ? block / 32 : 1, true};
  return true;
}
inline bool forward_shape(int64_t groups, int v, int acc_size, Shape* s) {
  if (v <= 2 && narrow_shape(groups, 8, 128, s)) return true;
  if (warp_shape(groups, v, v <= 2 ? 8 : (acc_size == 8 ? 32 : 64) / v, s, 128)) return true;
  for (int items = v >= 8 ? 4 : (v <= 2 ? 8 : 32 / v); items * v <= 32; items *= 2) {
    const int64_t threads = cdiv(cdiv(groups, items), 32) * 32;
    if (threads <= fwd_max_threads(items * v)) {
      *s = {static_cast<int>(threads), items, 1, false};
      return true;
    }
  }
  return false;
}
template <typename A> bool backward_shape(int64_t groups, int v, Shape* s) {
  if (v <= 2 && narrow_shape(groups, 8 / v, 256, s)) return true;
  if (warp_shape(groups, v, (sizeof(A) == 8 ? 8 : (v > 2 ? 32 : 16)) / v, s, 256)) return true;
  for (int items = v >= 8 ? 2 : (v <= 2 ? 8 : 16) / v; items * v <= 32; items *= 2) {
    const int64_t threads = cdiv(cdiv(groups, items), 32) * 32;
    if (threads <= bwd_max_threads<A>(v * items)) {
      *s = {static_cast<int>(threads), items, 1, false};
      return true;
    }
  }
  return false;
}

// fn(std::integral_constant<int, threads>) for the threads of narrow_shape.
template <typename F> int with_threads(int threads, F fn) {
  switch (threads) {
    case 32: return fn(std::integral_constant<int, 32>{});
    case 64: return fn(std::integral_constant<int, 64>{});
    case 128: return fn(std::integral_constant<int, 128>{});
    case 256: return fn(std::integral_constant<int, 256>{});
    case 512: return fn(std::integral_constant<int, 512>{});
    default: return FDWT_ERR_INVALID;
  }
}

// fn(std::integral_constant<int, items>); items V at most `MOST` elements.
template <int V, int MOST, typename F> int with_items(int items, F fn) {
  switch (items) {
    case 1: return fn(std::integral_constant<int, 1>{});
    case 2: return fn(std::integral_constant<int, 2>{});
    case 4:
      if constexpr (4 * V <= MOST) return fn(std::integral_constant<int, 4>{});
      break;
    case 8:
      if constexpr (8 * V <= MOST) return fn(std::integral_constant<int, 8>{});
      break;
    case 16:
      if constexpr (16 * V <= MOST) return fn(std::integral_constant<int, 16>{});
      break;
    case 32:
      if constexpr (32 * V <= MOST) return fn(std::integral_constant<int, 32>{});
      break;
    default: break;
  }
  return FDWT_ERR_INVALID;
}

template <typename T, typename P, int V>
int forward_v(int64_t rows, int64_t dim, const void* x, const void* w, const void* b, double eps,
              void* y, void* stats, bool* done, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  Shape s;
  if (!forward_shape(dim / V, V, sizeof(A), &s)) return FDWT_OK;
  *done = true;
  const dim3 block(s.threads, s.rows);
  const int64_t grid = cdiv(rows, s.rows);
  if (grid > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  const int st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  auto launch = [&](auto items, auto threads) {
    layer_norm_fwd_kernel<T, P, V, decltype(items)::value, decltype(threads)::value>
        <<<static_cast<unsigned>(grid), block, 0, stream>>>(
            static_cast<const T*>(x), static_cast<const P*>(w), static_cast<const P*>(b),
            static_cast<T*>(y), static_cast<A*>(stats), rows, static_cast<int>(dim),
            static_cast<A>(eps));
    return launch_status();
  };
  if constexpr (V <= 2) {
    if (s.narrow)
      return with_threads(s.threads, [&](auto threads) {
        return s.items == 6 ? launch(std::integral_constant<int, 6>{}, threads)
                            : launch(std::integral_constant<int, 8>{}, threads);
      });
  }
  return with_items<V, (V <= 2 ? 16 : sizeof(A) == 8 ? 32 : 64)>(
      s.items, [&](auto items) { return launch(items, std::integral_constant<int, 0>{}); });
}

// Elements of a group: 16 bytes, two elements or one, whatever rows and pointers are aligned to.
// Parameters of another type than the rows' have groups of another size (fp32 beside 16 bits: a
// pair is 8 bytes, not 4), so each of the two is tested by its own.
using Pointers = std::initializer_list<const void*>;
template <typename T, typename P> int group_of(int64_t dim, Pointers rows, Pointers params) {
  uintptr_t x = 0, p = 0;
  for (const void* q : rows) x |= reinterpret_cast<uintptr_t>(q);
  for (const void* q : params) p |= reinterpret_cast<uintptr_t>(q);
  constexpr int V = 16 / sizeof(T);
  if (dim % V == 0 && x % 16 == 0 && p % 16 == 0) return V;
  if (V > 2 && dim % 2 == 0 && x % (2 * sizeof(T)) == 0 && p % (2 * sizeof(P)) == 0) return 2;
  return 1;
}

template <typename T, typename P>
int forward(int64_t rows, int64_t dim, const void* x, const void* w, const void* b, double eps,
            void* y, void* stats, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  bool done = false;
  int st;
  const int v = group_of<T, P>(dim, {x, y}, {w, b});
  if (v == V) st = forward_v<T, P, V>(rows, dim, x, w, b, eps, y, stats, &done, stream);
  else if (v == 2) st = forward_v<T, P, 2>(rows, dim, x, w, b, eps, y, stats, &done, stream);
  else st = forward_v<T, P, 1>(rows, dim, x, w, b, eps, y, stats, &done, stream);
  if (done) return st;
  if (rows > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  layer_norm_fwd_long_kernel<T, P><<<static_cast<unsigned>(rows), 1024, 0, stream>>>(
      static_cast<const T*>(x), static_cast<const P*>(w), static_cast<const P*>(b),
      static_cast<T*>(y), static_cast<A*>(stats), dim, static_cast<A>(eps));
  return launch_status();
}

// Blocks of the backward pass: `resident` a multiprocessor, at most one a row group.  Their number
// is that of the partial rows, so the workspace takes the most that can be resident: at most 12
// (blocks of 64 threads, 65536 x 491 fp16: 63 us, and 68 us with at most 8; 16 gain nothing more).
constexpr int kLongParts = 64, kMostResident = 12;
inline int64_t backward_blocks(int64_t rows, const Shape& s, int resident) {
  const int64_t most = imin(kMostResident, 2048 / (s.threads * s.rows));
  return imin(cdiv(rows, s.rows), sm_count() * imin(resident, most));
}

// The largest of the counts that the forms for every alignment use: the query has no pointers.
inline int64_t backward_parts(int dtype, int64_t rows, int64_t dim) {
  const int v = static_cast<int>(16 / dtype_size(dtype));
  int64_t parts = 0;
  for (int per : {v, 2, 1}) {
    if (per > 1 && dim % per != 0) continue;
    Shape s;
    const bool fits = dtype == FDWT_F64 ? backward_shape<double>(dim / per, per, &s)
                                        : backward_shape<float>(dim / per, per, &s);
    parts = imax(parts, fits ? backward_blocks(rows, s, kMostResident) : imin(rows, kLongParts));
  }
  return parts;
}

template <typename T, typename P>
int params(const void* partial, int64_t parts, int64_t dim, void* dw, void* db,
           cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  const int st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  layer_norm_params_kernel<A, P><<<static_cast<unsigned>(cdiv(2 * dim, 32)), dim3(32, 8), 0,
                                   stream>>>(static_cast<const A*>(partial),
                                             static_cast<int>(parts), dim, static_cast<P*>(dw),
                                             static_cast<P*>(db));
  return launch_status();
}

template <typename T, typename P, int V>
int backward_v(int64_t rows, int64_t dim, const void* dy, const void* x, const void* w,
               const void* stats, void* dx, void* partial, int64_t* parts, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  Shape s;
  if (!backward_shape<A>(dim / V, V, &s)) return FDWT_OK;
  const dim3 block(s.threads, s.rows);
  const size_t smem =
      partial == nullptr || s.rows == 1 ? 0 : size_t(s.rows) * 2 * dim * sizeof(A);
  auto launch = [&](auto items, auto threads) -> int {
    auto kernel =
        layer_norm_bwd_kernel<T, P, V, decltype(items)::value, decltype(threads)::value>;
    int resident = 1;
    int st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
    if (st == FDWT_OK)
      st = occupancy(reinterpret_cast<const void*>(kernel), s.threads * s.rows, smem, &resident);
    if (st == FDWT_OK) st = pre_launch(stream);
    if (st != FDWT_OK) return st;
    const int64_t grid = backward_blocks(rows, s, resident < 1 ? 1 : resident);
    *parts = grid;
    kernel<<<static_cast<unsigned>(grid), block, smem, stream>>>(
        static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const P*>(w),
        static_cast<const A*>(stats), static_cast<T*>(dx), static_cast<A*>(partial), rows,
        static_cast<int>(dim));
    return launch_status();
  };
  if constexpr (V <= 2) {
    if (s.narrow)
      return with_threads(s.threads, [&](auto threads) {
        return s.items == 6 / V ? launch(std::integral_constant<int, 6 / V>{}, threads)
                                : launch(std::integral_constant<int, 8 / V>{}, threads);
      });
  }
  return with_items<V, (V <= 2 && sizeof(A) == 4 ? 16 : 32)>(
      s.items, [&](auto items) { return launch(items, std::integral_constant<int, 0>{}); });
}

template <typename T, typename P>
int backward(int64_t rows, int64_t dim, const void* dy, const void* x, const void* w,
             const void* stats, void* dx, void* dw, void* db, void* ws, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  void* partial = (dw != nullptr || db != nullptr) ? ws : nullptr;
  int64_t parts = 0;
  int st;
  const int v = group_of<T, P>(dim, {x, dy, dx}, {w});
  if (v == V) st = backward_v<T, P, V>(rows, dim, dy, x, w, stats, dx, partial, &parts, stream);
  else if (v == 2) st = backward_v<T, P, 2>(rows, dim, dy, x, w, stats, dx, partial, &parts, stream);
  else st = backward_v<T, P, 1>(rows, dim, dy, x, w, stats, dx, partial, &parts, stream);
  if (st != FDWT_OK) return st;
  if (parts == 0) {  // long rows
    if (rows > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
    if (dx != nullptr) {
      st = pre_launch(stream);
      if (st != FDWT_OK) return st;
      layer_norm_bwd_long_kernel<T, P><<<static_cast<unsigned>(rows), 1024, 0, stream>>>(
          static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const P*>(w),
          static_cast<const A*>(stats), static_cast<T*>(dx), dim);
      st = launch_status();
      if (st != FDWT_OK) return st;
    }
    parts = imin(rows, kLongParts);
    if (partial != nullptr) {
      st = pre_launch(stream);
      if (st != FDWT_OK) return st;
      layer_norm_columns_kernel<T><<<dim3(static_cast<unsigned>(cdiv(dim, 256)),
                                          static_cast<unsigned>(parts)), 256, 0, stream>>>(
          static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const A*>(stats),
          static_cast<A*>(partial), rows, dim);
      st = launch_status();
      if (st != FDWT_OK) return st;
    }
  }
  if (partial == nullptr) return FDWT_OK;
  return params<T, P>(partial, parts, dim, dw, db, stream);
}

inline bool types_ok(int dtype, int param_dtype) {
  if (dtype_size(dtype) == 0) return false;
  return param_dtype == dtype || (param_dtype == FDWT_F32 && dtype != FDWT_F64);
}

// fn(element type tag, parameter type tag)
template <typename F> int dispatch(int dtype, int param_dtype, F fn) {
  const bool same = dtype == param_dtype;
  switch (dtype) {
    case FDWT_F32: return fn(float{}, float{});
    case FDWT_F64: return fn(double{}, double{});
    case FDWT_F16: return same ? fn(__half{}, __half{}) : fn(__half{}, float{});
    default: return same ? fn(__nv_bfloat16{}, __nv_bfloat16{}) : fn(__nv_bfloat16{}, float{});
  }
}

}  // namespace
}  // namespace fdwt

using namespace fdwt;

extern "C" int fdwt_layer_norm_forward(int dtype, int param_dtype, int64_t rows, int64_t dim,
                                       const void* x, const void* weight, const void* bias,
                                       double eps, void* y, void* stats, void* stream) {
  FDWT_CHECK(types_ok(dtype, param_dtype) && rows >= 0 && dim >= 1 && eps >= 0);
  if (rows == 0) return FDWT_OK;
  FDWT_CHECK(x != nullptr && y != nullptr);
  return dispatch(dtype, param_dtype, [&](auto t, auto p) {
    return forward<decltype(t), decltype(p)>(rows, dim, x, weight, bias, eps, y, stats,
                                             static_cast<cudaStream_t>(stream));
  });
}

extern "C" size_t fdwt_layer_norm_backward_workspace(int dtype, int64_t rows, int64_t dim,
                                                     int need_params) {
  if (dtype_size(dtype) == 0 || rows <= 0 || dim < 1 || !need_params) return 0;
  return size_t(backward_parts(dtype, rows, dim)) * 2 * dim * (dtype == FDWT_F64 ? 8 : 4);
}

extern "C" int fdwt_layer_norm_backward(int dtype, int param_dtype, int64_t rows, int64_t dim,
                                        const void* dy, const void* x, const void* weight,
                                        const void* stats, void* dx, void* dweight, void* dbias,
                                        void* workspace, size_t workspace_bytes, void* stream) {
  FDWT_CHECK(types_ok(dtype, param_dtype) && rows >= 0 && dim >= 1);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t psize = dtype_size(param_dtype);
  if (rows == 0) {  // no rows: the sums over rows are zero
    if (dweight != nullptr) FDWT_CUDA(cudaMemsetAsync(dweight, 0, dim * psize, s));
    if (dbias != nullptr) FDWT_CUDA(cudaMemsetAsync(dbias, 0, dim * psize, s));
    return FDWT_OK;
  }
  FDWT_CHECK(dy != nullptr && x != nullptr && stats != nullptr);
  const bool need = dweight != nullptr || dbias != nullptr;
  if (dx == nullptr && !need) return FDWT_OK;
  const size_t bytes = fdwt_layer_norm_backward_workspace(dtype, rows, dim, need);
  if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes)) return FDWT_ERR_WORKSPACE;
  return dispatch(dtype, param_dtype, [&](auto t, auto p) {
    return backward<decltype(t), decltype(p)>(rows, dim, dy, x, weight, stats, dx, dweight, dbias,
                                              workspace, s);
  });
}
