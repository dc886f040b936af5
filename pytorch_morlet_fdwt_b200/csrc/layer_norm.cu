// Layer norm over the last axis: forward, and the gradients of its input, weight and bias.
//
//   m = mean x, r = 1 / sqrt(mean (x - m)^2 + eps), h = (x - m) r, y = h w + b
//   g = dy w, dx = r (g - mean g - h mean(g h)), dw = sum_rows dy h, db = sum_rows dy
//
// Both directions are bound by HBM (8 and 14 operations an element): each element is read once
// and kept in registers between the sums and the result.  The variance is the mean square of the
// centred values, a second pass over registers, since E x^2 - m^2 cancels for a large mean.
// Sums, statistics and the gradients' partial sums are 32 bits (64 for fp64 rows).
#include <type_traits>

#include "common.cuh"

namespace fdwt {
namespace {

// One aligned group of V elements of type T, loaded and stored as a whole.
template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

template <typename A> __device__ __forceinline__ A warp_sum(A v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of N values over the threads of a row (blockDim.x of them; a multiple of 32).  `slot`
// points at 32 * N cells of shared memory; consecutive calls take different slots, so that one
// barrier a call is enough.
template <typename A, int N>
__device__ __forceinline__ void row_sum(A (&v)[N], A* slot) {
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

template <typename A> __device__ __forceinline__ A inv_sqrt(A v);
template <> __device__ __forceinline__ float inv_sqrt(float v) { return 1.0f / sqrtf(v); }
template <> __device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

// ------------------------------------------------------------------------------ forward
// A row is held by blockDim.x threads, IT groups of V elements each (group i of thread t starts
// at (i * blockDim.x + t) * V: neighbouring lanes read neighbouring groups).  blockDim.y rows a
// block: more than one only where a single warp holds a row.
template <typename T, typename P, int V, int IT>
__global__ void __launch_bounds__(1024)
layer_norm_fwd_kernel(const T* __restrict__ x, const P* __restrict__ weight,
                      const P* __restrict__ bias, T* __restrict__ y,
                      typename AccOf<T>::type* __restrict__ stats, int64_t rows, int dim,
                      typename AccOf<T>::type eps) {
  using A = typename AccOf<T>::type;
  __shared__ A slots[2][32];
  const int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= rows) return;  // whole warps: blockDim.y > 1 only with one warp a row
  const T* xr = x + row * dim;
  Pack<T, V> in[IT];
  A sum[1] = {A(0)};
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * V;
    if (c < dim) {
      in[i] = *reinterpret_cast<const Pack<T, V>*>(xr + c);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] += to_acc(in[i].v[j]);
    }
  }
  row_sum(sum, slots[0]);
  const A mean = sum[0] / A(dim);
  A sq[1] = {A(0)};
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * V;
    if (c < dim) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const A d = to_acc(in[i].v[j]) - mean;
        sq[0] += d * d;
      }
    }
  }
  row_sum(sq, slots[1]);
  const A rstd = inv_sqrt(sq[0] / A(dim) + eps);
  if (stats != nullptr && threadIdx.x == 0) {
    stats[2 * row] = mean;
    stats[2 * row + 1] = rstd;
  }
  T* yr = y + row * dim;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * V;
    if (c < dim) {
      Pack<P, V> w, b;
      if (weight != nullptr) w = *reinterpret_cast<const Pack<P, V>*>(weight + c);
      if (bias != nullptr) b = *reinterpret_cast<const Pack<P, V>*>(bias + c);
      Pack<T, V> out;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        A h = (to_acc(in[i].v[j]) - mean) * rstd;
        if (weight != nullptr) h *= A(to_acc(w.v[j]));
        if (bias != nullptr) h += A(to_acc(b.v[j]));
        out.v[j] = from_acc<T>(h);
      }
      *reinterpret_cast<Pack<T, V>*>(yr + c) = out;
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
// Registers: 2 E sums, E weights and the current and next rows' groups (E / 2 each at 16 bits),
// E = V IT elements a thread; h and g are formed twice rather than kept.
template <typename A> constexpr int bwd_max_threads(int e) {
  const int words = e * int(sizeof(A) / 4);
  return words <= 4 ? 1024 : (words <= 16 ? 512 : 256);
}

template <typename T, typename P, int V, int IT>
__global__ void __launch_bounds__(bwd_max_threads<typename AccOf<T>::type>(V * IT))
layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                      const P* __restrict__ weight,
                      const typename AccOf<T>::type* __restrict__ stats, T* __restrict__ dx,
                      typename AccOf<T>::type* __restrict__ partial, int64_t rows, int dim) {
  using A = typename AccOf<T>::type;
  __shared__ A slots[2][64];
  extern __shared__ unsigned char smem_raw[];
  A* joined = reinterpret_cast<A*>(smem_raw);  // [blockDim.y - 1][2][dim], only blockDim.y > 1

  A dw[IT * V], db[IT * V], w[IT * V];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * V;
    Pack<P, V> pw;
    if (weight != nullptr && c < dim) pw = *reinterpret_cast<const Pack<P, V>*>(weight + c);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dw[i * V + j] = db[i * V + j] = A(0);
      w[i * V + j] = (weight != nullptr && c < dim) ? A(to_acc(pw.v[j])) : A(1);
    }
  }
  const int64_t step = int64_t(gridDim.x) * blockDim.y;
  int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  Pack<T, V> nx[IT], ny[IT];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * V;
      if (c < dim) {
        nx[i] = *reinterpret_cast<const Pack<T, V>*>(x + r * dim + c);
        ny[i] = *reinterpret_cast<const Pack<T, V>*>(dy + r * dim + c);
      }
    }
  };
  A mean = A(0), rstd = A(0);
  if (row < rows) {
    fetch(row);
    mean = stats[2 * row];
    rstd = stats[2 * row + 1];
  }
  int parity = 0;
  for (; row < rows; row += step, parity ^= 1) {
    Pack<T, V> cx[IT], cy[IT];
    const A m = mean, r = rstd;
    A s[2] = {A(0), A(0)};
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      const int c = (i * blockDim.x + threadIdx.x) * V;
      if (c < dim) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int e = i * V + j;
          const A d = to_acc(ny[i].v[j]);
          const A h = (to_acc(nx[i].v[j]) - m) * r;
          const A g = d * w[e];
          dw[e] += d * h;
          db[e] += d;
          s[0] += g;
          s[1] += g * h;
        }
        cx[i] = nx[i];
        cy[i] = ny[i];
      }
    }
    const int64_t next = row + step;
    if (next < rows) {
      fetch(next);
      mean = stats[2 * next];
      rstd = stats[2 * next + 1];
    }
    row_sum(s, slots[parity]);
    const A mg = s[0] / A(dim), mgh = s[1] / A(dim);
    if (dx != nullptr) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * V;
        if (c < dim) {
          Pack<T, V> out;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const A h = (to_acc(cx[i].v[j]) - m) * r;
            const A g = to_acc(cy[i].v[j]) * w[i * V + j];
            out.v[j] = from_acc<T>(r * (g - mg - h * mgh));
          }
          *reinterpret_cast<Pack<T, V>*>(dx + row * dim + c) = out;
        }
      }
    }
  }
  if (partial == nullptr) return;
  if (blockDim.y > 1) {
    if (threadIdx.y > 0) {
      A* mine = joined + int64_t(threadIdx.y - 1) * 2 * dim;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (i * blockDim.x + threadIdx.x) * V;
        if (c < dim) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            mine[c + j] = dw[i * V + j];
            mine[dim + c + j] = db[i * V + j];
          }
        }
      }
    }
    __syncthreads();
    if (threadIdx.y > 0) return;
  }
  A* out = partial + int64_t(blockIdx.x) * 2 * dim;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = (i * blockDim.x + threadIdx.x) * V;
    if (c < dim) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        A a = dw[i * V + j], b = db[i * V + j];
        for (int k = 1; k < blockDim.y; ++k) {
          a += joined[int64_t(k - 1) * 2 * dim + c + j];
          b += joined[int64_t(k - 1) * 2 * dim + dim + c + j];
        }
        out[c + j] = a;
        out[dim + c + j] = b;
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
};

// A thread takes about 8 elements where that fits (enough loads in flight, few threads to join);
// a warp holds a row of up to `warp_elems` elements a lane without any barrier; more items only
// where the row needs them.  False: the row does not fit (the long forms take it).
inline bool row_shape(int64_t groups, int v, int warp_elems, int (*limit)(int), Shape* s) {
  const int most = v > 1 ? 4 : 16;
  if (groups * v <= 32 * warp_elems) {
    int items = 1;
    while (32 * items < groups) items *= 2;
    if (items <= most) {
      *s = {32, items, 8};
      return true;
    }
  }
  for (int items = v >= 8 ? 1 : 8 / v > most ? most : 8 / v; items <= most; items *= 2) {
    const int64_t threads = cdiv(cdiv(groups, items), 32) * 32;
    if (threads <= limit(v * items)) {
      *s = {static_cast<int>(threads), items, 1};
      return true;
    }
  }
  return false;
}
inline int forward_limit(int) { return 1024; }
template <typename A> int backward_limit(int e) { return bwd_max_threads<A>(e); }
inline bool forward_shape(int64_t groups, int v, Shape* s) {
  return row_shape(groups, v, v > 1 ? 32 : 16, forward_limit, s);
}
template <typename A> bool backward_shape(int64_t groups, int v, Shape* s) {
  return row_shape(groups, v, 64 / int(sizeof(A)), backward_limit<A>, s);
}

// fn(std::integral_constant<int, items>) for the items that row_shape returns.
template <int V, typename F> int with_items(int items, F fn) {
  switch (items) {
    case 1: return fn(std::integral_constant<int, 1>{});
    case 2: return fn(std::integral_constant<int, 2>{});
    case 4: return fn(std::integral_constant<int, 4>{});
    default: break;
  }
  if constexpr (V == 1) {
    if (items == 8) return fn(std::integral_constant<int, 8>{});
    return fn(std::integral_constant<int, 16>{});
  }
  return FDWT_ERR_INVALID;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, typename P, int V>
int forward_v(int64_t rows, int64_t dim, const void* x, const void* w, const void* b, double eps,
              void* y, void* stats, bool* done, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  Shape s;
  if (!forward_shape(dim / V, V, &s)) return FDWT_OK;
  *done = true;
  const dim3 block(s.threads, s.rows);
  const int64_t grid = cdiv(rows, s.rows);
  if (grid > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  const int st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  return with_items<V>(s.items, [&](auto items) {
    constexpr int IT = decltype(items)::value;
    layer_norm_fwd_kernel<T, P, V, IT><<<static_cast<unsigned>(grid), block, 0, stream>>>(
        static_cast<const T*>(x), static_cast<const P*>(w), static_cast<const P*>(b),
        static_cast<T*>(y), static_cast<A*>(stats), rows, static_cast<int>(dim),
        static_cast<A>(eps));
    return launch_status();
  });
}

template <typename T, typename P>
int forward(int64_t rows, int64_t dim, const void* x, const void* w, const void* b, double eps,
            void* y, void* stats, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  bool done = false;
  int st;
  if (dim % V == 0 && aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b)) {
    st = forward_v<T, P, V>(rows, dim, x, w, b, eps, y, stats, &done, stream);
    if (done) return st;
  } else {
    st = forward_v<T, P, 1>(rows, dim, x, w, b, eps, y, stats, &done, stream);
    if (done) return st;
  }
  if (rows > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  layer_norm_fwd_long_kernel<T, P><<<static_cast<unsigned>(rows), 1024, 0, stream>>>(
      static_cast<const T*>(x), static_cast<const P*>(w), static_cast<const P*>(b),
      static_cast<T*>(y), static_cast<A*>(stats), dim, static_cast<A>(eps));
  return launch_status();
}

// Blocks of the backward pass: what is resident at once, at most one a row group.  The number
// of partial rows, so also a part of the workspace's size.
inline int64_t backward_blocks(int64_t rows, const Shape& s) {
  const int resident = s.rows > 1 ? 4 : (s.threads <= 256 ? 4 : (s.threads <= 512 ? 2 : 1));
  return imin(cdiv(rows, s.rows), int64_t(sm_count()) * resident);
}
constexpr int kLongParts = 64;

// The largest of the counts that the aligned and the unaligned form use, so that the query needs
// no pointers.
inline int64_t backward_parts(int dtype, int64_t rows, int64_t dim) {
  const int v = static_cast<int>(16 / dtype_size(dtype));
  int64_t parts = 0;
  for (int per : {v, 1}) {
    if (per > 1 && dim % per != 0) continue;
    Shape s;
    const bool fits = dtype == FDWT_F64 ? backward_shape<double>(dim / per, per, &s)
                                        : backward_shape<float>(dim / per, per, &s);
    parts = imax(parts, fits ? backward_blocks(rows, s) : imin(rows, kLongParts));
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
  const int64_t grid = backward_blocks(rows, s);
  *parts = grid;
  const dim3 block(s.threads, s.rows);
  const size_t smem = partial == nullptr ? 0 : size_t(s.rows - 1) * 2 * dim * sizeof(A);
  return with_items<V>(s.items, [&](auto items) -> int {
    constexpr int IT = decltype(items)::value;
    auto kernel = layer_norm_bwd_kernel<T, P, V, IT>;
    int st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
    if (st == FDWT_OK) st = pre_launch(stream);
    if (st != FDWT_OK) return st;
    kernel<<<static_cast<unsigned>(grid), block, smem, stream>>>(
        static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const P*>(w),
        static_cast<const A*>(stats), static_cast<T*>(dx), static_cast<A*>(partial), rows,
        static_cast<int>(dim));
    return launch_status();
  });
}

template <typename T, typename P>
int backward(int64_t rows, int64_t dim, const void* dy, const void* x, const void* w,
             const void* stats, void* dx, void* dw, void* db, void* ws, cudaStream_t stream) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  void* partial = (dw != nullptr || db != nullptr) ? ws : nullptr;
  int64_t parts = 0;
  int st;
  if (dim % V == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(w))
    st = backward_v<T, P, V>(rows, dim, dy, x, w, stats, dx, partial, &parts, stream);
  else
    st = backward_v<T, P, 1>(rows, dim, dy, x, w, stats, dx, partial, &parts, stream);
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
