// Root-mean-square norm over the last axis with the residual's addition: forward, gradients, and
// a result in 8 bits with scales.
//
//   t = x + r (rounded to r's type), i = 1 / sqrt(mean t^2 + eps), h = t i, y = h w
//   g = dy w, dt = i (g - h mean(g h)) + dtotal, dx = dr = dt, dw = sum_rows dy h
//   8 bits: s = max |y| / m over a group (m = 448 for e4m3, 127 for int8), q = round(y / s)
//
// t is rounded before the norm: y is the norm of the sum as it is stored, so that a fused call
// gives what an addition and a norm of its result give, and the backward pass, which reads t,
// differentiates the function that the forward pass computed.
//
// Bound by HBM (5, 8 and 16 operations an element): each element is read once and kept in
// registers between the sum and the result, 16 bytes a load.  Sums and statistics are 32 bits
// (64 for fp64 rows); y is rounded once, to its type or to 8 bits.
//
// Measured with the residual: 65536 x 2048 bf16 forward 170 us (6.3 TB/s), backward 171 us (6.3
// TB/s); 16384 x 8192 bf16 164 us both (6.5 TB/s); 40000 x 1001 fp32 106 and 90 us (6.0 and 7.1 TB/s
// with what L2 holds), bf16 72 and 78 us; 32768 x 2048 bf16 to e4m3 in groups of 128 84 us (5.6
// TB/s), 40000 x 1001 bf16 to e4m3 137 us.
#include <cuda_fp8.h>

#include "row_groups.cuh"

namespace fdwt {
namespace {

// V elements of the residual's type: a group of its own type, or 32 bytes of fp32 beside 16-bit
// rows in two loads.
template <typename R, int V> struct Stream : Group<R, V> {};
template <> struct Stream<float, 8> {
  struct Raw {
    float4 a, b;
  };
  static __device__ __forceinline__ Raw load(const float* p) {
    return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
  }
  static __device__ __forceinline__ void values(const Raw& r, float* x) {
    x[0] = r.a.x, x[1] = r.a.y, x[2] = r.a.z, x[3] = r.a.w;
    x[4] = r.b.x, x[5] = r.b.y, x[6] = r.b.z, x[7] = r.b.w;
  }
  static __device__ __forceinline__ void store(float* p, const float* x) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
};

// Values of 8 bits: the largest magnitude, and one value scaled and rounded.
struct E4m3 {
  uint8_t bits;
};
struct Int8 {
  int8_t value;
};
template <typename O> struct Quant;
template <> struct Quant<E4m3> {
  static constexpr float kMost = 448.0f;
  static __device__ __forceinline__ uint8_t one(float v) {
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
  }
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
};
template <> struct Quant<Int8> {
  static constexpr float kMost = 127.0f;
  // (NaN becomes some number: its scale is NaN)
  static __device__ __forceinline__ uint8_t one(float v) {
    return static_cast<uint8_t>(__float2int_rn(fminf(fmaxf(v, -127.0f), 127.0f)));
  }
  static __device__ __forceinline__ uint32_t pair(float a, float b) {
    return one(a) | uint32_t(one(b)) << 8;
  }
};
template <typename O> constexpr bool is_quant = false;
template <> constexpr bool is_quant<E4m3> = true;
template <> constexpr bool is_quant<Int8> = true;

// V values over their scale, rounded; 8, 4, 2 or 1 bytes in one store.  Both divisions, by the scale
// and of the largest magnitude, are products with reciprocals: two or three roundings in 32 bits more
// than one, which decide only between two neighbours in 8 bits as near as that (32768 x 2048 bf16 in
// groups of 128: 132 us with divisions, 90 us without).
template <typename O, int V>
__device__ __forceinline__ void store_quant(O* p, const float* x, float inv) {
  if constexpr (V == 1) {
    *reinterpret_cast<uint8_t*>(p) = Quant<O>::one(x[0] * inv);
  } else {
    static_assert(V == 4 || V == 8);
    uint32_t w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = Quant<O>::pair(x[4 * i] * inv, x[4 * i + 1] * inv) |
             Quant<O>::pair(x[4 * i + 2] * inv, x[4 * i + 3] * inv) << 16;
    if constexpr (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}
// The scale of a group whose largest magnitude is m: 1 where all are zero, else at least 2^-126 (the
// smallest normal number), so that its reciprocal is finite.  NaN stays NaN.
template <typename O> __device__ __forceinline__ float scale_of(float m) {
  return m == 0.0f ? 1.0f : max_nan(m * (1.0f / Quant<O>::kMost), 0x1p-126f);
}
__device__ __forceinline__ float inverse(float scale) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  return r;
}

// The largest over the threads of a row, as row_sum adds.
__device__ __forceinline__ float row_max(float v, float* slot) {
  const int lanes = blockDim.x < 32 ? blockDim.x : 32;
  for (int o = lanes / 2; o > 0; o >>= 1)
    v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (blockDim.x <= 32) return v;
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  v = lane < warps ? slot[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// ------------------------------------------------------------------------------ forward
// Rows by threads as in layer_norm_fwd_kernel.  O: the rows' type, or one of 8 bits, whose groups
// are the whole row (lanes = 0) or `lanes` neighbouring threads' groups (a power of two within a
// warp and a row).
template <typename T, typename R, typename P, typename O, int V, int IT, int NT>
__global__ void __launch_bounds__(fwd_threads(V * IT, NT),
                                  fwd_blocks(V * IT, NT, sizeof(typename AccOf<T>::type)))
rms_fwd_kernel(const T* __restrict__ x, const R* __restrict__ residual,
               const P* __restrict__ weight, O* __restrict__ y, R* __restrict__ total,
               typename AccOf<T>::type* __restrict__ rstd_out, float* __restrict__ scales,
               int lanes, int64_t rows, int dim, typename AccOf<T>::type eps) {
  using A = typename AccOf<T>::type;
  using G = Group<T, V>;
  using S = Stream<R, V>;
  __shared__ A slots[2][32];
  int64_t row = int64_t(blockIdx.x) * blockDim.y + threadIdx.y;
  const bool in = row < rows;
  if (!in) row = rows - 1;  // the lanes of a warp stay together
  const int64_t at = row * dim + threadIdx.x * V;
  const int step = (NT ? NT : int(blockDim.x)) * V, left = dim - threadIdx.x * V;
  constexpr int SURE = NT ? IT - 2 : 0;  // groups that every thread has
  typename G::Raw raw[IT];
  typename S::Raw more[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i)
    if (i < SURE || i * step < left) raw[i] = G::load(x + at + i * step);
  if (residual != nullptr) {
#pragma unroll
    for (int i = 0; i < IT; ++i)
      if (i < SURE || i * step < left) more[i] = S::load(residual + at + i * step);
  }
  A v[IT * V];
  A sum[1], part[4] = {A(0), A(0), A(0), A(0)};
#pragma unroll
  for (int i = 0; i < IT; ++i) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[i * V + j] = A(0);
    if (i < SURE || i * step < left) {
      A* d = v + i * V;
      G::values(raw[i], d);
      if (residual != nullptr) {
        A r[V];
        S::values(more[i], r);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = to_acc(from_acc<R>(d[j] + r[j]));
        if (in) S::store(total + at + i * step, d);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) part[(i * V + j) % 4] += d[j] * d[j];
    }
  }
  sum[0] = (part[0] + part[1]) + (part[2] + part[3]);
  if constexpr (NT) row_sum_of<NT>(sum, slots[0]);
  else row_sum(sum, slots[0]);
  const A rstd = inv_sqrt(sum[0] / A(dim) + eps);
  if (rstd_out != nullptr && in && threadIdx.x == 0) rstd_out[row] = rstd;
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
      if constexpr (!is_quant<O>) {
        if (in) Group<T, V>::store(y + at + i * step, d);
      }
    }
  }
  if constexpr (is_quant<O>) {
    float m[IT];
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      m[i] = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) m[i] = max_nan(m[i], fabsf(static_cast<float>(v[i * V + j])));
    }
    if (lanes == 0) {
#pragma unroll
      for (int i = 1; i < IT; ++i) m[0] = max_nan(m[0], m[i]);
      const float scale = scale_of<O>(row_max(m[0], reinterpret_cast<float*>(slots[1])));
      if (in && threadIdx.x == 0) scales[row] = scale;
      const float inv = inverse(scale);
#pragma unroll
      for (int i = 0; i < IT; ++i)
        if (in && i * step < left) store_quant<O, V>(y + at + i * step, v + i * V, inv);
    } else {
      const int group = lanes * V;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        for (int o = lanes / 2; o > 0; o >>= 1)
          m[i] = max_nan(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
        const float scale = scale_of<O>(m[i]);
        if (in && i * step < left) {
          if (threadIdx.x % lanes == 0) scales[(at + i * step) / group] = scale;
          store_quant<O, V>(y + at + i * step, v + i * V, inverse(scale));
        }
      }
    }
  }
}

// Rows too long for the registers of a block, rows off 16-byte boundaries with a result in 8 bits or an
// fp32 residual, and 8-bit groups that the lanes of a warp do not share evenly: element by element,
// the row kept in shared memory between the passes (CACHED) where that holds it, else found in L2.
constexpr int64_t kCachedBytes = 32768;
template <typename T, typename R, typename P, typename O, bool CACHED>
__global__ void __launch_bounds__(1024)
rms_fwd_long_kernel(const T* __restrict__ x, const R* __restrict__ residual,
                    const P* __restrict__ weight, O* __restrict__ y, R* total,
                    typename AccOf<T>::type* __restrict__ rstd_out, float* __restrict__ scales,
                    int64_t group, int64_t dim, typename AccOf<T>::type eps) {
  using A = typename AccOf<T>::type;
  __shared__ A slots[2][32];
  extern __shared__ __align__(16) unsigned char smem_raw[];
  A* cache = reinterpret_cast<A*>(smem_raw);
  const int64_t row = blockIdx.x, at = row * dim;
  A sum[1] = {A(0)};
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
    A v = to_acc(x[at + c]);
    if (residual != nullptr) {
      const R t = from_acc<R>(v + A(to_acc(residual[at + c])));
      total[at + c] = t;
      v = to_acc(t);
    }
    if (CACHED) cache[c] = v;
    sum[0] += v * v;
  }
  row_sum(sum, slots[0]);
  const A rstd = inv_sqrt(sum[0] / A(dim) + eps);
  if (rstd_out != nullptr && threadIdx.x == 0) rstd_out[row] = rstd;
  auto value = [&](int64_t c) {
    A v;
    if (CACHED) v = cache[c];
    else v = residual != nullptr ? A(to_acc(total[at + c])) : A(to_acc(x[at + c]));
    v *= rstd;
    if (weight != nullptr) v *= A(to_acc(weight[c]));
    return v;
  };
  if constexpr (!is_quant<O>) {
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) y[at + c] = from_acc<T>(value(c));
  } else if (group == dim) {
    float m = 0.0f;
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
      const A v = value(c);
      if (CACHED) cache[c] = v;
      m = max_nan(m, fabsf(static_cast<float>(v)));
    }
    const float scale = scale_of<O>(row_max(m, reinterpret_cast<float*>(slots[1])));
    if (threadIdx.x == 0) scales[row] = scale;
    const float inv = inverse(scale);
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
      const float v = static_cast<float>(CACHED ? cache[c] : value(c));
      store_quant<O, 1>(y + at + c, &v, inv);
    }
  } else {
    __syncthreads();  // a group's lanes read what other threads have stored
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    for (int64_t g = threadIdx.x >> 5; g < dim / group; g += warps) {
      float m = 0.0f;
      for (int64_t c = g * group + lane; c < (g + 1) * group; c += 32)
        m = max_nan(m, fabsf(static_cast<float>(value(c))));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float scale = scale_of<O>(m);
      if (lane == 0) scales[row * (dim / group) + g] = scale;
      const float inv = inverse(scale);
      for (int64_t c = g * group + lane; c < (g + 1) * group; c += 32) {
        const float v = static_cast<float>(value(c));
        store_quant<O, 1>(y + at + c, &v, inv);
      }
    }
  }
}

// ------------------------------------------------------------------------------ backward
// Persistent blocks walk the rows as in layer_norm_bwd_kernel: sums of dy h in registers, one
// partial row a block, added in a fixed order by rms_weight_kernel.
template <typename T, typename R, typename P, int V, int IT, int NT>
__global__ void __launch_bounds__(bwd_threads<typename AccOf<T>::type>(V * IT, NT))
rms_bwd_kernel(const T* __restrict__ dy, const R* __restrict__ dtotal,
               const R* __restrict__ total, const P* __restrict__ weight,
               const typename AccOf<T>::type* __restrict__ rstds, T* __restrict__ dx,
               R* __restrict__ dresidual, typename AccOf<T>::type* __restrict__ partial,
               int64_t rows, int dim) {
  using A = typename AccOf<T>::type;
  using G = Group<T, V>;
  using S = Stream<R, V>;
  __shared__ A slots[2][32];
  extern __shared__ __align__(16) unsigned char smem_raw[];
  A* joined = reinterpret_cast<A*>(smem_raw);  // [blockDim.y][dim], only blockDim.y > 1

  const int col = threadIdx.x * V, left = dim - col;
  const int step = (NT ? NT : int(blockDim.x)) * V;
  constexpr int SURE = NT ? IT - 2 / V : 0;  // groups that every thread has
  A dw[IT * V], w[IT * V];
#pragma unroll
  for (int e = 0; e < IT * V; ++e) {
    dw[e] = A(0);
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
  typename S::Raw nt[IT], ns[IT];
  typename G::Raw ny[IT];
  A rstd;
  auto fetch = [&](int64_t r) {
    if (r >= rows) r = rows - 1;
    const int64_t at = r * dim + col;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i < SURE || i * step < left) {
        nt[i] = S::load(total + at + i * step);
        ny[i] = G::load(dy + at + i * step);
        if (dtotal != nullptr) ns[i] = S::load(dtotal + at + i * step);
      }
    }
    rstd = rstds[r];
  };
  fetch(row);
  const A inv = A(1) / A(dim);
  for (int64_t k = 0; k < rounds; ++k, row += rows_step) {
    const bool in = row < rows;
    const A r = rstd;
    A h[IT * V], g[IT * V];
    typename S::Raw ds[IT];
    A s[1], part[2] = {A(0), A(0)};
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i < SURE || i * step < left) {
        A d[V];
        S::values(nt[i], h + i * V);
        G::values(ny[i], d);
        ds[i] = ns[i];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int e = i * V + j;
          h[e] *= r;
          if (!in) d[j] = A(0);
          g[e] = d[j] * w[e];
          dw[e] += d[j] * h[e];
          part[e % 2] += g[e] * h[e];
        }
      }
    }
    if (k + 1 < rounds) fetch(row + rows_step);
    s[0] = part[0] + part[1];
    if constexpr (NT) row_sum_of<NT>(s, slots[k & 1]);
    else row_sum(s, slots[k & 1]);
    const A mgh = s[0] * inv;
    if (dx != nullptr && in) {
      const int64_t at = row * dim + col;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        if (i < SURE || i * step < left) {
          A d[V];
#pragma unroll
          for (int j = 0; j < V; ++j) d[j] = r * (g[i * V + j] - h[i * V + j] * mgh);
          if (dtotal != nullptr) {
            A q[V];
            S::values(ds[i], q);
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] += q[j];
          }
          G::store(dx + at + i * step, d);
          if (dresidual != nullptr) S::store(dresidual + at + i * step, d);
        }
      }
    }
  }
  if (partial == nullptr) return;
  if (blockDim.y > 1) {  // join the block's rows in shared memory, a fixed order
    A* mine = joined + int64_t(threadIdx.y) * dim;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      if (i < SURE || i * step < left) {
#pragma unroll
        for (int j = 0; j < V; ++j) mine[col + i * step + j] = dw[i * V + j];
      }
    }
    __syncthreads();
    const int threads = blockDim.x * blockDim.y;
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < dim; c += threads) {
      A a = joined[c];
      for (int y = 1; y < blockDim.y; ++y) a += joined[int64_t(y) * dim + c];
      partial[int64_t(blockIdx.x) * dim + c] = a;
    }
    return;
  }
  A* out = partial + int64_t(blockIdx.x) * dim + col;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    if (i < SURE || i * step < left) {
#pragma unroll
      for (int j = 0; j < V; ++j) out[i * step + j] = dw[i * V + j];
    }
  }
}

// Rows too long for a block's registers: one block a row for dx, and dy h summed over the rows by
// a grid over the columns (each row group of it writes a partial row).
template <typename T, typename R, typename P>
__global__ void __launch_bounds__(1024)
rms_bwd_long_kernel(const T* __restrict__ dy, const R* __restrict__ dtotal,
                    const R* __restrict__ total, const P* __restrict__ weight,
                    const typename AccOf<T>::type* __restrict__ rstds, T* __restrict__ dx,
                    R* __restrict__ dresidual, int64_t dim) {
  using A = typename AccOf<T>::type;
  __shared__ A slots[32];
  const int64_t row = blockIdx.x;
  const A rstd = rstds[row];
  auto grad = [&](int64_t c) {
    A g = to_acc(dy[row * dim + c]);
    if (weight != nullptr) g *= A(to_acc(weight[c]));
    return g;
  };
  A s[1] = {A(0)};
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x)
    s[0] += grad(c) * (A(to_acc(total[row * dim + c])) * rstd);
  row_sum(s, slots);
  const A mgh = s[0] / A(dim);
  for (int64_t c = threadIdx.x; c < dim; c += blockDim.x) {
    A d = rstd * (grad(c) - A(to_acc(total[row * dim + c])) * rstd * mgh);
    if (dtotal != nullptr) d += A(to_acc(dtotal[row * dim + c]));
    dx[row * dim + c] = from_acc<T>(d);
    if (dresidual != nullptr) dresidual[row * dim + c] = from_acc<R>(d);
  }
}

template <typename T, typename R>
__global__ void __launch_bounds__(256)
rms_columns_kernel(const T* __restrict__ dy, const R* __restrict__ total,
                   const typename AccOf<T>::type* __restrict__ rstds,
                   typename AccOf<T>::type* __restrict__ partial, int64_t rows, int64_t dim) {
  using A = typename AccOf<T>::type;
  const int64_t c = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (c >= dim) return;
  A dw = A(0);
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y)
    dw += A(to_acc(dy[r * dim + c])) * (A(to_acc(total[r * dim + c])) * rstds[r]);
  partial[int64_t(blockIdx.y) * dim + c] = dw;
}

// dw from the partial rows: 32 columns by 8 row lanes a block, joined in a fixed order.
template <typename A, typename P>
__global__ void __launch_bounds__(256)
rms_weight_kernel(const A* __restrict__ partial, int parts, int64_t dim, P* __restrict__ dw) {
  __shared__ A cells[8][33];
  const int64_t c = int64_t(blockIdx.x) * 32 + threadIdx.x;
  A sum = A(0);
  if (c < dim) {
#pragma unroll 8
    for (int p = threadIdx.y; p < parts; p += 8) sum += partial[int64_t(p) * dim + c];
  }
  cells[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y != 0 || c >= dim) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) sum += cells[k][threadIdx.x];
  dw[c] = from_acc<P>(sum);
}

// ------------------------------------------------------------------------------ launches
struct ForwardCall {
  int64_t rows, dim, group;
  const void *x, *residual, *weight;
  double eps;
  void *y, *total, *rstd, *scales;
  cudaStream_t stream;
};

// Elements of a group as group_of, with the residual's rows beside: fp32 ones next to 16-bit rows
// take 16-byte loads or the long kernel (no forms of pairs for them).
template <typename T, typename R, typename P>
int rms_group(int64_t dim, Pointers rows, Pointers streams, Pointers params) {
  uintptr_t s = 0;
  for (const void* q : streams) s |= reinterpret_cast<uintptr_t>(q);
  const int v = group_of<T, P>(dim, rows, params);
  if constexpr (std::is_same_v<T, R>) {
    if (v == 1 || s % 16 == 0) return v;
    return dim % 2 == 0 && sizeof(T) == 2 && s % 4 == 0 && v > 1 ? 2 : 1;
  }
  return v == 16 / sizeof(T) && s % 16 == 0 ? v : 0;
}

// Threads of a row whose 8-bit groups are `lanes` threads wide: at least so many.  32 elements a
// thread: with the largest magnitudes beside the sums, 64 (as forward_shape takes) are slower
// (32768 x 2048 bf16: 125 us; 32: 90, 16: 92, 8: 100).
inline bool quant_shape(int64_t groups, int v, int lanes, Shape* s) {
  int threads = 32, items = 1;
  while (threads > 1 && threads / 2 >= groups && threads / 2 >= lanes) threads /= 2;
  while (threads * items < groups) items *= 2;
  if (items * v <= 32) {
    *s = {threads, items, 128 / threads, false};
    return lanes <= threads;
  }
  for (items = 4; items * v <= 32; items *= 2) {
    const int64_t wide = cdiv(cdiv(groups, items), 32) * 32;
    if (wide <= fwd_max_threads(items * v)) {
      *s = {static_cast<int>(wide), items, 1, false};
      return true;
    }
  }
  return false;
}

template <typename T, typename R, typename P, typename O, int V>
int rms_forward_v(const ForwardCall& c, bool* done) {
  using A = typename AccOf<T>::type;
  Shape s;
  int lanes = 0;
  if constexpr (is_quant<O>) {
    if (c.group != c.dim) {
      if (c.group % V != 0 || c.group / V > 32 || (c.group / V & (c.group / V - 1))) return FDWT_OK;
      lanes = static_cast<int>(c.group / V);
    }
    if (!quant_shape(c.dim / V, V, lanes, &s)) return FDWT_OK;
  } else {
    if (!forward_shape(c.dim / V, V, sizeof(A), &s)) return FDWT_OK;
  }
  *done = true;
  const dim3 block(s.threads, s.rows);
  const int64_t grid = cdiv(c.rows, s.rows);
  if (grid > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  const int st = pre_launch(c.stream);
  if (st != FDWT_OK) return st;
  auto launch = [&](auto items, auto threads) {
    rms_fwd_kernel<T, R, P, O, V, decltype(items)::value, decltype(threads)::value>
        <<<static_cast<unsigned>(grid), block, 0, c.stream>>>(
            static_cast<const T*>(c.x), static_cast<const R*>(c.residual),
            static_cast<const P*>(c.weight), static_cast<O*>(c.y), static_cast<R*>(c.total),
            static_cast<A*>(c.rstd), static_cast<float*>(c.scales), lanes, c.rows,
            static_cast<int>(c.dim), static_cast<A>(c.eps));
    return launch_status();
  };
  if constexpr (V <= 2 && !is_quant<O>) {
    if (s.narrow)
      return with_threads(s.threads, [&](auto threads) {
        return s.items == 6 ? launch(std::integral_constant<int, 6>{}, threads)
                            : launch(std::integral_constant<int, 8>{}, threads);
      });
  }
  constexpr int most = V <= 2 ? 16 : sizeof(A) == 8 ? 32 : 64;
  return with_items<V, most>(
      s.items, [&](auto items) { return launch(items, std::integral_constant<int, 0>{}); });
}

template <typename T, typename R, typename P, typename O> int rms_forward(const ForwardCall& c) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  constexpr bool same = std::is_same_v<T, R>;
  bool done = false;
  int st = FDWT_OK;
  const int v = rms_group<T, R, P>(c.dim, {c.x, c.y}, {c.residual, c.total}, {c.weight});
  if (v == V) st = rms_forward_v<T, R, P, O, V>(c, &done);
  if constexpr (same && !is_quant<O>) {
    if (v == 2 && V > 2) st = rms_forward_v<T, R, P, O, 2>(c, &done);
    else if (v == 1) st = rms_forward_v<T, R, P, O, 1>(c, &done);
  }
  if (done || st != FDWT_OK) return st;
  if (c.rows > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  st = pre_launch(c.stream);
  if (st != FDWT_OK) return st;
  auto launch = [&](auto cached) {
    constexpr bool CACHED = decltype(cached)::value;
    const int threads = c.dim <= 1024 ? 128 : (c.dim <= 4096 ? 256 : 1024);
    rms_fwd_long_kernel<T, R, P, O, CACHED>
        <<<static_cast<unsigned>(c.rows), threads, CACHED ? c.dim * sizeof(A) : 0, c.stream>>>(
            static_cast<const T*>(c.x), static_cast<const R*>(c.residual),
            static_cast<const P*>(c.weight), static_cast<O*>(c.y), static_cast<R*>(c.total),
            static_cast<A*>(c.rstd), static_cast<float*>(c.scales), c.group, c.dim,
            static_cast<A>(c.eps));
    return launch_status();
  };
  return c.dim * int64_t(sizeof(A)) <= kCachedBytes ? launch(std::true_type{})
                                                    : launch(std::false_type{});
}

struct BackwardCall {
  int64_t rows, dim;
  const void *dy, *dtotal, *total, *weight, *rstd;
  void *dx, *dresidual, *dweight, *partial;
  cudaStream_t stream;
};

// The largest of the counts that the forms for every alignment use: the query has no pointers.
inline int64_t rms_parts(int dtype, int64_t rows, int64_t dim) {
  const int v = static_cast<int>(16 / dtype_size(dtype));
  int64_t parts = imin(rows, kLongParts);
  for (int per : {v, 2, 1}) {
    if (per > 1 && dim % per != 0) continue;
    Shape s;
    const bool fits = dtype == FDWT_F64 ? backward_shape<double>(dim / per, per, &s)
                                        : backward_shape<float>(dim / per, per, &s);
    if (fits) parts = imax(parts, backward_blocks(rows, s, kMostResident));
  }
  return parts;
}

template <typename T, typename R, typename P, int V>
int rms_backward_v(const BackwardCall& c, int64_t* parts) {
  using A = typename AccOf<T>::type;
  Shape s;
  if (!backward_shape<A>(c.dim / V, V, &s)) return FDWT_OK;
  const dim3 block(s.threads, s.rows);
  const size_t smem = c.partial == nullptr || s.rows == 1 ? 0 : size_t(s.rows) * c.dim * sizeof(A);
  auto launch = [&](auto items, auto threads) -> int {
    auto kernel = rms_bwd_kernel<T, R, P, V, decltype(items)::value, decltype(threads)::value>;
    int resident = 1;
    int st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
    if (st == FDWT_OK)
      st = occupancy(reinterpret_cast<const void*>(kernel), s.threads * s.rows, smem, &resident);
    if (st == FDWT_OK) st = pre_launch(c.stream);
    if (st != FDWT_OK) return st;
    const int64_t grid = backward_blocks(c.rows, s, resident < 1 ? 1 : resident);
    *parts = grid;
    kernel<<<static_cast<unsigned>(grid), block, smem, c.stream>>>(
        static_cast<const T*>(c.dy), static_cast<const R*>(c.dtotal),
        static_cast<const R*>(c.total), static_cast<const P*>(c.weight),
        static_cast<const A*>(c.rstd), static_cast<T*>(c.dx), static_cast<R*>(c.dresidual),
        static_cast<A*>(c.partial), c.rows, static_cast<int>(c.dim));
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

template <typename T, typename R, typename P> int rms_backward(const BackwardCall& c) {
  using A = typename AccOf<T>::type;
  constexpr int V = 16 / sizeof(T);
  constexpr bool same = std::is_same_v<T, R>;
  int64_t parts = 0;
  int st = FDWT_OK;
  const int v = rms_group<T, R, P>(c.dim, {c.dy, c.dx}, {c.total, c.dtotal, c.dresidual},
                                   {c.weight});
  if (v == V) st = rms_backward_v<T, R, P, V>(c, &parts);
  if constexpr (same) {
    if (v == 2 && V > 2) st = rms_backward_v<T, R, P, 2>(c, &parts);
    else if (v == 1) st = rms_backward_v<T, R, P, 1>(c, &parts);
  }
  if (st != FDWT_OK) return st;
  if (parts == 0) {  // long rows
    if (c.rows > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
    if (c.dx != nullptr) {
      st = pre_launch(c.stream);
      if (st != FDWT_OK) return st;
      rms_bwd_long_kernel<T, R, P><<<static_cast<unsigned>(c.rows), 1024, 0, c.stream>>>(
          static_cast<const T*>(c.dy), static_cast<const R*>(c.dtotal),
          static_cast<const R*>(c.total), static_cast<const P*>(c.weight),
          static_cast<const A*>(c.rstd), static_cast<T*>(c.dx), static_cast<R*>(c.dresidual),
          c.dim);
      st = launch_status();
      if (st != FDWT_OK) return st;
    }
    parts = imin(c.rows, kLongParts);
    if (c.partial != nullptr) {
      st = pre_launch(c.stream);
      if (st != FDWT_OK) return st;
      rms_columns_kernel<T, R><<<dim3(static_cast<unsigned>(cdiv(c.dim, 256)),
                                      static_cast<unsigned>(parts)), 256, 0, c.stream>>>(
          static_cast<const T*>(c.dy), static_cast<const R*>(c.total),
          static_cast<const A*>(c.rstd), static_cast<A*>(c.partial), c.rows, c.dim);
      st = launch_status();
      if (st != FDWT_OK) return st;
    }
  }
  if (c.partial == nullptr) return FDWT_OK;
  st = pre_launch(c.stream);
  if (st != FDWT_OK) return st;
  rms_weight_kernel<A, P><<<static_cast<unsigned>(cdiv(c.dim, 32)), dim3(32, 8), 0, c.stream>>>(
      static_cast<const A*>(c.partial), static_cast<int>(parts), c.dim,
      static_cast<P*>(c.dweight));
  return launch_status();
}

inline bool rms_types_ok(int dtype, int residual_dtype, int param_dtype) {
  if (dtype_size(dtype) == 0) return false;
  for (int other : {residual_dtype, param_dtype})
    if (other != dtype && (other != FDWT_F32 || dtype == FDWT_F64)) return false;
  return true;
}

// fn(tags of the rows', the residual's and the parameter's type)
template <typename T, typename F> int rms_dispatch16(bool r, bool p, F fn) {
  if (r) return p ? fn(T{}, T{}, T{}) : fn(T{}, T{}, float{});
  return p ? fn(T{}, float{}, T{}) : fn(T{}, float{}, float{});
}
template <typename F> int rms_dispatch(int dtype, int residual_dtype, int param_dtype, F fn) {
  const bool r = residual_dtype == dtype, p = param_dtype == dtype;
  switch (dtype) {
    case FDWT_F32: return fn(float{}, float{}, float{});
    case FDWT_F64: return fn(double{}, double{}, double{});
    case FDWT_F16: return rms_dispatch16<__half>(r, p, fn);
    default: return rms_dispatch16<__nv_bfloat16>(r, p, fn);
  }
}

}  // namespace
}  // namespace fdwt

using namespace fdwt;

extern "C" int fdwt_rms_norm_forward(int dtype, int residual_dtype, int param_dtype, int64_t rows,
                                     int64_t dim, const void* x, const void* residual,
                                     const void* weight, double eps, void* y, void* total,
                                     void* rstd, void* stream) {
  FDWT_CHECK(rms_types_ok(dtype, residual_dtype, param_dtype) && rows >= 0 && dim >= 1 &&
             dim <= INT32_MAX && eps >= 0);
  if (rows == 0) return FDWT_OK;
  FDWT_CHECK(x != nullptr && y != nullptr && (residual == nullptr) == (total == nullptr));
  const ForwardCall c{rows, dim, dim, x, residual, weight, eps, y, total, rstd, nullptr,
                      static_cast<cudaStream_t>(stream)};
  return rms_dispatch(dtype, residual_dtype, param_dtype, [&](auto t, auto r, auto p) {
    using T = decltype(t);
    return rms_forward<T, decltype(r), decltype(p), T>(c);
  });
}

extern "C" int fdwt_rms_norm_quantized(int dtype, int residual_dtype, int param_dtype,
                                       int out_type, int64_t rows, int64_t dim, int64_t group,
                                       const void* x, const void* residual, const void* weight,
                                       double eps, void* q, void* scales, void* total,
                                       void* stream) {
  FDWT_CHECK(rms_types_ok(dtype, residual_dtype, param_dtype) && rows >= 0 && dim >= 1 &&
             dim <= INT32_MAX && eps >= 0 && group >= 1 && dim % group == 0);
  FDWT_CHECK(out_type == FDWT_E4M3 || out_type == FDWT_INT8);
  if (dtype == FDWT_F64) return FDWT_ERR_UNSUPPORTED;
  if (rows == 0) return FDWT_OK;
  FDWT_CHECK(x != nullptr && q != nullptr && scales != nullptr &&
             (residual == nullptr) == (total == nullptr));
  const ForwardCall c{rows, dim, group, x, residual, weight, eps, q, total, nullptr, scales,
                      static_cast<cudaStream_t>(stream)};
  return rms_dispatch(dtype, residual_dtype, param_dtype, [&](auto t, auto r, auto p) -> int {
    using T = decltype(t);
    if constexpr (std::is_same_v<T, double>) return FDWT_ERR_UNSUPPORTED;
    else
      return out_type == FDWT_E4M3 ? rms_forward<T, decltype(r), decltype(p), E4m3>(c)
                                   : rms_forward<T, decltype(r), decltype(p), Int8>(c);
  });
}

extern "C" size_t fdwt_rms_norm_backward_workspace(int dtype, int64_t rows, int64_t dim,
                                                   int need_weight) {
  if (dtype_size(dtype) == 0 || rows <= 0 || dim < 1 || !need_weight) return 0;
  return size_t(rms_parts(dtype, rows, dim)) * dim * (dtype == FDWT_F64 ? 8 : 4);
}

extern "C" int fdwt_rms_norm_backward(int dtype, int residual_dtype, int param_dtype, int64_t rows,
                                      int64_t dim, const void* dy, const void* dtotal,
                                      const void* total, const void* weight, const void* rstd,
                                      void* dx, void* dresidual, void* dweight, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  FDWT_CHECK(rms_types_ok(dtype, residual_dtype, param_dtype) && rows >= 0 && dim >= 1 &&
             dim <= INT32_MAX && (dx != nullptr || dresidual == nullptr));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (rows == 0) {  // no rows: the sum over rows is zero
    if (dweight != nullptr) FDWT_CUDA(cudaMemsetAsync(dweight, 0, dim * dtype_size(param_dtype), s));
    return FDWT_OK;
  }
  if (dx == nullptr && dweight == nullptr) return FDWT_OK;
  FDWT_CHECK(dy != nullptr && total != nullptr && rstd != nullptr);
  const size_t bytes = fdwt_rms_norm_backward_workspace(dtype, rows, dim, dweight != nullptr);
  if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes)) return FDWT_ERR_WORKSPACE;
  const BackwardCall c{rows, dim, dy, dtotal, total, weight, rstd, dx, dresidual, dweight,
                       dweight != nullptr ? workspace : nullptr, s};
  return rms_dispatch(dtype, residual_dtype, param_dtype, [&](auto t, auto r, auto p) {
    return rms_backward<decltype(t), decltype(r), decltype(p)>(c);
  });
}
