// What the norms over rows share (layer_norm.cu, rms_norm.cu): groups of neighbouring elements, sums
// over the threads of a row, and how many threads take a row of a given length.
#pragma once

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

// ------------------------------------------------------------------------------ backward
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

// Blocks of the backward pass: `resident` a multiprocessor, at most one a row group.  Their number
// is that of the partial rows, so the workspace takes the most that can be resident: at most 12
// (blocks of 64 threads, 65536 x 491 fp16: 63 us, and 68 us with at most 8; 16 gain nothing more).
constexpr int kLongParts = 64, kMostResident = 12;
inline int64_t backward_blocks(int64_t rows, const Shape& s, int resident) {
  const int64_t most = imin(kMostResident, 2048 / (s.threads * s.rows));
  return imin(cdiv(rows, s.rows), sm_count() * imin(resident, most));
}


}  // namespace
}  // namespace fdwt
