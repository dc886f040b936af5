// Linear attention with a decay for each head: entry points, the general kernels (every type,
// size and stride; products on the FMA pipes, or as pairs of TF32 values), the sum over segments,
// and the single-token form.
// The mathematics, the jobs and the segments are in linattn.cuh.
#include <type_traits>

#include "linattn.cuh"

namespace fdwt {
namespace linattn {
namespace {

template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// d^n for n >= 0.  d^0 = 1 also for d = 0 (log decay -inf).
__device__ __forceinline__ float decay_pow(float a, float n) {
  return n == 0.0f ? 1.0f : expf(a * n);
}
__device__ __forceinline__ double decay_pow(double a, double n) {
  return n == 0.0 ? 1.0 : exp(a * n);
}

__device__ __forceinline__ int64_t valid_tokens(const Call& c, int64_t b) {
  if (c.lengths == nullptr) return c.length;
  const int64_t n = c.lengths[b];
  return n < 0 ? 0 : (n > c.length ? c.length : n);
}

// Position in the tensors of token l of the job's order; rows past the end keep their place.
__device__ __forceinline__ int64_t token_of(int64_t l, int64_t n, int reverse) {
  return reverse && l < n ? n - 1 - l : l;
}

// rows x cols of a tensor (row l at base + token * stride) into shared memory, zeros past
// `valid` rows and `cols` columns.  256 threads; where no conversion is due and rows are aligned
// the copies are asynchronous (tiles_wait() below), else all loads are issued before the stores:
// one latency a tile instead of one a group (5 x 1537 tokens, 6 heads of 48 x 80, fp32: 163 -> 129 us
// for both launches at that step, 123 us now).
template <typename T, typename A, int ROWS, int COLS, int PITCH>
__device__ __forceinline__ void load_tile(A* dst, const T* base, int64_t stride, int64_t l0,
                                          int64_t n, int reverse, int valid, int cols, int vec) {
  constexpr int V = 16 / sizeof(T);
  if (vec) {
    constexpr int N = (ROWS * (COLS / V) + 255) / 256;
    if constexpr (std::is_same<T, A>::value) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = j * 256 + threadIdx.x, r = i / (COLS / V), c = i % (COLS / V) * V;
        if (r >= ROWS) break;
        const bool in = r < valid && c < cols;
        const T* src = in ? base + token_of(l0 + r, n, reverse) * stride + c : base;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         static_cast<uint32_t>(__cvta_generic_to_shared(dst + r * PITCH + c))),
                     "l"(src), "r"(in ? 16 : 0)
                     : "memory");
      }
    } else {
      Pack<T, V> p[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = j * 256 + threadIdx.x, r = i / (COLS / V), c = i % (COLS / V) * V;
        if (r < valid && c < cols)
          p[j] = *reinterpret_cast<const Pack<T, V>*>(base + token_of(l0 + r, n, reverse) * stride + c);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = j * 256 + threadIdx.x, r = i / (COLS / V), c = i % (COLS / V) * V;
        if (r >= ROWS) break;
#pragma unroll
        for (int e = 0; e < V; ++e)
          dst[r * PITCH + c + e] = r < valid && c < cols ? A(to_acc(p[j].v[e])) : A(0);
      }
    }
  } else {
    constexpr int N = 8;  // loads in flight
    for (int i0 = threadIdx.x; i0 < ROWS * COLS; i0 += 256 * N) {
      T x[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = i0 + 256 * j, r = i / COLS, c = i % COLS;
        if (r < valid && c < cols) x[j] = base[token_of(l0 + r, n, reverse) * stride + c];
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int i = i0 + 256 * j, r = i / COLS, c = i % COLS;
        if (r < ROWS) dst[r * PITCH + c] = r < valid && c < cols ? A(to_acc(x[j])) : A(0);
      }
    }
  }
}
__device__ __forceinline__ void tiles_wait() {
  asm volatile("cp.async.commit_group;\n cp.async.wait_group 0;" ::: "memory");
}

template <typename T, int DK, int C, int NV> struct Simt {
  using A = typename AccOf<T>::type;
  static constexpr int PK = DK + 4, PP = C + 4;
  static constexpr int words = 2 * C * PK + C * NV + C * PP + DK * NV + C;
  static constexpr size_t smem = words * sizeof(A);
};

// One block: one job's value tile of one head and segment, chunk after chunk.  256 threads as
// 16 x 16; thread (ty, tx) owns rows ty + 16 i and columns tx * TN + j (the scores: tx + 16 j),
// so that blocks of 16 rows above the causal diagonal drop out at compile time.
template <typename T, int DK, int C, int NV, bool STATES>
__global__ void __launch_bounds__(256)
linattn_simt_kernel(const __grid_constant__ Call call) {
  using Z = Simt<T, DK, C, NV>;
  using A = typename Z::A;
  constexpr int PK = Z::PK, PP = Z::PP, TM = C / 16, TN = NV / 16, TD = DK / 16;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  A* sq = reinterpret_cast<A*>(smem_raw);
  A* sk = sq + C * PK;
  A* sv = sk + C * PK;
  A* sp = sv + C * NV;
  A* ss = sp + C * PP;
  A* sw = ss + DK * NV;

  int tile = blockIdx.x % call.tiles;
  const int64_t rest = blockIdx.x / call.tiles;
  const int64_t heads = call.batch * call.heads;
  const int64_t bh = rest % heads;
  const int seg = static_cast<int>(rest / heads);
  int ji = 0;
  while (tile >= call.job[ji].tiles) tile -= call.job[ji++].tiles;
  const Job& job = call.job[ji];
  const int64_t b = bh / call.heads;
  const int h = static_cast<int>(bh % call.heads);
  const int v0 = tile * NV;
  const int vcols = job.dv - v0 < NV ? job.dv - v0 : NV;

  const int64_t n = valid_tokens(call, b);
  const int last = n == 0 ? 0 : static_cast<int>((n - 1) / call.seg_len);
  if (STATES && seg >= last) return;
  const A a = static_cast<const A*>(call.log_decay)[h];
  const int64_t begin = int64_t(seg) * call.seg_len;
  const int64_t row_end = imin(begin + call.seg_len, call.length);
  const int64_t end = imin(row_end, n);  // of the valid tokens; may lie before begin

  const T* q = static_cast<const T*>(job.q) + b * job.qs[0] + (h / job.q_group) * job.qs[2];
  const T* k = static_cast<const T*>(job.k) + b * job.ks[0] + (h / job.k_group) * job.ks[2];
  const T* v = static_cast<const T*>(job.v) + b * job.vs[0] + (h / job.v_group) * job.vs[2] + v0;
  const int64_t o_head = b * job.os[0] + h * job.os[2] + v0;
  T* o = static_cast<T*>(job.o) + o_head;
  float* wide = static_cast<float*>(job.o) + o_head;
  A* segs = static_cast<A*>(job.seg) + bh * (call.nseg - 1) * job.dk * job.dv;
  const int64_t state_size = int64_t(job.dk) * job.dv;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;

  A s[TD][TN];  // the state: rows ty + 16 i, columns tx * TN + j
#pragma unroll
  for (int i = 0; i < TD; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int r = ty + 16 * i, c = v0 + tx * TN + j;
      A x = A(0);
      if (!STATES && r < job.dk && c < job.dv) {
        if (seg > 0 && seg <= last) x = segs[(seg - 1) * state_size + int64_t(r) * job.dv + c];
        else if (seg == 0 && job.init != nullptr)
          x = static_cast<const A*>(job.init)[bh * state_size + r * job.init_row + c * job.init_col];
      }
      s[i][j] = x;
      if (!STATES) ss[r * NV + tx * TN + j] = x;
    }

  for (int64_t l0 = begin; l0 < end; l0 += C) {
    const int m = static_cast<int>(imin(C, end - l0));
    if (!STATES)
      load_tile<T, A, C, DK, PK>(sq, q, job.qs[1], l0, n, job.reverse, m, job.dk, job.q_vec);
    load_tile<T, A, C, DK, PK>(sk, k, job.ks[1], l0, n, job.reverse, m, job.dk, job.k_vec);
    load_tile<T, A, C, NV, NV>(sv, v, job.vs[1], l0, n, job.reverse, m, vcols, job.v_vec);
    if (threadIdx.x < C) {
      const int age = m - job.off - static_cast<int>(threadIdx.x);
      sw[threadIdx.x] = age < 0 ? A(0) : A(job.write) * decay_pow(a, A(age));
    }
    tiles_wait();
    __syncthreads();
    if (!STATES) {
      // scores, blocks on and below the diagonal
      A p[TM][TM];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) p[i][j] = A(0);
#pragma unroll 2
      for (int c = 0; c < DK; c += 4) {
        Pack<A, 4> x[TM], y[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          x[i] = *reinterpret_cast<const Pack<A, 4>*>(sq + (ty + 16 * i) * PK + c);
          y[i] = *reinterpret_cast<const Pack<A, 4>*>(sk + (tx + 16 * i) * PK + c);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j <= i; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) p[i][j] += x[i].v[e] * y[j].v[e];
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j <= i; ++j) {
          const int t = ty + 16 * i, u = tx + 16 * j;
          sp[t * PP + u] = u > t ? A(0) : p[i][j] * A(job.intra) * decay_pow(a, A(t - u));
        }
      A out[TM][TN];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) out[i][j] = A(0);
#pragma unroll 2
      for (int c = 0; c < DK; c += 4) {
        Pack<A, 4> x[TM];
        Pack<A, TN> y[4];
#pragma unroll
        for (int i = 0; i < TM; ++i)
          x[i] = *reinterpret_cast<const Pack<A, 4>*>(sq + (ty + 16 * i) * PK + c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = *reinterpret_cast<const Pack<A, TN>*>(ss + (c + e) * NV + tx * TN);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < TN; ++j) out[i][j] += x[i].v[e] * y[e].v[j];
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const A read = A(job.inter) * decay_pow(a, A(ty + 16 * i + job.off));
#pragma unroll
        for (int j = 0; j < TN; ++j) out[i][j] *= read;
      }
      __syncthreads();
      // scores times values; within the diagonal block a value after the token is left out, not
      // multiplied by zero: it may be an infinity
#pragma unroll
      for (int blk = 0; blk < TM; ++blk) {
#pragma unroll 2
        for (int u0 = 0; u0 < 16; u0 += 4) {
          const int u = blk * 16 + u0;
          Pack<A, TN> y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            y[e] = *reinterpret_cast<const Pack<A, TN>*>(sv + (u + e) * NV + tx * TN);
#pragma unroll
          for (int i = blk; i < TM; ++i) {
            const Pack<A, 4> x = *reinterpret_cast<const Pack<A, 4>*>(sp + (ty + 16 * i) * PP + u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (i == blk && u0 + e > ty) continue;
#pragma unroll
              for (int j = 0; j < TN; ++j) out[i][j] += x.v[e] * y[e].v[j];
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int t = ty + 16 * i;
        if (t < m) {
          const int64_t at = token_of(l0 + t, n, job.reverse) * job.os[1];
          T* row = o + at;
          if (job.o_wide) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
              if (tx * TN + j < vcols) wide[at + tx * TN + j] = static_cast<float>(out[i][j]);
          } else if (job.o_vec && TN * sizeof(T) % 8 == 0 && tx * TN + TN <= vcols) {
            Pack<T, TN> w;
#pragma unroll
            for (int j = 0; j < TN; ++j) w.v[j] = from_acc<T>(out[i][j]);
            *reinterpret_cast<Pack<T, TN>*>(row + tx * TN) = w;
          } else {
#pragma unroll
            for (int j = 0; j < TN; ++j)
              if (tx * TN + j < vcols) row[tx * TN + j] = from_acc<T>(out[i][j]);
          }
        }
      }
    }
    // state: the chunk's sum first, so that long sequences add up by chunks
    const A keep = decay_pow(a, A(m));
    A sum[TD][TN];
#pragma unroll
    for (int i = 0; i < TD; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) sum[i][j] = A(0);
#pragma unroll 4
    for (int u = 0; u < C; ++u) {
      Pack<A, TN> y = *reinterpret_cast<const Pack<A, TN>*>(sv + u * NV + tx * TN);
      const A w = sw[u];
#pragma unroll
      for (int j = 0; j < TN; ++j) y.v[j] *= w;
#pragma unroll
      for (int i = 0; i < TD; ++i) {
        const A x = sk[u * PK + ty + 16 * i];
#pragma unroll
        for (int j = 0; j < TN; ++j) sum[i][j] += x * y.v[j];
      }
    }
#pragma unroll
    for (int i = 0; i < TD; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) s[i][j] = keep * s[i][j] + sum[i][j];
    if (!STATES) {
#pragma unroll
      for (int i = 0; i < TD; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) ss[(ty + 16 * i) * NV + tx * TN + j] = s[i][j];
    }
    __syncthreads();
  }
  if (!STATES) {  // rows after the sequence's end
    for (int64_t l = imax(begin, n) + ty; l < row_end; l += 16)
      for (int c = tx; c < vcols; c += 16) {
        if (job.o_wide) wide[l * job.os[1] + c] = 0.0f;
        else o[l * job.os[1] + c] = from_acc<T>(A(0));
      }
  }
  A* dst = STATES ? segs + seg * state_size
                  : (seg == last && job.fin != nullptr ? static_cast<A*>(job.fin) + bh * state_size
                                                       : nullptr);
  if (dst != nullptr) {
#pragma unroll
    for (int i = 0; i < TD; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int r = ty + 16 * i, c = v0 + tx * TN + j;
        if (r < job.dk && c < job.dv) dst[int64_t(r) * job.dv + c] = s[i][j];
      }
  }
}

// ------------------------------------------------------------------------------ 32 bits, warps' MMA
// The same block for 32-bit precision on the tensor cores (warp-level TF32 products): each operand
// is the sum of two TF32 values, a b = ah bh + ah bl + al bh, which leaves 2^-21 of a product out,
// less than a 32-bit sum of this length rounds.  Three products at 275 TFLOP/s (measured) against
// the FMA pipes' 70; and a fragment serves 8 or 16 rows, where the FMA form above is bound by its
// shared-memory reads.  Also the 16-bit types where rows are not aligned for linattn_tc.cu.
//
// 8 warps, each of 16 rows and 32 columns of the scores and of o, and of every 64 rows of the state, which stays in its registers.  Pitches: rows 4 (8) words apart modulo 32
// put the 32 lanes of a fragment's read on different banks.
__device__ __forceinline__ void tf32_split(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;  // to nearest; the next binade is exact too
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4],
                                         const uint32_t (&b)[2]) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
struct FragA {
  uint32_t hi[4], lo[4];
  // element (row, k) of the 16 x 8 block at p[row * rs + k * ks]
  __device__ __forceinline__ void load(const float* p, int rs, int ks, int lane) {
    const float* q = p + lane / 4 * rs + lane % 4 * ks;
    tf32_split(q[0], hi[0], lo[0]);
    tf32_split(q[8 * rs], hi[1], lo[1]);
    tf32_split(q[4 * ks], hi[2], lo[2]);
    tf32_split(q[8 * rs + 4 * ks], hi[3], lo[3]);
  }
};
struct FragB {
  uint32_t hi[2], lo[2];
  // element (k, column) of the 8 x 8 block at p[k * ks + column * cs], times wk[k]
  __device__ __forceinline__ void load(const float* p, int ks, int cs, int lane) {
    const float* q = p + lane % 4 * ks + lane / 4 * cs;
    tf32_split(q[0], hi[0], lo[0]);
    tf32_split(q[4 * ks], hi[1], lo[1]);
  }
  // with zeros for infinities and NaN
  __device__ __forceinline__ void load_finite(const float* p, int ks, int cs, int lane) {
    const float* q = p + lane % 4 * ks + lane / 4 * cs;
    tf32_split(isfinite(q[0]) ? q[0] : 0.0f, hi[0], lo[0]);
    tf32_split(isfinite(q[4 * ks]) ? q[4 * ks] : 0.0f, hi[1], lo[1]);
  }
  __device__ __forceinline__ void load(const float* p, int ks, int cs, int lane, float w0,
                                       float w1) {
    const float* q = p + lane % 4 * ks + lane / 4 * cs;
    tf32_split(q[0] * w0, hi[0], lo[0]);
    tf32_split(q[4 * ks] * w1, hi[1], lo[1]);
  }
};
// A 16 x 8 block of a product.  The matrix unit's 32-bit sum is cut off, not rounded, at every
// step: the large products and the small ones are summed apart, each over one chunk or head only,
// and what is carried from chunk to chunk is added outside (6e-6 off on a long sequence else).
struct Block {
  float hi[4] = {0.0f, 0.0f, 0.0f, 0.0f}, lo[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  __device__ __forceinline__ void add(const FragA& a, const FragB& b) {
    mma_tf32(lo, a.lo, b.hi);
    mma_tf32(lo, a.hi, b.lo);
    mma_tf32(hi, a.hi, b.hi);
  }
  __device__ __forceinline__ float value(int e) const { return hi[e] + lo[e]; }
};

template <int DK> struct Tf32 {
  static constexpr int C = 64, NV = 64, PK = DK + 4, PV = NV + 8, PP = C + 4;
  static constexpr int words = 2 * C * PK + C * PV + DK * PV + C * PP + 2 * (C + 8);
  static constexpr size_t smem = words * sizeof(float);
};

// Two blocks leave 128 registers a thread, too few for 16-bit rows: 37 tokens of bf16 (off 16-byte
// boundaries) take 18 us with them and 11.5 us with more.
template <typename T, int DK, bool STATES>
__global__ void __launch_bounds__(256, DK == 64 && sizeof(T) == 4 ? 2 : 1)
linattn_tf32_kernel(const __grid_constant__ Call call) {
  using Z = Tf32<DK>;
  constexpr int C = Z::C, NV = Z::NV, PK = Z::PK, PV = Z::PV, PP = Z::PP, RT = DK / 64;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  float* sq = reinterpret_cast<float*>(smem_raw);
  float* sk = sq + C * PK;
  float* sv = sk + C * PK;
  float* ss = sv + C * PV;
  float* sp = ss + DK * PV;
  float* dpow = sp + C * PP;      // d^n, n = 0 .. 64
  float* weight = dpow + C + 8;   // of the chunk's values towards its end

  int tile = blockIdx.x % call.tiles;
  const int64_t rest = blockIdx.x / call.tiles;
  const int64_t heads = call.batch * call.heads;
  const int64_t bh = rest % heads;
  const int seg = static_cast<int>(rest / heads);
  int ji = 0;
  while (tile >= call.job[ji].tiles) tile -= call.job[ji++].tiles;
  const Job& job = call.job[ji];
  const int64_t b = bh / call.heads;
  const int h = static_cast<int>(bh % call.heads);
  const int v0 = tile * NV;
  const int vcols = job.dv - v0 < NV ? job.dv - v0 : NV;
  const int64_t n = valid_tokens(call, b);
  const int last = n == 0 ? 0 : static_cast<int>((n - 1) / call.seg_len);
  if (STATES && seg >= last) return;
  const float a = static_cast<const float*>(call.log_decay)[h];
  const int64_t begin = int64_t(seg) * call.seg_len;
  const int64_t row_end = imin(begin + call.seg_len, call.length);
  const int64_t end = imin(row_end, n);

  const T* q = static_cast<const T*>(job.q) + b * job.qs[0] + (h / job.q_group) * job.qs[2];
  const T* k = static_cast<const T*>(job.k) + b * job.ks[0] + (h / job.k_group) * job.ks[2];
  const T* v = static_cast<const T*>(job.v) + b * job.vs[0] + (h / job.v_group) * job.vs[2] + v0;
  const int64_t o_head = b * job.os[0] + h * job.os[2] + v0;
  T* o = static_cast<T*>(job.o) + o_head;
  float* wide = static_cast<float*>(job.o) + o_head;
  const int64_t state_size = int64_t(job.dk) * job.dv;
  float* segs = static_cast<float*>(job.seg) + bh * (call.nseg - 1) * state_size;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // the two warps of a scheduler share the work under the diagonal: rows 0 and 3, 1 and 2
  const int r0 = (warp < 4 ? warp : 7 - warp) * 16, c0 = warp / 4 * 32;
  const int g = lane / 4, t4 = lane % 4;

  for (int i = threadIdx.x; i <= C; i += 256) dpow[i] = decay_pow(a, float(i));
  float s[RT][4][4];  // the state: rows 64 rt + r0 + g (+ 8), columns c0 + 8 j + 2 t4 (+ 1)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 64 * rt + r0 + g + e / 2 * 8, col = c0 + 8 * j + 2 * t4 + e % 2;
        const int c = v0 + col;
        float x = 0.0f;
        if (!STATES && r < job.dk && c < job.dv) {
          if (seg > 0 && seg <= last) x = segs[(seg - 1) * state_size + int64_t(r) * job.dv + c];
          else if (seg == 0 && job.init != nullptr)
            x = static_cast<const float*>(job.init)[bh * state_size + r * job.init_row +
                                                    c * job.init_col];
        }
        s[rt][j][e] = x;
        if (!STATES) ss[r * PV + col] = x;
      }

  for (int64_t l0 = begin; l0 < end; l0 += C) {
    const int m = static_cast<int>(imin(C, end - l0));
    if (!STATES)
      load_tile<T, float, C, DK, PK>(sq, q, job.qs[1], l0, n, job.reverse, m, job.dk, job.q_vec);
    load_tile<T, float, C, DK, PK>(sk, k, job.ks[1], l0, n, job.reverse, m, job.dk, job.k_vec);
    load_tile<T, float, C, NV, PV>(sv, v, job.vs[1], l0, n, job.reverse, m, vcols, job.v_vec);
    if (threadIdx.x < C) {
      const int age = m - job.off - static_cast<int>(threadIdx.x);
      weight[threadIdx.x] = age < 0 ? 0.0f : decay_pow(a, float(age));
    }
    tiles_wait();
    __syncthreads();
    if (!STATES) {
      // scores: columns above the diagonal of these rows drop out
      Block acc[4];
      const int cols = r0 + 16 - c0 < 0 ? 0 : (r0 + 16 - c0 > 32 ? 4 : (r0 + 16 - c0) / 8);
      if (cols > 0) {
#pragma unroll 4
        for (int d = 0; d < DK; d += 8) {
          FragA x;
          x.load(sq + r0 * PK + d, PK, 1, lane);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < cols) {
              FragB y;
              y.load(sk + (c0 + 8 * j) * PK + d, 1, PK, lane);
              acc[j].add(x, y);
            }
          }
        }
      }
      const float intra = float(job.intra);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = r0 + g + e / 2 * 8, u = c0 + 8 * j + 2 * t4 + e % 2;
          sp[t * PP + u] = u > t ? 0.0f : acc[j].value(e) * (intra * dpow[t - u]);
        }
      // what the state gives
      Block state[4];
#pragma unroll 4
      for (int d = 0; d < DK; d += 8) {
        FragA x;
        x.load(sq + r0 * PK + d, PK, 1, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          FragB y;
          y.load(ss + d * PV + c0 + 8 * j, PV, 1, lane);
          state[j].add(x, y);
        }
      }
      const float inter = float(job.inter);
      const float f0 = inter * dpow[r0 + g + job.off], f1 = inter * dpow[r0 + g + 8 + job.off];
      float out[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        out[j][0] = f0 * state[j].value(0);
        out[j][1] = f0 * state[j].value(1);
        out[j][2] = f1 * state[j].value(2);
        out[j][3] = f1 * state[j].value(3);
      }
      __syncthreads();
      // and the chunk's own tokens, up to the end of these rows
      Block own[4];
#pragma unroll 4
      for (int u = 0; u < r0 + 16; u += 8) {
        FragA x;
        x.load(sp + r0 * PP + u, PP, 1, lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          FragB y;
          y.load(sv + u * PV + c0 + 8 * j, PV, 1, lane);
          own[j].add(x, y);
        }
      }
      float worst = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) worst += own[j].value(e) * 0.0f;
      if (__any_sync(0xffffffffu, worst != 0.0f)) {  // NaN
        // Infinities or NaN among the values (or scores): the masked scores of the block on the
        // diagonal, factors of zero, would bring them to earlier tokens.  Again with zeros in
        // their place, and NaN from their token on.
#pragma unroll
        for (int j = 0; j < 4; ++j) own[j] = Block();
#pragma unroll 1
        for (int u = 0; u < r0 + 16; u += 8) {
          FragA x;
          x.load(sp + r0 * PP + u, PP, 1, lane);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            FragB y;
            y.load_finite(sv + u * PV + c0 + 8 * j, PV, 1, lane);
            own[j].add(x, y);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int t = r0 + g + e / 2 * 8, col = c0 + 8 * j + 2 * t4 + e % 2;
#pragma unroll 1
            for (int u = 0; u <= t; ++u)
              if (!isfinite(sv[u * PV + col])) own[j].hi[e] = nanf("");
          }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) out[j][e] += own[j].value(e);
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const int t = r0 + g + e / 2 * 8;
        if (t < m) {
          const int64_t at = token_of(l0 + t, n, job.reverse) * job.os[1];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int col = c0 + 8 * j + 2 * t4;
            if (sizeof(T) == 4 && job.o_vec && col + 2 <= vcols) {
              *reinterpret_cast<float2*>(wide + at + col) = make_float2(out[j][e], out[j][e + 1]);
            } else {
#pragma unroll
              for (int i = 0; i < 2; ++i)
                if (col + i < vcols) {
                  if (job.o_wide) wide[at + col + i] = out[j][e + i];
                  else o[at + col + i] = from_acc<T>(out[j][e + i]);
                }
            }
          }
        }
      }
    }
    // state
    const float keep = dpow[m], write = float(job.write);
    Block update[RT][4];
#pragma unroll 4
    for (int u = 0; u < C; u += 8) {
      FragA x[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) x[rt].load(sk + u * PK + 64 * rt + r0, 1, PK, lane);
      const float w0 = write * weight[u + t4], w1 = write * weight[u + t4 + 4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        FragB y;
        y.load(sv + u * PV + c0 + 8 * j, PV, 1, lane, w0, w1);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) update[rt][j].add(x[rt], y);
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[rt][j][e] = keep * s[rt][j][e] + update[rt][j].value(e);
    if (!STATES) {  // (every read of the old one came before the barrier above)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
            *reinterpret_cast<float2*>(ss + (64 * rt + r0 + g + e / 2 * 8) * PV + c0 + 8 * j +
                                       2 * t4) = make_float2(s[rt][j][e], s[rt][j][e + 1]);
    }
    __syncthreads();
  }
  if (!STATES) {  // rows after the sequence's end
    for (int64_t l = imax(begin, n) + warp; l < row_end; l += 8)
      for (int c = lane; c < vcols; c += 32) {
        if (job.o_wide) wide[l * job.os[1] + c] = 0.0f;
        else o[l * job.os[1] + c] = from_acc<T>(0.0f);
      }
  }
  float* dst = STATES ? segs + seg * state_size
                      : (seg == last && job.fin != nullptr
                             ? static_cast<float*>(job.fin) + bh * state_size : nullptr);
  if (dst != nullptr) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 64 * rt + r0 + g + e / 2 * 8, c = v0 + c0 + 8 * j + 2 * t4 + e % 2;
          if (r < job.dk && c < job.dv) dst[int64_t(r) * job.dv + c] = s[rt][j][e];
        }
  }
}

// The states between segments: slot i of a head holds segment i's own end state and receives the
// state before segment i + 1.
template <typename A>
__global__ void __launch_bounds__(256)
linattn_scan_kernel(const __grid_constant__ Call call, int blocks) {  // blocks: a head's
  const Job& job = call.job[blockIdx.y];
  const int64_t size = int64_t(job.dk) * job.dv;
  const int64_t bh = blockIdx.x / blocks;
  const int64_t e = int64_t(blockIdx.x % blocks) * blockDim.x + threadIdx.x;
  if (e >= size) return;
  const int64_t n = valid_tokens(call, bh / call.heads);
  const int last = n == 0 ? 0 : static_cast<int>((n - 1) / call.seg_len);
  const A keep = decay_pow(static_cast<const A*>(call.log_decay)[bh % call.heads],
                           A(call.seg_len));
  A cur = A(0);
  if (job.init != nullptr)
    cur = static_cast<const A*>(job.init)[bh * size + e / job.dv * job.init_row +
                                          e % job.dv * job.init_col];
  A* slot = static_cast<A*>(job.seg) + bh * (call.nseg - 1) * size + e;
#pragma unroll 4
  for (int i = 0; i < last; ++i) {
    cur = keep * cur + slot[i * size];
    slot[i * size] = cur;
  }
}

// Gradients of shared key or value heads: the sum over the heads that read them, in the order of
// the heads; the heads' own gradients are 32 bits (64 for fp64), rounded once here.
// A thread takes W neighbouring columns.
template <typename T, int W>
__global__ void __launch_bounds__(256)
linattn_group_sum_kernel(const typename AccOf<T>::type* __restrict__ in, T* __restrict__ out,
                         int64_t rows, int group, int dim) {
  using A = typename AccOf<T>::type;
  const int per = dim / W, here = blockDim.x / per;  // whole rows a block
  const int64_t row = int64_t(blockIdx.x) * here + threadIdx.x / per;
  if (int(threadIdx.x) >= here * per || row >= rows) return;
  const int c = threadIdx.x % per * W;
  const A* p = in + row * group * dim + c;
  Pack<A, W> sum;
#pragma unroll
  for (int j = 0; j < W; ++j) sum.v[j] = A(0);
#pragma unroll 4
  for (int g = 0; g < group; ++g) {
    const Pack<A, W> x = *reinterpret_cast<const Pack<A, W>*>(p + int64_t(g) * dim);
#pragma unroll
    for (int j = 0; j < W; ++j) sum.v[j] += x.v[j];
  }
  Pack<T, W> y;
#pragma unroll
  for (int j = 0; j < W; ++j) y.v[j] = from_acc<T>(sum.v[j]);
  *reinterpret_cast<Pack<T, W>*>(out + row * dim + c) = y;
}

// ------------------------------------------------------------------------------ one token
// S <- d S + k v^T, o = scale q^T S.  Bound by reading and writing S: a block holds all rows of
// `lanes` groups of V columns, so that each S value is read and written once, in 16-byte
// accesses, 8 rows of a thread in flight; the products of the rows are joined in shared memory.
// Measured: 240 x 16 heads of 128 x 128 94 us (503 MB, 5.3 TB/s; streaming hints 92, but 20.1 in
// place of 18.7 us where the states fit L2); one head's 64 x 64 4.3 us.
template <typename T, int V>
__global__ void __launch_bounds__(256)
linattn_step_kernel(const __grid_constant__ fdwt_linattn_desc d, const T* __restrict__ q,
                    const T* __restrict__ k, const T* __restrict__ v,
                    const typename AccOf<T>::type* __restrict__ log_decay,
                    typename AccOf<T>::type* __restrict__ state, int64_t state_slots,
                    const int32_t* __restrict__ slots, T* __restrict__ out, int lanes,
                    int tiles) {
  using A = typename AccOf<T>::type;
  __shared__ A sq[256], sk[256];
  __shared__ __align__(16) A join[256 * V];
  const int tile = blockIdx.x % tiles;
  const int64_t bh = blockIdx.x / tiles;
  const int64_t b = bh / d.heads;
  const int h = static_cast<int>(bh % d.heads), hk = h / (d.heads / d.kv_heads);
  const int x = threadIdx.x % lanes, y = threadIdx.x / lanes, rows = blockDim.x / lanes;
  const int c = (tile * lanes + x) * V;
  T* o = out + b * d.o_stride[0] + h * d.o_stride[2] + c;
  const int64_t slot = slots == nullptr ? b : slots[b];
  if (slot < 0 || slot >= state_slots) {
    if (y == 0)
      for (int j = 0; j < V && c + j < d.dv; ++j) o[j] = from_acc<T>(A(0));
    return;
  }
  for (int i = threadIdx.x; i < d.dk; i += blockDim.x) {
    sq[i] = A(to_acc(q[b * d.q_stride[0] + h * d.q_stride[2] + i]));
    sk[i] = A(to_acc(k[b * d.k_stride[0] + hk * d.k_stride[2] + i]));
  }
  const A keep = decay_pow(log_decay[h], A(1));
  A vv[V], acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    vv[j] = c + j < d.dv ? A(to_acc(v[b * d.v_stride[0] + hk * d.v_stride[2] + c + j])) : A(0);
    acc[j] = A(0);
  }
  A* s = state + (slot * d.heads + h) * d.dk * d.dv + c;
  __syncthreads();
  if (c < d.dv) {
#pragma unroll 8
    for (int r = y; r < d.dk; r += rows) {
      Pack<A, V> p = *reinterpret_cast<const Pack<A, V>*>(s + int64_t(r) * d.dv);
      const A kr = sk[r], qr = sq[r];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        p.v[j] = keep * p.v[j] + kr * vv[j];
        acc[j] += qr * p.v[j];
      }
      *reinterpret_cast<Pack<A, V>*>(s + int64_t(r) * d.dv) = p;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) join[(y * lanes + x) * V + j] = acc[j];
  __syncthreads();
  for (int i = threadIdx.x; i < lanes * V; i += blockDim.x) {
    const int col = tile * lanes * V + i;
    if (col >= d.dv) break;
    A sum = A(0);
    for (int r = 0; r < rows; ++r) sum += join[r * lanes * V + i];
    out[b * d.o_stride[0] + h * d.o_stride[2] + col] = from_acc<T>(A(d.scale) * sum);
  }
}

// ------------------------------------------------------------------------------ launches
int block_chunk(int dtype, int dk) { return dtype == FDWT_F64 || dk > 128 ? 32 : 64; }

template <typename Kernel>
int launch_block(Kernel kernel, size_t smem, const Call& call, int64_t grid, cudaStream_t stream) {
  int st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
  if (st == FDWT_OK) st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  kernel<<<static_cast<unsigned>(grid), 256, smem, stream>>>(call);
  return launch_status();
}
template <typename T, int DK>
int simt_launch(const Call& call, bool states, int64_t grid, cudaStream_t stream) {
  return launch_block(states ? linattn_simt_kernel<T, DK, 32, 32, true>
                             : linattn_simt_kernel<T, DK, 32, 32, false>,
                      Simt<T, DK, 32, 32>::smem, call, grid, stream);
}
template <typename T, int DK>
int tf32_launch(const Call& call, bool states, int64_t grid, cudaStream_t stream) {
  return launch_block(states ? linattn_tf32_kernel<T, DK, true> : linattn_tf32_kernel<T, DK, false>,
                      Tf32<DK>::smem, call, grid, stream);
}

// fp64 and heads over 128 on the FMA pipes, the others by TF32 products.
template <typename T>
int general_launch(const Call& call, int dk, bool states, int64_t grid, cudaStream_t stream) {
  if constexpr (std::is_same<T, double>::value) {
    if (dk <= 64) return simt_launch<T, 64>(call, states, grid, stream);
    if (dk <= 128) return simt_launch<T, 128>(call, states, grid, stream);
  } else {
    if (dk <= 64) return tf32_launch<T, 64>(call, states, grid, stream);
    if (dk <= 128) return tf32_launch<T, 128>(call, states, grid, stream);
  }
  return simt_launch<T, 256>(call, states, grid, stream);
}

// Accesses of `bytes` along the last axis are aligned (and the axis ends on one).
inline bool vector_ok(const void* p, const int64_t* strides, int dim, size_t size,
                      size_t bytes = 16) {
  const int64_t v = static_cast<int64_t>(bytes / size);
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && dim % v == 0 && strides[0] % v == 0 &&
         strides[1] % v == 0 && strides[2] % v == 0;
}

struct Plan {
  bool tc;
  int chunk, tile, nseg;
  int64_t seg_len;
};

inline int max_dk(const Call& call) {
  int dk = 0;
  for (int j = 0; j < call.jobs; ++j) dk = call.job[j].dk > dk ? call.job[j].dk : dk;
  return dk;
}

// Chunk, value tile and segments of a call whose jobs have their sizes (pointers are looked at
// only for `tc`).
inline Plan make_plan(int dtype, const Call& call, bool tc) {
  Plan p{};
  p.tc = tc;
  const int dk = max_dk(call);
  p.chunk = tc ? kTcChunk : block_chunk(dtype, dk);
  p.tile = tc ? kTcTile : (p.chunk == 64 ? 64 : 32);
  int64_t tiles = 0;
  for (int j = 0; j < call.jobs; ++j) tiles += cdiv(call.job[j].dv, p.tile);
  const int64_t chunks = imax(1, cdiv(call.length, p.chunk));
  // Blocks a multiprocessor holds; two of the fp32 kernel up to heads of 64 (5 x 1537 tokens, 6
  // heads of 48 x 80: 120 us so, 132 us with one at that step).  Times in microseconds a chunk, all
  // multiprocessors busy: measured for the tensor cores (128 tokens).  For the general kernels one
  // set stands for all, near that of fp32 heads of 64 (64 tokens, 8.1 us with one block a
  // multiprocessor, 11.9 with two); others measure 10 to 26 us, 16-bit rows of 128 off 16-byte
  // boundaries 38 us.
  const int64_t slots = int64_t(sm_count()) * (dtype == FDWT_F32 && dk <= 64 ? 2 : 1);
  const int64_t units = tiles * call.batch * call.heads;
  const Cost cost = tc ? Cost{dk <= 64 ? 2.3 : 2.8, 0.75, 6.0, 4.0} : Cost{7.5, 3.0, 5.0, 4.0};
  const int64_t c = cdiv(chunks, plan_segments(units, chunks, slots, cost));
  p.nseg = static_cast<int>(cdiv(chunks, c));
  p.seg_len = c * p.chunk;
  return p;
}

// States between segments and the heads' own gradients are stored 32 bytes at a time.
constexpr uintptr_t kWorkspaceAlign = 32;

inline size_t seg_bytes(const Call& call, const Job& job, int nseg, int dtype) {
  const size_t bytes = size_t(call.batch) * call.heads * (nseg - 1) * job.dk * job.dv *
                       (dtype == FDWT_F64 ? 8 : 4);
  return (bytes + 255) & ~size_t(255);
}

inline size_t call_workspace(int dtype, const Call& call) {
  size_t most = 0;
  for (bool tc : {false, true}) {
    if (tc && (dtype == FDWT_F32 || dtype == FDWT_F64)) continue;
    const Plan p = make_plan(dtype, call, tc);
    size_t bytes = 0;
    for (int j = 0; j < call.jobs; ++j) bytes += seg_bytes(call, call.job[j], p.nseg, dtype);
    if (bytes > most) most = bytes;
  }
  return most;
}

int run(int dtype, Call& call, void* workspace, cudaStream_t stream) {
  const size_t size = dtype_size(dtype);
  for (int j = 0; j < call.jobs; ++j) {
    Job& job = call.job[j];
    // the stride of an axis of one element is whatever the caller had there
    auto normal = [&](int64_t* s, int group) {
      if (call.batch == 1) s[0] = 0;
      if (call.length == 1) s[1] = 0;
      if (call.heads / group == 1) s[2] = 0;
    };
    normal(job.qs, job.q_group);
    normal(job.ks, job.k_group);
    normal(job.vs, job.v_group);
    normal(job.os, 1);
    job.q_vec = vector_ok(job.q, job.qs, job.dk, size);
    job.k_vec = vector_ok(job.k, job.ks, job.dk, size);
    job.v_vec = vector_ok(job.v, job.vs, job.dv, size);
    const size_t o_size = job.o_wide ? 4 : size;
    job.o_vec = vector_ok(job.o, job.os, job.dv, o_size, 16) +
                vector_ok(job.o, job.os, job.dv, o_size, 32);
  }
  // The tensor cores wherever their kernel takes the call's types, sizes and strides: faster from
  // one token on (bf16, one sequence of 4 heads of 64: 1 token 10.3 us against the general
  // kernel's 12.4, 128 tokens 10.3 against 20.6; 32 sequences of 16 heads of 128: 79 against 117
  // and 85 against 223), and as exact.
  const bool tc = tc_supports(dtype, call);
  const Plan p = make_plan(dtype, call, tc);
  call.nseg = p.nseg;
  call.seg_len = p.seg_len;
  call.tiles = 0;
  char* ws = static_cast<char*>(workspace);
  int64_t elems = 0;
  for (int j = 0; j < call.jobs; ++j) {
    Job& job = call.job[j];
    job.tiles = static_cast<int>(cdiv(job.dv, p.tile));
    call.tiles += job.tiles;
    job.seg = ws;
    ws += seg_bytes(call, job, p.nseg, dtype);
    elems = imax(elems, int64_t(job.dk) * job.dv);
  }
  const int64_t heads = call.batch * call.heads;
  const int64_t grid = heads * call.tiles * p.nseg;
  if (grid > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
  const int dk = max_dk(call);
  auto launch = [&](bool states) -> int {
    if (p.tc) return tc_launch(dtype, call, states, stream);
    const int64_t blocks = states ? grid / p.nseg * (p.nseg - 1) : grid;
    switch (dtype) {
      case FDWT_F32: return general_launch<float>(call, dk, states, blocks, stream);
      case FDWT_F64: return general_launch<double>(call, dk, states, blocks, stream);
      case FDWT_F16: return general_launch<__half>(call, dk, states, blocks, stream);
      default: return general_launch<__nv_bfloat16>(call, dk, states, blocks, stream);
    }
  };
  call.scan_inside = p.tc && p.nseg <= kScanInside;
  if (p.nseg > 1) {
    int st = launch(true);
    if (st != FDWT_OK) return st;
  }
  if (p.nseg > 1 && !call.scan_inside) {
    int st = pre_launch(stream);
    if (st != FDWT_OK) return st;
    const int per = static_cast<int>(cdiv(elems, 256));
    if (per * heads > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
    const dim3 blocks(static_cast<unsigned>(per * heads), static_cast<unsigned>(call.jobs));
    if (dtype == FDWT_F64) linattn_scan_kernel<double><<<blocks, 256, 0, stream>>>(call, per);
    else linattn_scan_kernel<float><<<blocks, 256, 0, stream>>>(call, per);
    st = launch_status();
    if (st != FDWT_OK) return st;
  }
  return launch(false);
}

inline bool desc_ok(const fdwt_linattn_desc* d) {
  return d != nullptr && dtype_size(d->dtype) != 0 && d->heads >= 1 && d->kv_heads >= 1 &&
         d->heads % d->kv_heads == 0 && d->dk >= 1 && d->dv >= 1 && d->batch >= 0 &&
         d->length >= 0;
}
inline bool desc_supported(const fdwt_linattn_desc* d) {
  return d->dk <= 256 && d->dv <= 256;
}

inline void copy3(int64_t* dst, const int64_t* src) {
  for (int i = 0; i < 3; ++i) dst[i] = src[i];
}
inline void contiguous(int64_t* s, int64_t length, int64_t heads, int64_t dim) {
  s[0] = length * heads * dim;
  s[1] = heads * dim;
  s[2] = dim;
}

inline void fill_call(const fdwt_linattn_desc* d, Call* c) {
  c->batch = d->batch;
  c->length = d->length;
  c->heads = d->heads;
}

// Sizes, strides, order and scales of the jobs of the forward (1 job) or backward (3) pass.
inline void shape_jobs(const fdwt_linattn_desc* d, bool backward, Call* c) {
  fill_call(d, c);
  const int group = d->heads / d->kv_heads;
  const double scale = d->scale;
  auto set = [&](Job& j, const int64_t* qs, int qg, const int64_t* ks, int kg, const int64_t* vs,
                 int vg, int dk, int dv) {
    copy3(j.qs, qs);
    copy3(j.ks, ks);
    copy3(j.vs, vs);
    j.q_group = qg;
    j.k_group = kg;
    j.v_group = vg;
    j.dk = dk;
    j.dv = dv;
    contiguous(j.os, d->length, d->heads, dv);
    j.init_row = dv;
    j.init_col = 1;
    j.reverse = 0;
    j.off = 1;
    j.inter = j.intra = scale;
    j.write = 1.0;
  };
  if (!backward) {
    c->jobs = 1;
    set(c->job[0], d->q_stride, 1, d->k_stride, group, d->v_stride, group, d->dk, d->dv);
    copy3(c->job[0].os, d->o_stride);
    return;
  }
  c->jobs = 3;
  set(c->job[0], d->o_stride, 1, d->v_stride, group, d->k_stride, group, d->dv, d->dk);
  set(c->job[1], d->k_stride, group, d->q_stride, 1, d->o_stride, 1, d->dk, d->dv);
  set(c->job[2], d->v_stride, group, d->o_stride, 1, d->q_stride, 1, d->dv, d->dk);
  for (int j : {0, 2}) {  // states read transposed
    c->job[j].init_row = 1;
    c->job[j].init_col = d->dv;
  }
  for (int j : {1, 2}) {
    c->job[j].reverse = 1;
    c->job[j].off = 0;
    c->job[j].inter = 1.0;
    c->job[j].write = scale;
  }
}

inline size_t round256(size_t b) { return (b + 255) & ~size_t(255); }

// fn(element type tag)
template <typename F> int by_type(int dtype, F fn) {
  switch (dtype) {
    case FDWT_F32: return fn(float{});
    case FDWT_F64: return fn(double{});
    case FDWT_F16: return fn(__half{});
    default: return fn(__nv_bfloat16{});
  }
}

}  // namespace
}  // namespace linattn
}  // namespace fdwt

using namespace fdwt;
using namespace fdwt::linattn;

extern "C" size_t fdwt_linattn_forward_workspace(const fdwt_linattn_desc* desc) {
  if (!desc_ok(desc) || !desc_supported(desc) || desc->batch == 0 || desc->length == 0) return 0;
  Call call{};
  shape_jobs(desc, false, &call);
  return call_workspace(desc->dtype, call);
}

extern "C" int fdwt_linattn_forward(const fdwt_linattn_desc* desc, const void* q, const void* k,
                                    const void* v, const void* log_decay,
                                    const void* initial_state, const int32_t* lengths, void* out,
                                    void* final_state, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  FDWT_CHECK(desc_ok(desc));
  if (!desc_supported(desc)) return FDWT_ERR_UNSUPPORTED;
  if (desc->batch == 0) return FDWT_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (desc->length == 0) {  // the state passes through
    if (final_state == nullptr) return FDWT_OK;
    const size_t bytes = size_t(desc->batch) * desc->heads * desc->dk * desc->dv *
                         (desc->dtype == FDWT_F64 ? 8 : 4);
    if (initial_state == nullptr) FDWT_CUDA(cudaMemsetAsync(final_state, 0, bytes, s));
    else FDWT_CUDA(cudaMemcpyAsync(final_state, initial_state, bytes, cudaMemcpyDeviceToDevice, s));
    return FDWT_OK;
  }
  FDWT_CHECK(q != nullptr && k != nullptr && v != nullptr && log_decay != nullptr && out != nullptr);
  const size_t need = fdwt_linattn_forward_workspace(desc);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return FDWT_ERR_WORKSPACE;
  FDWT_CHECK(need == 0 || reinterpret_cast<uintptr_t>(workspace) % kWorkspaceAlign == 0);
  Call call{};
  shape_jobs(desc, false, &call);
  call.log_decay = log_decay;
  call.lengths = lengths;
  Job& j = call.job[0];
  j.q = q;
  j.k = k;
  j.v = v;
  j.o = out;
  j.init = initial_state;
  j.fin = final_state;
  return run(desc->dtype, call, workspace, s);
}

// A gradient of every query head in 32 bits (64 for fp64).
static size_t per_head_bytes(const fdwt_linattn_desc* desc, int dim) {
  return size_t(desc->batch) * desc->length * desc->heads * dim *
         (desc->dtype == FDWT_F64 ? 8 : 4);
}

extern "C" size_t fdwt_linattn_backward_workspace(const fdwt_linattn_desc* desc) {
  if (!desc_ok(desc) || !desc_supported(desc) || desc->batch == 0 || desc->length == 0) return 0;
  Call call{};
  shape_jobs(desc, true, &call);
  size_t bytes = call_workspace(desc->dtype, call);
  if (desc->heads != desc->kv_heads)
    bytes = round256(bytes) + round256(per_head_bytes(desc, desc->dk)) +
            per_head_bytes(desc, desc->dv);
  return bytes;
}

extern "C" int fdwt_linattn_backward(const fdwt_linattn_desc* desc, const void* q, const void* k,
                                     const void* v, const void* log_decay,
                                     const void* initial_state, const int32_t* lengths,
                                     const void* d_out, const void* d_final_state, void* dq,
                                     void* dk, void* dv, void* d_initial_state, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  FDWT_CHECK(desc_ok(desc));
  if (!desc_supported(desc)) return FDWT_ERR_UNSUPPORTED;
  if (desc->batch == 0) return FDWT_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (desc->length == 0) {
    if (d_initial_state == nullptr) return FDWT_OK;
    const size_t bytes = size_t(desc->batch) * desc->heads * desc->dk * desc->dv *
                         (desc->dtype == FDWT_F64 ? 8 : 4);
    if (d_final_state == nullptr) FDWT_CUDA(cudaMemsetAsync(d_initial_state, 0, bytes, s));
    else FDWT_CUDA(cudaMemcpyAsync(d_initial_state, d_final_state, bytes, cudaMemcpyDeviceToDevice, s));
    return FDWT_OK;
  }
  FDWT_CHECK(q != nullptr && k != nullptr && v != nullptr && log_decay != nullptr &&
             d_out != nullptr && dq != nullptr && dk != nullptr && dv != nullptr);
  const size_t need = fdwt_linattn_backward_workspace(desc);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return FDWT_ERR_WORKSPACE;
  FDWT_CHECK(need == 0 || reinterpret_cast<uintptr_t>(workspace) % kWorkspaceAlign == 0);
  Call call{};
  shape_jobs(desc, true, &call);
  call.log_decay = log_decay;
  call.lengths = lengths;
  const bool shared = desc->heads != desc->kv_heads;
  char* ws = static_cast<char*>(workspace);
  void *dk_all = dk, *dv_all = dv;
  if (shared) {  // per query head first
    char* p = ws + round256(call_workspace(desc->dtype, call));
    dk_all = p;
    dv_all = p + round256(per_head_bytes(desc, desc->dk));
    call.job[1].o_wide = call.job[2].o_wide = dtype_size(desc->dtype) == 2;
  }
  auto set = [&](Job& j, const void* jq, const void* jk, const void* jv, void* jo,
                 const void* init, void* fin) {
    j.q = jq;
    j.k = jk;
    j.v = jv;
    j.o = jo;
    j.init = init;
    j.fin = fin;
  };
  set(call.job[0], d_out, v, k, dq, initial_state, nullptr);
  set(call.job[1], k, q, d_out, dv_all, d_final_state, d_initial_state);
  set(call.job[2], v, d_out, q, dk_all, d_final_state, nullptr);
  int st = run(desc->dtype, call, ws, s);
  if (st != FDWT_OK || !shared) return st;
  const int group = desc->heads / desc->kv_heads;
  return by_type(desc->dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    for (int which = 0; which < 2; ++which) {
      const int dim = which == 0 ? desc->dk : desc->dv;
      const int64_t rows = desc->batch * desc->length * desc->kv_heads;
      void* to = which == 0 ? dk : dv;
      const bool wide = dim % 4 == 0 && reinterpret_cast<uintptr_t>(to) % (4 * sizeof(T)) == 0;
      const int64_t blocks = cdiv(rows, 256 / (wide ? dim / 4 : dim));
      if (blocks > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
      const int e = pre_launch(s);
      if (e != FDWT_OK) return e;
      auto go = [&](auto width) {
        linattn_group_sum_kernel<T, decltype(width)::value>
            <<<static_cast<unsigned>(blocks), 256, 0, s>>>(
                static_cast<const typename AccOf<T>::type*>(which == 0 ? dk_all : dv_all),
                static_cast<T*>(to), rows, group, dim);
      };
      if (wide) go(std::integral_constant<int, 4>{});
      else go(std::integral_constant<int, 1>{});
      const int l = launch_status();
      if (l != FDWT_OK) return l;
    }
    return FDWT_OK;
  });
}

extern "C" int fdwt_linattn_step(const fdwt_linattn_desc* desc, const void* q, const void* k,
                                 const void* v, const void* log_decay, void* state,
                                 int64_t state_slots, const int32_t* slots, void* out,
                                 void* stream) {
  FDWT_CHECK(desc_ok(desc) && desc->length == 1 && state_slots >= 0);
  FDWT_CHECK(slots != nullptr || state_slots >= desc->batch);
  if (desc->dk > 256 || desc->dv > 256) return FDWT_ERR_UNSUPPORTED;
  if (desc->batch == 0) return FDWT_OK;
  FDWT_CHECK(q != nullptr && k != nullptr && v != nullptr && log_decay != nullptr &&
             state != nullptr && out != nullptr);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return by_type(desc->dtype, [&](auto tag) -> int {
    using T = decltype(tag);
    using A = typename AccOf<T>::type;
    constexpr int W = 16 / sizeof(A);
    const bool vec = desc->dv % W == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0;
    const int groups = vec ? desc->dv / W : desc->dv;
    const int64_t bh = desc->batch * desc->heads;
    // columns a block: all of them (up to 32 groups) while the blocks fill the SMs, fewer when
    // they do not
    int lanes = 32;
    while (lanes > 4 && (lanes / 2 >= groups || bh * cdiv(groups, lanes) < sm_count())) lanes /= 2;
    const int64_t tiles = cdiv(groups, lanes);
    if (bh * tiles > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
    const int st = pre_launch(s);
    if (st != FDWT_OK) return st;
    auto go = [&](auto width) {
      linattn_step_kernel<T, decltype(width)::value>
          <<<static_cast<unsigned>(bh * tiles), 256, 0, s>>>(
              *desc, static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
              static_cast<const A*>(log_decay), static_cast<A*>(state), state_slots, slots,
              static_cast<T*>(out), lanes, static_cast<int>(tiles));
    };
    if (vec) go(std::integral_constant<int, W>{});
    else go(std::integral_constant<int, 1>{});
    return launch_status();
  });
}
