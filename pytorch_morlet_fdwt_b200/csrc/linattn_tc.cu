// Linear attention with a decay for each head on the tensor cores (tcgen05): fp16 and bf16,
// head sizes up to 128.  The mathematics, the jobs and the segments are in linattn.cuh.
//
// One block per SM runs one head's segment, 64 value columns of it, in chunks of 128 tokens:
//
//   Sc = Q K^T            (128 x 128)    shared x shared   -> TMEM, two buffers
//   P  = Sc * M           rounded to 16 bits, TMEM -> registers -> TMEM
//   Oi = P V              (128 x 64)     TMEM x shared     -> TMEM
//   Oe = Q S              (128 x 64)     shared x shared   -> TMEM, S the 16-bit copy of the state
//   U  = K^T (V' + V'')   (DK x 64)      shared x shared   -> TMEM
//   o  = diag(d^{l+off}) inter Oe + Oi,  S <- d^m S + write U   in registers, 32 bits
//
// V' + V'' is diag(d^{m-off-l}) V in two 16-bit parts: one part would leave the state 2^-9
// (bf16) off per token, two leave 2^-17.  The scores and the copy of S that multiplies Q are
// rounded once to the operands' type, as the products need it; their errors are of the size of
// the result's own rounding.  fp16 would overflow or lose small values there: each row of P and
// each copy of S is scaled by a power of two first, undone in the sum for o.
//
// Bound: 2 (2 Dk + 2 Dv) bytes of HBM a token and head against about 4 (Dk Dv + 128 (Dk + Dv))
// operations, 96 a byte at 128 x 128, under half of the tensor rate at the HBM rate.  What costs
// is the chain of dependent steps in a chunk, so every step has its own warps and the chunks
// overlap: four warps load (cp.async) and form V' + V'', one issues all products, four form P,
// four keep the state, four finish o.  Every wait on a barrier has a time limit.
#include <type_traits>

#include "linattn.cuh"

namespace fdwt {
namespace linattn {
namespace {

constexpr int C = kTcChunk;   // tokens a chunk (the M of the products over tokens)
constexpr int NV = kTcTile;   // value columns a block
constexpr int kPanel = C * 128;  // bytes of 128 rows of 64 elements, 128-byte swizzled

// ------------------------------------------------------------------------------ PTX
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void bar_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count)
               : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n"
      " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}
constexpr long long kWaitCycles = 4000000000LL;  // about two seconds
// False: the wait ran out here or elsewhere in the block; the block then ends early.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* failed) {
  if (bar_try(bar, parity)) return true;
  const long long start = clock64();
  while (!bar_try(bar, parity)) {
    if (*failed) return false;
    if (clock64() - start > kWaitCycles) {
      *failed = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void fence_async() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tc_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_addr(bar))
               : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
      : "memory");
}
// D = A B + 2^-11 D
__device__ __forceinline__ void mma_ss_shift11(uint32_t d, uint64_t a, uint64_t b,
                                               uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, 1, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, 11;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&r)[32]) {
  uint32_t u[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]),
        "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]),
        "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __uint_as_float(u[i]);
}
// Waits for the warp's loads; the values go through the statement so that no use moves above it.
template <int N> __device__ __forceinline__ void tmem_ld_wait(float (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(r[i]));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&r)[16]) {
  uint32_t u[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]),
        "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]),
        "=r"(u[14]), "=r"(u[15])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&u)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]),
      "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared-memory operand descriptor: 128-byte swizzle, 8-row groups 1024 bytes apart, panels of
// 64 elements `lead` bytes apart (used where the operand's rows run along the contraction).
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
  return uint64_t((addr & 0x3FFFF) >> 4) | (uint64_t(lead >> 4) << 16) |
         (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Instruction descriptor: fp32 result, 16-bit operands; a_mn / b_mn: the operand's contiguous
// axis is M / N instead of the contraction.
template <typename T> constexpr uint32_t instr(int m, int n, bool a_mn, bool b_mn) {
  const uint32_t type = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ type make(float a, float b) { return __floats2bfloat162_rn(a, b); }
  static __device__ __forceinline__ float2 split(type v) { return __bfloat1622float2(v); }
};
template <> struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ type make(float a, float b) { return __floats2half2_rn(a, b); }
  static __device__ __forceinline__ float2 split(type v) { return __half22float2(v); }
};
template <typename T> __device__ __forceinline__ uint32_t pack(float a, float b) {
  typename Pair<T>::type p = Pair<T>::make(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}
template <typename T> __device__ __forceinline__ float2 unpack(uint32_t u) {
  return Pair<T>::split(*reinterpret_cast<typename Pair<T>::type*>(&u));
}

// d^n for n >= 0; d^0 = 1 also for d = 0.
__device__ __forceinline__ float decay_pow(float a, float n) {
  return n == 0.0f ? 1.0f : expf(a * n);
}
// The power of two that brings `most` to 2^13 .. 2^14 (1 for 0, infinities and NaN), and its
// inverse.
__device__ __forceinline__ float scale_of(float most, float* inverse) {
  const int e = int((__float_as_uint(most) >> 23) & 255);
  if (e == 0 || e == 255) {
    *inverse = 1.0f;
    return 1.0f;
  }
  int s = 127 + 13 - e;  // exponent of the factor
  s = s > 100 ? 100 : (s < -100 ? -100 : s);
  *inverse = __uint_as_float(uint32_t(127 - s) << 23);
  return __uint_as_float(uint32_t(127 + s) << 23);
}

// ------------------------------------------------------------------------------ a block's work
struct Where {
  const Job* job;
  int64_t bh, n, begin, end, row_end;  // valid tokens [begin, end) and rows [begin, row_end)
  int h, b, seg, last, v0, vcols, chunks;
  float a;
};

__device__ __forceinline__ Where locate(const Call& call) {
  Where w;
  int tile = blockIdx.x % call.tiles;
  const int64_t rest = blockIdx.x / call.tiles;
  const int64_t heads = call.batch * call.heads;
  w.bh = rest % heads;
  w.seg = static_cast<int>(rest / heads);
  int ji = 0;
  while (tile >= call.job[ji].tiles) tile -= call.job[ji++].tiles;
  w.job = &call.job[ji];
  w.b = static_cast<int>(w.bh / call.heads);
  w.h = static_cast<int>(w.bh % call.heads);
  w.v0 = tile * NV;
  w.vcols = w.job->dv - w.v0 < NV ? w.job->dv - w.v0 : NV;
  int64_t n = call.length;
  if (call.lengths != nullptr) {
    n = call.lengths[w.b];
    n = n < 0 ? 0 : (n > call.length ? call.length : n);
  }
  w.n = n;
  w.last = n == 0 ? 0 : static_cast<int>((n - 1) / call.seg_len);
  w.a = static_cast<const float*>(call.log_decay)[w.h];
  w.begin = int64_t(w.seg) * call.seg_len;
  w.row_end = imin(w.begin + call.seg_len, call.length);
  w.end = imin(w.row_end, n);
  w.chunks = w.end > w.begin ? static_cast<int>(cdiv(w.end - w.begin, C)) : 0;
  return w;
}

// A loader thread's share of 128 rows x 64 PANELS columns: 16-byte column group `tid % 8` of the
// rows tid / 8 + 16 j of each panel, zeros past the valid rows and columns.
template <typename T, int PANELS> struct Loader {
  const T* base;     // row 0 of the head, this thread's first column
  int64_t stride;    // elements between tokens
  uint32_t in_mask;  // panels whose columns exist
  __device__ __forceinline__ void init(const void* p, const int64_t* s, int64_t b, int head,
                                       int first, int cols, int tid) {
    const int c = tid % 8 * 8;
    base = static_cast<const T*>(p) + b * s[0] + head * s[2] + first;
    stride = s[1];
    in_mask = 0;
#pragma unroll
    for (int i = 0; i < PANELS; ++i)
      if (c + 64 * i < cols) in_mask |= 1u << i;
    if (in_mask) base += c;
  }
  // rows l0 .. l0 + 127 of the job's order, `valid` of them
  __device__ __forceinline__ void load(uint32_t dst, int64_t l0, int64_t n, int reverse, int valid,
                                       int tid) const {
    const int r0 = tid / 8;
    const uint32_t cell = dst + r0 * 128 + (((tid % 8) ^ (r0 & 7)) << 4);
    const int64_t step = reverse ? -stride : stride;
    const T* row = base + (reverse ? n - 1 - l0 : l0) * stride;
#pragma unroll
    for (int j = 0; j < C / 16; ++j) {
      const bool in = r0 + 16 * j < valid;
      const T* src = in ? row + (r0 + 16 * j) * step : base;
#pragma unroll
      for (int i = 0; i < PANELS; ++i) {
        const bool ok = in && (in_mask >> i & 1);
        cp_async16(cell + i * kPanel + j * 16 * 128, ok ? src + 64 * i : base, ok);
      }
    }
  }
};

// The second part of a weighted value is held times 2^11 in fp16: where the first part is
// subnormal (a small value, far behind), an unscaled second part would have no bits left.
template <typename T> constexpr float kLowScale = std::is_same<T, __half>::value ? 2048.0f : 1.0f;

// diag(weight) V in two 16-bit parts.  A loader thread reads back the groups it copied itself.
template <typename T>
__device__ __forceinline__ void split_values(const unsigned char* v, unsigned char* high,
                                             unsigned char* low, const float (&weight)[C / 16],
                                             int tid) {
  const int r0 = tid / 8;
  const int cell = r0 * 128 + (((tid % 8) ^ (r0 & 7)) << 4);
#pragma unroll
  for (int j = 0; j < C / 16; ++j) {
    const int at = cell + j * 16 * 128;
    const uint4 x = *reinterpret_cast<const uint4*>(v + at);
    const uint32_t in[4] = {x.x, x.y, x.z, x.w};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f = unpack<T>(in[i]);
      f.x *= weight[j];
      f.y *= weight[j];
      hi[i] = pack<T>(f.x, f.y);
      const float2 g = unpack<T>(hi[i]);
      lo[i] = pack<T>((f.x - g.x) * kLowScale<T>, (f.y - g.y) * kLowScale<T>);
    }
    *reinterpret_cast<uint4*>(high + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(low + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
}

// D (+)= K^T B over a chunk: M runs along the heads' size, the contraction over the tokens.
// shift: D counts 2^-11 in the sum.
template <typename T, int DK, bool SHIFT>
__device__ __forceinline__ void issue_update(uint32_t d, uint32_t k, uint32_t b, bool add) {
  constexpr uint32_t id = instr<T>(DK, NV, true, true);
#pragma unroll
  for (int i = 0; i < C / 16; ++i) {
    const uint64_t x = operand(k + i * 2048, kPanel), y = operand(b + i * 2048, kPanel);
    if (SHIFT && i == 0) mma_ss_shift11(d, x, y, id);
    else mma_ss(d, x, y, id, add || i > 0);
  }
}

constexpr int kThreads = 544;  // 4 warps each: P, o, state, loads; one issues the products
constexpr uint32_t kColumns = 512;
// TMEM columns
constexpr uint32_t kSc = 0, kP = 256, kOe = 320, kOi = 384, kU = 448;

template <int DK> struct Smem {
  static constexpr int panels = DK / 64;
  static constexpr int stages = DK == 64 ? 3 : 2;
  static constexpr int q = 0, k = panels * kPanel, v = 2 * panels * kPanel;
  static constexpr int stage = (2 * panels + 1) * kPanel;
  static constexpr int high = stages * stage, low = high + kPanel, s = low + kPanel;
  static constexpr int out = s + DK * 128;
  static constexpr int bytes = out + kPanel + 1024;  // 1024: room to align the base
  // the state launch: K, V, and two buffers of V' + V''
  static constexpr int st_stage = (panels + 1) * kPanel;
  static constexpr int st_stages = 3;
  static constexpr int st_high = st_stages * st_stage;
  static constexpr int st_bytes = st_high + 4 * kPanel + 1024;
};

__device__ __forceinline__ unsigned char* align_smem(unsigned char* p) {
  return p + ((1024 - (smem_addr(p) & 1023)) & 1023);
}

__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(slot)),
               "r"(kColumns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(kColumns)
               : "memory");
}

// ------------------------------------------------------------------------------ main launch
template <typename T, int DK>
__global__ void __launch_bounds__(kThreads, 1)
linattn_tc_kernel(const __grid_constant__ Call call, int* error) {
  using Z = Smem<DK>;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr int S = Z::stages;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = align_smem(raw);
  __shared__ uint64_t full[S], empty[S], sc_full[2], sc_empty[2], p_full, o_full, o_empty, s_full,
      u_full, u_empty, vp_full, most_full, drain;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  __shared__ float power[64];          // power[31 + n] = intra d^n, n = 0 .. 31
  __shared__ float p_inv[2][C];        // fp16: inverse scales of P's rows
  __shared__ float s_inv[2];           // fp16: inverse scale of the state's copy
  __shared__ volatile float s_most[4];  // fp16: largest magnitude of each warp's rows

  const Where w = locate(call);
  const Job& job = *w.job;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      bar_init(&full[i], 128);
      bar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&sc_full[i], 1);
      bar_init(&sc_empty[i], 128);
    }
    bar_init(&p_full, 128);
    bar_init(&o_full, 1);
    bar_init(&o_empty, 128);
    bar_init(&s_full, 128);
    bar_init(&u_full, 1);
    bar_init(&u_empty, 128);
    bar_init(&vp_full, 128);
    bar_init(&most_full, 4);
    bar_init(&drain, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >= 64 && threadIdx.x < 128) {
    const int i = threadIdx.x - 64;
    power[i] = i < 31 ? 0.0f : float(job.intra) * decay_pow(w.a, float(i - 31));
  }
  if (warp == 16) tmem_alloc(&tmem_slot);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;
  const uint32_t base = smem_addr(sm);
  const int chunks = w.chunks;

  if (warp < 4) {
    // ---- P = Sc * M.  Row t = 32 warp + lane; 32 columns at a time, those above the diagonal
    // are zero once and for all.  Off the diagonal block d^{t-s} = (intra d^{32(w-j-1)+lane+1})
    // d^{31-c}: both powers are at least 0, nothing overflows.
    float tab[32];
#pragma unroll
    for (int c = 0; c < 32; ++c) tab[c] = decay_pow(w.a, float(31 - c));
    float lead = float(job.intra) * decay_pow(w.a, float(lane + 1));
    const float block = decay_pow(w.a, 32.0f);
    {
      uint32_t zero[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) zero[i] = 0;
      for (int j = warp + 1; j < 4; ++j) tmem_st16(tmem + lanes + kP + j * 16, zero);
      tmem_st_wait();
    }
    bool ok = true;
    for (int i = 0; i < chunks && ok; ++i) {
      ok = bar_wait(&sc_full[i & 1], (i >> 1) & 1, &failed);
      if (ok && i > 0) ok = bar_wait(&o_full, (i - 1) & 1, &failed);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_after();
      const uint32_t sc = tmem + lanes + kSc + (i & 1) * 128;
      float scale = 1.0f;
      if (kHalf) {
        float most = 0.0f, f = lead;
        for (int j = warp; j >= 0; --j) {
          float x[32];
          tmem_ld32(sc + j * 32, x);
          tmem_ld_wait(x);
          if (j == warp) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c <= lane) most = fmaxf(most, fabsf(x[c] * power[31 + lane - c]));
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) most = fmaxf(most, fabsf(x[c] * (f * tab[c])));
            f *= block;
          }
        }
        float inv;
        scale = scale_of(most, &inv);
        p_inv[i & 1][warp * 32 + lane] = inv;
      }
      float f = lead * scale;
      for (int j = warp; j >= 0; --j) {
        float x[32];
        uint32_t u[16];
        tmem_ld32(sc + j * 32, x);
        tmem_ld_wait(x);
        if (j == warp) {
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float p = x[c] * power[31 + lane - c];
            x[c] = c <= lane ? (kHalf ? p * scale : p) : 0.0f;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] *= f * tab[c];
          f *= block;
        }
#pragma unroll
        for (int c = 0; c < 16; ++c) u[c] = pack<T>(x[2 * c], x[2 * c + 1]);
        tmem_st16(tmem + lanes + kP + j * 16, u);
      }
      tmem_st_wait();
      tc_before();
      bar_arrive(&sc_empty[i & 1]);
      bar_arrive(&p_full);
    }
  } else if (warp < 8) {
    // ---- o = inter d^{t+off} Oe + Oi, through shared memory into whole 128-byte rows
    const int t = (warp - 4) * 32 + lane;
    const float read = float(job.inter) * decay_pow(w.a, float(t + job.off));
    unsigned char* stage = sm + Z::out + (warp - 4) * 4096;
    const size_t head = size_t(int64_t(w.b) * job.os[0] + int64_t(w.h) * job.os[2] + w.v0);
    bool ok = true;
    for (int i = 0; i < chunks && ok; ++i) {
      ok = __all_sync(0xffffffffu, bar_wait(&o_full, i & 1, &failed));
      if (!ok) break;
      tc_after();
      const int64_t l0 = w.begin + int64_t(i) * C;
      const int m = static_cast<int>(imin(C, w.end - l0));
      const float fe = kHalf ? read * s_inv[i & 1] : read;
      const float fi = kHalf ? p_inv[i & 1][t] : 1.0f;
      const int64_t first = job.reverse ? w.n - 1 - l0 : l0;  // token of row 0
      const int64_t step = job.reverse ? -job.os[1] : job.os[1];
      const int row0 = (warp - 4) * 32, rows = m - row0;  // rows of this warp
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float e[32], x[32];
        tmem_ld32(tmem + lanes + kOe + half * 32, e);
        tmem_ld32(tmem + lanes + kOi + half * 32, x);
        tmem_ld_wait(e);
        tmem_ld_wait(x);
        if (half == 1) {
          tc_before();
          bar_arrive(&o_empty);
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) x[c] = kHalf ? fe * e[c] + fi * x[c] : fe * e[c] + x[c];
        if (!job.o_wide) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float* y = x + g * 8;
            *reinterpret_cast<uint4*>(stage + lane * 128 + (((half * 4 + g) ^ (lane & 7)) << 4)) =
                make_uint4(pack<T>(y[0], y[1]), pack<T>(y[2], y[3]), pack<T>(y[4], y[5]),
                           pack<T>(y[6], y[7]));
          }
        } else {  // 32-bit results (added over heads later), 32 columns at a time
          float* o = static_cast<float*>(job.o) + head + first * job.os[1];
#pragma unroll
          for (int g = 0; g < 8; ++g)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((g ^ (lane & 7)) << 4)) =
                make_float4(x[g * 4], x[g * 4 + 1], x[g * 4 + 2], x[g * 4 + 3]);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = j * 4 + lane / 8, g = lane % 8, c = half * 32 + g * 4;
            if (r < rows && c < w.vcols)
              *reinterpret_cast<float4*>(o + (row0 + r) * step + c) =
                  *reinterpret_cast<const float4*>(stage + r * 128 + ((g ^ (r & 7)) << 4));
          }
          __syncwarp();
        }
      }
      if (!job.o_wide) {
        __syncwarp();
        T* o = static_cast<T*>(job.o) + head + first * job.os[1];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = j * 4 + lane / 8, g = lane % 8;
          if (r < rows && g * 8 < w.vcols) {
            const uint4 u = *reinterpret_cast<const uint4*>(stage + r * 128 + ((g ^ (r & 7)) << 4));
            T* dst = o + (row0 + r) * step + g * 8;
            if (job.o_vec) {
              *reinterpret_cast<uint4*>(dst) = u;
            } else {
              const T* e = reinterpret_cast<const T*>(&u);
              for (int c = 0; c < 8 && g * 8 + c < w.vcols; ++c) dst[c] = e[c];
            }
          }
        }
        __syncwarp();
      }
    }
  } else if (warp < 12) {
    // ---- the state, a row of 64 columns a thread (DK = 64: 16 rows a warp, the lanes that a
    // product with M = 64 fills)
    const int r = DK == 128 ? (warp - 8) * 32 + lane : (warp - 8) * 16 + (lane & 15);
    const bool mine = DK == 128 || lane < 16;
    const int64_t size = int64_t(job.dk) * job.dv;
    const float write = float(job.write);
    float s[2][32];
    {
      const float* src = nullptr;
      int64_t row = job.dv, col = 1;
      if (w.seg == 0) {
        if (job.init != nullptr) {
          src = static_cast<const float*>(job.init) + w.bh * size;
          row = job.init_row;
          col = job.init_col;
        }
      } else if (w.seg <= w.last) {
        src = static_cast<const float*>(job.seg) + (w.bh * (call.nseg - 1) + w.seg - 1) * size;
      }
      const bool in = src != nullptr && mine && r < job.dk;
#pragma unroll
      for (int c = 0; c < NV; ++c)
        s[c / 32][c % 32] = in && c < w.vcols ? src[r * row + (w.v0 + c) * col] : 0.0f;
    }
    bool ok = true;
    for (int i = 0; i <= chunks && ok; ++i) {
      if (i > 0) {
        ok = __all_sync(0xffffffffu, bar_wait(&u_full, (i - 1) & 1, &failed));
        if (!ok) break;
        tc_after();
        const int m = static_cast<int>(imin(C, w.end - (w.begin + int64_t(i - 1) * C)));
        const float keep = decay_pow(w.a, float(m));
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          float x[16];
          tmem_ld16(tmem + lanes + kU + part * 16, x);
          tmem_ld_wait(x);
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            float& y = s[part / 2][part % 2 * 16 + c];
            y = keep * y + write * x[c];
          }
        }
        tc_before();
        bar_arrive(&u_empty);
        if (i == chunks) break;
        ok = __all_sync(0xffffffffu, bar_wait(&o_full, (i - 1) & 1, &failed));
        if (!ok) break;
      }
      if (chunks == 0) break;
      float scale = 1.0f;
      if (kHalf) {
        float most = 0.0f;
        if (mine) {
#pragma unroll
          for (int c = 0; c < NV; ++c) most = fmaxf(most, fabsf(s[c / 32][c % 32]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        // (rewritten only after o_full of this chunk, which follows every warp's s_full)
        if (lane == 0) {
          s_most[warp - 8] = most;
          bar_arrive(&most_full);
        }
        ok = __all_sync(0xffffffffu, bar_wait(&most_full, i & 1, &failed));
        if (!ok) break;
        most = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
        float inv;
        scale = scale_of(most, &inv);
        if (warp == 8 && lane == 0) s_inv[i & 1] = inv;
      }
      if (mine) {
        unsigned char* row = sm + Z::s + r * 128;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float* y = &s[g / 4][g % 4 * 8];
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            u[e] = kHalf ? pack<T>(y[2 * e] * scale, y[2 * e + 1] * scale)
                         : pack<T>(y[2 * e], y[2 * e + 1]);
          *reinterpret_cast<uint4*>(row + ((g ^ (r & 7)) << 4)) = make_uint4(u[0], u[1], u[2], u[3]);
        }
      }
      fence_async();
      bar_arrive(&s_full);
    }
    if (ok && w.seg == w.last && job.fin != nullptr && mine && r < job.dk) {
      float* dst = static_cast<float*>(job.fin) + w.bh * size + int64_t(r) * job.dv + w.v0;
#pragma unroll
      for (int c = 0; c < NV; ++c)
        if (c < w.vcols) dst[c] = s[c / 32][c % 32];
    }
  } else if (warp < 16) {
    // ---- loads, and V' + V''
    const int tid = threadIdx.x - 384;
    Loader<T, Z::panels> lq, lk;
    Loader<T, 1> lv;
    lq.init(job.q, job.qs, w.b, w.h / job.q_group, 0, job.dk, tid);
    lk.init(job.k, job.ks, w.b, w.h / job.k_group, 0, job.dk, tid);
    lv.init(job.v, job.vs, w.b, w.h / job.v_group, w.v0, w.vcols, tid);
    auto load = [&](int i) {
      const int64_t l0 = w.begin + int64_t(i) * C;
      const int m = static_cast<int>(imin(C, w.end - l0));
      const uint32_t at = base + (i % S) * Z::stage;
      lq.load(at + Z::q, l0, w.n, job.reverse, m, tid);
      lk.load(at + Z::k, l0, w.n, job.reverse, m, tid);
      lv.load(at + Z::v, l0, w.n, job.reverse, m, tid);
    };
    float weight[C / 16];
    int weight_m = 0;
    for (int i = 0; i < S - 1; ++i) {
      if (i < chunks) load(i);
      cp_commit();
    }
    for (int i = 0; i < chunks; ++i) {
      cp_wait<S - 2>();
      fence_async();
      bar_arrive(&full[i % S]);
      const int m = static_cast<int>(imin(C, w.end - (w.begin + int64_t(i) * C)));
      if (m != weight_m) {
        weight_m = m;
#pragma unroll
        for (int j = 0; j < C / 16; ++j) {
          const int age = m - job.off - (tid / 8 + 16 * j);
          weight[j] = age < 0 ? 0.0f : decay_pow(w.a, float(age));
        }
      }
      if (i > 0 && !bar_wait(&u_full, (i - 1) & 1, &failed)) break;
      split_values<T>(sm + (i % S) * Z::stage + Z::v, sm + Z::high, sm + Z::low, weight, tid);
      fence_async();
      bar_arrive(&vp_full);
      const int next = i + S - 1;
      if (next < chunks) {
        if (i > 0 && !bar_wait(&empty[next % S], (next / S - 1) & 1, &failed)) break;
        load(next);
      }
      cp_commit();
    }
    cp_wait<0>();
  } else {
    // ---- all products, issued by one lane
    constexpr uint32_t id_sc = instr<T>(C, C, false, false);
    constexpr uint32_t id_o = instr<T>(C, NV, false, true);
    auto scores = [&](int i) {
      if (lane == 0) {
        tc_after();
        const uint32_t at = base + (i % S) * Z::stage;
#pragma unroll
        for (int j = 0; j < DK / 16; ++j) {
          const uint32_t off = j / 4 * kPanel + j % 4 * 32;
          mma_ss(tmem + kSc + (i & 1) * 128, operand(at + Z::q + off, kPanel),
                 operand(at + Z::k + off, kPanel), id_sc, j > 0);
        }
        tc_commit(&sc_full[i & 1]);
      }
      __syncwarp();
    };
    // true: chunk i's operands are there and its score buffer is free
    auto ready = [&](int i) {
      return bar_wait(&full[i % S], (i / S) & 1, &failed) &&
             (i < 2 || bar_wait(&sc_empty[i & 1], ((i >> 1) - 1) & 1, &failed));
    };
    bool ok = true;
    if (chunks > 0) {
      ok = __all_sync(0xffffffffu, ready(0));
      if (ok) scores(0);
    }
    for (int i = 0; i < chunks && ok; ++i) {
      const uint32_t at = base + (i % S) * Z::stage;
      ok = bar_wait(&vp_full, i & 1, &failed) &&
           (i == 0 || bar_wait(&u_empty, (i - 1) & 1, &failed));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        tc_after();
        issue_update<T, DK, false>(tmem + kU, at + Z::k, base + Z::low, false);
        issue_update<T, DK, kHalf>(tmem + kU, at + Z::k, base + Z::high, true);
        tc_commit(&u_full);
      }
      __syncwarp();
      ok = bar_wait(&s_full, i & 1, &failed) &&
           (i == 0 || bar_wait(&o_empty, (i - 1) & 1, &failed));
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        tc_after();
#pragma unroll
        for (int j = 0; j < DK / 16; ++j)
          mma_ss(tmem + kOe, operand(at + Z::q + j / 4 * kPanel + j % 4 * 32, kPanel),
                 operand(base + Z::s + j * 2048, kPanel), id_o, j > 0);
      }
      __syncwarp();
      // the next chunk's scores go before this one's P V where their operands are there already
      bool ahead = i + 1 < chunks && bar_try(&full[(i + 1) % S], ((i + 1) / S) & 1);
      ahead = __all_sync(0xffffffffu, ahead);
      if (ahead) {
        ok = __all_sync(0xffffffffu, ready(i + 1));
        if (!ok) break;
        scores(i + 1);
      }
      ok = __all_sync(0xffffffffu, bar_wait(&p_full, i & 1, &failed));
      if (!ok) break;
      if (lane == 0) {
        tc_after();
#pragma unroll
        for (int j = 0; j < C / 16; ++j)
          mma_ts(tmem + kOi, tmem + kP + j * 8, operand(at + Z::v + j * 2048, kPanel), id_o, j > 0);
        tc_commit(&o_full);
        tc_commit(&empty[i % S]);
      }
      __syncwarp();
      if (!ahead && i + 1 < chunks) {
        ok = __all_sync(0xffffffffu, ready(i + 1));
        if (ok) scores(i + 1);
      }
    }
    if (!ok) {  // let the products in flight end before TMEM goes
      if (lane == 0) tc_commit(&drain);
      __syncwarp();
      const long long start = clock64();
      while (!bar_try(&drain, 0) && clock64() - start < kWaitCycles) {
      }
    }
  }
  // rows after the sequence's end
  {
    const int64_t from = imax(w.begin, w.n);
    const int64_t cells = (w.row_end - from) * w.vcols;
    for (int64_t i = threadIdx.x; i < cells; i += kThreads) {
      const int64_t at = int64_t(w.b) * job.os[0] + int64_t(w.h) * job.os[2] + w.v0 +
                         (from + i / w.vcols) * job.os[1] + i % w.vcols;
      if (job.o_wide) static_cast<float*>(job.o)[at] = 0.0f;
      else static_cast<T*>(job.o)[at] = from_acc<T>(0.0f);
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 16) {
    tc_after();
    tmem_free(tmem);
    if (lane == 0 && failed) *error = kErrCopyTimeout;
  }
}

// ------------------------------------------------------------------------------ state launch
// A segment's own end state: U += K^T (V' + V''), V' + V'' = diag(d^{end-off-l}) V weighted
// towards the segment's end, so that the sum stays in TMEM over all chunks.
constexpr int kStateThreads = 288;  // loads, result, products: 4 + 4 + 1 warps

template <typename T, int DK>
__global__ void __launch_bounds__(kStateThreads, 1)
linattn_tc_state_kernel(const __grid_constant__ Call call, int* error) {
  using Z = Smem<DK>;
  constexpr int S = Z::st_stages;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = align_smem(raw);
  __shared__ uint64_t vp_full[2], used[S], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  const Where w = locate(call);
  const Job& job = *w.job;
  if (w.seg >= w.last) return;  // the whole block
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) bar_init(&vp_full[i], 128);
    for (int i = 0; i < S; ++i) bar_init(&used[i], 1);
    bar_init(&done, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) tmem_alloc(&tmem_slot);
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t base = smem_addr(sm);
  const int chunks = w.chunks;  // whole ones: every segment before the last is full

  if (warp < 4) {
    const int tid = threadIdx.x;
    Loader<T, Z::panels> lk;
    Loader<T, 1> lv;
    lk.init(job.k, job.ks, w.b, w.h / job.k_group, 0, job.dk, tid);
    lv.init(job.v, job.vs, w.b, w.h / job.v_group, w.v0, w.vcols, tid);
    auto load = [&](int i) {
      const int64_t l0 = w.begin + int64_t(i) * C;
      const uint32_t at = base + (i % S) * Z::st_stage;
      lk.load(at, l0, w.n, job.reverse, C, tid);
      lv.load(at + Z::panels * kPanel, l0, w.n, job.reverse, C, tid);
    };
    for (int i = 0; i < S - 1; ++i) {
      if (i < chunks) load(i);
      cp_commit();
    }
    for (int i = 0; i < chunks; ++i) {
      cp_wait<S - 2>();
      float weight[C / 16];
      const int64_t ages = w.end - job.off - (w.begin + int64_t(i) * C + tid / 8);
#pragma unroll
      for (int j = 0; j < C / 16; ++j) {
        const int64_t age = ages - 16 * j;
        weight[j] = age < 0 ? 0.0f : decay_pow(w.a, float(age));
      }
      // buffer i % 2 of V' + V'' is free when the products of chunk i - 2 have ended
      if (i >= 2 && !bar_wait(&used[(i - 2) % S], ((i - 2) / S) & 1, &failed)) break;
      unsigned char* high = sm + Z::st_high + (i & 1) * 2 * kPanel;
      split_values<T>(sm + (i % S) * Z::st_stage + Z::panels * kPanel, high, high + kPanel, weight,
                      tid);
      fence_async();
      bar_arrive(&vp_full[i & 1]);
      const int next = i + S - 1;
      if (next < chunks) {
        if (i > 0 && !bar_wait(&used[(i - 1) % S], ((i - 1) / S) & 1, &failed)) break;
        load(next);
      }
      cp_commit();
    }
    cp_wait<0>();
  } else if (warp < 8) {
    const bool ok = __all_sync(0xffffffffu, bar_wait(&done, 0, &failed));
    if (ok) {
      tc_after();
      const int r = DK == 128 ? (warp - 4) * 32 + lane : (warp - 4) * 16 + (lane & 15);
      const bool mine = (DK == 128 || lane < 16) && r < job.dk;
      float* dst = static_cast<float*>(job.seg) +
                   (w.bh * (call.nseg - 1) + w.seg) * (int64_t(job.dk) * job.dv) +
                   int64_t(r) * job.dv + w.v0;
      const float write = float(job.write);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[32], y[32];
        const uint32_t at = tmem + (uint32_t(warp % 4 * 32) << 16) + half * 32;
        tmem_ld32(at, x);
        tmem_ld32(at + NV, y);
        tmem_ld_wait(x);
        tmem_ld_wait(y);
        if (mine) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (half * 32 + c < w.vcols) dst[half * 32 + c] = write * (x[c] + y[c] / kLowScale<T>);
        }
      }
    }
  } else {
    bool ok = true;
    for (int i = 0; i < chunks && ok; ++i) {
      ok = __all_sync(0xffffffffu, bar_wait(&vp_full[i & 1], (i >> 1) & 1, &failed));
      if (!ok) break;
      if (lane == 0) {
        tc_after();
        const uint32_t high = base + Z::st_high + (i & 1) * 2 * kPanel;
        const uint32_t k = base + (i % S) * Z::st_stage;
        issue_update<T, DK, false>(tmem, k, high, i > 0);
        issue_update<T, DK, false>(tmem + NV, k, high + kPanel, i > 0);
        tc_commit(&used[i % S]);
      }
      __syncwarp();
    }
    // also after a failed wait: the products in flight end before TMEM goes
    if (lane == 0) tc_commit(&done);
    __syncwarp();
    const long long start = clock64();
    while (!bar_try(&done, 0) && clock64() - start < kWaitCycles) {
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 8) {
    tc_after();
    tmem_free(tmem);
    if (lane == 0 && failed) *error = kErrCopyTimeout;
  }
}

template <typename T, int DK>
int launch_as(const Call& call, bool states, cudaStream_t stream) {
  auto kernel = states ? linattn_tc_state_kernel<T, DK> : linattn_tc_kernel<T, DK>;
  const int64_t heads = call.batch * call.heads;
  const int64_t grid = heads * call.tiles * (states ? call.nseg - 1 : call.nseg);
  int* error = device_error_flag();
  if (error == nullptr) return FDWT_ERR_CUDA;
  int st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
  if (st == FDWT_OK) st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  kernel<<<static_cast<unsigned>(grid), states ? kStateThreads : kThreads,
           states ? Smem<DK>::st_bytes : Smem<DK>::bytes, stream>>>(call, error);
  return launch_status();
}

}  // namespace

bool tc_supports(int dtype, const Call& call) {
  if (dtype != FDWT_F16 && dtype != FDWT_BF16) return false;
  for (int j = 0; j < call.jobs; ++j) {
    const Job& job = call.job[j];
    if (job.dk > 128 || !job.q_vec || !job.k_vec || !job.v_vec) return false;
  }
  return true;
}

int tc_launch(int dtype, const Call& call, bool states, cudaStream_t stream) {
  int dk = 0;
  for (int j = 0; j < call.jobs; ++j) dk = call.job[j].dk > dk ? call.job[j].dk : dk;
  if (dtype == FDWT_F16)
    return dk <= 64 ? launch_as<__half, 64>(call, states, stream)
                    : launch_as<__half, 128>(call, states, stream);
  return dk <= 64 ? launch_as<__nv_bfloat16, 64>(call, states, stream)
                  : launch_as<__nv_bfloat16, 128>(call, states, stream);
}

}  // namespace linattn
}  // namespace fdwt
