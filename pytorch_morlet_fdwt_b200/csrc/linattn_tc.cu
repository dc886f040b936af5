// Linear attention with a decay for each head on the tensor cores (tcgen05): fp16 and bf16,
// head sizes up to 128.  The mathematics, the jobs and the segments are in linattn.cuh.
//
// One block per SM runs one head's segment, 64 value columns of it, in chunks of 128 tokens:
//
//   Sc = Q K^T            (128 x 128)    shared x shared   -> TMEM, two buffers
//   P  = Sc * M           two 16-bit parts, over Sc's columns
//   Oe = Q S              (128 x 64)     shared x shared   -> TMEM, S in two 16-bit parts
//   Oi = P V              (128 x 64)     TMEM x shared     -> TMEM, Oe's columns once it is taken
//   U  = K^T V'           (DK x 64 each part)  shared x shared -> TMEM
//   o  = diag(d^{l+off}) inter Oe + Oi,  S <- d^m S + write U   in registers, 32 bits
//
// What a product needs in 16 bits goes in as the sum of parts, so that the result is that of the
// operator in 32 bits, rounded once: two parts of the scores and of the state's copy that
// multiplies Q (one would put the result 1.41 times as far off as its own rounding does), and of
// V' = diag(d^{m-off-l}) V two (fp16) or three (bf16), which leave the 32-bit state as far off as
// its own sums.  fp16 would overflow or lose small values: each row of P and each copy of S is
// scaled by a power of two first, undone in the sum for o.
//
// Bound: 2 (2 Dk + 2 Dv) bytes of HBM a token and head against about 4 (Dk Dv + 128 (Dk + Dv))
// operations, 96 a byte at 128 x 128, under half of the tensor rate at the HBM rate.  What costs
// is the chain of dependent steps in a chunk, so every step has its own warps and the chunks
// overlap: one warp issues the loads (TMA), one all products, four form P, eight V', four finish
// o, four keep the state.  All parts of V' are one product (N = 64 parts), so that K is read once:
// the shared-memory rate binds the products more than the tensor rate.  Measured with all SMs
// busy, bf16: 2.3 us a chunk with heads of 64 (4 x 4096 tokens of 37 heads, 85 us; 304 KB a chunk
// through shared memory, 1.2 us at its rate), 2.8 us with heads of 128 (2 x 4096 of 37 heads, 102
// us; 448 KB, 1.8 us); 67 and 87 us with P and S in one part.  The first chunk is out after 10 us.
// Every wait on a barrier has a time limit.
#include <cuda.h>

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
// What a block needs to give up: a flag in shared memory and the time limit of a wait, about a
// second (less under the test hook).
struct Limit {
  volatile int* failed;
  long long cycles;
};
constexpr long long kWaitCycles = 2000000000LL, kTestCycles = 2000000LL;
// False: the wait ran out here or elsewhere in the block; the block then ends early.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, const Limit& limit) {
  if (bar_try(bar, parity)) return true;
  const long long start = clock64();
#pragma unroll 1
  while (!bar_try(bar, parity)) {
    if (*limit.failed) return false;
    if (clock64() - start > limit.cycles) {
      *limit.failed = 1;
      return false;
    }
  }
  return true;
}
// For what is in flight after a failure: no regard to the flag.
__device__ __forceinline__ void bar_drain(uint64_t* bar, uint32_t parity, const Limit& limit) {
  const long long start = clock64();
#pragma unroll 1
  while (!bar_try(bar, parity) && clock64() - start < limit.cycles) {
  }
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
// Shared-memory operands are given by the low word of their descriptor (operand() below); the
// high word is the same for all: 128-byte swizzle, 8-row groups 1024 bytes apart.
constexpr uint32_t kOperandHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
// D = A B (+ D), A in shared memory or (mma_ts) in TMEM
template <bool ADD>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 x, y;\n setp.ne.u32 p, %5, 0;\n"
      " mov.b64 x, {%1, %4};\n mov.b64 y, {%2, %4};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "n"(kOperandHigh), "n"(ADD ? 1 : 0)
      : "memory");
}
template <bool ADD>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 y;\n setp.ne.u32 p, %5, 0;\n"
      " mov.b64 y, {%2, %4};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "n"(kOperandHigh), "n"(ADD ? 1 : 0)
      : "memory");
}
// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(is));
  return is != 0;
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
__device__ __forceinline__ void tmem_ld8(uint32_t addr, float (&r)[8]) {
  uint32_t u[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]),
                 "=r"(u[6]), "=r"(u[7])
               : "r"(addr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = __uint_as_float(u[i]);
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
__device__ __forceinline__ void bar_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int token,
                                         int head, int batch, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(token), "r"(head), "r"(batch), "r"(smem_addr(bar))
      : "memory");
}
// (a, b) -= (c, d);  (a, b) += (c, d);  (a, b) = (a, b) * f + (c, d)
__device__ __forceinline__ void sub2(float& a, float& b, float c, float d) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n"
      " sub.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n"
      " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}
__device__ __forceinline__ void fma2(float& a, float& b, float f, float c, float d) {
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n"
      " mov.b64 z, {%4, %4};\n fma.rn.f32x2 x, x, z, y;\n mov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d), "f"(f));
}
// (a, b) * (c, d)
__device__ __forceinline__ void mul2(float& a, float& b, float c, float d) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n"
      " mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
}

// Low word of an operand's descriptor: its address, and `lead`, the distance of its panels of 64
// elements (used where the operand's rows run along the contraction).  An offset of n bytes adds
// n / 16 (addresses stay below 2^18).
__device__ __forceinline__ uint32_t operand(uint32_t addr, uint32_t lead) {
  return (addr >> 4) | ((lead >> 4) << 16);
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
// The first of the two 16-bit parts of (a, b), which keep what is left for the second one.  It is
// cut off rather than rounded: one conversion less, and the second part, rounded, takes up the
// rest (2^-16 of a value in bf16, 2^-21 in fp16).
template <typename T>
__device__ __forceinline__ uint32_t first_part(float& a, float& b) {
  constexpr uint32_t mask = std::is_same<T, __half>::value ? 0xffffe000u : 0xffff0000u;
  const float x = __uint_as_float(__float_as_uint(a) & mask);
  const float y = __uint_as_float(__float_as_uint(b) & mask);
  const uint32_t u = std::is_same<T, __half>::value
                         ? pack<T>(x, y)
                         : __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
  sub2(a, b, x, y);
  return u;
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
  int bh, n, begin, end, row_end;  // valid tokens [begin, end) and rows [begin, row_end)
  int h, b, seg, last, v0, vcols, chunks, ji;
  float a;
};

__device__ __forceinline__ bool first_block() { return blockIdx.x == 0 && blockIdx.y == 0; }

// Block (value tile of the jobs of a sequence and head, segment).
__device__ __forceinline__ Where locate(const Call& call, unsigned x, unsigned y) {
  Where w;
  w.bh = static_cast<int>(x / static_cast<unsigned>(call.tiles));
  int tile = static_cast<int>(x) - w.bh * call.tiles;
  w.seg = static_cast<int>(y);
  int ji = 0;
  while (tile >= call.job[ji].tiles) tile -= call.job[ji++].tiles;
  w.job = &call.job[ji];
  w.ji = ji;
  w.b = static_cast<int>(unsigned(w.bh) / static_cast<unsigned>(call.heads));
  w.h = w.bh - w.b * call.heads;
  w.v0 = tile * NV;
  w.vcols = w.job->dv - w.v0 < NV ? w.job->dv - w.v0 : NV;
  const int length = static_cast<int>(call.length), seg_len = static_cast<int>(call.seg_len);
  int n = length;
  if (call.lengths != nullptr) {
    n = call.lengths[w.b];
    n = n < 0 ? 0 : (n > length ? length : n);
  }
  w.n = n;
  w.last = n == 0 ? 0 : static_cast<int>(unsigned(n - 1) / unsigned(seg_len));
  w.a = static_cast<const float*>(call.log_decay)[w.h];
  w.begin = w.seg * seg_len;
  w.row_end = length - w.begin < seg_len ? length : w.begin + seg_len;
  w.end = w.row_end < n ? w.row_end : n;
  w.chunks = w.end > w.begin ? (w.end - w.begin + C - 1) / C : 0;
  return w;
}

// The operands of the jobs as 4-d tensors (column, token, head, batch), boxes of 64 columns x 64
// tokens, 128-byte swizzle; what lies outside reads as zeros.
constexpr int kBoxRows = 64, kBox = kBoxRows * 128;
struct Maps {
  CUtensorMap map[kMaxJobs][3];  // q, k, v
};
struct Source {
  const CUtensorMap* map;
  int head, batch;
  __device__ __forceinline__ Source(const CUtensorMap* m, const int64_t* stride, int h, int b)
      : map(m), head(stride[2] == 0 ? 0 : h), batch(stride[0] == 0 ? 0 : b) {}
  // ROWS tokens from `token` on, `columns` panels of 64 columns from x on, to dst
  template <int ROWS> __device__ __forceinline__ void load(uint32_t dst, int x, int panels,
                                                           int token, uint64_t* bar) const {
#pragma unroll 1
    for (int i = 0; i < panels; ++i)
#pragma unroll
      for (int r = 0; r < ROWS / kBoxRows; ++r)
        tma_load(dst + (i * (ROWS / kBoxRows) + r) * kBox, map, x + 64 * i,
                 token + r * kBoxRows, head, batch, bar);
  }
};

// Parts of a weighted value.  The second part is held times 2^11 in fp16: where the first part is
// subnormal (a small value, far behind), an unscaled second part would have no bits left.
template <typename T> constexpr bool kIsHalf = std::is_same<T, __half>::value;
template <typename T> constexpr int kParts = kIsHalf<T> ? 2 : 3;
constexpr float kLowScale = 2048.0f;

// V' = diag(weight) V in parts: one 16-byte group.
template <typename T>
__device__ __forceinline__ void split_group(const unsigned char* v, float weight,
                                            uint4 (&out)[kParts<T>]) {
  const uint4 x = *reinterpret_cast<const uint4*>(v);
  const uint32_t in[4] = {x.x, x.y, x.z, x.w};
  uint32_t u[kParts<T>][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f = unpack<T>(in[i]);
    mul2(f.x, f.y, weight, weight);
#pragma unroll
    for (int p = 0; p < kParts<T>; ++p) {
      u[p][i] = pack<T>(f.x, f.y);
      if (p + 1 == kParts<T>) break;
      const float2 g = unpack<T>(u[p][i]);
      sub2(f.x, f.y, g.x, g.y);
      if (kIsHalf<T>) mul2(f.x, f.y, kLowScale, kLowScale);
    }
  }
#pragma unroll
  for (int p = 0; p < kParts<T>; ++p) out[p] = make_uint4(u[p][0], u[p][1], u[p][2], u[p][3]);
}
// ROWS (64 or 32) rows of it by 128 threads: thread tid takes the column group tid % 8 of the rows
// tid / 8 + 16 j, whose weights are weight[from + j].  Part p goes to parts + p * ROWS * 128.
// `ready()` (false: give up) is asked for between forming the first two groups and storing them.
template <typename T, int ROWS, typename F>
__device__ __forceinline__ bool split_values(const unsigned char* v, unsigned char* parts,
                                             const float (&weight)[4], int from, int tid, F ready) {
  const int r0 = tid / 8;
  const int cell = r0 * 128 + (((tid % 8) ^ (r0 & 7)) << 4);
#pragma unroll 1
  for (int j = 0; j < ROWS / 16; j += 2) {
    uint4 a[2][kParts<T>];
    split_group<T>(v + cell + j * 2048, from + j == 0 ? weight[0] : weight[2], a[0]);
    split_group<T>(v + cell + j * 2048 + 2048, from + j == 0 ? weight[1] : weight[3], a[1]);
    if (j == 0 && !ready()) return false;
#pragma unroll
    for (int p = 0; p < kParts<T>; ++p) {
      *reinterpret_cast<uint4*>(parts + p * ROWS * 128 + cell + j * 2048) = a[0][p];
      *reinterpret_cast<uint4*>(parts + p * ROWS * 128 + cell + j * 2048 + 2048) = a[1][p];
    }
  }
  return true;
}

// D (+)= K^T V' over ROWS tokens, all parts at once, 64 columns each (FIRST: the first product does
// not add): M runs along the heads' size, the contraction over the tokens.  k, b: operand().
template <typename T, int DK, int ROWS, bool FIRST>
__device__ __forceinline__ void issue_update(uint32_t d, uint32_t k, uint32_t b) {
  constexpr uint32_t id = instr<T>(DK, NV * kParts<T>, true, true);
  mma_ss<!FIRST>(d, k, b, id);
#pragma unroll
  for (int i = 1; i < ROWS / 16; ++i) mma_ss<true>(d, k + i * 128, b + i * 128, id);
}
// 8 columns of U from the parts' sums.
template <typename T> __device__ __forceinline__ void load_update(uint32_t addr, float (&x)[8]) {
  float y[8], z[8];
  tmem_ld8(addr, x);
  tmem_ld8(addr + NV, y);
  if (!kIsHalf<T>) tmem_ld8(addr + 2 * NV, z);
  tmem_ld_wait(x);
  tmem_ld_wait(y);
#pragma unroll
  for (int c = 0; c < 8; c += 2) {
    if (kIsHalf<T>) {
      mul2(y[c], y[c + 1], 1.0f / kLowScale, 1.0f / kLowScale);
    } else {
      if (c == 0) tmem_ld_wait(z);
      add2(y[c], y[c + 1], z[c], z[c + 1]);
    }
    add2(x[c], x[c + 1], y[c], y[c + 1]);
  }
}

// Products: warp 0, loads: 1 (2 and 3 only give registers; the first warps go first where several
// could), P: 4 warps, V': 8, o: 4, state: 4.
constexpr int kThreads = 768;
// Registers a thread: 768 threads leave 80 each; the six groups of four warps share the 480 as
// 96 (P), 2 x 56 (V'), 96 (o), 136 (state, 64 of it its rows) and 40.
template <int N> __device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N> __device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
constexpr uint32_t kColumns = 512;
// TMEM columns: two buffers of Sc (both parts of P over it), Oe and after it Oi, U
constexpr uint32_t kSc = 0, kO = 256, kU = 320;
// The state launch takes 64 tokens at a time.  A stage is held from its load to the end of its
// product, some 2.5 us, so what counts is their number (4: 140 us for 1 x 65536 x 16 x 128).
constexpr int kStateRows = 64, kStatePanel = kStateRows * 128, kStateGroups = 4, kStateParts = 2;

template <typename T, int DK> struct Smem {
  static constexpr int panels = DK / 64;
  static constexpr int stages = DK == 64 ? 3 : 2;
  static constexpr int q = 0, k = stages * panels * kPanel, v = 2 * k;  // rings of stages
  // V' is formed and multiplied by blocks of v_rows tokens, two of them in turn; the smaller ones
  // are what heads of 128 have room for
  static constexpr int v_rows = DK == 64 ? 64 : 32, v_block = kParts<T> * v_rows * 128;
  static constexpr int parts = v + stages * kPanel, s = parts + 2 * v_block;
  static constexpr int s_part = DK * 128;              // two parts of the state's copy
  static constexpr int bytes = s + 2 * s_part + 1024;  // 1024: room to align the base
  static constexpr int st_stages = DK == 64 ? 8 : 6;
  static constexpr int st_stage = (panels + 1) * kStatePanel;
  static constexpr int st_parts = st_stages * st_stage;
  static constexpr int st_bytes = st_parts + kStateParts * kParts<T> * kStatePanel + 1024;
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

// 16 columns of a row (`cols` of them exist, a multiple of 8), in whole 32-byte sectors where
// these are aligned (vec 2), else in 16 bytes.
__device__ __forceinline__ void store8(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d,
                                       uint32_t e, uint32_t f, uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(a), "r"(b),
               "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void store_row(T* dst, const float (&x)[16], int cols, int vec) {
  uint32_t u[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) u[c] = pack<T>(x[2 * c], x[2 * c + 1]);
  if (vec == 2) {
    if (cols > 0) store8(dst, u[0], u[1], u[2], u[3], u[4], u[5], u[6], u[7]);
  } else {
    if (cols > 0) *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
    if (cols > 8) *reinterpret_cast<uint4*>(dst + 8) = make_uint4(u[4], u[5], u[6], u[7]);
  }
}
// The 32-bit form (results that are added over heads later): contiguous, columns in eights.
__device__ __forceinline__ void store_wide(float* dst, const float (&x)[16], int cols) {
#pragma unroll
  for (int g = 0; g < 2; ++g)
    if (g * 8 < cols)
      store8(dst + g * 8, __float_as_uint(x[g * 8]), __float_as_uint(x[g * 8 + 1]),
             __float_as_uint(x[g * 8 + 2]), __float_as_uint(x[g * 8 + 3]),
             __float_as_uint(x[g * 8 + 4]), __float_as_uint(x[g * 8 + 5]),
             __float_as_uint(x[g * 8 + 6]), __float_as_uint(x[g * 8 + 7]));
}

// ------------------------------------------------------------------------------ non-finite values
// P V takes an infinity or NaN among a chunk's values to the chunk's earlier tokens too (a masked
// score is a factor zero of the product).  Such a value also makes its column of the segment's end
// state NaN, which costs nothing to see; what it spoilt, its column's outputs in its chunk before
// its token, is then formed again by the recurrence.  The warp looks for column c's first such
// token and walks to it from the segment's first one, lanes taking rows of the column:
//   R_l = d R_{l-1} + k_l v_l,   o_l = q_l . (inter d^{l+off} S_0 + intra R_l).
template <typename T, int DK>
__device__ __forceinline__ void restore_column(const Call& call, const Where& w, int c, int lane) {
  constexpr int N = DK / 32;
  const Job& job = *w.job;
  auto token = [&](int l) { return int64_t(job.reverse ? w.n - 1 - l : l); };
  const T* v = static_cast<const T*>(job.v) + w.b * job.vs[0] + w.h / job.v_group * job.vs[2] +
               w.v0 + c;
  int first = w.begin;  // of the tokens not known to be finite
  for (; first < w.end; first += 32) {
    const int l = first + lane;
    const unsigned odd = __ballot_sync(
        0xffffffffu, l < w.end && !isfinite(to_acc(v[token(l < w.end ? l : first) * job.vs[1]])));
    if (odd != 0) {
      first += __ffs(odd) - 1;
      break;
    }
  }
  const int from = w.begin + (first - w.begin) / C * C;  // its chunk's first token
  if (first >= w.end || first == from) return;
  const T* q = static_cast<const T*>(job.q) + w.b * job.qs[0] + w.h / job.q_group * job.qs[2];
  const T* k = static_cast<const T*>(job.k) + w.b * job.ks[0] + w.h / job.k_group * job.ks[2];
  const int64_t size = int64_t(job.dk) * job.dv, head = w.bh * size;
  const float* seg = static_cast<const float*>(job.seg) + head * (call.nseg - 1);
  const bool inside = call.scan_inside != 0;
  const float whole = inside ? decay_pow(w.a, float(call.seg_len)) : 0.0f;
  const float keep = decay_pow(w.a, 1.0f);
  float s0[N], r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {  // the state before the segment
    const int row = lane + 32 * i;
    s0[i] = r[i] = 0.0f;
    if (row >= job.dk) continue;
    if (job.init != nullptr && (w.seg == 0 || inside))
      s0[i] = static_cast<const float*>(job.init)[head + row * job.init_row +
                                                  (w.v0 + c) * job.init_col];
    for (int j = inside ? 0 : w.seg - 1; j < w.seg; ++j)
      if (j >= 0) s0[i] = whole * s0[i] + seg[j * size + int64_t(row) * job.dv + w.v0 + c];
  }
  for (int l = w.begin; l < first; ++l) {
    const float x = to_acc(v[token(l) * job.vs[1]]);
    float sum = 0.0f;
    const float read = float(job.inter) * decay_pow(w.a, float(l - w.begin + job.off));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = lane + 32 * i;
      if (row >= job.dk) continue;
      r[i] = keep * r[i] + to_acc(k[token(l) * job.ks[1] + row]) * x;
      if (l >= from)
        sum += to_acc(q[token(l) * job.qs[1] + row]) * (read * s0[i] + float(job.intra) * r[i]);
    }
    if (l < from) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int64_t at = w.b * job.os[0] + w.h * job.os[2] + w.v0 + c + token(l) * job.os[1];
    if (lane == 0) {
      if (job.o_wide) static_cast<float*>(job.o)[at] = sum;
      else static_cast<T*>(job.o)[at] = from_acc<T>(sum);
    }
  }
}

// ------------------------------------------------------------------------------ main launch
template <typename T, int DK>
__global__ void __launch_bounds__(kThreads, 1)
linattn_tc_kernel(const __grid_constant__ Call call, const __grid_constant__ Maps maps,
                  int* error, unsigned extra_tx) {
  using Z = Smem<T, DK>;
  constexpr bool kHalf = kIsHalf<T>;
  constexpr int S = Z::stages;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = align_smem(raw);
  __shared__ uint64_t k_full[S], q_full[S], v_in[S], k_empty[S], q_empty[S], v_empty[S];
  __shared__ uint64_t sc_full[2], p_full[2], oe_full, oe_empty, o_full, o_empty, s_full, u_full,
      u_empty, v_full[2], v_free[2], most_full, drain;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  __shared__ float power[64];          // at 31 + t - s: intra d^|t-s|, 0 for a masked pair
  __shared__ float p_inv[2][C];        // fp16: inverse scales of P's rows
  __shared__ float s_inv[2];           // fp16: inverse scale of the state's copy
  __shared__ volatile float s_most[4];  // fp16: largest magnitude of each warp's rows

  __shared__ float dpow[C + 1];  // d^n
  __shared__ unsigned odd[2];    // columns of the end state with infinities or NaN

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  if (warp == 0) tmem_alloc(&tmem_slot);
  const Limit limit{&failed, extra_tx == 0 ? kWaitCycles : kTestCycles};
  const Where w = locate(call, blockIdx.x, blockIdx.y);
  const Job& job = *w.job;
  const uint32_t base = smem_addr(sm);
  const int chunks = w.chunks;
  // loads: j = 3 i + (0: K, 1: Q, 2: V) of chunk i
  auto load = [&](int j) {
    const int i = j / 3, which = j % 3, st = i % S;
    const CUtensorMap* map = maps.map[w.ji];
    const int l0 = w.begin + i * C, token = job.reverse ? w.n - C - l0 : l0;
    if (which == 2) {
      // (test hook: block 0 waits for bytes that never come)
      bar_expect(&v_in[st], kPanel + (j == 2 && first_block() ? extra_tx : 0));
      Source(map + 2, job.vs, w.h / job.v_group, w.b)
          .template load<C>(base + Z::v + st * kPanel, w.v0, 1, token, &v_in[st]);
    } else {
      const bool k = which == 0;
      uint64_t* bar = k ? &k_full[st] : &q_full[st];
      bar_expect(bar, Z::panels * kPanel);
      Source(k ? map + 1 : map, k ? job.ks : job.qs, w.h / (k ? job.k_group : job.q_group), w.b)
          .template load<C>(base + (k ? Z::k : Z::q) + st * Z::panels * kPanel, 0, Z::panels, token,
                            bar);
    }
  };
  const int first_loads = 3 * (chunks < S ? chunks : S);
  if (threadIdx.x == 32) {
    for (int i = 0; i < S; ++i) {
      bar_init(&k_full[i], 1);
      bar_init(&q_full[i], 1);
      bar_init(&v_in[i], 1);
      bar_init(&k_empty[i], 1);
      bar_init(&q_empty[i], 1);
      bar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&sc_full[i], 1);
      bar_init(&p_full[i], 128);
      bar_init(&v_full[i], 128);
      bar_init(&v_free[i], 1);
    }
    bar_init(&oe_full, 1);
    bar_init(&oe_empty, 128);
    bar_init(&o_full, 1);
    bar_init(&o_empty, 128);
    bar_init(&s_full, 128);
    bar_init(&u_full, 1);
    bar_init(&u_empty, 128);
    bar_init(&most_full, 4);
    bar_init(&drain, 1);
    failed = 0;
    odd[0] = odd[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
#pragma unroll 1
    for (int j = 0; j < first_loads; ++j) load(j);
  }
  if (threadIdx.x >= 64 && threadIdx.x < 128) {
    const int i = threadIdx.x - 64;
    const int n = job.reverse ? 31 - i : i - 31;
    power[i] = n < 0 ? 0.0f : float(job.intra) * decay_pow(w.a, float(n));
  }
  if (threadIdx.x >= 128 && threadIdx.x <= 128 + C)
    dpow[threadIdx.x - 128] = decay_pow(w.a, float(threadIdx.x - 128));
  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t lanes = uint32_t(warp % 4 * 32) << 16;

  if (warp >= 4 && warp < 8) {
    take_registers<96>();
    const int row_warp = warp - 4;
    // ---- P = Sc * M.  Row t = 32 row_warp + lane, 32 columns at a time: their two 16-bit parts (16
    // columns each) go over the scores.  Off the diagonal block (forward; the mirror image back
    // in time) d^{t-s} = d^{32(w-j-1)+lane+1} d^{31-c}: both powers are at least 0, nothing
    // overflows.
    const bool rev = job.reverse != 0;
    float tab[32], lead[4];
#pragma unroll
    for (int c = 0; c < 32; ++c) tab[c] = dpow[rev ? c + 1 : 31 - c];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = rev ? 32 * (j - row_warp - 1) + 31 - lane : 32 * (row_warp - j - 1) + lane + 1;
      lead[j] = n < 0 || n > C ? 0.0f : float(job.intra) * dpow[n];
    }
    const float* diagonal = power + 31 + lane;
    bool ok = true;
    for (int i = 0; i < chunks && ok; ++i) {
      ok = __all_sync(0xffffffffu, bar_wait(&sc_full[i & 1], (i >> 1) & 1, limit));
      if (!ok) break;
      tc_after();
      const uint32_t sc = tmem + lanes + kSc + (i & 1) * 128;
      float scale = 1.0f;
      if (kHalf) {
        float most = 0.0f;
#pragma unroll 1
        for (int j = rev ? row_warp : 0; j <= (rev ? 3 : row_warp); ++j) {
          const float f = j == 0 ? lead[0] : (j == 1 ? lead[1] : (j == 2 ? lead[2] : lead[3]));
          float x[32], block = 0.0f;
          tmem_ld32(sc + j * 32, x);
          tmem_ld_wait(x);
          if (j == row_warp) {
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float p = diagonal[-c];
              if (p != 0.0f) most = fmaxf(most, fabsf(x[c] * p));
            }
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) block = fmaxf(block, fabsf(x[c] * tab[c]));
            most = fmaxf(most, block * fabsf(f));
          }
        }
        float inv;
        scale = scale_of(most, &inv);
        p_inv[i & 1][row_warp * 32 + lane] = inv;
      }
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        uint32_t u[16];
        if (rev ? j < row_warp : j > row_warp) {  // all masked
#pragma unroll
          for (int c = 0; c < 16; ++c) u[c] = 0;
          tmem_st16(sc + j * 32, u);
        } else {
          float x[32];
          tmem_ld32(sc + j * 32, x);
          tmem_ld_wait(x);
          if (j == row_warp) {
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const float p = diagonal[-c];
              x[c] = p != 0.0f ? (kHalf ? x[c] * p * scale : x[c] * p) : 0.0f;
            }
          } else {
            const float f =
                (j == 0 ? lead[0] : (j == 1 ? lead[1] : (j == 2 ? lead[2] : lead[3]))) * scale;
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              mul2(x[c], x[c + 1], tab[c], tab[c + 1]);
              mul2(x[c], x[c + 1], f, f);
            }
          }
#pragma unroll
          for (int c = 0; c < 16; ++c) u[c] = first_part<T>(x[2 * c], x[2 * c + 1]);
          tmem_st16(sc + j * 32, u);
#pragma unroll
          for (int c = 0; c < 16; ++c) u[c] = pack<T>(x[2 * c], x[2 * c + 1]);
        }
        tmem_st16(sc + j * 32 + 16, u);
      }
      tmem_st_wait();
      tc_before();
      bar_arrive(&p_full[i & 1]);
    }
  } else if (warp >= 8 && warp < 16) {
    give_registers<56>();
    // ---- V', two groups of four warps take blocks of v_rows tokens by turns, each with its own
    // buffer: a block is formed while the other group's is multiplied.  idx = 0 .. 3 are a
    // thread's rows of a chunk, kIn of them in a block.
    constexpr int R = Z::v_rows, kBlocks = C / R / 2, kIn = 4 / kBlocks;
    const int tid = threadIdx.x % 128, group = (warp - 8) / 4;
    auto row = [&](int idx) { return (group + idx / kIn * 2) * R + tid / 8 + idx % kIn * 16; };
    float weight[4];
    int weight_m = 0;
    bool ok = true;
    for (int i = 0; i < chunks && ok; ++i) {
      const int left = w.end - (w.begin + i * C), m = left < C ? left : C;
      if (m != weight_m) {
        weight_m = m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = row(j), age = m - job.off - (job.reverse ? C - 1 - r : r);
          weight[j] = age < 0 ? 0.0f : dpow[age];
        }
      }
      if (!bar_wait(&v_in[i % S], (i / S) & 1, limit)) break;
      unsigned char* v = sm + Z::v + (i % S) * kPanel;
      if (m < C && !job.reverse && w.n < call.length) {
        // padding after the sequence's end: the products take zeros for its keys and values
        // (scores with them are masked, whichever of the two they read).  A thread clears the
        // values that it reads below.
        if (!bar_wait(&k_full[i % S], (i / S) & 1, limit)) break;
        unsigned char* k = sm + Z::k + (i % S) * Z::panels * kPanel;
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          const int r = row(j);
          if (r < m) continue;
          const int at = r * 128 + (((tid % 8) ^ (r & 7)) << 4);
#pragma unroll
          for (int p = 0; p < Z::panels; ++p)
            *reinterpret_cast<uint4*>(k + p * kPanel + at) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(v + at) = make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll 1
      for (int b = 0; b < kBlocks && ok; ++b) {
        const int turn = i * kBlocks + b;
        ok = split_values<T, R>(v + (group + 2 * b) * R * 128, sm + Z::parts + group * Z::v_block,
                                weight, b * kIn, tid, [&] {
          return turn == 0 || bar_wait(&v_free[group], (turn - 1) & 1, limit);
        });
        if (!ok) break;
        fence_async();
        bar_arrive(&v_full[group]);
      }
    }
  } else if (warp >= 16 && warp < 20) {
    take_registers<96>();
    // ---- o = inter d^{l+off} Oe + Oi, a row of 64 columns a thread; Oe is taken as soon as it is
    // there, so that Oi can take its place
    const int t = warp % 4 * 32 + lane, l = job.reverse ? C - 1 - t : t;
    const float read = float(job.inter) * dpow[l + job.off];
    const int64_t head = int64_t(w.b) * job.os[0] + int64_t(w.h) * job.os[2] + w.v0;
    for (int i = 0; i < chunks; ++i) {
      if (!__all_sync(0xffffffffu, bar_wait(&oe_full, i & 1, limit))) break;
      tc_after();
      const int l0 = w.begin + i * C;
      const bool in = l0 + l < w.end;
      const int token = (job.reverse ? w.n - C - l0 : l0) + t;
      const int64_t at = head + int64_t(token) * job.os[1];
      const float fe = kHalf ? read * s_inv[i & 1] : read;
      float y[NV / 16][16];
#pragma unroll
      for (int g = 0; g < NV / 16; ++g) tmem_ld16(tmem + lanes + kO + g * 16, y[g]);
#pragma unroll
      for (int g = 0; g < NV / 16; ++g) tmem_ld_wait(y[g]);
      tc_before();
      bar_arrive(&oe_empty);
      if (!__all_sync(0xffffffffu, bar_wait(&o_full, i & 1, limit))) break;
      tc_after();
      const float fi = kHalf ? p_inv[i & 1][t] : 1.0f;
#pragma unroll
      for (int g = 0; g < NV / 16; ++g) {
        float x[16];
        tmem_ld16(tmem + lanes + kO + g * 16, x);
        tmem_ld_wait(x);
        if (g == NV / 16 - 1) {
          tc_before();
          bar_arrive(&o_empty);
        }
#pragma unroll
        for (int c = 0; c < 16; c += 2) {
          if (kHalf) mul2(x[c], x[c + 1], fi, fi);
          fma2(y[g][c], y[g][c + 1], fe, x[c], x[c + 1]);
        }
        if (in) {
          if (job.o_wide)
            store_wide(static_cast<float*>(job.o) + at + g * 16, y[g], w.vcols - g * 16);
          else
            store_row(static_cast<T*>(job.o) + at + g * 16, y[g], w.vcols - g * 16, job.o_vec);
        }
      }
    }
    asm volatile("bar.arrive 1, 256;" ::: "memory");
  } else if (warp >= 20) {
    take_registers<136>();
    // ---- the state, a row of 64 columns a thread (DK = 64: 16 rows a warp, the lanes that a
    // product with M = 64 fills)
    const int r = DK == 128 ? (warp - 20) * 32 + lane : (warp - 20) * 16 + (lane & 15);
    const bool mine = DK == 128 || lane < 16;
    const int64_t size = int64_t(job.dk) * job.dv;
    const float write = float(job.write);
    float s[2][32];
    {
      // the first state, or what the segments before leave: their own end states are added up
      // here where there are few, by a launch before this one where there are many
      const bool inside = call.scan_inside != 0;
      const int cols = mine && r < job.dk && w.seg <= w.last ? w.vcols : 0;
      const int64_t first = int64_t(w.bh) * size;
      if (job.init != nullptr && (w.seg == 0 || inside)) {
        const float* src = static_cast<const float*>(job.init) + first + r * job.init_row +
                           w.v0 * job.init_col;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          s[c / 32][c % 32] = c < cols ? *src : 0.0f;
          src += job.init_col;
        }
      } else {
#pragma unroll
        for (int c = 0; c < NV; ++c) s[c / 32][c % 32] = 0.0f;
      }
      // the main launch may begin before the state launch has ended (launch_as): only this waits
      if (w.seg > 0) asm volatile("griddepcontrol.wait;" ::: "memory");
      const float* src = static_cast<const float*>(job.seg) + first * (call.nseg - 1) +
                         int64_t(r) * job.dv + w.v0;
      const float keep = inside ? decay_pow(w.a, float(call.seg_len)) : 0.0f;
#pragma unroll 1
      for (int j = inside ? 0 : w.seg - 1; j < w.seg; ++j) {
        if (j < 0) continue;
#pragma unroll
        for (int c = 0; c < NV; c += 4) {
          if (c < cols) {
            const float4 u = *reinterpret_cast<const float4*>(src + j * size + c);
            float* y = &s[c / 32][c % 32];
            y[0] = keep * y[0] + u.x;
            y[1] = keep * y[1] + u.y;
            y[2] = keep * y[2] + u.z;
            y[3] = keep * y[3] + u.w;
          }
        }
      }
    }
    bool ok = true;
    for (int i = 0; i <= chunks && ok; ++i) {
      if (i > 0) {
        ok = __all_sync(0xffffffffu, bar_wait(&u_full, (i - 1) & 1, limit));
        if (!ok) break;
        tc_after();
        const int left = w.end - (w.begin + (i - 1) * C);
        const float keep = dpow[left < C ? left : C];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          float x[8];
          load_update<T>(tmem + lanes + kU + g * 8, x);
          float* y = &s[g / 4][g % 4 * 8];
#pragma unroll
          for (int c = 0; c < 8; c += 2) {
            mul2(x[c], x[c + 1], write, write);
            fma2(y[c], y[c + 1], keep, x[c], x[c + 1]);
          }
        }
        tc_before();
        bar_arrive(&u_empty);
        if (i == chunks) break;
        ok = __all_sync(0xffffffffu, bar_wait(&oe_full, (i - 1) & 1, limit));
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
        // (rewritten only after oe_full of this chunk, which follows every warp's s_full)
        if (lane == 0) {
          s_most[warp - 20] = most;
          bar_arrive(&most_full);
        }
        ok = __all_sync(0xffffffffu, bar_wait(&most_full, i & 1, limit));
        if (!ok) break;
        most = fmaxf(fmaxf(s_most[0], s_most[1]), fmaxf(s_most[2], s_most[3]));
        float inv;
        scale = scale_of(most, &inv);
        if (warp == 20 && lane == 0) s_inv[i & 1] = inv;
      }
      if (mine) {
        unsigned char* row = sm + Z::s + r * 128;
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const float* y = &s[g / 4][g % 4 * 8];
          uint32_t u[4], low[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float a = y[2 * e], b = y[2 * e + 1];
            if (kHalf) mul2(a, b, scale, scale);
            u[e] = first_part<T>(a, b);
            low[e] = pack<T>(a, b);
          }
          const int at = (g ^ (r & 7)) << 4;
          *reinterpret_cast<uint4*>(row + at) = make_uint4(u[0], u[1], u[2], u[3]);
          *reinterpret_cast<uint4*>(row + Z::s_part + at) =
              make_uint4(low[0], low[1], low[2], low[3]);
        }
      }
      fence_async();
      bar_arrive(&s_full);
    }
    float zeros[2] = {0.0f, 0.0f};  // 0 s: NaN for what is not finite
#pragma unroll
    for (int c = 0; c < NV; c += 2) {
      float x = s[c / 32][c % 32], y = s[c / 32][c % 32 + 1];
      fma2(x, y, 0.0f, zeros[0], zeros[1]);
      zeros[0] = x;
      zeros[1] = y;
    }
    if (ok && mine && r < job.dk && zeros[0] + zeros[1] != 0.0f) {
#pragma unroll
      for (int c = 0; c < NV; ++c)
        if (!isfinite(s[c / 32][c % 32])) atomicOr(&odd[c / 32], 1u << (c % 32));
    }
    if (ok && w.seg == w.last && job.fin != nullptr && mine && r < job.dk) {
      float* dst = static_cast<float*>(job.fin) + w.bh * size + int64_t(r) * job.dv + w.v0;
#pragma unroll
      for (int c = 0; c < NV; ++c)
        if (c < w.vcols) dst[c] = s[c / 32][c % 32];
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");  // o is stored, odd is whole
    if ((odd[0] | odd[1]) != 0) {
#pragma unroll 1
      for (int c = warp - 20; c < w.vcols; c += 4)
        if (odd[c / 32] >> (c % 32) & 1) restore_column<T, DK>(call, w, c, lane);
    }
  } else if (warp == 1) {
    give_registers<40>();
    // ---- loads: an operand's buffer is loaded again as soon as its own last product has ended
    const bool one = elect_one();
    int issued = first_loads;
    bool ok = true;
    for (; issued < 3 * chunks; ++issued) {
      const int i = issued / 3, which = issued % 3, st = i % S;
      uint64_t* empty = which == 0 ? k_empty : (which == 1 ? q_empty : v_empty);
      ok = __all_sync(0xffffffffu, bar_wait(&empty[st], (i / S - 1) & 1, limit));
      if (!ok) break;
      if (one) load(issued);
      __syncwarp();
    }
    if (!ok || failed) {  // copies in flight land before the block ends
      for (int j = issued > 3 * S ? issued - 3 * S : 0; j < issued; ++j) {
        const int i = j / 3, which = j % 3;
        uint64_t* bar = which == 0 ? k_full : (which == 1 ? q_full : v_in);
        bar_drain(&bar[i % S], (i / S) & 1, limit);
      }
    }
  } else if (warp > 1) {
    give_registers<40>();
  } else {
    give_registers<40>();
    // ---- all products, issued by one lane
    constexpr uint32_t id_sc = instr<T>(C, C, false, false);
    constexpr uint32_t id_o = instr<T>(C, NV, false, true);
    // operands of stage 0, and of what has one buffer
    const uint32_t oq = operand(base + Z::q, kPanel), ok0 = operand(base + Z::k, kPanel);
    const uint32_t ov = operand(base + Z::v, kPanel);
    const uint32_t os = operand(base + Z::s, kPanel);
    const uint32_t op = operand(base + Z::parts, Z::v_rows * 128);
    const bool one = elect_one();
    bool ok = true;
    // each turn: U, Oe of chunk i, the scores of chunk i + 1, Oi of chunk i (turn -1: the scores
    // alone), so that P of the next chunk is formed beside the rest
    for (int i = -1; i < chunks; ++i) {
      if (i >= 0) {
        const uint32_t q = oq + (i % S) * (Z::panels * kPanel / 16);
        const uint32_t k = ok0 + (i % S) * (Z::panels * kPanel / 16);
        constexpr int kBlocks = C / Z::v_rows;  // of V', in turn from the two groups that form them
        ok = __all_sync(0xffffffffu, i == 0 || bar_wait(&u_empty, (i - 1) & 1, limit));
        if (!ok) break;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
          const int turn = i * (kBlocks / 2) + b / 2;
          ok = __all_sync(0xffffffffu, bar_wait(&v_full[b % 2], turn & 1, limit));
          if (!ok) break;
          if (one) {
            tc_after();
            const uint32_t kb = k + b * (Z::v_rows * 128 / 16), pb = op + b % 2 * (Z::v_block / 16);
            if (b == 0) issue_update<T, DK, Z::v_rows, true>(tmem + kU, kb, pb);
            else issue_update<T, DK, Z::v_rows, false>(tmem + kU, kb, pb);
            tc_commit(&v_free[b % 2]);
            if (b + 1 == kBlocks) {
              tc_commit(&u_full);
              tc_commit(&k_empty[i % S]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        // o of the chunk before is out: its columns take this chunk's, and its scores' buffer the
        // next scores
        ok = bar_wait(&s_full, i & 1, limit) &&
             (i == 0 || bar_wait(&o_empty, (i - 1) & 1, limit));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (one) {
          tc_after();
          mma_ss<false>(tmem + kO, q, os, id_o);
#pragma unroll
          for (int j = 1; j < DK / 8; ++j) {  // both parts of the state's copy
            const int d = j % (DK / 16);
            mma_ss<true>(tmem + kO, q + d / 4 * (kPanel / 16) + d % 4 * 2,
                         os + j / (DK / 16) * (Z::s_part / 16) + d * 128, id_o);
          }
          tc_commit(&oe_full);
          tc_commit(&q_empty[i % S]);
        }
        __syncwarp();
      }
      const int n = i + 1;
      if (n < chunks) {
        ok = bar_wait(&k_full[n % S], (n / S) & 1, limit) &&
             bar_wait(&q_full[n % S], (n / S) & 1, limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (one) {
          tc_after();
          const uint32_t q = oq + (n % S) * (Z::panels * kPanel / 16);
          const uint32_t k = ok0 + (n % S) * (Z::panels * kPanel / 16);
          const uint32_t d = tmem + kSc + (n & 1) * 128;
          mma_ss<false>(d, q, k, id_sc);
#pragma unroll
          for (int j = 1; j < DK / 16; ++j)
            mma_ss<true>(d, q + j / 4 * (kPanel / 16) + j % 4 * 2,
                         k + j / 4 * (kPanel / 16) + j % 4 * 2, id_sc);
          tc_commit(&sc_full[n & 1]);
        }
        __syncwarp();
      }
      if (i < 0) continue;
      // (no barrier may be two phases ahead of who waits for it: each Oe and Oi is taken before the
      // next one is issued)
      ok = bar_wait(&p_full[i & 1], (i >> 1) & 1, limit) && bar_wait(&oe_empty, i & 1, limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (one) {
        tc_after();
        const uint32_t v = ov + (i % S) * (kPanel / 16);
        const uint32_t p = tmem + kSc + (i & 1) * 128;
        mma_ts<false>(tmem + kO, p, v, id_o);
#pragma unroll
        for (int j = 1; j < C / 8; ++j) {  // the first part of P, then the second
          const int t = j % (C / 16);
          mma_ts<true>(tmem + kO, p + t / 2 * 32 + t % 2 * 8 + j / (C / 16) * 16, v + t * 128, id_o);
        }
        tc_commit(&o_full);
        tc_commit(&v_empty[i % S]);
      }
      __syncwarp();
    }
    if (!ok) {  // let the products in flight end before TMEM goes
      if (one) tc_commit(&drain);
      __syncwarp();
      bar_drain(&drain, 0, limit);
    }
  }
  // rows after the sequence's end
  {
    const int from = w.begin > w.n ? w.begin : w.n;
    const int64_t cells = int64_t(w.row_end - from) * w.vcols;
    for (int64_t i = threadIdx.x; i < cells; i += kThreads) {
      const unsigned row = unsigned(i) / unsigned(w.vcols), c = unsigned(i) - row * w.vcols;
      const int64_t at = int64_t(w.b) * job.os[0] + int64_t(w.h) * job.os[2] + w.v0 +
                         (from + int64_t(row)) * job.os[1] + c;
      if (job.o_wide) static_cast<float*>(job.o)[at] = 0.0f;
      else static_cast<T*>(job.o)[at] = from_acc<T>(0.0f);
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 0) {
    tc_after();
    tmem_free(tmem);
    if (lane == 0 && failed) *error = kErrCopyTimeout;
  }
}

// ------------------------------------------------------------------------------ state launch
// A segment's own end state: U += K^T V' with V' = diag(d^{end-off-l}) V weighted towards the
// segment's end, so that the sums stay in TMEM over all tokens.
constexpr int kStateThreads = 576;  // V' (and the result): 16 warps, products: 1, loads: 1

template <typename T, int DK>
__global__ void __launch_bounds__(kStateThreads, 1)
linattn_tc_state_kernel(const __grid_constant__ Call call, const __grid_constant__ Maps maps,
                        int* error, unsigned extra_tx) {
  using Z = Smem<T, DK>;
  constexpr int R = kStateRows;
  constexpr int S = Z::st_stages;
  extern __shared__ unsigned char raw[];
  unsigned char* sm = align_smem(raw);
  constexpr int NB = kStateParts, kGroups = kStateGroups;
  __shared__ uint64_t full[S], v_full[NB], used[S], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int failed;
  const Limit limit{&failed, extra_tx == 0 ? kWaitCycles : kTestCycles};
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  const Where w = locate(call, blockIdx.x, blockIdx.y);
  const Job& job = *w.job;
  if (w.seg >= w.last) return;  // the whole block
  if (warp == 16) tmem_alloc(&tmem_slot);
  const uint32_t base = smem_addr(sm);
  const int chunks = w.chunks * (C / R);  // whole ones: every segment before the last is full
  auto load = [&](int i) {
    const int st = i % S, l0 = w.begin + i * R;
    const int token = job.reverse ? w.n - R - l0 : l0;
    const uint32_t at = base + st * Z::st_stage;
    const CUtensorMap* map = maps.map[w.ji];
    bar_expect(&full[st], Z::st_stage + (i == 0 && first_block() ? extra_tx : 0));
    Source(map + 1, job.ks, w.h / job.k_group, w.b)
        .template load<R>(at, 0, Z::panels, token, &full[st]);
    Source(map + 2, job.vs, w.h / job.v_group, w.b)
        .template load<R>(at + Z::panels * kStatePanel, w.v0, 1, token, &full[st]);
  };
  const int first_loads = chunks < S ? chunks : S;
  if (threadIdx.x == 17 * 32) {
    for (int i = 0; i < NB; ++i) bar_init(&v_full[i], 128);
    for (int i = 0; i < S; ++i) {
      bar_init(&full[i], 1);
      bar_init(&used[i], 1);
    }
    bar_init(&done, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async();
#pragma unroll 1
    for (int i = 0; i < first_loads; ++i) load(i);
  }
  __syncwarp();
  tc_before();
  __syncthreads();
  tc_after();
  // every block is on its way: blocks of the main launch may take the multiprocessors left over
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t tmem = tmem_slot;

  if (warp < 4 * kGroups) {
    // groups of four warps take the blocks of 64 tokens by turns
    const int tid = threadIdx.x % 128, mine = warp / 4;
    for (int i = mine; i < chunks; i += kGroups) {
      float weight[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = tid / 8 + 16 * j;
        const int age = w.end - job.off - (w.begin + i * R + (job.reverse ? R - 1 - r : r));
        weight[j] = age < 0 ? 0.0f : decay_pow(w.a, float(age));
      }
      if (!bar_wait(&full[i % S], (i / S) & 1, limit)) break;
      const bool ok = split_values<T, R>(
          sm + (i % S) * Z::st_stage + Z::panels * kStatePanel,
          sm + Z::st_parts + i % NB * kParts<T> * kStatePanel, weight, 0, tid,
          // the products of block i - NB have ended
          [&] { return i < NB || bar_wait(&used[(i - NB) % S], ((i - NB) / S) & 1, limit); });
      if (!ok) break;
      fence_async();
      bar_arrive(&v_full[i % NB]);
    }
    if (warp < 4 && __all_sync(0xffffffffu, bar_wait(&done, 0, limit)) && !failed) {
      tc_after();
      const int r = DK == 128 ? warp * 32 + lane : warp * 16 + (lane & 15);
      const bool in = (DK == 128 || lane < 16) && r < job.dk;
      float* dst = static_cast<float*>(job.seg) +
                   (int64_t(w.bh) * (call.nseg - 1) + w.seg) * (int64_t(job.dk) * job.dv) +
                   int64_t(r) * job.dv + w.v0;
      const float write = float(job.write);
      for (int g = 0; g < NV; g += 8) {
        float x[8];
        load_update<T>(tmem + (uint32_t(warp * 32) << 16) + g, x);
        if (in) {
#pragma unroll
          for (int c = 0; c < 8; ++c) x[c] *= write;
          if (g < w.vcols)
            store8(dst + g, __float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                   __float_as_uint(x[3]), __float_as_uint(x[4]), __float_as_uint(x[5]),
                   __float_as_uint(x[6]), __float_as_uint(x[7]));
        }
      }
    }
  } else if (warp == 17) {
    const bool one = elect_one();
    int issued = first_loads;
    bool ok = true;
    for (; issued < chunks; ++issued) {
      ok = __all_sync(0xffffffffu, bar_wait(&used[issued % S], (issued / S - 1) & 1, limit));
      if (!ok) break;
      if (one) load(issued);
      __syncwarp();
    }
    if (!ok || failed) {  // copies in flight land before the block ends
      for (int i = issued > S ? issued - S : 0; i < issued; ++i) bar_drain(&full[i % S], (i / S) & 1, limit);
    }
  } else {
    const uint32_t ok0 = operand(base, kStatePanel), op0 = operand(base + Z::st_parts, kStatePanel);
    const bool one = elect_one();
    bool ok = true;
    for (int i = 0; i < chunks && ok; ++i) {
      ok = __all_sync(0xffffffffu, bar_wait(&v_full[i % NB], (i / NB) & 1, limit));
      if (!ok) break;
      const uint32_t k = ok0 + (i % S) * (Z::st_stage / 16);
      const uint32_t parts = op0 + (i % NB) * (kParts<T> * kStatePanel / 16);
      if (one) {
        tc_after();
        if (i == 0) issue_update<T, DK, R, true>(tmem, k, parts);
        else issue_update<T, DK, R, false>(tmem, k, parts);
        tc_commit(&used[i % S]);
      }
      __syncwarp();
    }
    // also after a failed wait: the products in flight end before TMEM goes
    if (one) tc_commit(&done);
    __syncwarp();
    bar_drain(&done, 0, limit);
  }
  tc_before();
  __syncthreads();
  if (warp == 16) {
    tc_after();
    tmem_free(tmem);
    if (lane == 0 && failed) *error = kErrCopyTimeout;
  }
}

// ------------------------------------------------------------------------------ launches
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                            const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                            CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                            CUtensorMapFloatOOBfill);
Encode encoder() {
  static const Encode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<Encode>(p);
  }();
  return fn;
}

int encode(Encode fn, int dtype, CUtensorMap* map, const void* p, const int64_t* stride, int dim,
           int64_t length, int64_t heads, int64_t batch) {
  // an axis of one element, or broadcast with stride 0, is one coordinate
  const int64_t some = (dim + 7) / 8 * 16;
  const cuuint64_t dims[4] = {cuuint64_t(dim), cuuint64_t(stride[1] == 0 ? 1 : length),
                              cuuint64_t(stride[2] == 0 ? 1 : heads),
                              cuuint64_t(stride[0] == 0 ? 1 : batch)};
  const cuuint64_t strides[3] = {cuuint64_t(stride[1] == 0 ? some : stride[1] * 2),
                                 cuuint64_t(stride[2] == 0 ? some : stride[2] * 2),
                                 cuuint64_t(stride[0] == 0 ? some : stride[0] * 2)};
  const cuuint32_t box[4] = {64, kBoxRows, 1, 1}, one[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type =
      dtype == FDWT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int tries = 0; tries < 2; ++tries) {
    if (fn(map, type, 4, const_cast<void*>(p), dims, strides, box, one,
           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS)
      return FDWT_OK;
    // a thread's first CUDA call (autograd's) finds no current context: bind the device's
    if (tries == 0) FDWT_CUDA(cudaFree(nullptr));
  }
  return FDWT_ERR_UNSUPPORTED;
}

template <typename T, int DK>
int launch_as(const Call& call, const Maps& maps, bool states, cudaStream_t stream) {
  auto kernel = states ? linattn_tc_state_kernel<T, DK> : linattn_tc_kernel<T, DK>;
  const int64_t heads = call.batch * call.heads;
  const dim3 grid(static_cast<unsigned>(heads * call.tiles),
                  static_cast<unsigned>(states ? call.nseg - 1 : call.nseg));
  int* error = device_error_flag();
  if (error == nullptr) return FDWT_ERR_CUDA;
  int st = allow_max_dynamic_smem(reinterpret_cast<const void*>(kernel));
  if (st == FDWT_OK) st = pre_launch(stream);
  if (st != FDWT_OK) return st;
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(states ? kStateThreads : kThreads);
  config.dynamicSmemBytes = states ? Smem<T, DK>::st_bytes : Smem<T, DK>::bytes;
  config.stream = stream;
  // The main launch right after the state launch starts beside its end (1 x 1024 x 8 heads of 64:
  // 19.0 us one after the other, 16.8 us so).  Its state warps wait for the state launch; nothing
  // else in it touches what that one reads or writes.
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = !states && call.nseg > 1 && call.scan_inside ? 1 : 0;
  FDWT_CUDA(cudaLaunchKernelEx(&config, kernel, call, maps, error, copy_wait_test().extra_tx));
  return launch_status();
}

}  // namespace

bool tc_supports(int dtype, const Call& call) {
  if (dtype != FDWT_F16 && dtype != FDWT_BF16) return false;
  if (call.length > INT32_MAX - 2 * C || call.batch > INT32_MAX || encoder() == nullptr) return false;
  for (int j = 0; j < call.jobs; ++j) {
    const Job& job = call.job[j];
    if (job.dk > 128 || !job.q_vec || !job.k_vec || !job.v_vec || !job.o_vec) return false;
    // tensor maps: no broadcast tokens, no negative strides, strides below 2^40 bytes
    for (const int64_t* s : {job.qs, job.ks, job.vs}) {
      if (call.length > 1 && s[1] == 0) return false;
      for (int i = 0; i < 3; ++i)
        if (s[i] < 0 || s[i] >= int64_t(1) << 39) return false;
    }
  }
  return true;
}

int tc_launch(int dtype, const Call& call, bool states, cudaStream_t stream) {
  const Encode fn = encoder();
  Maps maps;
  int dk = 0;
  for (int j = 0; j < call.jobs; ++j) {
    const Job& job = call.job[j];
    dk = job.dk > dk ? job.dk : dk;
    const void* p[3] = {job.q, job.k, job.v};
    const int64_t* stride[3] = {job.qs, job.ks, job.vs};
    const int group[3] = {job.q_group, job.k_group, job.v_group};
    for (int i = states ? 1 : 0; i < 3; ++i) {
      const int st = encode(fn, dtype, &maps.map[j][i], p[i], stride[i], i == 2 ? job.dv : job.dk,
                            call.length, call.heads / group[i], call.batch);
      if (st != FDWT_OK) return st;
    }
  }
  if (dtype == FDWT_F16)
    return dk <= 64 ? launch_as<__half, 64>(call, maps, states, stream)
                    : launch_as<__half, 128>(call, maps, states, stream);
  return dk <= 64 ? launch_as<__nv_bfloat16, 64>(call, maps, states, stream)
                  : launch_as<__nv_bfloat16, 128>(call, maps, states, stream);
}

}  // namespace linattn
}  // namespace fdwt
