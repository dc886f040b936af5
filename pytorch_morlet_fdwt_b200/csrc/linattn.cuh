// Linear attention with a decay for each head: the call that its kernels share.
//
// With a = log_decay[h] and d = e^a, one job computes over the tokens l = 0 .. n-1 of a sequence
//
//   o_l = d^{l+off} inter q_l^T S_0 + intra sum_{s<=l} d^{l-s} (q_l . k_s) v_s,
//   S_n = d^n S_0 + write sum_l d^{n-off-l} k_l v_l^T                       (inter, q of S_s alike)
//
// in chunks of C tokens: from the state S before a chunk of m <= C tokens,
//
//   o = inter diag(d^{l+off}) Q S + intra (Q K^T * M) V,   M_ls = d^{l-s} for s <= l, else 0
//   S <- d^m S + write (diag(d^{m-off-l}) K)^T V.
//
// The forward pass is one job (off = 1, inter = intra = scale, write = 1).  The gradients are the
// same job with other operands: with g = dL/do and R the gradient of the state,
//
//   dq: q := g, k := v, v := k, S_0 := S_0^T                      forward in time
//   dv: q := k, k := q, v := g   (intra = write = scale, inter = 1, off = 0)   back in time
//   dk: q := v, k := g, v := q   (the same, from R^T)                          back in time
//
// where back in time l = 0 is the last token, and the dv job's last state is dL/dS_0.
//
// Few sequences and heads leave most SMs without work, so a long sequence is cut into segments:
// one launch forms every segment's own end state (K and V only), a second one adds these up to
// the state before each segment, and the main launch runs all segments at once.
#pragma once

#include "common.cuh"

namespace fdwt {
namespace linattn {

struct Job {
  const void *q, *k, *v;
  void* o;
  const void* init;  // state before the first token, null: zeros
  void* fin;         // state after the last one, contiguous (dk, dv), null: not wanted
  void* seg;         // workspace: states between segments, (batch * heads, nseg - 1, dk, dv)
  int64_t qs[3], ks[3], vs[3], os[3];  // strides (batch, token, head) in elements
  int64_t init_row, init_col;          // strides of init inside a head's dk * dv values
  int q_group, k_group, v_group;       // operand head = h / group
  int dk, dv, tiles;                   // tiles: column tiles of the value axis
  int reverse, off;
  int q_vec, k_vec, v_vec, o_vec;      // 16-byte accesses are aligned (o_vec 2: 32-byte too)
  int o_wide;                          // o is fp32 though the operands are 16 bits
  double inter, intra, write;
};

constexpr int kMaxJobs = 3;

struct Call {
  Job job[kMaxJobs];
  int jobs, tiles;  // tiles: of all jobs
  const void* log_decay;
  const int32_t* lengths;
  int64_t batch, length, seg_len;
  int heads, nseg;
  int scan_inside;  // the main launch adds up the segments' end states itself
};

// Times of the launches, in any unit: a block of c chunks takes `fixed + c chunk` in the main launch
// and `fixed + c state` in the state launch, each launch `launch` once.
struct Cost {
  double chunk, state, fixed, launch;
};
// Up to this many segments the main launch adds up their end states, beyond it a launch of its own.
constexpr int kScanInside = 8;

// Segments for `units` independent blocks of `chunks` chunks, `slots` of them resident.
inline int plan_segments(int64_t units, int64_t chunks, int64_t slots, const Cost& k) {
  int best = 1;
  double best_time = double(cdiv(units, slots)) * (k.fixed + double(chunks) * k.chunk);
  const int64_t most = imin(chunks, 64);
  for (int64_t s = 2; s <= most; ++s) {
    const int64_t c = cdiv(chunks, s);
    const int64_t real = cdiv(chunks, c);
    const double time = double(cdiv(units * real, slots)) * (k.fixed + double(c) * k.chunk) +
                        double(cdiv(units * (real - 1), slots)) * (k.fixed + double(c) * k.state) +
                        k.launch * (real > kScanInside ? 2 : 1);
    if (time < best_time) {
      best_time = time;
      best = static_cast<int>(real);
    }
  }
  return best;
}

// The tensor-core form (linattn_tc.cu), 16-bit types.
constexpr int kTcChunk = 128, kTcTile = 64;
bool tc_supports(int dtype, const Call& call);
// states: the state launch, else the main one.
int tc_launch(int dtype, const Call& call, bool states, cudaStream_t stream);

}  // namespace linattn
}  // namespace fdwt
