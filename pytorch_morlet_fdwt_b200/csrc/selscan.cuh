// Selective state space scan.  A channel d has `states` numbers h[n] that a token moves on by
//
//   v = dt + dt_bias,  delta = v or log(1 + e^v)
//   h_t[n] = e^(delta_t a[n]) h_{t-1}[n] + delta_t x_t b_t[n]
//   p_t = sum_n c_t[n] h_t[n] + skip x_t,   y_t = p_t, or p_t gate sigmoid(gate)
//
// with b and c shared by the channels of a group.  Its gradients, with dp = dy silu(gate):
//
//   g_t[n] = c_t[n] dp_t + r_{t+1}[n],   r_t[n] = e^(delta_t a[n]) g_t[n]     (back in time)
//   k_t[n] = r_t[n] h_{t-1}[n]
//   da[n] = sum_t delta_t k_t[n]            dx_t = delta_t sum_n g_t[n] b_t[n] + skip dp_t
//   db_t[n] = sum_d g_t[n] delta_t x_t      ddelta_t = sum_n (a[n] k_t[n]) + x_t sum_n g_t[n] b_t[n]
//   dc_t[n] = sum_d dp_t h_t[n]             dgate_t = dy_t p_t silu'(gate_t),  dskip = sum_t dp_t x_t
//
// The decays depend on channel, state and token, so there is no product of matrices in it: a state
// and token cost one exponential (16 a clock and SM, 4.65e12 a second on 148 SMs) and 4 (backward
// 12) operations of the FMA pipes; bytes are 8 and 22 a token and channel in 16 bits, 0.3 of the
// exponentials' time with 16 states.
//
// Split.  A thread keeps 4 neighbouring states of 2 channels; LN lanes hold a channel's states (up to
// 4 LN) and the 32 / LN groups of lanes of a warp neighbouring channels.  Sums over states cross LN
// lanes, those over channels (db, dc) the others; each step of such a sum halves the values a lane
// holds.  A block of 4 warps stages some tokens of its channels in shared memory in 32 bits: delta
// and delta x, b and c.  Long sequences of few channels are cut into segments: a state launch forms
// each segment's end state from zero and its sum of delta, and the main launch's blocks add up those
// before them.
//
// Measured (bf16, 16 states, a gate; ncu and events).  64 x 1024 x 2048, one launch: 794 us, 2.7e12
// exponentials a second, 0.58 of their rate, 0.73 with those of the steps and gates counted.
// 1 x 65536 x 2048, 37 segments: state launch 642 us, main launch 838 us.  4 x 4096 x 2048 with
// gradients, 9 and 16 segments: 154 + 235 us forward, 173 us of states back in time, 637 us backward,
// 29 us of sums.  240 single tokens of 2048 channels: 15.4 us (4.4 TB/s).  With few states the steps and
// gates, some 35 instructions and 4 exponentials or reciprocals a token and channel, are as much work as
// the states: 64 x 1024 x 1024 with 4 states 238 us, 1.1e12 exponentials of decays a second.
// What was tried on the forward launches and changed nothing or made them slower: a quarter of the
// exponentials by a polynomial on the FMA pipes (state launch 640 us either way, main launch 6 %
// slower), 5 and 6 blocks an SM (5 % and 9 % slower), a second copy of the staged steps for wider
// loads.  It is the mix of exponentials, shared memory and FMA instructions that fills the issue
// slots; a 16-bit load that is taken apart where it is issued, and so waited for, cost 1.7 times.
#pragma once

#include "row_groups.cuh"

namespace fdwt {

constexpr int kScanCheck = 8;  // tokens from one kept state to the next (for the backward pass)

struct ScanArgs {
  const void *x, *dt, *a, *b, *c, *skip, *gate, *dt_bias, *initial;
  const int32_t* lengths;
  int64_t batch, length, dim;
  int groups, states;
  int softplus;
  int64_t xs[2], dts[2], gs[2], dys[2], bs[3], cs[3];
  int vec, vec_states;  // rows of channels, of b and c begin on boundaries of 4 elements
  int64_t per, tiles; // channels of a group, tiles of one
  int64_t tile0, tile_count;  // the launch's tiles among those of all groups
  int segments;
  int64_t seg_len;    // tokens, a multiple of kScanCheck and of the staged tokens
  void *seg_state, *seg_sum;  // [batch][segments][dim][padded states], [batch][segments][dim]
  void *y, *final_state;
  void* check;        // states before tokens 0, 8, 16, ...: [batch][ceil(length / 8)][dim][padded]
  // backward
  const void *dy, *d_final;
  void *dx, *ddt, *dgate, *d_initial;
  void *part_bc;      // [tile_count][batch][length][2][padded states]; null where none are wanted
  void *part_a;       // [batch][segments][dim][padded states]
  void *part_ch;      // [batch][segments][2][dim]: dskip, ddt_bias
};

// Launchers by element type (selscan_*.cu).  `lanes` is LN, 1 to 32.
template <typename T> int scan_forward(const ScanArgs& p, int lanes, cudaStream_t stream);
template <typename T> int scan_states(const ScanArgs& p, int lanes, bool reverse, cudaStream_t stream);
template <typename T> int scan_backward(const ScanArgs& p, int lanes, cudaStream_t stream);
// Blocks of the forward and the backward launch that are resident on the device.
template <typename T> int64_t scan_resident(int lanes, bool backward);
template <typename T> int scan_step(const ScanArgs& p, int lanes, const int32_t* slots, int64_t pool,
                                    void* state, cudaStream_t stream);

// Channels of a thread, and of a block.
constexpr int scan_fwd_channels(int ln) { return ln == 1 ? 1 : 2; }
constexpr int scan_fwd_tile(int ln) { return 4 * (32 / ln) * scan_fwd_channels(ln); }
constexpr int scan_bwd_channels(int ln, bool fp64) { return ln <= 2 || (fp64 && ln <= 8) ? 1 : 2; }
constexpr int scan_bwd_tile(int ln, bool fp64) {
  return 4 * (32 / ln) * scan_bwd_channels(ln, fp64);
}

}  // namespace fdwt
