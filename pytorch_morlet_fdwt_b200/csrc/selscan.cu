// Selective state space scan: the C entry points, how a call is cut, and the sums over blocks.
#include "selscan.cuh"

namespace fdwt {
namespace {

// db and dc (batch, length, groups, states) of the groups from group0 on, from the parts of the tiles
// tile0 ... tile1 - 1, added in a fixed order: a group's sum goes on from `sums` where earlier tiles of it
// were in another launch, and into it where later ones are.
template <typename T>
__global__ void __launch_bounds__(256)
scan_bc_kernel(const typename AccOf<T>::type* __restrict__ part,
               typename AccOf<T>::type* __restrict__ sums, const int32_t* __restrict__ lengths,
               int64_t batch, int64_t length, int groups, int group0, int64_t tiles, int64_t tile0,
               int64_t tile1, int states, int padded, T* __restrict__ db, T* __restrict__ dc) {
  using A = typename AccOf<T>::type;
  const int64_t id = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int e = static_cast<int>(id % (2 * padded));
  const int64_t row = id / (2 * padded) + group0 * batch * length;  // (group, batch, token)
  const int n = e % padded;
  if (row >= groups * batch * length || n >= states) return;
  T* out = e < padded ? db : dc;
  if (out == nullptr) return;
  const int64_t t = row % length, b = row / length % batch, g = row / length / batch;
  const int64_t first = g * tiles > tile0 ? g * tiles : tile0;
  const int64_t end = (g + 1) * tiles < tile1 ? (g + 1) * tiles : tile1;
  if (first >= end) return;
  A sum = A(0);
  if (lengths == nullptr || t < lengths[b]) {
    if (first != g * tiles) sum = sums[row * 2 * padded + e];
    const int64_t step = batch * length * 2 * padded;
    const A* q = part + (first - tile0) * step + (b * length + t) * 2 * padded + e;
#pragma unroll 4
    for (int64_t k = first; k < end; ++k, q += step) sum += *q;
  }
  if (end == (g + 1) * tiles) out[((b * length + t) * groups + g) * states + n] = from_acc<T>(sum);
  else sums[row * 2 * padded + e] = sum;
}

// da, dskip and ddt_bias: columns summed over the rows (sequences and segments) in a fixed order, 32
// columns by 8 row lanes a block.  A row of `parts_a` has dim x padded columns, one of `parts_ch`
// 2 dim.
template <typename A>
__global__ void __launch_bounds__(256)
scan_rows_kernel(const A* __restrict__ parts_a, const A* __restrict__ parts_ch, int64_t rows,
                 int64_t dim, int states, int padded, A* __restrict__ da, A* __restrict__ dskip,
                 A* __restrict__ dbias) {
  __shared__ A cells[8][33];
  const int64_t c = int64_t(blockIdx.x) * 32 + threadIdx.x, cols_a = dim * padded;
  const bool of_a = c < cols_a;
  A* out = nullptr;
  if (of_a) {
    if (da != nullptr && c % padded < states) out = da + c / padded * states + c % padded;
  } else if (c < cols_a + dim) {
    if (dskip != nullptr) out = dskip + (c - cols_a);
  } else if (c < cols_a + 2 * dim && dbias != nullptr) {
    out = dbias + (c - cols_a - dim);
  }
  A sum = A(0);
  if (out != nullptr) {
    const A* q = of_a ? parts_a + c : parts_ch + (c - cols_a);
    const int64_t stride = of_a ? cols_a : 2 * dim;
#pragma unroll 4
    for (int64_t r = threadIdx.y; r < rows; r += 8) sum += q[r * stride];
  }
  cells[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  if (threadIdx.y != 0 || out == nullptr) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) sum += cells[k][threadIdx.x];
  *out = sum;
}

constexpr int64_t kMostTokens = int64_t(1) << 30;

bool scan_ok(const fdwt_scan_desc* d) {
  return d != nullptr && dtype_size(d->dtype) != 0 && d->groups >= 1 && d->states >= 1 &&
         d->batch >= 0 && d->length >= 0 && d->dim >= 1 && d->dim % d->groups == 0 &&
         d->batch < kMostTokens && d->length < kMostTokens && d->dim < kMostTokens;
}
int lanes_of(int states) {
  int lanes = 1;
  while (4 * lanes < states) lanes *= 2;
  return lanes;
}
size_t acc_size(int dtype) { return dtype == FDWT_F64 ? 8 : 4; }
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

template <typename F> auto with_type(int dtype, F fn) {
  switch (dtype) {
    case FDWT_F32: return fn(float{});
    case FDWT_F64: return fn(double{});
    case FDWT_F16: return fn(__half{});
    default: return fn(__nv_bfloat16{});
  }
}

// How a launch is cut: channels into tiles, sequences into segments.
struct Cut {
  int64_t tiles;  // of one group
  int segments;
  int64_t seg_len;
};
constexpr int64_t kSegmentStep = 16;  // segments are multiples of the staged tokens
constexpr int kMostSegments = 64;
// Microseconds of a token for each of the k blocks that share an SM, base + each k, and of a block's
// beginning, start (with what it does for every other segment, other): fitted to calls of 64 channels
// a block, 16 states, cut in 1 to 64 ways, in 16 bits.  Other counts of states (8 to 128 channels a block)
// and 64 bits go by the same numbers; nothing has shown how near the best cut those come.
struct Pace {
  double base, each, start, other;
};
double launch_time(double blocks, double resident, int64_t tokens, int segments, const Pace& pace) {
  const double sms = sm_count(), whole = static_cast<double>(static_cast<int64_t>(blocks / resident));
  const double rest = blocks - whole * resident, start = pace.start + pace.other * segments;
  double t = whole * (tokens * (pace.base + pace.each * resident / sms) + start);
  if (rest > 0) t += tokens * (pace.base + pace.each * (rest > sms ? rest / sms : 1.0)) + start;
  // blocks that all begin together stage and compute together, and overlap less
  return whole > 0 ? t : 1.1 * t;
}
// The number of segments with the shortest modelled time: more of them fill the device, but cost a
// state launch (for all segments but one) and beginnings.
Cut cut_of(const fdwt_scan_desc* d, int tile, int state_tile, int64_t resident, const Pace& pace,
           const Pace& state_pace) {
  Cut best{cdiv(d->dim / d->groups, tile), 1,
           imax(kSegmentStep, cdiv(d->length, kSegmentStep) * kSegmentStep)};
  const double blocks = double(best.tiles) * d->groups * d->batch;
  const double state_blocks = double(cdiv(d->dim / d->groups, state_tile)) * d->groups * d->batch;
  if (blocks == 0) return best;
  double least = launch_time(blocks, resident, best.seg_len, 1, pace);
  for (int n = 2; n <= kMostSegments; ++n) {
    const int64_t len = cdiv(cdiv(d->length, n), kSegmentStep) * kSegmentStep;
    if (len < 4 * kSegmentStep || cdiv(d->length, len) != n) continue;
    const double t = launch_time(blocks * n, resident, len, n, pace) + 3.0 +
                     launch_time(state_blocks * (n - 1), 4.0 * sm_count(), len, n, state_pace);
    if (t < least) least = t, best.segments = n, best.seg_len = len;
  }
  return best;
}
Cut forward_cut(const fdwt_scan_desc* d) {
  const int lanes = lanes_of(d->states), tile = scan_fwd_tile(lanes);
  return with_type(d->dtype, [&](auto t) {
    return cut_of(d, tile, tile, scan_resident<decltype(t)>(lanes, false),
                  {0.08, 0.0355, 1.0, 0.1}, {0.04, 0.0363, 0.5, 0.0});
  });
}
Cut backward_cut(const fdwt_scan_desc* d) {
  const int lanes = lanes_of(d->states);
  return with_type(d->dtype, [&](auto t) {
    return cut_of(d, scan_bwd_tile(lanes, d->dtype == FDWT_F64), scan_fwd_tile(lanes),
                  scan_resident<decltype(t)>(lanes, true), {0.107, 0.133, 1.0, 0.04},
                  {0.045, 0.037, 0.5, 0.0});
  });
}
struct Segments {
  size_t state, sum, bytes;
};
Segments segment_bytes(const fdwt_scan_desc* d, const Cut& c) {
  Segments s{0, 0, 0};
  if (c.segments == 1) return s;
  const size_t rows = size_t(d->batch) * c.segments * d->dim, a = acc_size(d->dtype);
  s.sum = up256(rows * 4 * lanes_of(d->states) * a);
  s.bytes = s.sum + up256(rows * a);
  return s;
}
// Parts of db and dc: one for each tile and token.  Tiles are the narrower the more states there are, so
// with all of them at once this would take 4 KB a token of 2048 channels at 16 states and 256 KB at 128.
// Above kMostPartBytes the backward pass is launched for some tiles at a time, and the sums go on from one
// launch's tiles to the next's, in the same order.
constexpr size_t kMostPartBytes = size_t(1) << 30;
struct Parts {
  size_t a, ch, bc, sums, least, bytes;  // least: without db and dc
  int64_t tiles;  // of a launch
};
Parts part_bytes(const fdwt_scan_desc* d, const Cut& c) {
  const size_t size = acc_size(d->dtype), np = 4 * lanes_of(d->states);
  const size_t rows = size_t(d->batch) * c.segments;
  const int64_t all = c.tiles * d->groups;
  const size_t tile = size_t(d->batch) * d->length * 2 * np * size;
  Parts p;
  p.tiles = tile == 0 ? all : imax(1, imin(all, static_cast<int64_t>(kMostPartBytes / tile)));
  p.a = segment_bytes(d, c).bytes;
  p.ch = p.a + up256(rows * d->dim * np * size);
  p.bc = p.least = p.ch + up256(rows * 2 * d->dim * size);
  p.sums = p.bc + up256(p.tiles * tile);
  p.bytes = p.sums + (p.tiles < all ? up256(d->groups * tile) : 0);
  return p;
}

bool aligned32(std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* q : pointers) bits |= reinterpret_cast<uintptr_t>(q);
  return bits % 32 == 0;
}

ScanArgs args_of(const fdwt_scan_desc* d, const void* x, const void* dt, const void* a,
                 const void* b, const void* c, const void* skip, const void* gate,
                 const void* dt_bias, const void* initial, const int32_t* lengths) {
  ScanArgs p{};
  p.x = x, p.dt = dt, p.a = a, p.b = b, p.c = c, p.skip = skip, p.gate = gate;
  p.dt_bias = dt_bias, p.initial = initial, p.lengths = lengths;
  p.batch = d->batch, p.length = d->length, p.dim = d->dim;
  p.groups = d->groups, p.states = d->states, p.softplus = d->dt_softplus != 0;
  for (int i = 0; i < 2; ++i) {
    p.xs[i] = d->x_stride[i], p.dts[i] = d->dt_stride[i];
    p.gs[i] = d->gate_stride[i], p.dys[i] = d->dy_stride[i];
  }
  for (int i = 0; i < 3; ++i) p.bs[i] = d->b_stride[i], p.cs[i] = d->c_stride[i];
  p.per = d->dim / d->groups;
  p.segments = 1;
  return p;
}
// Whether rows of channels, and of b and c, begin on boundaries of 4 elements (and channels and
// states come in whole fours).
bool in_fours(const fdwt_scan_desc* d, int64_t counts, std::initializer_list<const void*> pointers) {
  uintptr_t bits = 0;
  for (const void* q : pointers) bits |= reinterpret_cast<uintptr_t>(q);
  return counts % 4 == 0 && bits % (4 * dtype_size(d->dtype)) == 0;
}
void see_alignment(ScanArgs* p, const fdwt_scan_desc* d, bool backward) {
  int64_t rows = p->per | p->xs[0] | p->xs[1] | p->dts[0] | p->dts[1];
  if (p->gate != nullptr) rows |= p->gs[0] | p->gs[1];
  if (backward) rows |= p->dys[0] | p->dys[1];
  p->vec = in_fours(d, rows, {p->x, p->dt, p->gate, p->y, p->dy, p->dx, p->ddt, p->dgate});
  int64_t states = p->states;
  for (int i = 0; i < 3; ++i) states |= p->bs[i] | p->cs[i];
  p->vec_states = in_fours(d, states, {p->b, p->c});
}
void cut_into(ScanArgs* p, const fdwt_scan_desc* d, const Cut& c, void* ws) {
  const Segments s = segment_bytes(d, c);
  p->tiles = c.tiles, p->segments = c.segments, p->seg_len = c.seg_len;
  p->tile_count = c.tiles * d->groups;
  p->seg_state = static_cast<char*>(ws) + s.state;
  p->seg_sum = static_cast<char*>(ws) + s.sum;
}

}  // namespace
}  // namespace fdwt

using namespace fdwt;

extern "C" size_t fdwt_selscan_forward_workspace(const fdwt_scan_desc* desc) {
  if (!scan_ok(desc) || desc->states > FDWT_MAX_SCAN_STATES) return 0;
  return segment_bytes(desc, forward_cut(desc)).bytes;
}

extern "C" size_t fdwt_selscan_checkpoint_bytes(const fdwt_scan_desc* desc) {
  if (!scan_ok(desc) || desc->states > FDWT_MAX_SCAN_STATES) return 0;
  return size_t(desc->batch) * cdiv(desc->length, kScanCheck) * desc->dim * 4 *
         lanes_of(desc->states) * acc_size(desc->dtype);
}

extern "C" int fdwt_selscan_forward(const fdwt_scan_desc* desc, const void* x, const void* dt,
                                    const void* a, const void* b, const void* c, const void* skip,
                                    const void* gate, const void* dt_bias,
                                    const void* initial_state, const int32_t* lengths, void* y,
                                    void* final_state, void* checkpoints, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  FDWT_CHECK(scan_ok(desc));
  if (desc->states > FDWT_MAX_SCAN_STATES) return FDWT_ERR_UNSUPPORTED;
  if (desc->batch == 0 || (desc->length == 0 && final_state == nullptr)) return FDWT_OK;
  FDWT_CHECK(a != nullptr);
  FDWT_CHECK(desc->length == 0 || (x != nullptr && dt != nullptr && b != nullptr && c != nullptr &&
                                   y != nullptr));
  const Cut cut = forward_cut(desc);
  const size_t bytes = segment_bytes(desc, cut).bytes;
  if (bytes > 0 && (workspace == nullptr || workspace_bytes < bytes)) return FDWT_ERR_WORKSPACE;
  FDWT_CHECK(aligned32({workspace, checkpoints}));
  ScanArgs p = args_of(desc, x, dt, a, b, c, skip, gate, dt_bias, initial_state, lengths);
  p.y = y, p.final_state = final_state, p.check = checkpoints;
  see_alignment(&p, desc, false);
  cut_into(&p, desc, cut, workspace);
  const int lanes = lanes_of(desc->states);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return with_type(desc->dtype, [&](auto t) {
    using T = decltype(t);
    if (cut.segments > 1) {
      const int st = scan_states<T>(p, lanes, false, s);
      if (st != FDWT_OK) return st;
    }
    return scan_forward<T>(p, lanes, s);
  });
}

extern "C" size_t fdwt_selscan_backward_workspace(const fdwt_scan_desc* desc) {
  if (!scan_ok(desc) || desc->states > FDWT_MAX_SCAN_STATES) return 0;
  return part_bytes(desc, backward_cut(desc)).bytes;
}

extern "C" size_t fdwt_selscan_backward_workspace_least(const fdwt_scan_desc* desc) {
  if (!scan_ok(desc) || desc->states > FDWT_MAX_SCAN_STATES) return 0;
  return part_bytes(desc, backward_cut(desc)).least;
}

extern "C" int fdwt_selscan_backward(const fdwt_scan_desc* desc, const void* x, const void* dt,
                                     const void* a, const void* b, const void* c, const void* skip,
                                     const void* gate, const void* dt_bias, const int32_t* lengths,
                                     const void* checkpoints, const void* dy,
                                     const void* d_final_state, void* dx, void* ddt, void* da,
                                     void* db, void* dc, void* dskip, void* dgate, void* ddt_bias,
                                     void* d_initial_state, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  FDWT_CHECK(scan_ok(desc));
  if (desc->states > FDWT_MAX_SCAN_STATES) return FDWT_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t size = acc_size(desc->dtype);
  if (desc->batch == 0) {  // no sequences: the sums over them are zero
    if (da != nullptr) FDWT_CUDA(cudaMemsetAsync(da, 0, size * desc->dim * desc->states, s));
    if (dskip != nullptr) FDWT_CUDA(cudaMemsetAsync(dskip, 0, size * desc->dim, s));
    if (ddt_bias != nullptr) FDWT_CUDA(cudaMemsetAsync(ddt_bias, 0, size * desc->dim, s));
    return FDWT_OK;
  }
  FDWT_CHECK(a != nullptr && (gate == nullptr || dgate != nullptr || desc->length == 0));
  FDWT_CHECK(desc->length == 0 || (x != nullptr && dt != nullptr && b != nullptr && c != nullptr &&
                                   checkpoints != nullptr && dy != nullptr && dx != nullptr &&
                                   ddt != nullptr));
  const Cut cut = backward_cut(desc);
  const Parts parts = part_bytes(desc, cut);
  const bool want_bc = db != nullptr || dc != nullptr;
  if (workspace == nullptr || workspace_bytes < (want_bc ? parts.bytes : parts.least))
    return FDWT_ERR_WORKSPACE;
  FDWT_CHECK(aligned32({workspace, checkpoints}));
  ScanArgs p = args_of(desc, x, dt, a, b, c, skip, gate, dt_bias, nullptr, lengths);
  p.check = const_cast<void*>(checkpoints);
  p.dy = dy, p.d_final = d_final_state, p.dx = dx, p.ddt = ddt, p.dgate = dgate;
  p.d_initial = d_initial_state;
  char* ws = static_cast<char*>(workspace);
  p.part_a = ws + parts.a, p.part_ch = ws + parts.ch;
  p.part_bc = want_bc ? ws + parts.bc : nullptr;
  see_alignment(&p, desc, true);
  cut_into(&p, desc, cut, workspace);
  const int lanes = lanes_of(desc->states), np = 4 * lanes;
  return with_type(desc->dtype, [&](auto t) -> int {
    using T = decltype(t);
    using A = typename AccOf<T>::type;
    int st = FDWT_OK;
    if (cut.segments > 1) {
      // the state launch has tiles of its own
      ScanArgs r = p;
      r.tiles = cdiv(p.per, scan_fwd_tile(lanes));
      r.tile_count = r.tiles * desc->groups;
      st = scan_states<T>(r, lanes, true, s);
      if (st != FDWT_OK) return st;
    }
    const int64_t all = cut.tiles * desc->groups, each = want_bc ? parts.tiles : all;
    for (int64_t tile = 0; tile < all; tile += each) {
      const int64_t end = imin(all, tile + each);
      p.tile0 = tile, p.tile_count = end - tile;
      st = scan_backward<T>(p, lanes, s);
      if (st != FDWT_OK) return st;
      if (desc->length == 0 || !want_bc) continue;
      const int64_t group0 = tile / cut.tiles, count = cdiv(end, cut.tiles) - group0;
      const int64_t n = count * desc->batch * desc->length * 2 * np;
      if (cdiv(n, 256) > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
      st = pre_launch(s);
      if (st != FDWT_OK) return st;
      scan_bc_kernel<T><<<static_cast<unsigned>(cdiv(n, 256)), 256, 0, s>>>(
          static_cast<const A*>(p.part_bc), reinterpret_cast<A*>(ws + parts.sums), lengths,
          desc->batch, desc->length, desc->groups, static_cast<int>(group0), cut.tiles, tile, end,
          desc->states, np, static_cast<T*>(db), static_cast<T*>(dc));
      st = launch_status();
      if (st != FDWT_OK) return st;
    }
    const int64_t rows = desc->batch * cut.segments;
    if (da == nullptr && dskip == nullptr && ddt_bias == nullptr) return FDWT_OK;
    const int64_t columns = cdiv(desc->dim * (np + 2), 32);
    if (columns > INT32_MAX) return FDWT_ERR_UNSUPPORTED;
    st = pre_launch(s);
    if (st != FDWT_OK) return st;
    scan_rows_kernel<A><<<static_cast<unsigned>(columns), dim3(32, 8), 0, s>>>(
        static_cast<const A*>(p.part_a), static_cast<const A*>(p.part_ch), rows, desc->dim,
        desc->states, np, static_cast<A*>(da), static_cast<A*>(dskip), static_cast<A*>(ddt_bias));
    return launch_status();
  });
}

extern "C" int fdwt_selscan_step(const fdwt_scan_desc* desc, const void* x, const void* dt,
                                 const void* a, const void* b, const void* c, const void* skip,
                                 const void* gate, const void* dt_bias, void* state,
                                 int64_t state_slots, const int32_t* slots, void* y, void* stream) {
  FDWT_CHECK(scan_ok(desc) && desc->length == 1 && state_slots >= 0);
  FDWT_CHECK(slots != nullptr || state_slots >= desc->batch);
  if (desc->states > FDWT_MAX_SCAN_STATES) return FDWT_ERR_UNSUPPORTED;
  if (desc->batch == 0) return FDWT_OK;
  FDWT_CHECK(x != nullptr && dt != nullptr && a != nullptr && b != nullptr && c != nullptr &&
             y != nullptr && (state != nullptr || state_slots == 0));
  ScanArgs p = args_of(desc, x, dt, a, b, c, skip, gate, dt_bias, nullptr, nullptr);
  p.y = y;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(state);
  p.vec = desc->states % 4 == 0 && bits % (4 * acc_size(desc->dtype)) == 0;
  int64_t states = p.states;
  for (int i : {0, 2}) states |= p.bs[i] | p.cs[i];
  p.vec_states = in_fours(desc, states, {p.b, p.c});
  return with_type(desc->dtype, [&](auto t) {
    return scan_step<decltype(t)>(p, lanes_of(desc->states), slots, state_slots, state,
                                  static_cast<cudaStream_t>(stream));
  });
}
