// Launches of the gated linear recurrence and its single-token step (gated_kernel.hpp).
#include "column_sum.hpp"
#include "gated_kernel.hpp"
#include "workspace.hpp"

namespace linrec {
namespace {

// d_rate from the segments' sums of P: the last launch of a backward.
__global__ __launch_bounds__(64 * SUM_WAVES) void rate_sum_kernel(const float* in, int64_t rows, int64_t channels, int64_t per_chunk,
                                                                  float* out) {
  column_sum_block(in, rows, channels, per_chunk, [&](int64_t c, float s) { out[blockIdx.y * channels + c] = s; });
}
__global__ __launch_bounds__(64 * SUM_WAVES) void rate_gradient_kernel(const float* in, int64_t rows, int64_t channels, const float* rate,
                                                                       float* d_rate) {
  column_sum_block(in, rows, channels, rows, [&](int64_t c, float s) {
    // sigmoid / softplus of the rate, 1 where both vanish
    const float v = rate[c], sp = fast_softplus(v);
    d_rate[c] = sp > 0.0f ? s * (fast_sigmoid(v) / sp) : s;
  });
}

// Sequences of no positions at all: what enters leaves.
__global__ void hand_on_kernel(const float* from, float* to, int64_t n) {
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.0f;
}
int hand_on(const float* from, float* to, int64_t n, void* stream) {
  return to ? launch_kernel(hand_on_kernel, cdiv(n, 256), 1, 256, stream, from, to, n) : LINREC_OK;
}

// One position: a lane has VEC channels of a row.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void gated_step_kernel(linrec_gated_step_t p, int blocks) {
  const int64_t n = blockIdx.x / unsigned(blocks);
  const int64_t c0 = (int64_t(blockIdx.x - unsigned(n) * unsigned(blocks)) * 256 + threadIdx.x) * VEC;
  if (c0 >= p.channels) return;
  const int64_t last = p.channels - VEC, c = c0 < last ? c0 : last;  // (a lane that starts early stores what is its own)
  const int own = int(c0 - c);
  T* h = static_cast<T*>(p.h) + n * p.channels + c;
  const int64_t slot = p.slots ? p.slots[n] : n;
  Lanes<VEC> v;
  if (slot < 0 || slot >= p.slots_total) {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e >= own) h[e] = T(0.0f);
    return;
  }
  const Lanes<VEC> x = widen(ld_any<VEC, false>(static_cast<const T*>(p.x) + n * p.x_stride + c));
  const Lanes<VEC> ga = widen(ld_any<VEC, false>(static_cast<const T*>(p.gate_a) + n * p.gate_a_stride + c));
  const Lanes<VEC> gx = widen(ld_any<VEC, false>(static_cast<const T*>(p.gate_x) + n * p.gate_x_stride + c));
  float* state = p.state + slot * p.state_stride + c;
  const Lanes<VEC> rate = ld_any<VEC, false>(p.rate + c).q, s = ld_any<VEC, false>(state).q;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const Gate g = gate_of(ga.v[e], gx.v[e], LOG2E * p.scale * fast_softplus(rate.v[e]));
    v.v[e] = fmaf(g.a, s.v[e], taken_in(g, x.v[e]));
  }
  if (own == 0) {
    st_any<VEC>(state, v);
    st_any<VEC>(h, v);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e >= own) {
        state[e] = v.v[e];
        h[e] = T(v.v[e]);
      }
  }
}

int check_gated(const linrec_gated_t* p) {
  if (!p || p->batch < 0 || p->time < 0 || p->channels < 0 || p->sequences < 0) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->cu_seqlens ? p->batch != 1 : p->sequences != p->batch) return LINREC_E_INVALID;
  if (p->time > 2147483647LL - 4096 || p->channels > 2147483647LL - 4096 || p->batch > 2147483647LL || p->sequences > 2147483647LL)
    return LINREC_E_TOO_LARGE;
  if (p->channels > 0 && p->batch > 0 && p->time > 0 && (!p->x || !p->gate_a || !p->gate_x || !p->rate)) return LINREC_E_INVALID;
  return LINREC_OK;
}

// Channels of a lane: 4 bytes' worth, one where there are no two.
int lane_width(int dtype, int64_t channels) { return dtype == LINREC_DTYPE_F32 || channels < 2 ? 1 : 2; }

constexpr int kFwdRun = 16, kFwdWaves = 4, kBwdRun = 8, kBwdWaves = 8;
struct Geometry {
  int64_t segments, channel_blocks, grid, tiles;
  int save;
};
Geometry geometry(int dtype, int64_t batch, int64_t time, int64_t channels, bool bwd) {
  Geometry g;
  const int64_t rows = 64 * lane_width(dtype, channels);
  g.channel_blocks = cdiv(channels, rows);
  const int64_t blocks = g.channel_blocks * batch;
  g.save = kBwdRun * kBwdWaves;
  g.segments = cdiv(time, bwd ? g.save : kFwdWaves * kFwdRun);
  g.grid = g.segments * blocks;
  g.tiles = chain_places(g.segments) * blocks * rows;  // places of words
  return g;
}

// Rows are whole lines of 128 bytes.
bool whole_lines(const linrec_gated_t& p) { return p.channels * (p.dtype == LINREC_DTYPE_F32 ? 4 : 2) % 128 == 0; }

int fill_args(const linrec_gated_t* p, const Geometry& g, GatedArgs* a) {
  a->p = *p;
  a->chain = TileArgs{};
  a->segments = int(g.segments);
  a->channel_blocks = int(g.channel_blocks);
  a->save = g.save;
  a->side = whole_lines(*p) ? GROUP : 8;
  if (a->side > g.segments) a->side = int(g.segments);
  if (g.grid > 2147483647LL) return LINREC_E_TOO_LARGE;
  if (g.segments <= 1) return LINREC_OK;
  if (!p->workspace || (reinterpret_cast<uintptr_t>(p->workspace) & 15u)) return LINREC_E_WORKSPACE;
  const WorkspaceLayout lay = workspace_layout(size_t(p->workspace_bytes));
  if (lay.tiles < g.tiles) return LINREC_E_WORKSPACE;
  a->chain.num_tiles = g.grid;
  a->chain.ws = static_cast<CarryHeader*>(p->workspace);
  a->chain.counters = reinterpret_cast<uint32_t*>(static_cast<char*>(p->workspace) + lay.counters_offset);
  a->chain.desc = reinterpret_cast<uint64_t*>(static_cast<char*>(p->workspace) + lay.desc_offset);
  a->chain.ws_tiles = lay.tiles;
  a->chain.spin_limit = linrec_set_spin_limit(0);  // (asks)
  return LINREC_OK;
}

template <typename T, int VEC, bool PACKED, bool LINES>
int launch_pass(const GatedArgs& a, const Geometry& g, bool bwd) {
  return bwd ? launch_kernel(gated_bwd_kernel<T, VEC, kBwdRun, kBwdWaves, PACKED, LINES>, g.grid, 1, 64 * kBwdWaves, a.p.stream, a)
             : launch_kernel(gated_fwd_kernel<T, VEC, kFwdRun, kFwdWaves, PACKED, LINES>, g.grid, 1, 64 * kFwdWaves, a.p.stream, a);
}
template <typename T, int VEC>
int launch_pass(const GatedArgs& a, const Geometry& g, bool bwd) {
  if constexpr (VEC * sizeof(T) == 2)  // (rows of one value)
    return a.p.cu_seqlens ? launch_pass<T, VEC, true, false>(a, g, bwd) : launch_pass<T, VEC, false, false>(a, g, bwd);
  else if (a.p.cu_seqlens) return whole_lines(a.p) ? launch_pass<T, VEC, true, true>(a, g, bwd) : launch_pass<T, VEC, true, false>(a, g, bwd);
  else
    return whole_lines(a.p) ? launch_pass<T, VEC, false, true>(a, g, bwd) : launch_pass<T, VEC, false, false>(a, g, bwd);
}

int launch_pass(const GatedArgs& a, const Geometry& g, bool bwd) {
  return with_dtype(a.p.dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (sizeof(T) == 2) {
      if (lane_width(a.p.dtype, a.p.channels) == 2) return launch_pass<T, 2>(a, g, bwd);
    }
    return launch_pass<T, 1>(a, g, bwd);
  });
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

int64_t linrec_gated_saved_floats(int dtype, int64_t batch, int64_t time, int64_t channels) {
  if (batch <= 0 || time <= 0 || channels <= 0) return 0;
  return batch * geometry(dtype, batch, time, channels, true).segments * channels;
}

// a row for every backward segment, and the sums of their chunks
int64_t linrec_gated_partial_floats(int dtype, int64_t batch, int64_t time, int64_t channels) {
  if (batch <= 0 || time <= 0 || channels <= 0) return 0;
  const int64_t rows = batch * geometry(dtype, batch, time, channels, true).segments, chunks = column_sum_chunks(rows);
  return (rows + (chunks > 1 ? chunks : 0)) * channels;
}

size_t linrec_gated_workspace_bytes(int dtype, int64_t batch, int64_t time, int64_t channels, int is_bwd) {
  if (batch <= 0 || time <= 0 || channels <= 0) return 0;
  const Geometry g = geometry(dtype, batch, time, channels, is_bwd != 0);
  return g.segments > 1 ? linrec_workspace_bytes_for_tiles(g.tiles) : 0;
}

int linrec_gated_fwd(const linrec_gated_t* p) {
  if (const int rc = check_gated(p)) return rc;
  if (p->channels == 0 || p->batch == 0 || p->sequences == 0) return LINREC_OK;
  if (p->time == 0) return hand_on(p->h0, p->state, p->sequences * p->channels, p->stream);
  if (!p->h) return LINREC_E_INVALID;
  const Geometry g = geometry(p->dtype, p->batch, p->time, p->channels, false);
  GatedArgs a;
  if (const int rc = fill_args(p, g, &a)) return rc;
  return launch_pass(a, g, false);
}

int linrec_gated_bwd(const linrec_gated_t* p) {
  if (const int rc = check_gated(p)) return rc;
  if (p->channels == 0) return LINREC_OK;
  if (!p->d_rate || !p->rate) return LINREC_E_INVALID;
  if (p->batch == 0 || p->time == 0 || p->sequences == 0) {
    if (const int rc = hand_on(p->d_state, p->d_h0, p->sequences * p->channels, p->stream)) return rc;
    return hand_on(nullptr, p->d_rate, p->channels, p->stream);
  }
  if (!p->saved || !p->d_h || !p->d_x || !p->d_gate_a || !p->d_gate_x || !p->partial) return LINREC_E_INVALID;
  const Geometry g = geometry(p->dtype, p->batch, p->time, p->channels, true);
  GatedArgs a;
  if (const int rc = fill_args(p, g, &a)) return rc;
  if (const int rc = launch_pass(a, g, true)) return rc;
  int64_t rows = p->batch * g.segments;
  const int64_t chunks = column_sum_chunks(rows), columns = cdiv(p->channels, 64);
  const float* sums = p->partial;
  if (chunks > 1) {
    float* out = p->partial + rows * p->channels;
    if (const int rc = launch_kernel(rate_sum_kernel, columns, chunks, 64 * SUM_WAVES, p->stream, sums, rows, p->channels, SUM_ROWS, out))
      return rc;
    sums = out;
    rows = chunks;
  }
  return launch_kernel(rate_gradient_kernel, columns, 1, 64 * SUM_WAVES, p->stream, sums, rows, p->channels, p->rate, p->d_rate);
}

int linrec_gated_step(const linrec_gated_step_t* p) {
  if (!p || p->batch < 0 || p->channels < 0 || p->slots_total < 0) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->batch == 0 || p->channels == 0) return LINREC_OK;
  if (!p->x || !p->gate_a || !p->gate_x || !p->rate || !p->h || (!p->state && p->slots_total > 0)) return LINREC_E_INVALID;
  if (!p->slots && p->slots_total < p->batch) return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto kernel, int vec) {
      const int64_t blocks = cdiv(p->channels, 256 * vec);
      return launch_kernel(kernel, p->batch * blocks, 1, 256, p->stream, *p, int(blocks));
    };
    return p->channels >= 4 ? launch(gated_step_kernel<T, 4>, 4) : launch(gated_step_kernel<T, 1>, 1);
  });
}

}  // extern "C"
