// Launches of group norm with an activation (group_norm_kernel.hpp).
#include "group_norm_kernel.hpp"

namespace linrec {
namespace {

// d_bias and d_weight from rows of (sums of e, sums of e xh).
__global__ __launch_bounds__(64 * SUM_WAVES) void param_sum_kernel(const float* in, int64_t rows, int64_t columns, int64_t per_chunk, float* out) {
  column_sum_block(in, rows, columns, per_chunk, [&](int64_t c, float s) { out[blockIdx.y * columns + c] = s; });
}
__global__ __launch_bounds__(64 * SUM_WAVES) void param_gradient_kernel(const float* in, int64_t rows, int64_t channels, int dtype, void* d_weight,
                                                                        void* d_bias) {
  column_sum_block(in, rows, 2 * channels, rows, [&](int64_t c, float s) {
    void* to = c < channels ? d_bias : d_weight;
    if (c >= channels) c -= channels;
    if (dtype == LINREC_DTYPE_F32) static_cast<float*>(to)[c] = s;
    else if (dtype == LINREC_DTYPE_F16) static_cast<_Float16*>(to)[c] = _Float16(s);
    else static_cast<__bf16*>(to)[c] = __bf16(s);
  });
}

enum class Shape { tokens, held, chunks };
struct NormPlan {
  Shape shape;
  int vec;
  int lanes;           // of a workgroup
  int64_t grid;
  int64_t param_rows;  // rows of partial sums of d_weight and d_bias
  int64_t pieces;      // floats of partial statistics
  TokenArgs tokens;
  int items_per_lane;  // tokens: slots of a lane
  bool parts;          // held: a workgroup's rows are fp32 and not whole lines
  BlockArgs block;
};

int pow2_at_least(int64_t n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

NormPlan make_norm_plan(int dtype, int64_t batch, int64_t positions, int64_t channels, int64_t groups, bool bwd) {
  NormPlan pl{};
  const int64_t width = channels / groups;
  const int size = dtype == LINREC_DTYPE_F32 ? 4 : 2;
  pl.vec = 16 / size;
  while (width % pl.vec) pl.vec >>= 1;
  const int64_t columns = width / pl.vec;  // of a group

  // 16 channels to a lane, at most eight waves to a group (32768 x 1024 in 16 groups bf16 31 and 49 us, as a workgroup's columns 61
  // and 165)
  if (positions == 1 && width <= 16 * 64 * TOKEN_WAVES) {
    pl.shape = Shape::tokens;
    TokenArgs& t = pl.tokens;
    // one slot to a lane while eight waves hold a group so: the registers of more cost rows under way
    const int64_t slots_of_lane = columns <= 64 * TOKEN_WAVES ? 1 : 16 / pl.vec;
    pl.items_per_lane = int(slots_of_lane);
    t.team = pow2_at_least(cdiv(columns, slots_of_lane));
    const int64_t waves = t.team < 64 ? cdiv(groups, 64 / t.team) : groups * (t.team / 64);  // of a row
    t.column_waves = waves < TOKEN_WAVES ? pow2_at_least(waves) : TOKEN_WAVES;
    t.column_blocks = int(cdiv(waves, t.column_waves));
    const int64_t slots = TOKEN_WAVES / t.column_waves;
    // enough workgroups for the chip; in the backward each leaves a row of sums behind, 8 bytes a channel, so a wave walks eight
    // rows first (2048 x 4096 in bf16: 32 us with a row of sums to every four)
    int64_t row_blocks = cdiv(batch, slots);
    int64_t most = 1024;
    if (bwd) {
      most = cdiv(batch, slots * 8);
      most = most < 128 ? 128 : most > 512 ? 512 : most;
    }
    const int64_t cap = most / t.column_blocks > 1 ? most / t.column_blocks : 1;
    if (row_blocks > cap) row_blocks = cap;
    t.row_blocks = int(row_blocks);
    pl.lanes = 64 * TOKEN_WAVES;
    pl.grid = int64_t(t.row_blocks) * t.column_blocks;
    pl.param_rows = t.row_blocks;
    return pl;
  }

  BlockArgs& a = pl.block;
  a.whole = int(columns);
  // held: whole groups in registers, side by side where one is narrower than a line (16 x 2048 x 512 in 32 groups fp32 38 and 62 us,
  // in chunks 49 and 92; 512 x 64 x 256 in 8 groups bf16 12 and 27, in chunks 16 and 29)
  const int bytes = pl.vec * size;
  const int keep = (bwd && size == 2 ? 24 : 32) / (bytes >= 4 ? bytes / 4 : 1);
  auto rows_of = [](int lanes, int64_t wide) { return wide <= lanes ? lanes / wide : int64_t(0); };
  auto rounds = [&](int lanes, int64_t wide) { return rows_of(lanes, wide) ? cdiv(positions, rows_of(lanes, wide)) : int64_t(1) << 40; };
  for (const int line : {128, 64}) {
    int64_t g = cdiv(line, columns * bytes);
    if (g > groups) g = groups;
    while (g > 1 && cdiv(groups, g) * batch < 256) g = g / 2;  // (so few that the chip idles: latency, not lines)
    for (const int lanes : {256, 1024}) {
      if (rounds(lanes, g * columns) > keep) continue;
      // few workgroups: more lanes to each
      if (lanes == 256 && cdiv(groups, g) * batch <= 256 && rounds(lanes, g * columns) > 2) continue;
      // a backward whose few workgroups hold much is better shared out (1 x 700 x 512 in 8 groups bf16 26 us held, 20 in chunks,
      // 2 x 2048 x 512 in 32 fp32 26 and 23; of 24 values to a lane 22 and 22, of 128 workgroups and 24 values 24 and 25)
      if (bwd && cdiv(groups, g) * batch <= 64 && rounds(lanes, g * columns) * pl.vec > 24) continue;
      int64_t items = 1;
      // lanes that have nothing to do take more groups, or more batch items; so do short walks while the chip stays full
      auto grows = [&](int64_t gg, int64_t it) {
        const int64_t n = rounds(lanes, gg * columns * it);
        return n == 1 || (n <= (bwd ? keep : keep / 2) && cdiv(groups, gg) * cdiv(batch, it) >= (bwd ? 512 : 1024));
      };
      while (2 * g <= groups && grows(2 * g, 1)) g *= 2;
      if (g < groups && 2 * g > groups && grows(groups, 1)) g = groups;
      if (g == groups)
        while (2 * items <= batch && grows(g, 2 * items)) items *= 2;
      pl.shape = Shape::held;
      pl.lanes = lanes;
      a.per_group = int(columns); a.groups = int(g); a.items = int(items); a.parts = 1; a.chunks = 1;
      a.blocks = int(cdiv(groups, g));
      a.columns = int(items * g * columns);
      a.R = int(rows_of(lanes, a.columns));
      a.rows = int(positions);
      pl.parts = size == 4 && (g * columns * bytes % 128 != 0 || channels * size % 128 != 0);
      pl.param_rows = cdiv(batch, items);
      pl.grid = pl.param_rows * a.blocks;
      return pl;
    }
  }

  pl.shape = Shape::chunks;
  pl.lanes = 256;
  a.parts = int(cdiv(columns, 256));
  a.per_group = int(cdiv(columns, a.parts));
  a.parts = int(cdiv(columns, a.per_group));  // (none of them empty)
  a.groups = a.parts > 1 ? 1 : int(256 / columns < groups ? 256 / columns : groups);
  a.items = 1;
  a.blocks = int(cdiv(groups, a.groups) * a.parts);
  a.columns = a.groups * a.per_group;
  a.R = 256 / a.columns;
  const int64_t side = batch * a.blocks;
  int64_t chunks = cdiv(2048, side), most = cdiv(positions, int64_t(a.R) * 8);
  if (chunks > most) chunks = most;
  if (chunks > 256) chunks = 256;
  if (chunks < 1) chunks = 1;
  a.rows = int(cdiv(cdiv(positions, chunks), a.R) * a.R);
  a.chunks = int(cdiv(positions, a.rows));
  pl.grid = side * a.chunks;
  pl.param_rows = batch * a.chunks;
  pl.pieces = 2 * batch * a.chunks * a.parts * groups;
  return pl;
}

int64_t partial_floats(const NormPlan& pl, int64_t channels, bool bwd) {
  if (!bwd) return pl.pieces;
  const int64_t chunks = column_sum_chunks(pl.param_rows);
  return pl.pieces + 2 * channels * (pl.param_rows + (chunks > 1 ? chunks : 0));
}

template <typename T, int VEC, bool BWD>
int launch_tokens(const linrec_group_norm_t& p, const NormPlan& pl) {
  TokenArgs a = pl.tokens;
  a.p = p;
  if (BWD) a.p.partial = p.partial + pl.pieces;
  return pl.items_per_lane == 1 ? launch_kernel(norm_tokens_kernel<T, VEC, 1, BWD>, pl.grid, 1, pl.lanes, p.stream, a)
                                : launch_kernel(norm_tokens_kernel<T, VEC, 16 / VEC, BWD>, pl.grid, 1, pl.lanes, p.stream, a);
}

template <typename T, int VEC, int LANES, int PHASE>
int launch_held(const BlockArgs& a, const NormPlan& pl, bool bwd, float* sums) {
  return bwd ? launch_kernel(norm_bwd_kernel<T, VEC, LANES, PHASE>, pl.grid, 1, LANES, a.p.stream, a, sums)
             : launch_kernel(norm_fwd_kernel<T, VEC, LANES, PHASE>, pl.grid, 1, LANES, a.p.stream, a);
}
template <typename T, int VEC, int PHASE>
int launch_held(const BlockArgs& a, const NormPlan& pl, bool bwd, float* sums) {
  return pl.lanes == 256 ? launch_held<T, VEC, 256, PHASE>(a, pl, bwd, sums) : launch_held<T, VEC, 1024, PHASE>(a, pl, bwd, sums);
}

template <typename T, int VEC>
int launch_norm(const linrec_group_norm_t& p, const NormPlan& pl, bool bwd) {
  if (pl.shape == Shape::tokens) return bwd ? launch_tokens<T, VEC, true>(p, pl) : launch_tokens<T, VEC, false>(p, pl);
  BlockArgs a = pl.block;
  a.p = p;
  float* sums = p.partial + pl.pieces;
  if (pl.shape == Shape::held) {
    if constexpr (sizeof(T) == 4) {
      if (pl.parts) return launch_held<T, VEC, NORM_HELD_PARTS>(a, pl, bwd, sums);
    }
    return launch_held<T, VEC, NORM_HELD>(a, pl, bwd, sums);
  }
  if (!bwd) {
    if (const int rc = launch_kernel(norm_fwd_kernel<T, VEC, 256, NORM_STATS>, pl.grid, 1, 256, p.stream, a)) return rc;
    return launch_kernel(norm_fwd_kernel<T, VEC, 256, NORM_APPLY>, pl.grid, 1, 256, p.stream, a);
  }
  if (const int rc = launch_kernel(norm_bwd_kernel<T, VEC, 256, NORM_STATS>, pl.grid, 1, 256, p.stream, a, sums)) return rc;
  return launch_kernel(norm_bwd_kernel<T, VEC, 256, NORM_APPLY>, pl.grid, 1, 256, p.stream, a, sums);
}

int launch_norm(const linrec_group_norm_t& p, const NormPlan& pl, bool bwd) {
  return with_dtype(p.dtype, [&](auto t) {
    using T = decltype(t);
    switch (pl.vec) {
      case 1: return launch_norm<T, 1>(p, pl, bwd);
      case 2: return launch_norm<T, 2>(p, pl, bwd);
      case 4: return launch_norm<T, 4>(p, pl, bwd);
    }
    if constexpr (sizeof(T) == 2) return launch_norm<T, 8>(p, pl, bwd);
    return int(LINREC_E_UNSUPPORTED);
  });
}

int check_norm(const linrec_group_norm_t* p) {
  if (!p || p->batch < 0 || p->positions < 0 || p->channels < 0 || p->groups < 1 || p->channels % p->groups) return LINREC_E_INVALID;
  if (p->act < LINREC_ACT_NONE || p->act > LINREC_ACT_GELU || !p->weight != !p->bias) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16 || p->weight_dtype < LINREC_DTYPE_F32 || p->weight_dtype > LINREC_DTYPE_BF16)
    return LINREC_E_UNSUPPORTED;
  if (p->batch > 2147483647LL || p->positions > 2147483647LL - 65536 || p->channels > 2147483647LL - 65536) return LINREC_E_TOO_LARGE;
  if (p->batch > 0 && p->positions > 0 && p->channels > 0 && (!p->x || !p->mean || !p->rstd)) return LINREC_E_INVALID;
  return LINREC_OK;
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

int64_t linrec_group_norm_partial_floats(int dtype, int64_t batch, int64_t positions, int64_t channels, int64_t groups, int is_bwd) {
  if (batch <= 0 || positions <= 0 || channels <= 0 || groups <= 0 || channels % groups) return is_bwd ? 2 * (channels > 0 ? channels : 0) : 0;
  return partial_floats(make_norm_plan(dtype, batch, positions, channels, groups, is_bwd != 0), channels, is_bwd != 0);
}

int linrec_group_norm_fwd(const linrec_group_norm_t* p) {
  if (const int rc = check_norm(p)) return rc;
  if (p->batch == 0 || p->positions == 0 || p->channels == 0) return LINREC_OK;
  const NormPlan pl = make_norm_plan(p->dtype, p->batch, p->positions, p->channels, p->groups, false);
  if (!p->y || (partial_floats(pl, p->channels, false) && !p->partial)) return LINREC_E_INVALID;
  return launch_norm(*p, pl, false);
}

int linrec_group_norm_bwd(const linrec_group_norm_t* p) {
  if (const int rc = check_norm(p)) return rc;
  if (p->channels == 0) return LINREC_OK;
  if (p->weight && (!p->d_weight || !p->d_bias)) return LINREC_E_INVALID;
  int64_t rows = 0;
  const float* sums = p->partial;
  if (p->batch > 0 && p->positions > 0) {
    if (!p->d_y || !p->d_x || !p->partial) return LINREC_E_INVALID;
    const NormPlan pl = make_norm_plan(p->dtype, p->batch, p->positions, p->channels, p->groups, true);
    if (const int rc = launch_norm(*p, pl, true)) return rc;
    rows = pl.param_rows;
    sums += pl.pieces;
  }
  if (!p->weight) return LINREC_OK;
  const int64_t chunks = column_sum_chunks(rows), columns = 2 * p->channels;
  if (chunks > 1) {
    float* out = const_cast<float*>(sums) + rows * columns;
    if (const int rc = launch_kernel(param_sum_kernel, cdiv(columns, 64), chunks, 64 * SUM_WAVES, p->stream, sums, rows, columns, SUM_ROWS, out))
      return rc;
    sums = out;
    rows = chunks;
  }
  return launch_kernel(param_gradient_kernel, cdiv(columns, 64), 1, 64 * SUM_WAVES, p->stream, sums, rows, p->channels, p->weight_dtype,
                       p->d_weight, p->d_bias);
}

}  // extern "C"
