// Launches of the root-mean-square norm (rms_norm_kernel.hpp).
#include "rms_norm_kernel.hpp"

namespace linrec {
namespace {

__global__ __launch_bounds__(64 * SUM_WAVES) void rms_sum_kernel(const float* in, int64_t rows, int64_t columns, int64_t per_chunk, float* out) {
  column_sum_block(in, rows, columns, per_chunk, [&](int64_t c, float s) { out[blockIdx.y * columns + c] = s; });
}
__global__ __launch_bounds__(64 * SUM_WAVES) void rms_weight_gradient_kernel(const float* in, int64_t rows, int64_t channels, int dtype, void* to) {
  column_sum_block(in, rows, channels, rows, [&](int64_t c, float s) {
    if (dtype == LINREC_DTYPE_F32) static_cast<float*>(to)[c] = s;
    else if (dtype == LINREC_DTYPE_F16) static_cast<_Float16*>(to)[c] = _Float16(s);
    else static_cast<__bf16*>(to)[c] = __bf16(s);
  });
}

struct RmsPlan {
  int vec, items, team, lanes, blocks;
};

RmsPlan plan_rms(int dtype, int64_t rows, int64_t channels, bool bwd) {
  RmsPlan pl{};
  const int whole = dtype == LINREC_DTYPE_F32 ? 4 : 8;
  pl.vec = channels >= whole ? whole : 1;
  const int64_t slots = cdiv(channels, pl.vec);
  const int most_items = bwd ? 4 : 8;
  auto team_of = [&](int items) {
    int team = 1;
    while (int64_t(team) * items < slots) team <<= 1;
    return team;
  };
  // Two loads of a lane to a row, and as many more as keep a row within a workgroup of 256: many waves hide the latency better than
  // many loads of few (20011 x 4096 bf16 with a residual to 8 bits: teams of 256 lanes with 2 loads 147 us, 64 with 8 212, 512 with 1 231,
  // all three before the weights came as vectors, with which the first is 117; 40000 x 1024: 64 with 2 32, 128 with 1 36, 32 with 4 45)
  pl.items = slots < 64 ? 1 : 2;
  while (pl.items < most_items && team_of(pl.items) > RMS_LANES) pl.items *= 2;
  // few rows: more lanes to each, so that one load's latency is all that a row takes
  while (pl.items > 1 && rows * team_of(pl.items) < 65536 && team_of(pl.items / 2) <= RMS_WIDE) pl.items /= 2;
  // a wide workgroup has half the registers for a lane
  while (pl.items > 1 && team_of(pl.items) > RMS_LANES && team_of(pl.items / 2) <= RMS_WIDE) pl.items /= 2;
  pl.team = team_of(pl.items);
  pl.lanes = pl.team > RMS_LANES ? pl.team : RMS_LANES;
  // A backward's workgroups each leave a row of sums behind: no more of them than a million sums, but twice the CUs (32768 x 2048 bf16: 512
  // 106 us, 1024 127, 4096 138; 262144 x 64 fp32: 4096 49 us, 1024 71).
  const int64_t sums = (int64_t(1) << 20) / channels;
  const int64_t needed = cdiv(rows, pl.lanes / pl.team), most = (!bwd || sums > 4096 ? 4096 : sums < 512 ? 512 : sums) * RMS_LANES / pl.lanes;
  pl.blocks = int(needed < most ? needed : most);
  return pl;
}

int check_rms(const linrec_rms_norm_t* p) {
  if (!p || p->rows < 0 || p->channels < 1 || p->inner < 1) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->weight && (p->weight_dtype < LINREC_DTYPE_F32 || p->weight_dtype > LINREC_DTYPE_BF16)) return LINREC_E_UNSUPPORTED;
  if (p->quantized < LINREC_QUANTIZED_NONE || p->quantized > LINREC_QUANTIZED_E4M3) return LINREC_E_UNSUPPORTED;
  if (p->channels > LINREC_RMS_NORM_CHANNELS_MAX) return LINREC_E_TOO_LARGE;
  if (p->rows > 0 && !p->x) return LINREC_E_INVALID;
  return LINREC_OK;
}

template <int VEC, int MOST, typename F>
int with_items(int items, F&& f) {
  auto of = [&](auto n) { return f(std::integral_constant<int, VEC>{}, n); };
  if (items == 1) return of(std::integral_constant<int, 1>{});
  if (items == 2) return of(std::integral_constant<int, 2>{});
  if constexpr (MOST > 4)
    if (items == 8) return of(std::integral_constant<int, 8>{});
  return of(std::integral_constant<int, 4>{});
}

template <typename T, int KIND>
int launch_fwd(const RmsArgs& a, const RmsPlan& pl) {
  auto go = [&](auto vec, auto items) {
    if constexpr (vec() > 1 && vec() * items() <= 16)  // (16384 channels are 16 to each of 1024 lanes)
      if (pl.lanes > RMS_LANES) return launch_kernel(rms_fwd_kernel<T, vec(), items(), KIND, RMS_WIDE>, pl.blocks, 1, pl.lanes, a.p.stream, a);
    return launch_kernel(rms_fwd_kernel<T, vec(), items(), KIND, RMS_LANES>, pl.blocks, 1, RMS_LANES, a.p.stream, a);
  };
  if (pl.vec == 1) return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});  // (fewer channels than a lane holds)
  return with_items<16 / int(sizeof(T)), 8>(pl.items, go);
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

int64_t linrec_rms_norm_partial_floats(int dtype, int64_t rows, int64_t channels) {
  if (rows <= 0 || channels <= 0) return 0;
  const int64_t n = plan_rms(dtype, rows, channels, true).blocks, chunks = column_sum_chunks(n);
  return (n + (chunks > 1 ? chunks : 0)) * channels;
}

int linrec_rms_norm_fwd(const linrec_rms_norm_t* p) {
  if (const int rc = check_rms(p)) return rc;
  if (p->rows == 0) return LINREC_OK;
  if (!p->y || (p->residual && !p->total) || (p->quantized != LINREC_QUANTIZED_NONE && !p->scales)) return LINREC_E_INVALID;
  const RmsPlan pl = plan_rms(p->dtype, p->rows, p->channels, false);
  const RmsArgs a{*p, pl.team, pl.blocks};
  return with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    if (p->quantized == LINREC_QUANTIZED_INT8) return launch_fwd<T, LINREC_QUANTIZED_INT8>(a, pl);
    if (p->quantized == LINREC_QUANTIZED_E4M3) return launch_fwd<T, LINREC_QUANTIZED_E4M3>(a, pl);
    return launch_fwd<T, LINREC_QUANTIZED_NONE>(a, pl);
  });
}

int linrec_rms_norm_bwd(const linrec_rms_norm_t* p) {
  if (const int rc = check_rms(p)) return rc;
  if (p->rows > 0 && (!p->d_y || !p->d_x || !p->rstd)) return LINREC_E_INVALID;
  if (p->d_weight && (!p->weight || (p->rows > 0 && !p->partial))) return LINREC_E_INVALID;
  RmsPlan pl{};
  if (p->rows > 0) {
    pl = plan_rms(p->dtype, p->rows, p->channels, true);
    RmsArgs a{*p, pl.team, pl.blocks};
    if (!p->d_weight) a.p.partial = nullptr;
    const int rc = with_dtype(p->dtype, [&](auto t) {
      using T = decltype(t);
      auto go = [&](auto vec, auto items) {
        if constexpr (vec() > 1 && vec() * items() <= 16)
          if (pl.lanes > RMS_LANES) return launch_kernel(rms_bwd_kernel<T, vec(), items(), RMS_WIDE>, pl.blocks, 1, pl.lanes, p->stream, a);
        return launch_kernel(rms_bwd_kernel<T, vec(), items(), RMS_LANES>, pl.blocks, 1, RMS_LANES, p->stream, a);
      };
      if (pl.vec == 1) return go(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
      return with_items<16 / int(sizeof(T)), 4>(pl.items, go);
    });
    if (rc) return rc;
  }
  if (!p->d_weight) return LINREC_OK;
  int64_t rows = pl.blocks;
  const int64_t columns = cdiv(p->channels, 64), chunks = column_sum_chunks(rows);
  const float* sums = p->partial;
  if (chunks > 1) {
    float* out = p->partial + rows * p->channels;
    if (const int rc = launch_kernel(rms_sum_kernel, columns, chunks, 64 * SUM_WAVES, p->stream, sums, rows, p->channels, SUM_ROWS, out)) return rc;
    sums = out;
    rows = chunks;
  }
  return launch_kernel(rms_weight_gradient_kernel, columns, 1, 64 * SUM_WAVES, p->stream, sums, rows, p->channels, p->weight_dtype, p->d_weight);
}

}  // extern "C"
