// Group norm with an activation, channels last, forward and backward.
//
//   xh = (x - mean) rstd,  z = xh w + b,  y = act(z)
//   e = d_y act'(z),  d_x = rstd (e w - s1 - xh s2),  s1 = sum e w / M,  s2 = sum e w xh / M  over the M values of a group,
//   d_b = sum e,  d_w = sum e xh  over all rows
//
// What bounds it: memory, and the launches where little is normed.  Forward and backward: 32768 x 1024 in 16 groups, bf16, 31 and
// 49 us (134 and 201 MB: 4.4 and 4.1 TB/s of the 5.2 that a copy reaches), fp32 52 and 76 (5.1 and 5.3); 16 x 2048 x 512 in 32 groups,
// fp32, gelu 38 and 62 us (3.5 and 3.3 TB/s): one round of workgroups that all load, then add up, then store; 8 x 16384 x 512 in 32
// groups, bf16, in chunks 96 and 157 us, for three and five tensors' worth of memory traffic.  3 x 333 x 222 in 6 groups: 12 us, of
// which an empty kernel takes 6.  Three shapes, by how much one group is:
//   tokens  one position: a team of 1 .. 64 adjacent lanes holds a group in registers; waves keep their channels and walk down
//           the rows, so weights are read once and the sums of d_w and d_b stay in registers.
//   held    a workgroup holds all positions of one or more groups (and batch items) in registers: every value is read once.
//   chunks  larger groups: partial statistics of chunks of positions, and a second launch that puts them together and reads
//           the values again.
//
// Statistics: tokens and held take the mean first and the squares of the differences then.  Chunks cannot; a lane goes through
// its values in runs of batches of four slots, none longer than all before it, and sums differences to one value, d and d^2: to the mean of
// its first batch in the first run of 8, to the mean of all that it has had in the others.  What cancels in M2 = sum d^2 - (sum d)^2 / n
// is then at most seven times the M2 of the values so far: a run's mean is D off the value it is taken to, where n D^2 cancels, only if
// the values before and in it spread by at least n D^2 / 7, whatever the mean and wherever a value lies far from the others.  (Differences to a
// lane's first value cancel n times M2 where that is the one far off; they cost 2 % less in groups that idle lanes leave to latency.)  Runs,
// lanes and chunks are merged as (count, mean, M2) (T. F. Chan, G. H. Golub, R. J. LeVeque, "Updating formulae and a pairwise algorithm for
// computing sample variances", 1979).  All sums are trees whose shape depends on the sizes alone: the same bits in every run.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/linrec_layers.h"
#include "collook_kernel.hpp"  // Held, ld_any, st_any, widen
#include "column_sum.hpp"

namespace linrec {

// ---- activation -------------------------------------------------------------------------------
// erfc(|v|) / exp(-v^2) as a polynomial in t = 1 / (1 + p |v|): M. Abramowitz, I. A. Stegun, "Handbook of Mathematical
// Functions", 7.1.26, at most 1.5e-7 off in erf.
__device__ __forceinline__ float erfc_scaled(float abs_v) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, abs_v, 1.0f));
  return t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
}
__device__ __forceinline__ float norm_exp(float v) { return __builtin_amdgcn_exp2f(1.4426950408889634f * v); }

template <int N>
__device__ __forceinline__ void activate(int act, float (&z)[N]) {
  switch (act) {  // (the same for all lanes)
    case LINREC_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = z[i] < 0.0f ? 0.0f : z[i];  // (NaN stays)
      break;
    case LINREC_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] *= __builtin_amdgcn_rcpf(1.0f + norm_exp(-z[i]));
      break;
    case LINREC_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float half = 0.5f * erfc_scaled(0.70710678118654752f * fabsf(z[i])) * norm_exp(-0.5f * z[i] * z[i]);
        z[i] *= z[i] > 0.0f ? 1.0f - half : half;
      }
      break;
    default: break;
  }
}
// e[i] *= act'(z[i])
template <int N>
__device__ __forceinline__ void activate_slope(int act, const float (&z)[N], float (&e)[N]) {
  switch (act) {
    case LINREC_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = z[i] > 0.0f ? e[i] : (z[i] != z[i] ? z[i] : 0.0f) * e[i];  // (NaN stays, not what -inf hides)
      break;
    case LINREC_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float s = __builtin_amdgcn_rcpf(1.0f + norm_exp(-z[i]));
        e[i] *= s * fmaf(z[i], 1.0f - s, 1.0f);
      }
      break;
    case LINREC_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float g = norm_exp(-0.5f * z[i] * z[i]);
        const float half = 0.5f * erfc_scaled(0.70710678118654752f * fabsf(z[i])) * g;
        e[i] *= fmaf(z[i], 0.39894228040143268f * g, z[i] > 0.0f ? 1.0f - half : half);
      }
      break;
    default: break;
  }
}

template <int VEC, typename T>
__device__ __forceinline__ void widen_params(const void* p, int64_t c, float (&out)[VEC]) {
  const Lanes<VEC> v = widen(ld_any<VEC, false>(static_cast<const T*>(p) + c));
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[e] = v.v[e];
}
template <int VEC>
__device__ __forceinline__ void load_params(const void* p, int dtype, int64_t c, float none, float (&out)[VEC]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = none;
  } else if (dtype == LINREC_DTYPE_F32) {
    widen_params<VEC, float>(p, c, out);
  } else if (dtype == LINREC_DTYPE_F16) {
    widen_params<VEC, _Float16>(p, c, out);
  } else {
    widen_params<VEC, __bf16>(p, c, out);
  }
}

// ---- sums over the lanes of a team ------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// Sum over teams of `lanes` (a power of two) adjacent lanes, in all of them.
__device__ __forceinline__ float team_sum(float v, int lanes) {
  if (lanes > 1) v = dpp_add<0xb1>(v);   // quad_perm 1 0 3 2
  if (lanes > 2) v = dpp_add<0x4e>(v);   // quad_perm 2 3 0 1
  if (lanes > 4) v = dpp_add<0x141>(v);  // row_half_mirror: the other quad of eight
  if (lanes > 8) v = dpp_add<0x140>(v);  // row_mirror: the other eight of a row
  if (lanes > 16) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
  }
  if (lanes > 32) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
  }
  return v;
}

// ---- tokens: one position ---------------------------------------------------------------------
constexpr int TOKEN_WAVES = 8;
struct TokenArgs {
  linrec_group_norm_t p;
  int team;          // lanes of a group: a power of two up to 64, or whole waves side by side
  int column_waves;  // waves of a workgroup side by side over the channels (a power of two), the others take other rows
  int column_blocks;
  int row_blocks;
};

// Sums over a team; one of several waves goes through LDS (`turn` alternates, so that one barrier a sum is enough).
template <int N>
__device__ __forceinline__ void team_sums(float (&v)[N], int team, float (*sh)[TOKEN_WAVES][N], int& turn, int wave) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = team_sum(v[i], team);
  if (team > 64) {
    float(*mine)[N] = sh[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) mine[wave][i] = v[i];
    }
    __syncthreads();
    const int waves = team >> 6, first = wave & ~(waves - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
      for (int w = 0; w < waves; ++w) v[i] += mine[first + w][i];
    }
  }
}

template <typename T, int VEC, int ITEMS, bool BWD>
__global__ __launch_bounds__(64 * TOKEN_WAVES) void norm_tokens_kernel(TokenArgs args) {
  constexpr int N = VEC * ITEMS;
  __shared__ float sh_team[2][TOKEN_WAVES][BWD ? 2 : 1];
  const linrec_group_norm_t& p = args.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int block = int(blockIdx.x % unsigned(args.column_blocks)), row_block = int(blockIdx.x / unsigned(args.column_blocks));
  const int cw = wave & (args.column_waves - 1), row_slot = wave / args.column_waves, row_slots = TOKEN_WAVES / args.column_waves;
  const int width = int(p.channels / p.groups);
  const int64_t column = (int64_t(block) * args.column_waves + cw) * 64 + lane;  // lane of the row
  const int64_t g = column / args.team;
  const int in_team = int(column - g * args.team);
  const bool there = g < p.groups;
  const int64_t c0 = (there ? g : 0) * width;
  bool has[ITEMS];
  int64_t c[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int o = (i * args.team + in_team) * VEC;  // (VEC divides the width: a slot lies in the group or not)
    has[i] = there && o < width;
    c[i] = c0 + (has[i] ? o : 0);
  }
  const int64_t step = int64_t(args.row_blocks) * row_slots;
  const float inv_count = 1.0f / float(width);
  const T* x = static_cast<const T*>(p.x);
  const T* dy = static_cast<const T*>(p.d_y);
  Held<T, VEC> hx[ITEMS], hd[BWD ? ITEMS : 1];
  float mean = 0.0f, rstd = 0.0f;
  auto load = [&](int64_t n) __attribute__((always_inline)) {
    if (n >= p.batch) n = p.batch - 1;  // (read and not used)
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      hx[i] = ld_any<VEC, true>(x + n * p.x_stride[0] + c[i]);
      if constexpr (BWD) hd[i] = ld_any<VEC, true>(dy + n * p.d_y_stride[0] + c[i]);
    }
    if constexpr (BWD) {
      mean = p.mean[n * p.groups + (there ? g : 0)];
      rstd = p.rstd[n * p.groups + (there ? g : 0)];
    }
  };
  int64_t base = int64_t(row_block) * row_slots;  // the same for all waves: they meet at barriers
  load(base + row_slot);
  float w[N], b[N];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    float wi[VEC], bi[VEC];
    load_params<VEC>(p.weight, p.weight_dtype, c[i], 1.0f, wi);
    load_params<VEC>(p.bias, p.weight_dtype, c[i], 0.0f, bi);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      w[i * VEC + e] = wi[e];
      b[i * VEC + e] = bi[e];
    }
  }
  float dw[BWD ? N : 1], db[BWD ? N : 1];
#pragma unroll
  for (int i = 0; i < (BWD ? N : 1); ++i) dw[i] = db[i] = 0.0f;

  int turn = 0;
  for (; base < p.batch; base += step) {
    const int64_t n = base + row_slot;
    const bool row = n < p.batch;
    float v[N], d[BWD ? N : 1];
    float m = mean, r = rstd;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const Lanes<VEC> t = widen(hx[i]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = t.v[e];
      if constexpr (BWD) {
        const Lanes<VEC> u = widen(hd[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) d[i * VEC + e] = u.v[e];
      }
    }
    load(n + step);  // (under way while this row is worked on; two rows ahead gained nothing)
    if constexpr (!BWD) {
      float s[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < N; ++i) s[0] += has[i / VEC] ? v[i] : 0.0f;
      team_sums<1>(s, args.team, sh_team, turn, wave);
      m = s[0] * inv_count;
      s[0] = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] -= m;
        s[0] = fmaf(has[i / VEC] ? v[i] : 0.0f, v[i], s[0]);
      }
      team_sums<1>(s, args.team, sh_team, turn, wave);
      r = __builtin_amdgcn_rsqf(fmaf(s[0], inv_count, p.eps));
      if (row && there && in_team == 0) {
        p.mean[n * p.groups + g] = m;
        p.rstd[n * p.groups + g] = r;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = fmaf(v[i] * r, w[i], b[i]);
      activate<N>(p.act, v);
    } else {
      float z[N], s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] = (v[i] - m) * r;
        z[i] = fmaf(v[i], w[i], b[i]);
      }
      activate_slope<N>(p.act, z, d);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!(has[i / VEC] && row)) d[i] = v[i] = 0.0f;
        dw[i] = fmaf(d[i], v[i], dw[i]);
        db[i] += d[i];
        d[i] *= w[i];
        s[0] += d[i];
        s[1] = fmaf(d[i], v[i], s[1]);
      }
      team_sums<2>(s, args.team, sh_team, turn, wave);
      const float s1 = s[0] * inv_count, s2 = s[1] * inv_count;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = r * (d[i] - fmaf(v[i], s2, s1));
    }
    T* out = static_cast<T*>(BWD ? p.d_x : p.y) + n * p.channels;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      Lanes<VEC> t;
#pragma unroll
      for (int e = 0; e < VEC; ++e) t.v[e] = v[i * VEC + e];
      if (has[i] && row) st_any<VEC>(out + c[i], t);
    }
  }
  if constexpr (BWD) {
    if (!p.weight) return;
    // the waves that had the same channels
    __shared__ float sh[TOKEN_WAVES][64];
    float* to = p.partial + int64_t(row_block) * 2 * p.channels;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
        sh[wave][lane] = which ? dw[i] : db[i];
        __syncthreads();
        if (row_slot == 0 && has[i / VEC]) {
          float s = sh[cw][lane];
          for (int q = 1; q < row_slots; ++q) s += sh[q * args.column_waves + cw][lane];
          to[which * p.channels + c[i / VEC] + i % VEC] = s;
        }
      }
    }
  }
}

// ---- held and chunks: the lanes of a workgroup over (row, batch item, column) --------------------
// A column is a slot of VEC channels; a group is `per_group` columns.  A workgroup has `groups` whole groups of `items` batch
// items side by side (or one of `parts` parts of one group's columns) and R rows of positions at a time.
struct BlockArgs {
  linrec_group_norm_t p;
  int per_group;   // columns of a group (of a part of it)
  int groups;      // of a workgroup
  int items;       // batch items of a workgroup
  int parts;       // workgroups that share a group's columns
  int blocks;      // workgroups over the channels
  int chunks;      // workgroups over the positions
  int rows;        // positions of a chunk
  int columns;     // items * groups * per_group: lanes of a row
  int R;           // rows at a time
  int whole;       // columns of a whole group
};

struct BlockLane {
  int vc, r, q, g;  // column and row; column in its group; group of the workgroup (over all its items)
  int64_t n, group, channel, first, end;  // batch item, group, first channel; positions of the chunk
  bool there;
};
// Workgroups are dealt to the eight XCDs in turn; numbered so that neighbours run on one of them, groups narrower than a
// 128-byte line share its lines in one L2.
__device__ __forceinline__ unsigned block_number() {
  const unsigned xcd = blockIdx.x & 7u, whole = gridDim.x >> 3, rest = gridDim.x & 7u;
  return xcd * whole + (xcd < rest ? xcd : rest) + (blockIdx.x >> 3);
}
template <int VEC>
__device__ __forceinline__ BlockLane block_lane(const BlockArgs& a) {
  BlockLane l;
  const int tid = int(threadIdx.x);
  unsigned id = block_number();
  const int chunk = int(id % unsigned(a.chunks));
  id /= unsigned(a.chunks);
  const int block = int(id % unsigned(a.blocks));
  const int64_t item_block = id / unsigned(a.blocks);
  l.r = tid / a.columns;
  l.vc = tid - l.r * a.columns;
  l.g = l.vc / a.per_group;
  l.q = l.vc - l.g * a.per_group;
  const int item = l.g / a.groups, g = l.g - item * a.groups;
  const int part = block % a.parts;
  l.n = item_block * a.items + item;
  l.group = int64_t(block / a.parts) * a.groups + g;
  const int column = part * a.per_group + l.q;
  l.channel = (l.group * a.whole + column) * VEC;
  l.there = l.r < a.R && l.n < a.p.batch && l.group < a.p.groups && column < a.whole;
  l.first = int64_t(chunk) * a.rows + l.r;
  l.end = int64_t(chunk + 1) * a.rows;
  if (l.end > a.p.positions) l.end = a.p.positions;
  return l;
}

// Columns that are a power of two up to a wave: sums go over the lanes of a wave first.
__device__ __forceinline__ bool columns_in_wave(const BlockArgs& a) { return (a.columns & (a.columns - 1)) == 0 && a.columns <= 64; }
// Sum over the lanes of a wave that are a multiple of `columns` apart (a power of two), in all of them.
__device__ __forceinline__ float same_column_sum(float v, int columns) {
  if (columns < 2) v = dpp_add<0x121>(v);   // row_ror:1
  if (columns < 4) v = dpp_add<0x122>(v);   // row_ror:2
  if (columns < 8) v = dpp_add<0x124>(v);   // row_ror:4
  if (columns < 16) v = dpp_add<0x128>(v);  // row_ror:8
  if (columns < 32) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
  }
  if (columns < 64) {
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v = __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
  }
  return v;
}
// Sums over the rows: v of row 0 (of all rows if columns_in_wave) becomes the sum of its column.  sh: N * blockDim floats.
template <int N>
__device__ __forceinline__ void sum_rows(float (&v)[N], float* sh, const BlockArgs& a, const BlockLane& l) {
  const int lanes = int(blockDim.x), tid = int(threadIdx.x);
  if (a.R == 1) return;
  if (columns_in_wave(a)) {
    const int lane = tid & 63, wave = tid >> 6, waves = lanes >> 6, total = a.columns * N;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = same_column_sum(v[i], a.columns);
    __syncthreads();
    if (lane < a.columns) {
#pragma unroll
      for (int i = 0; i < N; ++i) sh[wave * total + i * a.columns + lane] = v[i];
    }
    for (int j = tid; j - tid < total; j += lanes) {
      __syncthreads();
      float t = 0.0f;
      if (j < total) {
        t = sh[j];
        for (int w = 1; w < waves; ++w) t += sh[w * total + j];
      }
      if (j < total) sh[j] = t;  // (no other lane reads it)
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sh[i * a.columns + l.vc];
    return;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) sh[i * lanes + tid] = v[i];
  int s = 1;
  while (s < a.R) s <<= 1;
  for (s >>= 1; s > 0; s >>= 1) {
    __syncthreads();
    if (l.r < s && l.r + s < a.R) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] += sh[i * lanes + tid + s * a.columns];
        sh[i * lanes + tid] = v[i];
      }
    }
  }
}
// Sums over the columns of a group among the lanes of row 0; every lane gets its group's sum.
template <int N>
__device__ __forceinline__ void sum_group(float (&v)[N], float* sh, const BlockArgs& a, const BlockLane& l) {
  const int lanes = int(blockDim.x), tid = int(threadIdx.x);
  if (columns_in_wave(a) && (a.per_group & (a.per_group - 1)) == 0) {  // (every row has the columns' sums)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = team_sum(v[i], a.per_group);
    return;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) sh[i * lanes + tid] = v[i];
  for (int s = 1; s < a.per_group; s <<= 1) {
    __syncthreads();
    if (l.r == 0 && (l.q & (2 * s - 1)) == 0 && l.q + s < a.per_group) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        v[i] += sh[i * lanes + tid + s];
        sh[i * lanes + tid] = v[i];
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = sh[i * lanes + l.g * a.per_group];
}

// Sums over all rows and columns of a group, in all its lanes.  sh: N * blockDim floats.
template <int N>
__device__ __forceinline__ void sum_all(float (&v)[N], float* sh, const BlockArgs& a, const BlockLane& l) {
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6, waves = int(blockDim.x) >> 6;
  if (columns_in_wave(a)) {  // (so is the width of a group a power of two)
    // every wave has all groups
    const int groups = a.columns / a.per_group, total = groups * N;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = team_sum(same_column_sum(v[i], a.columns), a.per_group);
    __syncthreads();
    if (lane < a.columns && l.q == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) sh[wave * total + i * groups + l.g] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
      for (int w = 0; w < waves; ++w) v[i] += sh[w * total + i * groups + l.g];
    }
  } else if (a.columns == a.per_group) {
    // all waves have the one group
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = team_sum(v[i], 64);
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) sh[i * waves + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
      for (int w = 0; w < waves; ++w) v[i] += sh[i * waves + w];
    }
  } else if ((a.per_group & 63) == 0) {
    // a wave has one group
    const int per_row = a.columns >> 6, per_group = a.per_group >> 6, first = l.g * per_group;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = team_sum(v[i], 64);
    __syncthreads();
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) sh[i * waves + wave] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
      for (int r = 0; r < a.R; ++r)
        for (int w = 0; w < per_group; ++w) v[i] += sh[i * waves + r * per_row + first + w];
    }
  } else {
    sum_rows<N>(v, sh, a, l);
    sum_group<N>(v, sh, a, l);
  }
}

struct Moments {
  float count, mean, m2;
};
__device__ __forceinline__ Moments merge(Moments a, Moments b) {
  if (b.count == 0.0f) return a;
  if (a.count == 0.0f) return b;
  const float n = a.count + b.count, f = b.count / n, d = b.mean - a.mean;
  return {n, fmaf(d, f, a.mean), fmaf(d * d, a.count * f, a.m2 + b.m2)};
}
// The moments of all lanes of a group, in all of them.  sh: 3 * blockDim floats.
__device__ __forceinline__ Moments merge_group(Moments v, float* sh, const BlockArgs& a, const BlockLane& l) {
  const int lanes = int(blockDim.x), tid = int(threadIdx.x);
  auto put = [&](const Moments& m) {
    sh[tid] = m.count;
    sh[lanes + tid] = m.mean;
    sh[2 * lanes + tid] = m.m2;
  };
  auto get = [&](int i) { return Moments{sh[i], sh[lanes + i], sh[2 * lanes + i]}; };
  __syncthreads();
  put(v);
  int s = 1;
  while (s < a.R) s <<= 1;
  for (s >>= 1; s > 0; s >>= 1) {
    __syncthreads();
    if (l.r < s && l.r + s < a.R) put(v = merge(v, get(tid + s * a.columns)));
  }
  for (s = 1; s < a.per_group; s <<= 1) {
    __syncthreads();
    if (l.r == 0 && (l.q & (2 * s - 1)) == 0 && l.q + s < a.per_group) put(v = merge(v, get(tid + s)));
  }
  __syncthreads();
  return get(l.g * a.per_group);
}

// The number of this workgroup's part of its groups' statistics, and where it lies.
__device__ __forceinline__ int64_t piece_of(const BlockArgs& a) {
  const unsigned id = block_number(), chunk = id % unsigned(a.chunks), block = id / unsigned(a.chunks) % unsigned(a.blocks);
  return int64_t(chunk) * a.parts + block % unsigned(a.parts);
}
__device__ __forceinline__ int64_t piece_index(const BlockArgs& a, int64_t n, int64_t group, int64_t piece) {
  return ((n * a.chunks * a.parts + piece) * a.p.groups + group) * 2;
}

// NORM_HELD_PARTS: the workgroup's rows are fp32 and not whole lines of 128 bytes.  Its results go through the caches, where the parts
// of a line that neighbours write come together, all others past them: 16 x 2048 x 512 in 32 groups fp32 38 and 62 us, past the caches 40
// and 66; whole lines, 512 x 64 x 256 in 8 groups bf16, 11 and 27 us past them and 14 and 29 through them; parts of 16 bits gain nothing,
// 16 x 2048 x 510 in 30 groups bf16 39 and 52 us through them and 38 and 52 past them (an odd width, one channel of 2 bytes to a lane: that
// is what bounds it), 32 x 1024 x 256 in 32 groups 15 and 27, 13 and 27.
constexpr int NORM_HELD = 0, NORM_STATS = 1, NORM_APPLY = 2, NORM_HELD_PARTS = 3;
constexpr bool holds(int phase) { return phase == NORM_HELD || phase == NORM_HELD_PARTS; }
template <int PHASE, int VEC, typename T>
__device__ __forceinline__ void store_result(T* to, const Lanes<VEC>& v) {
  if constexpr (PHASE != NORM_HELD_PARTS) {
    st_any<VEC>(to, v);
  } else if constexpr (VEC == 1) {
    *to = T(v.v[0]);
  } else {
    using A = typename AnyPack<T, VEC>::type;
    A q;
#pragma unroll
    for (int e = 0; e < VEC; ++e) q[e] = T(v.v[e]);
    *reinterpret_cast<A*>(to) = q;
  }
}
// Batches of four slots between two merges of a lane's statistics: of the first two runs, and of the longest (all runs of 8: 1 x 131072 x 516
// fp32 in one group, 128 batches to a lane, 354 us instead of 335).
constexpr int STATS_RUN = 8, STATS_RUN_MOST = 32;
template <int VEC, typename T>
constexpr int held_rows(bool two) {  // of a lane: 32 registers' worth, 24 of each of two 16-bit tensors (what they widen to needs more)
  return (two && sizeof(T) == 2 ? 24 : 32) / (VEC * int(sizeof(T)) >= 4 ? VEC * int(sizeof(T)) / 4 : 1);
}

template <typename T, int VEC, int LANES, int PHASE>
__global__ __launch_bounds__(LANES) void norm_fwd_kernel(BlockArgs args) {
  constexpr int KEEP = held_rows<VEC, T>(false);
  __shared__ float sh[(holds(PHASE) ? 1 : 3) * LANES];
  const linrec_group_norm_t& p = args.p;
  const BlockLane l = block_lane<VEC>(args);
  const T* x = static_cast<const T*>(p.x) + l.n * p.x_stride[0] + l.channel;
  T* y = static_cast<T*>(p.y) + l.n * p.positions * p.channels + l.channel;
  float w[VEC], b[VEC];
  auto params = [&]() __attribute__((always_inline)) {
    if (l.there) {
      load_params<VEC>(p.weight, p.weight_dtype, l.channel, 1.0f, w);
      load_params<VEC>(p.bias, p.weight_dtype, l.channel, 0.0f, b);
    }
  };
  float mean, rstd;
  auto apply = [&](const Held<T, VEC>& h, int64_t pos) __attribute__((always_inline)) {
    Lanes<VEC> v = widen(h);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v.v[e] = fmaf((v.v[e] - mean) * rstd, w[e], b[e]);
    activate<VEC>(p.act, v.v);
    store_result<PHASE>(y + pos * p.channels, v);
  };
  const bool writes = l.there && l.r == 0 && l.q == 0 && (PHASE != NORM_APPLY || (l.first == 0 && l.channel == l.group * args.whole * VEC));

  if constexpr (holds(PHASE)) {
    Held<T, VEC> held[KEEP];
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int64_t pos = l.first + i * args.R;
      if (l.there && pos < l.end) held[i] = ld_any<VEC, true>(x + pos * p.x_stride[1]);
    }
    params();
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (l.there && l.first + i * args.R < l.end) {
        const Lanes<VEC> v = widen(held[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[0] += v.v[e];
      }
    const float inv_count = 1.0f / (float(p.positions) * float(args.whole * VEC));
    sum_all<1>(s, sh, args, l);
    mean = s[0] * inv_count;
    s[0] = 0.0f;
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (l.there && l.first + i * args.R < l.end) {
        const Lanes<VEC> v = widen(held_again(held[i]));
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = v.v[e] - mean;
          s[0] = fmaf(d, d, s[0]);
        }
      }
    sum_all<1>(s, sh, args, l);
    rstd = __builtin_amdgcn_rsqf(fmaf(s[0], inv_count, p.eps));
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (l.there && l.first + i * args.R < l.end) apply(held_again(held[i]), l.first + i * args.R);
  } else if constexpr (PHASE == NORM_STATS) {
    Moments m{0.0f, 0.0f, 0.0f};
    if (l.there) {
      int run = STATS_RUN;
      for (int64_t pos = l.first; pos < l.end;) {
        float shift = m.mean, s = 0.0f, s2 = 0.0f, count = 0.0f;
        for (int n = 0; n < run && pos < l.end; ++n, pos += 4 * args.R) {
          Held<T, VEC> h[4];
          float t = 0.0f, t2 = 0.0f, more = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pos + i * args.R < l.end) {
              h[i] = ld_any<VEC, false>(x + (pos + i * args.R) * p.x_stride[1]);
              more += float(VEC);
            }
          if (m.count == 0.0f && n == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (pos + i * args.R < l.end) {
                const Lanes<VEC> v = widen(h[i]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) shift += v.v[e];
              }
            shift /= more;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pos + i * args.R < l.end) {
              const Lanes<VEC> v = widen(h[i]);
#pragma unroll
              for (int e = 0; e < VEC; ++e) {
                const float d = v.v[e] - shift;
                t += d;
                t2 = fmaf(d, d, t2);
              }
            }
          s += t;
          s2 += t2;
          count += more;
        }
        if (m.count != 0.0f && run < STATS_RUN_MOST) run *= 2;
        const float off = s / count, m2 = fmaf(-off, s, s2);
        m = merge(m, {count, shift + off, m2 < 0.0f ? 0.0f : m2});  // (NaN stays)
      }
    }
    m = merge_group(m, sh, args, l);
    if (writes) {
      const int64_t piece = piece_of(args);
      float* out = p.partial + piece_index(args, l.n, l.group, piece);
      out[0] = m.mean;
      out[1] = m.m2;
    }
    return;
  } else {
    params();
    // the lanes of a group share its pieces out
    Moments m{0.0f, 0.0f, 0.0f};
    const int pieces = args.chunks * args.parts;
    if (l.there) {
      for (int i = l.r * args.per_group + l.q; i < pieces; i += args.R * args.per_group) {
        const int chunk = i / args.parts, part = i - chunk * args.parts;
        const int64_t first = int64_t(chunk) * args.rows, rows = first + args.rows < p.positions ? args.rows : p.positions - first;
        const int columns = (part + 1) * args.per_group < args.whole ? args.per_group : args.whole - part * args.per_group;
        const float* in = p.partial + piece_index(args, l.n, l.group, i);
        m = merge(m, {float(rows) * float(columns * VEC), in[0], in[1]});
      }
    }
    m = merge_group(m, sh, args, l);
    mean = m.mean;
    rstd = __builtin_amdgcn_rsqf(m.m2 / m.count + p.eps);
    if (l.there)
      for (int64_t pos = l.first; pos < l.end; pos += 4 * args.R) {
        Held<T, VEC> h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (pos + i * args.R < l.end) h[i] = ld_any<VEC, false>(x + (pos + i * args.R) * p.x_stride[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (pos + i * args.R < l.end) apply(h[i], pos + i * args.R);
      }
  }
  if (writes) {
    p.mean[l.n * p.groups + l.group] = mean;
    p.rstd[l.n * p.groups + l.group] = rstd;
  }
}

// PARTIAL layout of the backward: the pieces' sums (chunks only), then a row of 2 * channels sums for every (item block, chunk).
template <typename T, int VEC, int LANES, int PHASE>
__global__ __launch_bounds__(LANES) void norm_bwd_kernel(BlockArgs args, float* param_sums) {
  constexpr int KEEP = held_rows<VEC, T>(true);
  __shared__ float sh[(PHASE == NORM_APPLY ? 2 : 2 * VEC) * LANES];
  const linrec_group_norm_t& p = args.p;
  const BlockLane l = block_lane<VEC>(args);
  const T* x = static_cast<const T*>(p.x) + l.n * p.x_stride[0] + l.channel;
  const T* dy = static_cast<const T*>(p.d_y) + l.n * p.d_y_stride[0] + l.channel;
  T* dx = static_cast<T*>(p.d_x) + l.n * p.positions * p.channels + l.channel;
  float w[VEC], b[VEC];
  float mean = 0.0f, rstd = 0.0f;
  if (l.there) {
    load_params<VEC>(p.weight, p.weight_dtype, l.channel, 1.0f, w);
    load_params<VEC>(p.bias, p.weight_dtype, l.channel, 0.0f, b);
    mean = p.mean[l.n * p.groups + l.group];
    rstd = p.rstd[l.n * p.groups + l.group];
  }
  // xh and e of one slot
  auto expand = [&](const Held<T, VEC>& hx, const Held<T, VEC>& hd, float (&xh)[VEC], float (&e)[VEC]) __attribute__((always_inline)) {
    const Lanes<VEC> vx = widen(hx), vd = widen(hd);
    float z[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      xh[i] = (vx.v[i] - mean) * rstd;
      z[i] = fmaf(xh[i], w[i], b[i]);
      e[i] = vd.v[i];
    }
    activate_slope<VEC>(p.act, z, e);
  };
  float sums[2 * VEC], s[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 2 * VEC; ++i) sums[i] = 0.0f;
  auto add = [&](const Held<T, VEC>& hx, const Held<T, VEC>& hd) __attribute__((always_inline)) {
    float xh[VEC], e[VEC];
    expand(hx, hd, xh, e);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      sums[i] += e[i];
      sums[VEC + i] = fmaf(e[i], xh[i], sums[VEC + i]);
    }
  };
  auto apply = [&](const Held<T, VEC>& hx, const Held<T, VEC>& hd, int64_t pos) __attribute__((always_inline)) {
    float xh[VEC], e[VEC];
    expand(hx, hd, xh, e);
    Lanes<VEC> out;
#pragma unroll
    for (int i = 0; i < VEC; ++i) out.v[i] = rstd * (fmaf(e[i], w[i], -s[0]) - xh[i] * s[1]);
    store_result<PHASE>(dx + pos * p.channels, out);
  };
  // the columns' sums, from there those of d_weight and d_bias and the group's
  auto finish_sums = [&]() __attribute__((always_inline)) {
    sum_rows<2 * VEC>(sums, sh, args, l);
    if (l.there && (l.r == 0 || columns_in_wave(args))) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        s[0] = fmaf(sums[i], w[i], s[0]);
        s[1] = fmaf(sums[VEC + i], w[i], s[1]);
      }
    }
    if (p.weight) {
      __syncthreads();
      if (l.r == 0) {
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) sh[i * LANES + l.vc] = l.there ? sums[i] : 0.0f;
      }
      __syncthreads();
      const int width = args.groups * args.per_group;
      if (l.there && l.r == 0 && l.vc < width) {  // (the lanes of the first batch item)
#pragma unroll
        for (int i = 0; i < 2 * VEC; ++i) {
          float t = sh[i * LANES + l.vc];
          for (int q = 1; q < args.items; ++q) t += sh[i * LANES + q * width + l.vc];
          const unsigned id = block_number();
          const int64_t row = int64_t(id / unsigned(args.chunks) / unsigned(args.blocks)) * args.chunks + id % unsigned(args.chunks);
          param_sums[(row * 2 + i / VEC) * p.channels + l.channel + i % VEC] = t;
        }
      }
    }
    if (!columns_in_wave(args) && (args.columns == args.per_group || (args.per_group & 63) == 0))
      sum_all<2>(s, sh, args, l);  // (nothing in the rows but the first)
    else sum_group<2>(s, sh, args, l);
  };
  const float inv_count = 1.0f / (float(p.positions) * float(args.whole * VEC));

  if constexpr (holds(PHASE)) {
    Held<T, VEC> hx[KEEP], hd[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      const int64_t pos = l.first + i * args.R;
      if (l.there && pos < l.end) {
        hx[i] = ld_any<VEC, true>(x + pos * p.x_stride[1]);
        hd[i] = ld_any<VEC, true>(dy + pos * p.d_y_stride[1]);
      }
    }
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (l.there && l.first + i * args.R < l.end) add(hx[i], hd[i]);
    finish_sums();
    s[0] *= inv_count;
    s[1] *= inv_count;
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
      if (l.there && l.first + i * args.R < l.end) apply(held_again(hx[i]), held_again(hd[i]), l.first + i * args.R);
  } else {
    auto walk = [&](auto&& f, auto&& then) __attribute__((always_inline)) {
      if (!l.there) return;
      for (int64_t pos = l.first; pos < l.end; pos += 2 * args.R) {
        Held<T, VEC> hx[2], hd[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (pos + i * args.R < l.end) {
            hx[i] = ld_any<VEC, false>(x + (pos + i * args.R) * p.x_stride[1]);
            hd[i] = ld_any<VEC, false>(dy + (pos + i * args.R) * p.d_y_stride[1]);
          }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (pos + i * args.R < l.end) f(hx[i], hd[i], pos + i * args.R);
        then();
      }
    };
    if constexpr (PHASE == NORM_STATS) {
      // two levels: a sum that adds the same value again and again is off the same way at every step
      float before[2 * VEC];
      int n = 0;
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) before[i] = 0.0f;
      walk([&](const Held<T, VEC>& hx, const Held<T, VEC>& hd, int64_t) { add(hx, hd); },
           [&] {
             if (++n < 32) return;  // (of two positions)
#pragma unroll
             for (int i = 0; i < 2 * VEC; ++i) {
               before[i] += sums[i];
               sums[i] = 0.0f;
             }
             n = 0;
           });
#pragma unroll
      for (int i = 0; i < 2 * VEC; ++i) sums[i] += before[i];
      finish_sums();
      if (l.there && l.r == 0 && l.q == 0) {
        const int64_t piece = piece_of(args);
        float* out = p.partial + piece_index(args, l.n, l.group, piece);
        out[0] = s[0];
        out[1] = s[1];
      }
    } else {
      const int pieces = args.chunks * args.parts;
      if (l.there) {
        for (int i = l.r * args.per_group + l.q; i < pieces; i += args.R * args.per_group) {
          const float* in = p.partial + piece_index(args, l.n, l.group, i);
          s[0] += in[0];
          s[1] += in[1];
        }
      }
      sum_all<2>(s, sh, args, l);
      s[0] *= inv_count;
      s[1] *= inv_count;
      walk([&](const Held<T, VEC>& hx, const Held<T, VEC>& hd, int64_t pos) { apply(hx, hd, pos); }, [] {});
    }
  }
}

}  // namespace linrec
