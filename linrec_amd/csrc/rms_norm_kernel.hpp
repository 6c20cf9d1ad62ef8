// Root-mean-square norm of rows, with the residual's addition before it and an output in 8 bits after it.
//
//   s = x + residual (rounded to the storage type, which is what the next layer adds to),  y = s w / sqrt(mean s^2 + eps)
//
// and backwards, with h = s rstd, the gradient of x and of the residual is d_total + rstd (w dy - h mean(w dy h)), that of w the
// sum of dy h over the rows.  8 bits: a scale a row, the largest |y| over the largest value of the type, and y over the scale
// rounded to even.
//
// Memory is all there is to it: each row is read once and stays in the registers of a team of lanes, a power of two of them, up to
// 64 in a wave (several rows to a wave where they are short), above it the waves of a workgroup that meet at a barrier.  A
// lane's weights stay with it from row to row.  Sums are fp32, in an order that depends on sizes alone.
//
// Measured against what the bytes take at the rate of a large copy (5.1 TB/s): 32768 x 2048 bf16 with a residual 95 us (105) and back 102
// (105; some of it is still in the caches), 262144 x 64 fp32 31 (26) and 46 (39), 20011 x 4096 bf16 with a residual to 8 bits 117
// (112); 64 x 4096 5.3 us, the latency of three loads and two meetings of a workgroup.
#pragma once
#include "collook_kernel.hpp"
#include "column_sum.hpp"

namespace linrec {

constexpr int RMS_LANES = 256, RMS_WIDE = 1024;  // of a workgroup: whose teams are not wider, and the most of others, which have one team

struct RmsArgs {
  linrec_rms_norm_t p;
  int team;    // lanes of a row
  int blocks;  // workgroups
};

// Which of a row's values a lane has: VEC from c[i] on, of which the first skip[i] are another lane's (the last lane of a row starts
// early; it computes and stores the same values there).
template <int VEC, int ITEMS>
struct RmsLane {
  bool has[ITEMS];
  int c[ITEMS], skip[ITEMS];
  __device__ __forceinline__ RmsLane(int in_team, int team, int channels) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int o = (i * team + in_team) * VEC;
      has[i] = o < channels;
      c[i] = !has[i] ? 0 : o < channels - VEC ? o : channels - VEC;
      skip[i] = has[i] ? o - c[i] : VEC;
    }
  }
};

template <int N>
__device__ __forceinline__ void rms_weights(const void* weight, int dtype, int64_t c, float (&w)[N]) {
  auto of = [&](auto t) {
    const auto x = widen(ld_any<N, false>(static_cast<const decltype(t)*>(weight) + c));
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = x.v[e];
  };
  if (!weight) {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = 1.0f;
  } else if (dtype == LINREC_DTYPE_F32) {
    of(float());
  } else if (dtype == LINREC_DTYPE_F16) {
    of(_Float16());
  } else {
    of(__bf16());
  }
}

// Of all lanes of a team; `sh` has a place for every wave and is free again at the next barrier but one.
template <typename F>
__device__ __forceinline__ float over_team(float x, int team, float* sh, F&& join) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1)
    if (d < team) x = join(x, __shfl_xor(x, d));
  if (team > 64) {
    const int wave = threadIdx.x >> 6, waves = team >> 6, first = wave & ~(waves - 1);
    if ((threadIdx.x & 63) == 0) sh[wave] = x;
    __syncthreads();
    x = sh[first];
    for (int k = 1; k < waves; ++k) x = join(x, sh[first + k]);
  }
  return x;
}

__device__ __forceinline__ int64_t rms_row(const int64_t (&stride)[2], int64_t row, int64_t inner) {
  const int64_t outer = row / inner;
  return outer * stride[0] + (row - outer * inner) * stride[1];
}

// up: a power of two that keeps the reciprocal of a small scale finite, `inverse` that of scale * up (0 where the scale is 0).  (Scales
// that are subnormal are rounded, and values over them can be more than the type's largest.)
template <int KIND, int VEC>
__device__ __forceinline__ void store_quantized(void* y, int64_t at, const float (&v)[VEC], float up, float inverse) {
  typedef uint8_t any __attribute__((ext_vector_type(VEC), aligned(1)));
  any q;
  constexpr float MOST = KIND == LINREC_QUANTIZED_INT8 ? 127.0f : 448.0f;
  float t[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) t[e] = __builtin_amdgcn_fmed3f(v[e] * up * inverse, -MOST, MOST);
  if constexpr (KIND == LINREC_QUANTIZED_INT8) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) q[e] = uint8_t(int8_t(int(rintf(t[e]))));
  } else if constexpr (VEC % 4 == 0) {
    int words[VEC / 4];
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) {
      words[k] = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * k], t[4 * k + 1], 0, false);
      words[k] = __builtin_amdgcn_cvt_pk_fp8_f32(t[4 * k + 2], t[4 * k + 3], words[k], true);
    }
    __builtin_memcpy(&q, words, VEC);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) q[e] = uint8_t(__builtin_amdgcn_cvt_pk_fp8_f32(t[e], 0.0f, 0, false) & 0xff);
  }
  *reinterpret_cast<any*>(static_cast<uint8_t*>(y) + at) = q;
}

// KIND: LINREC_QUANTIZED_*
template <typename T, int VEC, int ITEMS, int KIND, int LANES>
__global__ __launch_bounds__(LANES) void rms_fwd_kernel(RmsArgs a) {
  __shared__ float sh[2][16];
  const linrec_rms_norm_t& p = a.p;
  const int channels = int(p.channels), rows_side = int(blockDim.x) / a.team;
  const int in_team = threadIdx.x & (a.team - 1), row_slot = threadIdx.x / a.team;
  const RmsLane<VEC, ITEMS> l(in_team, a.team, channels);
  float w[ITEMS][VEC];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) rms_weights<VEC>(p.weight, p.weight_dtype, l.c[i], w[i]);
  const T* x = static_cast<const T*>(p.x);
  const T* residual = static_cast<const T*>(p.residual);
  for (int64_t base = int64_t(blockIdx.x) * rows_side; base < p.rows; base += int64_t(a.blocks) * rows_side) {
    const bool there = base + row_slot < p.rows;
    const int64_t row = there ? base + row_slot : p.rows - 1;
    const T* from = x + rms_row(p.x_stride, row, p.inner);
    Held<T, VEC> hx[ITEMS], hr[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (l.has[i]) hx[i] = ld_any<VEC, true>(from + l.c[i]);
    if (residual) {
      const T* more = residual + rms_row(p.residual_stride, row, p.inner);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (l.has[i]) hr[i] = ld_any<VEC, true>(more + l.c[i]);
    }
    float v[ITEMS][VEC], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!l.has[i]) continue;
      Lanes<VEC> t = widen(hx[i]);
      if (residual) {
        const Lanes<VEC> u = widen(hr[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) t.v[e] = float(T(t.v[e] + u.v[e]));
        if (there) st_any<VEC>(static_cast<T*>(p.total) + row * p.channels + l.c[i], t);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        v[i][e] = t.v[e];
        if (e >= l.skip[i]) sum = fmaf(t.v[e], t.v[e], sum);
      }
    }
    sum = over_team(sum, a.team, sh[0], [](float f, float g) { return f + g; });
    const float rstd = 1.0f / sqrtf(sum / float(channels) + p.eps);
    if (p.rstd && there && in_team == 0) p.rstd[row] = rstd;
    float up = 1.0f, inverse = 0.0f;
    if constexpr (KIND != LINREC_QUANTIZED_NONE) {
      unsigned most = 0;  // as bits, whose order is that of the values, and a NaN is over them all
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (l.has[i])
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            v[i][e] = v[i][e] * rstd * w[i][e];
            const unsigned m = __float_as_uint(v[i][e]) & 0x7fffffffu;
            most = m > most ? m : most;
          }
      most = __float_as_uint(over_team(__uint_as_float(most), a.team, sh[1], [](float f, float g) {
        const unsigned m = __float_as_uint(f), n = __float_as_uint(g);
        return __uint_as_float(m > n ? m : n);
      }));
      const bool bad = most >= 0x7f800000u;
      const float scale = bad ? __builtin_nanf("") : __uint_as_float(most) * (1.0f / (KIND == LINREC_QUANTIZED_INT8 ? 127.0f : 448.0f));
      if (bad) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i][e] = 0.0f;
      } else if (scale > 0.0f) {
        up = scale < 1e-30f ? 0x1p60f : 1.0f;
        inverse = 1.0f / (scale * up);
      }
      if (there && in_team == 0) p.scales[row] = scale;
    } else if (a.team > 64) {
      __syncthreads();  // (the sums' places are written again in the next row)
    }
    if (there)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (!l.has[i]) continue;
        const int64_t at = row * p.channels + l.c[i];
        if constexpr (KIND != LINREC_QUANTIZED_NONE) {
          store_quantized<KIND, VEC>(p.y, at, v[i], up, inverse);
        } else {
          Lanes<VEC> t;
#pragma unroll
          for (int e = 0; e < VEC; ++e) t.v[e] = v[i][e] * rstd * w[i][e];
          st_any<VEC>(static_cast<T*>(p.y) + at, t);
        }
      }
  }
}

// A workgroup leaves a row of sums for d_weight behind.
template <typename T, int VEC, int ITEMS, int LANES>
__global__ __launch_bounds__(LANES) void rms_bwd_kernel(RmsArgs a) {
  __shared__ float sh[2][16];
  __shared__ float sh_w[LANES * VEC];
  const linrec_rms_norm_t& p = a.p;
  const int channels = int(p.channels), rows_side = int(blockDim.x) / a.team;
  const int in_team = threadIdx.x & (a.team - 1), row_slot = threadIdx.x / a.team;
  const RmsLane<VEC, ITEMS> l(in_team, a.team, channels);
  float w[ITEMS][VEC], d_w[ITEMS][VEC];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    rms_weights<VEC>(p.weight, p.weight_dtype, l.c[i], w[i]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) d_w[i][e] = 0.0f;
  }
  const T* x = static_cast<const T*>(p.x);
  const T* d_y = static_cast<const T*>(p.d_y);
  const T* d_total = static_cast<const T*>(p.d_total);
  const float inv_channels = 1.0f / float(channels);
  int turn = 0;
  for (int64_t base = int64_t(blockIdx.x) * rows_side; base < p.rows; base += int64_t(a.blocks) * rows_side, turn ^= 1) {
    const bool there = base + row_slot < p.rows;
    const int64_t row = there ? base + row_slot : p.rows - 1;
    const T* from = x + rms_row(p.x_stride, row, p.inner);
    const T* grad = d_y + rms_row(p.d_y_stride, row, p.inner);
    Held<T, VEC> hx[ITEMS], hd[ITEMS], ht[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (l.has[i]) {
        hx[i] = ld_any<VEC, true>(from + l.c[i]);
        hd[i] = ld_any<VEC, true>(grad + l.c[i]);
      }
    if (d_total) {
      const T* more = d_total + rms_row(p.d_total_stride, row, p.inner);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
        if (l.has[i]) ht[i] = ld_any<VEC, true>(more + l.c[i]);
    }
    const float rstd = p.rstd[row];
    float h[ITEMS][VEC], g[ITEMS][VEC], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (!l.has[i]) continue;
      const Lanes<VEC> vx = widen(hx[i]), vd = widen(hd[i]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        h[i][e] = vx.v[e] * rstd;
        g[i][e] = vd.v[e] * w[i][e];
        if (e >= l.skip[i]) {
          sum = fmaf(g[i][e], h[i][e], sum);
          if (there) d_w[i][e] = fmaf(vd.v[e], h[i][e], d_w[i][e]);
        }
      }
    }
    sum = over_team(sum, a.team, sh[turn], [](float f, float s) { return f + s; }) * inv_channels;
    if (there)
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if (!l.has[i]) continue;
        Lanes<VEC> t;
#pragma unroll
        for (int e = 0; e < VEC; ++e) t.v[e] = rstd * (g[i][e] - h[i][e] * sum);
        if (d_total) {
          const Lanes<VEC> u = widen(ht[i]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) t.v[e] += u.v[e];
        }
        st_any<VEC>(static_cast<T*>(p.d_x) + row * p.channels + l.c[i], t);
      }
  }
  if (!p.partial) return;
  float* out = p.partial + int64_t(blockIdx.x) * p.channels;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) sh_w[threadIdx.x * VEC + e] = d_w[i][e];
    __syncthreads();
    if (row_slot == 0 && l.has[i])
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float s = d_w[i][e];
        for (int k = 1; k < rows_side; ++k) s += sh_w[(k * a.team + in_team) * VEC + e];
        if (e >= l.skip[i]) out[l.c[i] + e] = s;
      }
  }
}

}  // namespace linrec
