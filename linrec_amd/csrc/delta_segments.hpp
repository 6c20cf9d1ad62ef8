// Gated delta rule where few sequences and heads would leave most of the chip idle: sequences are cut into segments of chunks.
//
// The state behind a segment is T S + N with a key_dim x key_dim matrix T, since every position maps the state linearly.  A first
// pass (SCAN_CARRY) lets all segments run side by side from nothing, which gives N, and from the unit matrix without values, which gives
// T: to a segment these are key_dim columns more.  The kernel here goes from segment to segment with the states that enter
// them, and the second pass runs all of them side by side again, each from its state.  Backwards the gradient of the state goes
// through T^T.  That is two passes and more columns instead of one pass, for as many times fewer chunks one after another.
#pragma once
#include "delta_scan.hpp"

namespace linrec {

// A workgroup has 16 columns of a (sequence, head), a wave a quarter of the rows; fp32 products, the state in LDS between them.
// REVERSE: from the last segment to the first, with T^T.
//
// T lies column by column, and a lane loads 16 bytes of it at a time: of one row of T^T, or of one column of T, whose rows then belong to a
// product each (row n of product t stands for row TILES n + t).  It comes a quarter or half ahead of the products, all that the next ones
// wait for but the state: 147 us for 20 segments of 256 x 128, 178 back (one value a lane and load, and a wave's part of T at once, which
// went through scratch, 927 and 232).
template <int DK, bool REVERSE>
__global__ __launch_bounds__(256) void delta_segments_kernel(DeltaArgs a) {
  constexpr int TILES = DK / 64, STEPS = DK / 16, PAD = 17, SHARE = STEPS >= 8 ? 4 : 2, SHARES = STEPS / SHARE;
  static_assert(SHARES % 2 == 0, "");
  __shared__ float sh[2][DK * PAD];
  const linrec_delta_t& p = a.p;
  const int blocks = a.columns / 16;
  const int64_t pair = blockIdx.x / unsigned(blocks), n = pair / p.heads;
  const int head = int(pair - n * p.heads), lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = int(blockIdx.x - pair * unsigned(blocks)) * 16 + r;
  const Span span = span_of(p, n);
  const int64_t count = count_of_parts(a, span), first = first_part(a, n, span);
  const float* from = REVERSE ? p.d_state : p.h0;
  auto place = [&](int64_t g) { return (first + (REVERSE ? count - 1 - g : g)) * p.heads + head; };
  auto dim = [&](int t, int row) { return wave * (16 * TILES) + (REVERSE ? 16 * t + row : TILES * row + t); };
  v4f s[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = dim(t, 4 * q + e);
      s[t][e] = from && col < p.value_dim && d < p.key_dim ? from[(pair * p.key_dim + d) * int64_t(p.value_dim) + col] : 0.0f;
    }
  float m[2][SHARE][4][TILES];  // T (or T^T): row dim(t, r), columns 16 i + 4 q + e
  v4f next[TILES];
  auto fetch = [&](int64_t g, auto share) __attribute__((always_inline)) {
    const float* c = a.carry + place(g) * (a.columns + DK) * DK;
    const float* unit = c + int64_t(a.columns) * DK;
#pragma unroll
    for (int t = 0; t < (share() == 0 ? TILES : 0); ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) next[t][e] = c[int64_t(col) * DK + dim(t, 4 * q + e)];
    auto& to = m[share() & 1];
#pragma unroll
    for (int i = 0; i < SHARE; ++i) {
      const int j = 16 * (share() * SHARE + i) + 4 * q;
      if constexpr (REVERSE) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const v4f x = *reinterpret_cast<const v4f*>(unit + dim(t, r) * DK + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) to[i][e][t] = x[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          typedef float vt __attribute__((ext_vector_type(TILES)));
          const vt x = *reinterpret_cast<const vt*>(unit + (j + e) * DK + dim(0, r));
#pragma unroll
          for (int t = 0; t < TILES; ++t) to[i][e][t] = x[t];
        }
      }
    }
  };
  if (count > 1) fetch(0, std::integral_constant<int, 0>{});
  for (int64_t g = 0; g < count; ++g) {
    float* to = a.start + (place(g) * a.columns + col) * DK;
    float* mine = sh[g & 1];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = dim(t, 4 * q + e);
        to[d] = s[t][e];
        mine[d * PAD + r] = s[t][e];
      }
    if (g + 1 == count) break;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TILES; ++t) s[t] = next[t];
    static_for<SHARES>([&](auto share) __attribute__((always_inline)) {
      if constexpr (share() + 1 < SHARES) fetch(g, std::integral_constant<int, share() + 1>{});
      else if (g + 2 < count) fetch(g + 1, std::integral_constant<int, 0>{});
#pragma unroll
      for (int i = 0; i < SHARE; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = mine[(16 * (share() * SHARE + i) + 4 * q + e) * PAD + r];
#pragma unroll
          for (int t = 0; t < TILES; ++t) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[share() & 1][i][e][t], x, s[t], 0, 0, 0);
        }
    });
  }
}

}  // namespace linrec
