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
template <int DK, bool REVERSE>
__global__ __launch_bounds__(256) void delta_segments_kernel(DeltaArgs a) {
  constexpr int TILES = DK / 64, STEPS = DK / 16, PAD = 17;
  constexpr bool AHEAD = DK <= 128;  // (a quarter of a larger T is more than the registers hold beside the one in use)
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
  v4f s[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * (wave * TILES + t) + 4 * q + e;
      s[t][e] = from && col < p.value_dim && d < p.key_dim ? from[(pair * p.key_dim + d) * int64_t(p.value_dim) + col] : 0.0f;
    }
  float m[TILES][STEPS][4];  // T (or T^T) of the next segment: row r, columns 16 i + 4 q + e
  v4f next[TILES];
  auto fetch = [&](int64_t g) __attribute__((always_inline)) {
    const float* c = a.carry + place(g) * (a.columns + DK) * DK;
    const float* unit = c + int64_t(a.columns) * DK;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int d = 16 * (wave * TILES + t);
      next[t] = *reinterpret_cast<const v4f*>(c + int64_t(col) * DK + d + 4 * q);
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 16 * i + 4 * q + e;
          m[t][i][e] = REVERSE ? unit[(d + r) * DK + j] : unit[j * DK + d + r];
        }
    }
  };
  if (AHEAD && count > 1) fetch(0);
  for (int64_t g = 0; g < count; ++g) {
    float* to = a.start + (place(g) * a.columns + col) * DK;
    float* mine = sh[g & 1];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      const int d = 16 * (wave * TILES + t) + 4 * q;
      *reinterpret_cast<v4f*>(to + d) = s[t];
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(d + e) * PAD + r] = s[t][e];
    }
    if (g + 1 == count) break;
    if (!AHEAD) fetch(g);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      s[t] = next[t];
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[t][i][e], mine[(16 * i + 4 * q + e) * PAD + r], s[t], 0, 0, 0);
    }
    if (AHEAD && g + 2 < count) fetch(g + 1);
  }
}

}  // namespace linrec
