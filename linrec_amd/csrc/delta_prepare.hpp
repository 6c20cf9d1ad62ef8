// Gated delta rule, what a chunk needs that does not depend on the state: M = (1 + A)^-1, C and the decays.
//
// A workgroup for every (chunk, head).  K K^T and Q K^T are matrix instructions, a wave for 16 rows; their operands lie in LDS where M
// and C are put together afterwards.  1 + A is unit lower triangular; its inverse is put together in fp32: blocks of 16 by substitution, a lane for a column,
// then of 32 and of 64 by M21 = -M22 A21 M11 with the fp32 matrix instruction.  (Substitution over all 64 rows would be 64 dependent
// steps; powers of A, whose binomials cancel, lose all digits where keys are alike.)
//
// 8 x 4096, 16 heads of 128 x 128 bf16: 130 us forward and 145 backward for 0.34 and 0.44 GB (66 and 86 us at the rate of a copy); ten meetings
// of a workgroup, three of which fit into a CU.
#pragma once
#include "delta_core.hpp"

namespace linrec {

constexpr int PREPARE_STRIDE = 68;  // floats of a row in LDS

// Rows of 64 values in LDS to a [64][64] block, without the quarter above the diagonal; TRANSPOSED: columns, without that below.
template <bool TRANSPOSED>
__device__ __forceinline__ void store_triangle(float* to, const float* from) {
  constexpr int S = PREPARE_STRIDE;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int i = n * 256 + int(threadIdx.x), row = i >> 4, c = (i & 15) * 4;
    if (TRANSPOSED ? row >= 32 && c < 32 : row < 32 && c >= 32) continue;
    v4f x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = TRANSPOSED ? from[(c + e) * S + row] : from[row * S + c + e];
    *reinterpret_cast<v4f*>(to + row * 64 + c) = x;
  }
}

// e^{G_63 - G} and so on of a chunk by its first wave, a lane for a position; G in fp64, where differences of large sums keep
// their digits.
__device__ __forceinline__ double chunk_sum(float g, int lane) {
  if (g < DELTA_LEAST_LOG) g = DELTA_LEAST_LOG;
  double sum = double(g);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double up = __shfl_up(sum, d);
    if (lane >= d) sum += up;
  }
  return sum;
}

template <typename T, int DK, bool BWD>
__global__ __launch_bounds__(256) void delta_prepare_kernel(DeltaArgs a) {
  using TK = Tile<T, DK>;
  constexpr int S = PREPARE_STRIDE, SQUARES = 2 * 64 * S * 4;
  __shared__ __align__(16) float sh_a[64 * S];
  __shared__ __align__(16) char sh_keys[2 * TK::BYTES > SQUARES ? 2 * TK::BYTES : SQUARES];
  float *sh_m = reinterpret_cast<float*>(sh_keys), *sh_c = sh_m + 64 * S;
  __shared__ double sh_g[64];
  __shared__ float sh_beta[64];
  const linrec_delta_t& p = a.p;
  const int64_t slot = blockIdx.x / unsigned(p.heads);
  const int head = int(blockIdx.x - slot * unsigned(p.heads)), key_head = head / a.shared;
  const Chunk ch = chunk_of(p, slot);
  if (ch.length == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, q = lane >> 4;
  const int64_t block = slot * p.heads + head;

  {
    Stager<T, DK, 256> k, qq;
    k.fetch(head_rows<T>(p.k, p.k_stride, ch.batch, ch.first, key_head), p.k_stride[1], ch.length, p.key_dim, threadIdx.x);
    qq.fetch(head_rows<T>(p.q, p.q_stride, ch.batch, ch.first, key_head), p.q_stride[1], ch.length, p.key_dim, threadIdx.x);
    k.put(sh_keys, threadIdx.x);
    qq.put(sh_keys + TK::BYTES, threadIdx.x);
  }
  if (wave == 0) {
    const bool there = lane < ch.length;
    const float g = there ? *(head_rows<float>(p.log_decay, p.log_decay_stride, ch.batch, ch.first + lane, head)) : 0.0f;
    const float beta = there ? *(head_rows<float>(p.beta, p.beta_stride, ch.batch, ch.first + lane, head)) : 0.0f;
    const double sum = chunk_sum(g, lane), last = __shfl(sum, 63);
    sh_g[lane] = sum;
    sh_beta[lane] = beta;
    float* gates = a.gates + block * 192;
    gates[lane] = expf(float(sum));
    gates[64 + lane] = expf(float(last - sum));
    gates[128 + lane] = beta;
    if constexpr (BWD) a.sums[block * 64 + lane] = sum;
  }
  __syncthreads();
  v4f kk[4], qk[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) kk[t] = v4f{0, 0, 0, 0}, qk[t] = v4f{0, 0, 0, 0};
  const int rows = TK::natural_rows(r, q);
  // wave w has rows 16 w and up; tile t of columns from 16 t on, none above the diagonal
#pragma unroll
  for (int b = 0; b < DK / 32; ++b) {
    const Frag<T> rk = TK::frag(sh_keys + wave * (16 * TK::ROW), rows, 0, b), rq = TK::frag(sh_keys + TK::BYTES + wave * (16 * TK::ROW), rows, 0, b);
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t <= wave) {
        const Frag<T> other = TK::frag(sh_keys, rows, 16 * t, b);
        kk[t] = mma(rk, other, kk[t]);
        qk[t] = mma(rq, other, qk[t]);
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * S; i += 256) sh_m[i] = 0.0f, sh_c[i] = 0.0f;
  __syncthreads();
#pragma unroll
  for (int t = 0; t < 4; ++t)
    if (t <= wave) {
      const int j = 16 * t + r;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * wave + 4 * q + e;
        const float d = i >= j ? fast_exp(float(sh_g[i] - sh_g[j])) : 0.0f;
        sh_a[i * S + j] = i > j ? sh_beta[i] * d * kk[t][e] : 0.0f;
        sh_c[i * S + j] = i >= j ? p.scale * d * qk[t][e] : 0.0f;
      }
    }
  __syncthreads();
  // blocks of 16: lane 16 q + r has column r of block q
  if (wave == 0) {
    const float* from = sh_a + 16 * q * S + 16 * q;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == r ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) s = fmaf(-from[i * S + j], x[j], s);
      x[i] = s;
      sh_m[(16 * q + i) * S + 16 * q + r] = s;
    }
  }
  __syncthreads();
  auto product = [&](const float* left, const float* right, v4f c) __attribute__((always_inline)) {  // 16 x 16 x 16
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(left[r * S + 4 * q + e], right[(4 * q + e) * S + r], c, 0, 0, 0);
    return c;
  };
  auto product_of = [&](const float* left, const v4f& right, v4f c) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(left[r * S + 4 * q + e], right[e], c, 0, 0, 0);
    return c;
  };
  if (wave < 2) {
    const int at = 32 * wave * S + 32 * wave;
    const v4f x = product(sh_a + at + 16 * S, sh_m + at, v4f{0, 0, 0, 0});
    const v4f y = product_of(sh_m + at + 16 * S + 16, x, v4f{0, 0, 0, 0});
#pragma unroll
    for (int e = 0; e < 4; ++e) sh_m[at + (16 + 4 * q + e) * S + r] = -y[e];
  }
  __syncthreads();
  {
    const int rt = wave >> 1, ct = wave & 1;
    v4f x[2], y = v4f{0, 0, 0, 0};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      x[n] = product(sh_a + (32 + 16 * n) * S, sh_m + 16 * ct, v4f{0, 0, 0, 0});
      x[n] = product(sh_a + (32 + 16 * n) * S + 16, sh_m + 16 * S + 16 * ct, x[n]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) y = product_of(sh_m + (32 + 16 * rt) * S + 32 + 16 * n, x[n], y);
#pragma unroll
    for (int e = 0; e < 4; ++e) sh_m[(32 + 16 * rt + 4 * q + e) * S + 16 * ct + r] = -y[e];
  }
  __syncthreads();
  store_triangle<false>(a.m + block * 4096, sh_m);
  if constexpr (BWD) store_triangle<true>(a.m_t + block * 4096, sh_m);
  store_triangle<BWD>(a.c + block * 4096, sh_c);
}

}  // namespace linrec
