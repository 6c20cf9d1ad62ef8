// Gated delta rule, the gradients of q, k and the gates of a chunk (delta_core.hpp):
//
//   F_ij = scale e^{G_i - G_j} dO_i.N_j (i >= j)      E_ij = -e^{G_i - G_j} dB_i.N_j (i > j)
//   dQ = scale e^G dO S^T + F K
//   X  = E K - e^G dB S^T,  Z = e^{G_63 - G} N dS'^T,  Y = Z + F^T Q + E^T (beta K);      dK = beta X + Y
//   dbeta = dB.V + K.X      dG = Q.dQ + beta K.X - K.Y  (row by row),   dG_63 += sum K.Z + e^{G_63} <S, dS'>
//
// and the gradient of log_decay is the sum of dG from a position to the chunk's end.
//
// A workgroup has a (chunk, key head) and walks over the value heads that share it, so that nothing is added by atomics; a wave has
// 16 rows of dQ and dK.  Value channels come 32 at a time through LDS.  The four 64 x 64 products F, F^T, E, E^T are computed as they
// are needed as operands: what a lane gets of a product is its part of an operand over the product's rows.
#pragma once
#include "delta_prepare.hpp"
#include "delta_scan.hpp"

namespace linrec {

template <typename T, int DK>
struct GradientShared {
  using U = Inner<T>;
  static constexpr int P = planes_of<U>(), IN = input_planes<T>();
  static constexpr int IN_V = 64 * 32 * int(sizeof(U)), BY_V = 32 * 64 * int(sizeof(U)), STATE = 32 * DK * int(sizeof(U)),
                       KEYS = Tile<U, DK>::BYTES;
  static constexpr int O = 0, V = O + IN * IN_V, B = V + IN * IN_V, N = B + P * BY_V, S = N + P * BY_V, D = S + P * STATE, FIRST = D + P * STATE;
  static constexpr int K = 0, Q = K + IN * KEYS, SECOND = Q + IN * KEYS;
  static constexpr int BYTES = FIRST > SECOND ? FIRST : SECOND;
};

// COLS columns of 64 rows of an input on their way to IN tiles of the inner type.
template <typename T, int COLS, int LANES>
struct InputStager {
  using U = Inner<T>;
  Stager<T, COLS, LANES> s;
  __device__ __forceinline__ void fetch(const T* from, int64_t stride, int rows, int cols) { s.fetch(from, stride, rows, cols, threadIdx.x); }
  __device__ __forceinline__ void put(char* tile) const {
    if constexpr (std::is_same_v<T, U>) {
      s.put(tile, threadIdx.x);
    } else {  // fp16 as two bf16
      Stager<U, COLS, LANES> hi, lo;
#pragma unroll
      for (int n = 0; n < decltype(s)::N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          hi.v[n][e] = U(float(s.v[n][e]));
          lo.v[n][e] = U(float(s.v[n][e]) - float(hi.v[n][e]));
        }
      hi.put(tile, threadIdx.x);
      lo.put(tile + 64 * Tile<U, COLS>::ROW, threadIdx.x);
    }
  }
};

__device__ __forceinline__ float sum_of_16(float x) {
  x += __shfl_xor(x, 1);
  x += __shfl_xor(x, 2);
  x += __shfl_xor(x, 4);
  return x + __shfl_xor(x, 8);
}

// DK: columns of dQ and dK at a time; WIDE: key_dim is more than that and they come in turns.
template <typename T, int DK, bool WIDE>
__global__ __launch_bounds__(256) void delta_gradient_kernel(DeltaArgs a) {
  using U = Inner<T>;
  using Sh = GradientShared<T, DK>;
  using TI = Tile<U, 32>;  // dO, V
  using TB = Tile<U, 64>;  // dB, N: rows are channels
  using TK = Tile<U, DK>;  // K, Q; S, dS': rows are channels
  constexpr int P = Sh::P, IN = Sh::IN, KT = DK / 16;
  constexpr int64_t ROW = WIDE ? 2 * DK : DK;  // of the kept states
  __shared__ __align__(16) char smem[Sh::BYTES];
  __shared__ double sh_g[64];
  __shared__ float sh_gamma[64], sh_rest[64], sh_beta[64], sh_total[64], sh_sum[4];
  const linrec_delta_t& p = a.p;
  const int64_t slot = blockIdx.x / unsigned(p.key_heads);
  const int key_head = int(blockIdx.x - slot * unsigned(p.key_heads));
  const Chunk ch = chunk_of(p, slot);
  if (ch.length == 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, q = lane >> 4;
  const int row0 = 16 * wave + 4 * q;  // this lane's rows of a result
  auto natural = [&](int t) { return [t](int j) { return 16 * t + 4 * j; }; };
  auto mapped = [&](int t) { return [t](int j) { return row_of_result(t, j); }; };

  for (int d0 = 0; d0 < (WIDE ? p.key_dim : 1); d0 += DK) {
    v4f dq_all[KT], dk_all[KT];
#pragma unroll
    for (int u = 0; u < KT; ++u) dq_all[u] = v4f{0, 0, 0, 0}, dk_all[u] = v4f{0, 0, 0, 0};
    for (int h = 0; h < a.shared; ++h) {
      const int head = key_head * a.shared + h;
      const int64_t block = slot * p.heads + head;
      __syncthreads();
      if (wave == 0) {
        const bool there = lane < ch.length;
        const float g = there ? *(head_rows<float>(p.log_decay, p.log_decay_stride, ch.batch, ch.first + lane, head)) : 0.0f;
        sh_g[lane] = chunk_sum(g, lane);
        sh_gamma[lane] = a.gates[block * 192 + lane];
        sh_rest[lane] = a.gates[block * 192 + 64 + lane];
        sh_beta[lane] = a.gates[block * 192 + 128 + lane];
      }
      v4f f[4], ft[4], ee[4], et[4], dq[KT], x[KT], y[KT], bv = v4f{0, 0, 0, 0}, inner = v4f{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = ft[t] = ee[t] = et[t] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < KT; ++u) dq[u] = x[u] = y[u] = v4f{0, 0, 0, 0};
      const T* d_o = head_rows<T>(p.d_o, p.d_o_stride, ch.batch, ch.first, head);
      const T* v = head_rows<T>(p.v, p.v_stride, ch.batch, ch.first, head);
      for (int v0 = 0; v0 < p.value_dim; v0 += 32) {
        __syncthreads();
        {
          InputStager<T, 32, 256> so, sv;
          Stager<U, 64, 256, 32> sb[P], sn[P];
          Stager<U, DK, 256, 32> ss[P], sd[P];
          so.fetch(d_o + v0, p.d_o_stride[1], ch.length, p.value_dim - v0);
          sv.fetch(v + v0, p.v_stride[1], ch.length, p.value_dim - v0);
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const int64_t row = (block * P + k) * a.columns + v0;
            sb[k].fetch_dense(reinterpret_cast<const U*>(a.d_b) + row * 64, threadIdx.x);
            sn[k].fetch_dense(reinterpret_cast<const U*>(a.n) + row * 64, threadIdx.x);
            ss[k].fetch(reinterpret_cast<const U*>(a.s) + row * ROW + d0, ROW, 32, DK, threadIdx.x);
            sd[k].fetch(reinterpret_cast<const U*>(a.d_s) + row * ROW + d0, ROW, 32, DK, threadIdx.x);
          }
          so.put(smem + Sh::O);
          sv.put(smem + Sh::V);
#pragma unroll
          for (int k = 0; k < P; ++k) {
            sb[k].put(smem + Sh::B + k * Sh::BY_V, threadIdx.x);
            sn[k].put(smem + Sh::N + k * Sh::BY_V, threadIdx.x);
            ss[k].put(smem + Sh::S + k * Sh::STATE, threadIdx.x);
            sd[k].put(smem + Sh::D + k * Sh::STATE, threadIdx.x);
          }
        }
        __syncthreads();
        auto rows_in = [&](int at, int row) __attribute__((always_inline)) {
          Planes<U, IN> out;
#pragma unroll
          for (int k = 0; k < IN; ++k) out.p[k] = TI::frag(smem + at + k * Sh::IN_V, row, 0, q);
          return out;
        };
        auto by_v = [&](int at, auto col) __attribute__((always_inline)) {
          Planes<U> out;
#pragma unroll
          for (int k = 0; k < P; ++k) out.p[k] = TB::column_frag(smem + at + k * Sh::BY_V, 0, q, col);
          return out;
        };
        auto state = [&](int at, auto col) __attribute__((always_inline)) {
          Planes<U> out;
#pragma unroll
          for (int k = 0; k < P; ++k) out.p[k] = TK::column_frag(smem + at + k * Sh::STATE, 0, q, col);
          return out;
        };
        const Planes<U, IN> do_w = rows_in(Sh::O, 16 * wave + r), v_w = rows_in(Sh::V, 16 * wave + r);
        const Planes<U> db_w = by_v(Sh::B, natural(wave)), n_w = by_v(Sh::N, natural(wave));
        bv = mma(db_w, v_w, bv);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (t / 2 <= wave / 2) {  // rows j of F^T and E^T up to this wave's columns i
            const Planes<U> n_t = by_v(Sh::N, mapped(t));
            ft[t] = mma(n_t, do_w, ft[t]);
            et[t] = mma(n_t, db_w, et[t]);
          }
          if (t / 2 >= wave / 2) {
            f[t] = mma(rows_in(Sh::O, row_of_tile(t, r)), n_w, f[t]);
            ee[t] = mma(by_v(Sh::B, mapped(t)), n_w, ee[t]);
          }
        }
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          const Planes<U> s_u = state(Sh::S, natural(u));
          dq[u] = mma(do_w, s_u, dq[u]);
          x[u] = mma(db_w, s_u, x[u]);
          y[u] = mma(n_w, state(Sh::D, natural(u)), y[u]);
        }
        // <S, dS'> on the diagonal of S^T dS', 16 channels at a time
        {
          const int row = 16 * (wave & 1) + r;
#pragma unroll
          for (int b = 0; b < DK / 32; ++b)
            if ((b & 1) == wave >> 1) {
              Planes<U> s_v, d_v;
#pragma unroll
              for (int k = 0; k < P; ++k) {
                s_v.p[k] = TK::frag(smem + Sh::S + k * Sh::STATE, row, b, q);
                d_v.p[k] = TK::frag(smem + Sh::D + k * Sh::STATE, row, b, q);
              }
              inner = mma(s_v, d_v, inner);
            }
        }
      }
      // the masks and decays; rows of results to operands
      Planes<U> fp[2], ftp[2], ep[2], etp[2];
      {
        const int own = 16 * wave + r;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = row_of_result(t, q) + e;
            const float down = i >= own ? expf(float(sh_g[i] - sh_g[own])) : 0.0f;  // i after this lane's column
            const float up = own >= i ? expf(float(sh_g[own] - sh_g[i])) : 0.0f;
            f[t][e] = i >= own ? p.scale * down * f[t][e] : 0.0f;
            ee[t][e] = i > own ? -sh_beta[i] * down * ee[t][e] : 0.0f;
            ft[t][e] = own >= i ? p.scale * up * ft[t][e] : 0.0f;
            et[t][e] = own > i ? -up * et[t][e] : 0.0f;
          }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          fp[b] = split<U>(f[2 * b], f[2 * b + 1]);
          ftp[b] = split<U>(ft[2 * b], ft[2 * b + 1]);
          ep[b] = split<U>(ee[2 * b], ee[2 * b + 1]);
          etp[b] = split<U>(et[2 * b], et[2 * b + 1]);
        }
      }
      __syncthreads();
      const T* k_rows = head_rows<T>(p.k, p.k_stride, ch.batch, ch.first, key_head) + d0;
      const T* q_rows = head_rows<T>(p.q, p.q_stride, ch.batch, ch.first, key_head) + d0;
      {
        InputStager<T, DK, 256> sk, sq;
        sk.fetch(k_rows, p.k_stride[1], ch.length, p.key_dim - d0);
        sq.fetch(q_rows, p.q_stride[1], ch.length, p.key_dim - d0);
        sk.put(smem + Sh::K);
        sq.put(smem + Sh::Q);
      }
      __syncthreads();
      float dot_q[4], dot_x[4], dot_y[4], dot_z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) dot_q[e] = dot_x[e] = dot_y[e] = dot_z[e] = 0.0f;
      const v4f gamma = *reinterpret_cast<const v4f*>(sh_gamma + row0), rest = *reinterpret_cast<const v4f*>(sh_rest + row0),
                beta = *reinterpret_cast<const v4f*>(sh_beta + row0);
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        v4f kv = v4f{0, 0, 0, 0}, qv = v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < IN; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            kv[e] += TK::value(smem + Sh::K + k * Sh::KEYS, row0 + e, 16 * u + r);
            qv[e] += TK::value(smem + Sh::Q + k * Sh::KEYS, row0 + e, 16 * u + r);
          }
        v4f dqu = dq[u] * gamma * p.scale, xu = -gamma * x[u], yu = rest * y[u];
#pragma unroll
        for (int e = 0; e < 4; ++e) dot_z[e] = fmaf(kv[e], yu[e], dot_z[e]);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          Planes<U, IN> k_b, q_b;
#pragma unroll
          for (int k = 0; k < IN; ++k) {
            k_b.p[k] = TK::column_frag(smem + Sh::K + k * Sh::KEYS, b, q, natural(u));
            q_b.p[k] = TK::column_frag(smem + Sh::Q + k * Sh::KEYS, b, q, natural(u));
          }
          if (b <= wave / 2) {
            dqu = mma(ftp[b], k_b, dqu);
            xu = mma(etp[b], k_b, xu);
          }
          if (b >= wave / 2) {
            yu = mma(fp[b], q_b, yu);
            yu = mma(ep[b], k_b, yu);
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dot_q[e] = fmaf(qv[e], dqu[e], dot_q[e]);
          dot_x[e] = fmaf(kv[e], xu[e], dot_x[e]);
          dot_y[e] = fmaf(kv[e], yu[e], dot_y[e]);
        }
        dq_all[u] += dqu;
        dk_all[u] += beta * xu + yu;
      }
      float z = 0.0f;
      float* dots = a.dots + block * 192;  // (every place is written and read by one lane)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float qq = sum_of_16(dot_q[e]), xx = sum_of_16(dot_x[e]), yy = sum_of_16(dot_y[e]);
        z += sum_of_16(dot_z[e]);
        // dB.V stands on the diagonal of a product, lane 16 q + 4 q + e
        const float own = __shfl(bv[e], 16 * q + 4 * q + e);
        float total = qq + beta[e] * xx - yy, d_beta = xx;
        if (r == 0) {
          if (WIDE && d0 > 0) {
            total += dots[row0 + e];
            d_beta += dots[64 + row0 + e];
          } else {
            d_beta += own;
          }
          if (WIDE && d0 + DK < p.key_dim) {
            dots[row0 + e] = total;
            dots[64 + row0 + e] = d_beta;
          } else if (row0 + e < ch.length) {
            p.d_beta[((ch.batch * p.time + ch.first + row0 + e) * p.heads) + head] = d_beta;
          }
          sh_total[row0 + e] = total;
        }
      }
      // z of four rows in every lane of a group of 16; <S, dS'> on diagonals
      float sum = r == 0 ? z : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (r == 4 * q + e) sum = fmaf(sh_gamma[63], inner[e], sum);
      sum = sum_of_16(sum);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lane == 0) sh_sum[wave] = sum;
      __syncthreads();
      if (wave == 0) {
        double total = double(sh_total[lane]);
        if (lane == 63) {
          float ends = (sh_sum[0] + sh_sum[1]) + (sh_sum[2] + sh_sum[3]);
          if (WIDE && d0 > 0) ends += dots[128];
          if (WIDE && d0 + DK < p.key_dim) dots[128] = ends;
          total += double(ends);
        }
        if (!WIDE || d0 + DK >= p.key_dim) {
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) {
            const double up = __shfl_down(total, d);
            if (lane + d < 64) total += up;
          }
          if (lane < ch.length) p.d_log_decay[((ch.batch * p.time + ch.first + lane) * p.heads) + head] = float(total);
        }
      }
    }
    // what the value heads' shares add up to
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row0 + e < ch.length) {
        const int64_t at = ((ch.batch * p.time + ch.first + row0 + e) * p.key_heads + key_head) * int64_t(p.key_dim) + d0;
#pragma unroll
        for (int u = 0; u < KT; ++u)
          if (d0 + 16 * u + r < p.key_dim) {
            static_cast<T*>(p.d_q)[at + 16 * u + r] = T(dq_all[u][e]);
            static_cast<T*>(p.d_k)[at + 16 * u + r] = T(dk_all[u][e]);
          }
      }
  }
}

}  // namespace linrec
