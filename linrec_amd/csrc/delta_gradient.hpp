// Gated delta rule, the gradients of q, k and the gates of a chunk (delta_core.hpp):
//
//   F_ij = scale e^{G_i - G_j} dO_i.N_j (i >= j)      E_ij = -e^{G_i - G_j} dB_i.N_j (i > j)
//   dQ = scale e^G dO S^T + F K
//   X  = E K - e^G dB S^T,  Z = e^{G_63 - G} N dS'^T,  Y = Z + F^T Q + E^T (beta K);      dK = beta X + Y
//   dbeta = dB.V + K.X,  dG = Q.dQ + beta K.X - K.Y (row by row),  dG_63 += sum K.Z + e^{G_63} <S, dS'>
//
// and the gradient of log_decay is the sum of dG from a position to the chunk's end.
//
// A workgroup has a (chunk, key head) and walks over the value heads that share it, so that nothing is added by atomics.  Value
// channels come 32 at a time through LDS, the next ones on their way in registers meanwhile.  Its waves have three parts, four waves
// of 16 rows each: dQ, X and Y.  (One wave for all three holds twice the registers that three waves to a SIMD leave it, and what
// then goes through scratch costs more than the products: 2.4 ms instead of the time below.)  The 64 x 64 products F, F^T, E, E^T are
// computed as they are needed as operands: what a lane gets of a product is its part of an operand over the product's rows.
#pragma once
#include "delta_prepare.hpp"
#include "delta_scan.hpp"

namespace linrec {

constexpr int GRADIENT_LANES = 768, GRADIENT_PART = 256;

template <typename T, int DK>
struct GradientShared {
  using U = Inner<T>;
  static constexpr int P = planes_of<U>(), IN = input_planes<T>();
  static constexpr int IN_V = 64 * 32 * int(sizeof(U)), BY_V = 32 * 64 * int(sizeof(U)), STATE = 32 * DK * int(sizeof(U)),
                       KEYS = Tile<U, DK>::BYTES;
  // one step's values, then both inputs of key channels
  static constexpr int O = 0, V = O + IN * IN_V, B = V + IN * IN_V, N = B + P * BY_V, S = N + P * BY_V, D = S + P * STATE, STEP = D + P * STATE;
  static constexpr int BUFFERS = 2 * STEP + 2 * IN * KEYS + 4096 <= 160 * 1024 ? 2 : 1;
  static constexpr int K = BUFFERS * STEP, Q = K + IN * KEYS, BYTES = Q + IN * KEYS;
  static_assert(64 * DK * 4 <= BUFFERS * STEP, "room to hand dK over");
};

// COLS columns of 64 rows of an input on their way to IN tiles of the inner type.
template <typename T, int COLS, int LANES>
struct InputStager {
  using U = Inner<T>;
  Stager<T, COLS, LANES> s;
  __device__ __forceinline__ void fetch(const T* from, int64_t stride, int rows, int cols, int lane) { s.fetch(from, stride, rows, cols, lane); }
  __device__ __forceinline__ void put(char* tile, int lane) const {
    if constexpr (std::is_same_v<T, U>) {
      s.put(tile, lane);
    } else {  // fp16 as two bf16
      Stager<U, COLS, LANES> hi, lo;
#pragma unroll
      for (int n = 0; n < decltype(s)::N; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          hi.v[n][e] = U(float(s.v[n][e]));
          lo.v[n][e] = U(float(s.v[n][e]) - float(hi.v[n][e]));
        }
      hi.put(tile, lane);
      lo.put(tile + 64 * Tile<U, COLS>::ROW, lane);
    }
  }
};

enum GradientPart { GRADIENT_Q, GRADIENT_X, GRADIENT_Y };

template <typename T, int DK>
struct GradientScratch {  // LDS beside GradientShared
  double g[64];
  alignas(16) float gamma[64], rest[64], beta[64], q[64], x[64], y[64], bv[64], sum[8];
};

// What the waves of one part do.  All parts meet at the same barriers.
template <typename T, int DK, bool WIDE, GradientPart PART>
__device__ __forceinline__ void gradient_part(const DeltaArgs& a, const Chunk& ch, int64_t slot, int key_head, char* smem, GradientScratch<T, DK>& sh) {
  using U = Inner<T>;
  using Sh = GradientShared<T, DK>;
  using TI = Tile<U, 32>;  // dO, V
  using TB = Tile<U, 64>;  // dB, N: rows are channels
  using TK = Tile<U, DK>;  // K, Q; S, dS': rows are channels
  constexpr int P = Sh::P, IN = Sh::IN, KT = DK / 16, LANES = GRADIENT_PART;
  constexpr int64_t ROW = WIDE ? 2 * DK : DK;  // of the kept states
  const linrec_delta_t& p = a.p;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, by0 = threadIdx.x & (LANES - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int row0 = 16 * wave + 4 * q;  // this lane's rows of a result
  const int rows_w0 = TI::natural_rows(r, q) + wave * (16 * TI::ROW), rows_m0 = TI::mapped_rows(r, q);
  const int cols_w0 = TB::template column_tile<false>(TB::template columns<false>(r, q), wave), cols_m0 = TB::template columns<true>(r, q);
  const int cols_k0 = TK::template columns<false>(r, q), rows_v0 = TK::natural_rows(r, q) + (wave & 1) * (16 * TK::ROW),
            points0 = TK::points(r, q) + wave * (16 * TK::ROW);

  // each part loads some of a step: the rows of dO and V with dB and N, S, dS'
  InputStager<T, 32, LANES> so, sv;
  Stager<U, 64, LANES, 32> sb[P], sn[P];
  Stager<U, DK, LANES, 32> ss[P];
  // one wave has what belongs to the positions, a lane for each
  const bool keeper = PART == GRADIENT_Y && wave == 0;
  double sum = 0.0;
  float gamma = 0.0f, rest = 0.0f, beta = 0.0f;
  auto fetch = [&](int head, int v0, int d0) __attribute__((always_inline)) {
    const int64_t block = slot * p.heads + head;
    const int by = anew(by0);
    if (keeper && v0 == 0) {
      const int own = anew(lane);
      sum = a.sums[block * 64 + own];
      gamma = a.gates[block * 192 + own];
      rest = a.gates[block * 192 + 64 + own];
      beta = a.gates[block * 192 + 128 + own];
    }
    if constexpr (PART == GRADIENT_Q) {
      so.fetch(head_rows<T>(p.d_o, p.d_o_stride, ch.batch, ch.first, head) + v0, p.d_o_stride[1], ch.length, p.value_dim - v0, by);
      sv.fetch(head_rows<T>(p.v, p.v_stride, ch.batch, ch.first, head) + v0, p.v_stride[1], ch.length, p.value_dim - v0, by);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int64_t row = int64_t(k) * a.columns + v0;
      if constexpr (PART == GRADIENT_Q) {
        sb[k].fetch_dense(reinterpret_cast<const U*>(a.d_b + block * a.rows) + row * 64, by);
        sn[k].fetch_dense(reinterpret_cast<const U*>(a.n + block * a.rows) + row * 64, by);
      } else {
        const U* from = reinterpret_cast<const U*>((PART == GRADIENT_X ? a.s : a.d_s) + block * a.state) + row * ROW;
        if constexpr (WIDE) ss[k].fetch(from + d0, ROW, 32, DK, by);
        else ss[k].fetch_dense(from, by);
      }
    }
  };
  auto put = [&](char* to) __attribute__((always_inline)) {
    const int by = anew(by0);
    if constexpr (PART == GRADIENT_Q) {
      so.put(to + Sh::O, by);
      sv.put(to + Sh::V, by);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if constexpr (PART == GRADIENT_Q) {
        sb[k].put(to + Sh::B + k * Sh::BY_V, by);
        sn[k].put(to + Sh::N + k * Sh::BY_V, by);
      } else {
        ss[k].put(to + (PART == GRADIENT_X ? Sh::S : Sh::D) + k * Sh::STATE, by);
      }
    }
  };

  for (int d0 = 0; d0 < (WIDE ? p.key_dim : 1); d0 += DK) {
    v4f all[KT];  // this part's share of dQ or dK over the value heads
    v4f before = v4f{0, 0, 0, 0};  // Y: K times what it was before this head, row by row
#pragma unroll
    for (int u = 0; u < KT; ++u) all[u] = v4f{0, 0, 0, 0};
    {
      InputStager<T, DK, LANES> keys;
      if constexpr (PART == GRADIENT_X)
        keys.fetch(head_rows<T>(p.k, p.k_stride, ch.batch, ch.first, key_head) + d0, p.k_stride[1], ch.length, p.key_dim - d0, by0);
      if constexpr (PART == GRADIENT_Y)
        keys.fetch(head_rows<T>(p.q, p.q_stride, ch.batch, ch.first, key_head) + d0, p.q_stride[1], ch.length, p.key_dim - d0, by0);
      fetch(key_head * a.shared, 0, d0);
      __syncthreads();
      if constexpr (PART != GRADIENT_Q) keys.put(smem + (PART == GRADIENT_X ? Sh::K : Sh::Q), by0);
    }
    int turn = 0;
    for (int h = 0; h < a.shared; ++h) {
      const int head = key_head * a.shared + h;
      const int64_t block = slot * p.heads + head;
      // (of the head before, others read these before the last barrier)
      if (keeper) {
        const int own = anew(lane);
        sh.g[own] = sum;
        sh.gamma[own] = gamma;
        sh.rest[own] = rest;
        sh.beta[own] = beta;
      }
      // F^T, dQ; E^T, X; F, E, Y
      // (Y has the most operands: its rows of N are scaled on their way, so that it adds to the share itself)
      v4f f[4], ee[4], acc[PART == GRADIENT_Y ? 1 : KT], bv = v4f{0, 0, 0, 0}, inner = v4f{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = ee[t] = v4f{0, 0, 0, 0};
      if constexpr (PART != GRADIENT_Y)
#pragma unroll
        for (int u = 0; u < KT; ++u) acc[u] = v4f{0, 0, 0, 0};
      for (int v0 = 0; v0 < p.value_dim; v0 += 32) {
        char* at = smem + (Sh::BUFFERS == 2 ? turn * Sh::STEP : 0);
        if constexpr (Sh::BUFFERS == 1) __syncthreads();
        put(at);
        __syncthreads();
        if (v0 + 32 < p.value_dim) fetch(head, v0 + 32, d0);
        else if (h + 1 < a.shared) fetch(head + 1, 0, d0);
        turn ^= 1;
        const int rows_w = anew(rows_w0), rows_m = anew(rows_m0), cols_w = anew(cols_w0), cols_m = anew(cols_m0), cols_k = anew(cols_k0),
                  rows_v = anew(rows_v0);
        auto rows_in = [&](int part, int view, int row) __attribute__((always_inline)) {
          Planes<U, IN> out;
#pragma unroll
          for (int k = 0; k < IN; ++k) out.p[k] = TI::frag(at + part + k * Sh::IN_V, view, row, 0);
          return out;
        };
        auto by_v = [&](int part) __attribute__((always_inline)) {  // this wave's rows
          Planes<U> out;
#pragma unroll
          for (int k = 0; k < P; ++k) out.p[k] = TB::template column_frag<false>(at + part + k * Sh::BY_V, cols_w, 0, 0);
          return out;
        };
        auto by_v_mapped = [&](int part, int t) __attribute__((always_inline)) {
          Planes<U> out;
#pragma unroll
          for (int k = 0; k < P; ++k) out.p[k] = TB::template column_frag<true>(at + part + k * Sh::BY_V, cols_m, 0, t);
          return out;
        };
        auto state = [&](int part, int u) __attribute__((always_inline)) {
          Planes<U> out;
#pragma unroll
          for (int k = 0; k < P; ++k) out.p[k] = TK::template column_frag<false>(at + part + k * Sh::STATE, cols_k, 0, u);
          return out;
        };
        if constexpr (PART == GRADIENT_Q) {
          const Planes<U, IN> do_w = rows_in(Sh::O, rows_w, 0);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (t / 2 <= wave / 2) f[t] = mma(by_v_mapped(Sh::N, t), do_w, f[t]);  // rows j up to this wave's columns i
#pragma unroll
          for (int u = 0; u < KT; ++u) acc[u] = mma(do_w, state(Sh::S, u), acc[u]);
        } else if constexpr (PART == GRADIENT_X) {
          const Planes<U> db_w = by_v(Sh::B);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (t / 2 <= wave / 2) ee[t] = mma(by_v_mapped(Sh::N, t), db_w, ee[t]);
#pragma unroll
          for (int u = 0; u < KT; ++u) acc[u] = mma(db_w, state(Sh::S, u), acc[u]);
          bv = mma(db_w, rows_in(Sh::V, rows_w, 0), bv);
          // <S, dS'> on the diagonal of S^T dS', 16 channels at a time
#pragma unroll
          for (int b = 0; b < DK / 32; ++b)
            if ((b & 1) == wave >> 1) {
              Planes<U> s_v, d_v;
#pragma unroll
              for (int k = 0; k < P; ++k) {
                s_v.p[k] = TK::frag(at + Sh::S + k * Sh::STATE, rows_v, 0, b);
                d_v.p[k] = TK::frag(at + Sh::D + k * Sh::STATE, rows_v, 0, b);
              }
              inner = mma(s_v, d_v, inner);
            }
        } else {
          const Planes<U> n_w = by_v(Sh::N);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (t / 2 >= wave / 2) {
              f[t] = mma(rows_in(Sh::O, rows_m, TI::mapped_row(t)), n_w, f[t]);
              ee[t] = mma(by_v_mapped(Sh::B, t), n_w, ee[t]);
            }
          Planes<U> scaled;
          {
            const float by = sh.rest[16 * wave + anew(r)];
            v4f n[2];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float x = float(n_w.p[0][e]);
              if constexpr (P == 2) x += float(n_w.p[1][e]);
              n[e >> 2][e & 3] = by * x;
            }
            scaled = split<U>(n[0], n[1]);
          }
#pragma unroll
          for (int u = 0; u < KT; ++u) all[u] = mma(scaled, state(Sh::D, u), all[u]);
        }
      }
      int cols_k = anew(cols_k0), points = anew(points0);
      const int r1 = anew(r), row1 = 16 * wave + 4 * anew(q);
      // the masks and decays; rows of results to operands
      Planes<U> fp[2], ep[2];
      {
        const int own = 16 * wave + anew(r), q1 = anew(q);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int other = row_of_result(t, q1) + e, i = PART == GRADIENT_Y ? other : own, j = PART == GRADIENT_Y ? own : other;
            const float d = i >= j ? fast_exp(float(sh.g[i] - sh.g[j])) : 0.0f;
            if constexpr (PART != GRADIENT_X) f[t][e] = i >= j ? p.scale * d * f[t][e] : 0.0f;
            if constexpr (PART != GRADIENT_Q) ee[t][e] = i > j ? -(PART == GRADIENT_Y ? sh.beta[i] : 1.0f) * d * ee[t][e] : 0.0f;
          }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if constexpr (PART != GRADIENT_X) fp[b] = split<U>(f[2 * b], f[2 * b + 1]);
          if constexpr (PART != GRADIENT_Q) ep[b] = split<U>(ee[2 * b], ee[2 * b + 1]);
        }
      }
      auto keys = [&](int part, int b, int u) __attribute__((always_inline)) {
        Planes<U, IN> out;
#pragma unroll
        for (int k = 0; k < IN; ++k) out.p[k] = TK::template column_frag<false>(smem + part + k * Sh::KEYS, cols_k, b, u);
        return out;
      };
      auto values = [&](int part, int u) __attribute__((always_inline)) {
        v4f out = v4f{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < IN; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) out[e] += TK::point(smem + part + k * Sh::KEYS, points, 0, e, u);
        return out;
      };
      v4f dot = v4f{0, 0, 0, 0}, ends = v4f{0, 0, 0, 0};
      v4f by_row = *reinterpret_cast<const v4f*>(sh.gamma + row1);
      if constexpr (PART == GRADIENT_Q) by_row *= p.scale;
      if constexpr (PART == GRADIENT_X) by_row = -by_row;
      const v4f beta_of = *reinterpret_cast<const v4f*>(sh.beta + row1);
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        v4f z;
        if constexpr (PART == GRADIENT_Y) z = all[u];
        else z = by_row * acc[u];
        const v4f x = values(PART == GRADIENT_Q ? Sh::Q : Sh::K, u);
        if constexpr (PART == GRADIENT_Y) ends += x * z;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if constexpr (PART == GRADIENT_Q) {
            if (b <= wave / 2) z = mma(fp[b], keys(Sh::K, b, u), z);
          } else if constexpr (PART == GRADIENT_X) {
            if (b <= wave / 2) z = mma(ep[b], keys(Sh::K, b, u), z);
          } else if (b >= wave / 2) {
            z = mma(fp[b], keys(Sh::Q, b, u), z);
            z = mma(ep[b], keys(Sh::K, b, u), z);
          }
        }
        dot += x * z;
        // (reads of the next columns, all ahead of their products, would push other values out of the registers)
        points = anew_after(points, dot);
        cols_k = anew_after(cols_k, z);
        if constexpr (PART == GRADIENT_X) z *= beta_of;
        if constexpr (PART == GRADIENT_Y) all[u] = z;
        else all[u] += z;
      }
      if constexpr (PART == GRADIENT_Y) {
        const v4f now = dot;
        dot -= before;
        ends -= before;
        before = now;
      }
      float* to = PART == GRADIENT_Q ? sh.q : PART == GRADIENT_X ? sh.x : sh.y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = sum_of_16(dot[e]);
        if (r1 == 0) to[row1 + e] = d;
      }
      if constexpr (PART == GRADIENT_X) {
        // dB.V and <S, dS'> stand on diagonals, lane 16 q + 4 q + e
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r1 == row1 - 16 * wave + e) {
            sh.bv[row1 + e] = bv[e];
            ends[0] = sh.gamma[63] * inner[e];
          }
      }
      if constexpr (PART != GRADIENT_Q) {
        float whole = sum_of_16((ends[0] + ends[1]) + (ends[2] + ends[3]));
        whole += __shfl_xor(whole, 16);
        whole += __shfl_xor(whole, 32);
        if (lane == 0) sh.sum[PART == GRADIENT_X ? wave : 4 + wave] = whole;
      }
      __syncthreads();
      if (keeper) {
        const int own = anew(lane);
        float* dots = a.dots + block * 192;  // (every place is written and read by one own)
        float total = sh.q[own] + sh.beta[own] * sh.x[own] - sh.y[own], d_beta = sh.x[own] + (d0 == 0 ? sh.bv[own] : 0.0f);
        if (own == 63) total += ((sh.sum[0] + sh.sum[1]) + (sh.sum[2] + sh.sum[3])) + ((sh.sum[4] + sh.sum[5]) + (sh.sum[6] + sh.sum[7]));
        if (WIDE && d0 > 0) {
          total += dots[own];
          d_beta += dots[64 + own];
        }
        if (WIDE && d0 + DK < p.key_dim) {
          dots[own] = total;
          dots[64 + own] = d_beta;
        } else {
          double after = double(total);
#pragma unroll
          for (int d = 1; d < 64; d <<= 1) {
            const double up = __shfl_down(after, d);
            if (own + d < 64) after += up;
          }
          if (own < ch.length) {
            const int64_t at = (ch.batch * p.time + ch.first + own) * p.heads + head;
            p.d_log_decay[at] = float(after);
            p.d_beta[at] = d_beta;
          }
        }
      }
    }
    // the two shares of dK together
    __syncthreads();
    float* sh_k = reinterpret_cast<float*>(smem);
    if constexpr (PART == GRADIENT_Y)
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) sh_k[(row0 + e) * DK + 16 * u + r] = all[u][e];
    __syncthreads();
    if constexpr (PART != GRADIENT_Y) {
      T* out = static_cast<T*>(PART == GRADIENT_Q ? p.d_q : p.d_k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (row0 + e < ch.length) {
          const int64_t at = ((ch.batch * p.time + ch.first + row0 + e) * p.key_heads + key_head) * int64_t(p.key_dim) + d0;
#pragma unroll
          for (int u = 0; u < KT; ++u)
            if (d0 + 16 * u + r < p.key_dim)
              out[at + 16 * u + r] = T(PART == GRADIENT_Q ? all[u][e] : all[u][e] + sh_k[(row0 + e) * DK + 16 * u + r]);
        }
    }
  }
}

// DK: columns of dQ and dK at a time; WIDE: key_dim is more than that and they come in turns.
template <typename T, int DK, bool WIDE>
__global__ __launch_bounds__(GRADIENT_LANES) void delta_gradient_kernel(DeltaArgs a) {
  __shared__ __align__(16) char smem[GradientShared<T, DK>::BYTES];
  __shared__ GradientScratch<T, DK> sh;
  const int64_t slot = blockIdx.x / unsigned(a.p.key_heads);
  const int key_head = int(blockIdx.x - slot * unsigned(a.p.key_heads));
  const Chunk ch = chunk_of(a.p, slot);
  if (ch.length == 0) return;
  const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  if (part == 0) gradient_part<T, DK, WIDE, GRADIENT_Q>(a, ch, slot, key_head, smem, sh);
  else if (part == 1) gradient_part<T, DK, WIDE, GRADIENT_X>(a, ch, slot, key_head, smem, sh);
  else gradient_part<T, DK, WIDE, GRADIENT_Y>(a, ch, slot, key_head, smem, sh);
}

}  // namespace linrec
