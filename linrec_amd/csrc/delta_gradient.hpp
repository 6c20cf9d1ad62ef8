// Gated delta rule, the gradients of q, k and the gates of a chunk (delta_core.hpp):
//
//   F_ij = scale e^{G_i - G_j} dO_i.N_j (i >= j)      E_ij = -e^{G_i - G_j} dB_i.N_j (i > j)
//   dQ = scale e^G dO S^T + F K
//   X  = E K - e^G dB S^T,  Z = e^{G_63 - G} N dS'^T,  Y = Z + F^T Q + E^T (beta K);      dK = beta X + Y
//   dbeta = dB.V + K.X,  dG = Q.dQ + beta K.X - K.Y (row by row),  dG_63 += sum K.Z + e^{G_63} <S, dS'>
//
// and the gradient of log_decay is the sum of dG from a position to the chunk's end.  The dots are those of one value head; the gradients of
// q and k are the sums of dQ and dK over the heads that share them.
//
// A workgroup has a (chunk, key head) and walks over the value heads that share it, so that nothing is added by atomics.  Value
// channels come 32 at a time through LDS, the next ones on their way in registers meanwhile.  Its waves have two parts, four waves
// of 16 rows each: dQ and X, which multiply S, and Y, which multiplies dS'.  One wave for all three would hold more than its share of the
// registers (with two numbers an operand 2.4 ms for 8 x 4096, 16 heads of 128 x 128 bf16, what went through scratch cost more than the products), three
// parts read S from LDS twice (0.79 ms); two 0.70 ms.  Now all that is not an input is three numbers (delta_core.hpp), with which two steps
// no longer fit into LDS above 64 key channels: 0.87 to 0.94 ms, for 2.1 GB of states, operands and results (0.42 at the rate of a
// copy).  beta X goes from the one part to the other through LDS, head by head, and is added to Y there, so each part keeps one sum over
// the heads and what its head alone has (with differences of running sums for the latter, which took as long, a small head lost its
// digits).  The 64 x 64 products F, F^T, E, E^T are computed as they are needed as operands: what a lane gets of a product is its part of an
// operand over the product's rows.
#pragma once
#include "delta_prepare.hpp"
#include "delta_scan.hpp"

namespace linrec {

constexpr int GRADIENT_LANES = 512, GRADIENT_PART = 256;

template <typename T, int DK>
struct GradientShared {
  using U = Inner<T>;
  static constexpr int CHAIN = chain_planes<U>(), IN = input_planes<T>();
  static constexpr int IN_V = 64 * 32 * int(sizeof(U)), BY_V = 32 * 64 * int(sizeof(U)), STATE = 32 * DK * int(sizeof(U)),
                       KEYS = Tile<U, DK>::BYTES;
  // one step's values, then both inputs of key channels
  static constexpr int O = 0, V = O + IN * IN_V, B = V + IN * IN_V, N = B + CHAIN * BY_V, S = N + CHAIN * BY_V, D = S + CHAIN * STATE, STEP = D + CHAIN * STATE;
  static constexpr int BUFFERS = 2 * STEP + 2 * IN * KEYS + 4096 <= 160 * 1024 ? 2 : 1;
  static constexpr int K = BUFFERS * STEP, Q = K + IN * KEYS, BYTES = Q + IN * KEYS;
  static_assert(64 * DK * 4 <= STEP, "room to hand beta X over");
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

struct GradientScratch {  // LDS beside GradientShared
  alignas(32) double g[64];
  alignas(16) float gamma[64], rest[64], beta[64], q[64], x[64], y[64], bv[64], sum[8];
};

// An operand with its rows scaled.
template <typename U, int OUT, int N>
__device__ __forceinline__ Planes<U, OUT> scaled(const Planes<U, N>& f, float by) {
  v4f x[2];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v = float(f.p[0][e]);
    if constexpr (N >= 2) v += float(f.p[1][e]);
    if constexpr (N >= 3) v += float(f.p[2][e]);
    x[e >> 2][e & 3] = by * v;
  }
  return split<U, OUT>(x[0], x[1]);
}

// What the waves of one part do: dQ and X, or (BEHIND) Y.  Both parts meet at the same barriers.
template <typename T, int DK, bool WIDE, bool BEHIND>
__device__ __forceinline__ void gradient_part(const DeltaArgs& a, const Chunk& ch, int64_t slot, int key_head, char* smem, GradientScratch& sh) {
  using U = Inner<T>;
  using Sh = GradientShared<T, DK>;
  using TI = Tile<U, 32>;  // dO, V
  using TB = Tile<U, 64>;  // dB, N: rows are channels
  using TK = Tile<U, DK>;  // K, Q; S, dS': rows are channels
  constexpr int CHAIN = Sh::CHAIN, IN = Sh::IN, KT = DK / 16, LANES = GRADIENT_PART;
  constexpr int64_t ROW = WIDE ? 2 * DK : DK;  // of the kept states
  const linrec_delta_t& p = a.p;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4, by0 = threadIdx.x & (LANES - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int rows_w0 = TI::natural_rows(r, q) + wave * (16 * TI::ROW), rows_m0 = TI::mapped_rows(r, q);
  const int cols_w0 = TB::template column_tile<false>(TB::template columns<false>(r, q), wave), cols_m0 = TB::template columns<true>(r, q);
  const int cols_k0 = TK::template columns<false>(r, q), rows_v0 = TK::natural_rows(r, q) + (wave & 1) * (16 * TK::ROW),
            points0 = TK::points(r, q) + wave * (16 * TK::ROW);

  // what a step needs on its way: the rows of dO and V with dB and N, or S and dS'
  InputStager<T, 32, LANES> so, sv;
  SplitStager<U, 64, LANES, 32> sb, sn;
  SplitStager<U, DK, LANES, 32> ss, sd;
  // one wave has what belongs to the positions, a lane for each
  const bool keeper = BEHIND && wave == 0;
  double sum = 0.0;
  float gamma = 0.0f, rest = 0.0f, beta = 0.0f;
  // (loads are issued one part after the other between products; all at once at the step's start 879 us instead of 870)
  constexpr int LOADS = decltype(ss)::N, PARTS = BEHIND ? 2 * LOADS : 4;
  static_assert(decltype(sb)::N == 1, "");
  auto fetch_gates = [&](int head) __attribute__((always_inline)) {
    if (keeper) {
      const int64_t block = slot * p.heads + head;
      const int own = anew(lane);
      sum = a.sums[block * 64 + own];
      gamma = a.gates[block * 192 + own];
      rest = a.gates[block * 192 + 64 + own];
      beta = a.gates[block * 192 + 128 + own];
    }
  };
  auto fetch_part = [&](auto part, int head, int v0, int d0, int by) __attribute__((always_inline)) {
    const int64_t block = slot * p.heads + head;
    if constexpr (!BEHIND) {
      if constexpr (part() == 0) {
        so.fetch(head_rows<T>(p.d_o, p.d_o_stride, ch.batch, ch.first, head) + v0, p.d_o_stride[1], ch.length, p.value_dim - v0, by);
      } else if constexpr (part() == 1) {
        sv.fetch(head_rows<T>(p.v, p.v_stride, ch.batch, ch.first, head) + v0, p.v_stride[1], ch.length, p.value_dim - v0, by);
      } else if constexpr (part() == 2) {
        sb.template fetch_pieces<4>(0, a.d_b + block * a.rows + v0 * 64, 0, by);
      } else {
        sn.template fetch_pieces<4>(0, a.n + block * a.rows + v0 * 64, 0, by);
      }
    } else {
      const float* from = (part() < LOADS ? a.s : a.d_s) + block * a.state + v0 * ROW;
      (part() < LOADS ? ss : sd).template fetch_pieces<int(ROW / 16)>(part() % LOADS, from, WIDE ? d0 / 16 : 0, by);
    }
  };
  auto put = [&](char* to) __attribute__((always_inline)) {
    const int by = anew(by0);
    if constexpr (!BEHIND) {
      so.put(to + Sh::O, by);
      sv.put(to + Sh::V, by);
      sb.put_pieces(to + Sh::B, by);
      sn.put_pieces(to + Sh::N, by);
    } else {
      ss.put_pieces(to + Sh::S, by);
      sd.put_pieces(to + Sh::D, by);
    }
  };

  for (int d0 = 0; d0 < (WIDE ? p.key_dim : 1); d0 += DK) {
    v4f all[KT];  // dQ, or dK, over the value heads
#pragma unroll
    for (int u = 0; u < KT; ++u) all[u] = v4f{0, 0, 0, 0};
    {
      InputStager<T, DK, LANES> keys;
      const T* from = BEHIND ? head_rows<T>(p.q, p.q_stride, ch.batch, ch.first, key_head) : head_rows<T>(p.k, p.k_stride, ch.batch, ch.first, key_head);
      keys.fetch(from + d0, BEHIND ? p.q_stride[1] : p.k_stride[1], ch.length, p.key_dim - d0, by0);
      fetch_gates(key_head * a.shared);
      static_for<PARTS>([&](auto part) __attribute__((always_inline)) { fetch_part(part, key_head * a.shared, 0, d0, anew(by0)); });
      __syncthreads();
      keys.put(smem + (BEHIND ? Sh::Q : Sh::K), by0);
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
      // dQ, or Y, of this head alone (rows are scaled on their way, so that products add to it), which the gates' gradients are dots of: a
      // difference of sums over heads would lose the digits of a small head beside a large one, and all of them beside one that is not finite
      v4f z[KT];
      v4f f[4], ee[4], x[BEHIND ? 1 : KT], bv = v4f{0, 0, 0, 0}, inner = v4f{0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < KT; ++u) z[u] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = ee[t] = v4f{0, 0, 0, 0};
      if constexpr (!BEHIND)
#pragma unroll
        for (int u = 0; u < KT; ++u) x[u] = v4f{0, 0, 0, 0};
      char* at = smem;
      for (int v0 = 0; v0 < p.value_dim; v0 += 32) {
        at = smem + (Sh::BUFFERS == 2 ? turn * Sh::STEP : 0);
        if constexpr (Sh::BUFFERS == 1) __syncthreads();
        put(at);
        __syncthreads();
        turn ^= 1;
        const bool same = v0 + 32 < p.value_dim;
        const int next = same ? head : head + 1, next_v0 = same ? v0 + 32 : 0;
        if (!same && h + 1 < a.shared) fetch_gates(next);
        const bool more = same || h + 1 < a.shared;
        // the parts of a sixth of the step, not before a product is there: at its start, behind F and E, and with the first four column tiles
        auto fetch_beside = [&](auto sixth, v4f& after) __attribute__((always_inline)) {
          if (more) {
            static_for<PARTS>([&](auto part) __attribute__((always_inline)) {
              if constexpr (part() * 6 / PARTS == sixth()) fetch_part(part, next, next_v0, d0, anew_after(by0, after));
            });
          }
        };
        const int rows_w = anew(rows_w0), rows_m = anew(rows_m0), cols_w = anew(cols_w0), cols_m = anew(cols_m0), cols_k = anew(cols_k0),
                  rows_v = anew(rows_v0);
        auto rows_in = [&](int part, int view, int row) __attribute__((always_inline)) {
          Planes<U, IN> out;
#pragma unroll
          for (int k = 0; k < IN; ++k) out.p[k] = TI::frag(at + part + k * Sh::IN_V, view, row, 0);
          return out;
        };
        auto by_v = [&](int part) __attribute__((always_inline)) {  // this wave's rows
          Planes<U, CHAIN> out;
#pragma unroll
          for (int k = 0; k < CHAIN; ++k) out.p[k] = TB::template column_frag<false>(at + part + k * Sh::BY_V, cols_w, 0, 0);
          return out;
        };
        auto by_v_mapped = [&](int part, int t) __attribute__((always_inline)) {
          Planes<U, CHAIN> out;
#pragma unroll
          for (int k = 0; k < CHAIN; ++k) out.p[k] = TB::template column_frag<true>(at + part + k * Sh::BY_V, cols_m, 0, t);
          return out;
        };
        auto state = [&](int part, int u) __attribute__((always_inline)) {
          Planes<U, CHAIN> out;
#pragma unroll
          for (int k = 0; k < CHAIN; ++k) out.p[k] = TK::template column_frag<false>(at + part + k * Sh::STATE, cols_k, 0, u);
          return out;
        };
        const int own = 16 * wave + anew(r);
        fetch_beside(std::integral_constant<int, 0>{}, z[0]);
        if constexpr (!BEHIND) {
          const Planes<U, CHAIN> db_w = by_v(Sh::B);
          const Planes<U, IN> do_w = rows_in(Sh::O, rows_w, 0);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (t / 2 <= wave / 2) {  // rows j of F^T and E^T up to this wave's columns i
              const Planes<U, CHAIN> n_t = by_v_mapped(Sh::N, t);
              f[t] = mma_up_to<2>(n_t, do_w, f[t]);
              ee[t] = mma_up_to<2>(n_t, db_w, ee[t]);
            }
          fetch_beside(std::integral_constant<int, 1>{}, z[0]);
          const Planes<U, CHAIN> do_s = scaled<U, CHAIN>(do_w, p.scale * sh.gamma[own]);
          static_for<KT>([&](auto u) __attribute__((always_inline)) {
            const Planes<U, CHAIN> s_u = state(Sh::S, u);
            // (the products of two rests too: without them the gradients of the gates are 1.2e-6 to 4e-6 off instead of 2e-7 to 7e-7, for 50 of 870 us)
            z[u] = mma_up_to<2>(do_s, s_u, z[u]);
            x[u] = mma_up_to<2>(db_w, s_u, x[u]);
            fetch_beside(std::integral_constant<int, 2 + u()>{}, z[u]);
          });
          bv = mma_up_to<2>(db_w, rows_in(Sh::V, rows_w, 0), bv);
          // <S, dS'> on the diagonal of S^T dS', 16 channels at a time
#pragma unroll
          for (int b = 0; b < DK / 32; ++b)
            if ((b & 1) == wave >> 1) {
              Planes<U, CHAIN> s_v, d_v;
#pragma unroll
              for (int k = 0; k < CHAIN; ++k) {
                s_v.p[k] = TK::frag(at + Sh::S + k * Sh::STATE, rows_v, 0, b);
                d_v.p[k] = TK::frag(at + Sh::D + k * Sh::STATE, rows_v, 0, b);
              }
              inner = mma_up_to<2>(s_v, d_v, inner);
            }
        } else {
          const Planes<U, CHAIN> n_w = by_v(Sh::N);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (t / 2 >= wave / 2) {
              f[t] = mma_up_to<2>(rows_in(Sh::O, rows_m, TI::mapped_row(t)), n_w, f[t]);
              ee[t] = mma_up_to<2>(by_v_mapped(Sh::B, t), n_w, ee[t]);
            }
          fetch_beside(std::integral_constant<int, 1>{}, z[0]);
          const Planes<U, CHAIN> n_s = scaled<U, CHAIN>(n_w, sh.rest[own]);
          static_for<KT>([&](auto u) __attribute__((always_inline)) {
            z[u] = mma(n_s, state(Sh::D, u), z[u]);
            fetch_beside(std::integral_constant<int, 2 + u()>{}, z[u]);
          });
        }
      }
      int cols_k = anew(cols_k0), points = anew(points0);
      const int r1 = anew(r), row1 = 16 * wave + 4 * anew(q);
      // the masks and decays; rows of results to operands
      Planes<U, CHAIN> fp[2];
      Planes<U, CHAIN> ep[2];
      {
        // (all reads ahead of what they are compared for: a read that waits in a branch of its own costs its latency, 16 times over)
        typedef double v4d __attribute__((ext_vector_type(4)));
        const int own = 16 * wave + anew(r), q1 = anew(q);
        const double g_own = sh.g[own];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int first = row_of_result(t, q1);
          const v4d g_other = *reinterpret_cast<const v4d*>(sh.g + first);
          const v4f beta_of = BEHIND ? *reinterpret_cast<const v4f*>(sh.beta + first) : v4f{1, 1, 1, 1};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = BEHIND ? first + e : own, j = BEHIND ? own : first + e;
            const float apart = float(BEHIND ? g_other[e] - g_own : g_own - g_other[e]);
            const float d = fast_exp(i >= j ? apart : -__builtin_inff());
            f[t][e] = i >= j ? p.scale * d * f[t][e] : 0.0f;
            ee[t][e] = i > j ? -beta_of[e] * d * ee[t][e] : 0.0f;
          }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          fp[b] = split<U, CHAIN>(f[2 * b], f[2 * b + 1]);
          ep[b] = split<U, CHAIN>(ee[2 * b], ee[2 * b + 1]);
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
      v4f dot = v4f{0, 0, 0, 0}, dot_x = v4f{0, 0, 0, 0}, ends = v4f{0, 0, 0, 0};
      const v4f down = -*reinterpret_cast<const v4f*>(sh.gamma + row1), beta_of = *reinterpret_cast<const v4f*>(sh.beta + row1);
#pragma unroll
      for (int u = 0; u < KT; ++u) {
        const v4f kv = values(Sh::K, u);
        if constexpr (!BEHIND) {
          const v4f qv = values(Sh::Q, u);
          v4f xu = down * x[u];
#pragma unroll
          for (int b = 0; b < 2; ++b)
            if (b <= wave / 2) {
              const Planes<U, IN> k_b = keys(Sh::K, b, u);
              z[u] = mma_up_to<2>(fp[b], k_b, z[u]);
              xu = mma_up_to<2>(ep[b], k_b, xu);
            }
          dot += qv * z[u];
          dot_x += kv * xu;
          x[u] = beta_of * xu;
        } else {
          ends += kv * z[u];
#pragma unroll
          for (int b = 0; b < 2; ++b)
            if (b >= wave / 2) {
              z[u] = mma_up_to<2>(fp[b], keys(Sh::Q, b, u), z[u]);
              z[u] = mma_up_to<2>(ep[b], keys(Sh::K, b, u), z[u]);
            }
          dot += kv * z[u];
        }
        // (reads of the next columns, all ahead of their products, would push other values out of the registers)
        if constexpr (!BEHIND) {
          points = anew_after(points, dot);
          cols_k = anew_after(cols_k, z[u]);
        }
        all[u] += z[u];
      }
      float* to = BEHIND ? sh.y : sh.q;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = sum_of_16(dot[e]);
        if (r1 == 0) to[row1 + e] = d;
        if constexpr (!BEHIND) {
          const float dx = sum_of_16(dot_x[e]);
          if (r1 == 0) sh.x[row1 + e] = dx;
        }
      }
      // sum K.Z, or (on the diagonal, lane 16 q + 4 q + e, where dB.V stands too) <S, dS'>
      float whole = 0.0f;
      if constexpr (BEHIND) {
        whole = (ends[0] + ends[1]) + (ends[2] + ends[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (r1 == row1 - 16 * wave + e) {
            sh.bv[row1 + e] = bv[e];
            whole = sh.gamma[63] * inner[e];
          }
      }
      whole = sum_of_16(whole);
      whole += __shfl_xor(whole, 16);
      whole += __shfl_xor(whole, 32);
      if (lane == 0) sh.sum[BEHIND ? 4 + wave : wave] = whole;
      __syncthreads();
      // beta X for the other part's dK, to the wave and lane that have the same rows and columns, through what was this step's place (nobody
      // reads it any more, and it is written next behind a barrier more)
      v4f* hand = reinterpret_cast<v4f*>(at) + wave * 64 + anew(lane);
      if constexpr (!BEHIND)
#pragma unroll
        for (int u = 0; u < KT; ++u) hand[u * 256] = x[u];
      __syncthreads();
      if constexpr (BEHIND)
#pragma unroll
        for (int u = 0; u < KT; ++u) all[u] += hand[u * 256];
      if (keeper) {
        const int own = anew(lane);
        float* dots = a.dots + block * 192;  // (every place is written and read by one lane)
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
    const int r2 = anew(r), row2 = 16 * wave + 4 * anew(q);
    T* to = static_cast<T*>(BEHIND ? p.d_k : p.d_q);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (row2 + e < ch.length) {
        const int64_t at = ((ch.batch * p.time + ch.first + row2 + e) * p.key_heads + key_head) * int64_t(p.key_dim) + d0;
#pragma unroll
        for (int u = 0; u < KT; ++u)
          if (d0 + 16 * u + r2 < p.key_dim) to[at + 16 * u + r2] = T(all[u][e]);
      }
  }
}

// DK: columns of dQ and dK at a time; WIDE: key_dim is more than that and they come in turns.
template <typename T, int DK, bool WIDE>
__global__ __launch_bounds__(GRADIENT_LANES) void delta_gradient_kernel(DeltaArgs a) {
  __shared__ __align__(16) char smem[GradientShared<T, DK>::BYTES];
  __shared__ GradientScratch sh;
  const int64_t slot = blockIdx.x / unsigned(a.p.key_heads);
  const int key_head = int(blockIdx.x - slot * unsigned(a.p.key_heads));
  const Chunk ch = chunk_of(a.p, slot);
  if (ch.length == 0) return;
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 8) == 0) gradient_part<T, DK, WIDE, false>(a, ch, slot, key_head, smem, sh);
  else gradient_part<T, DK, WIDE, true>(a, ch, slot, key_head, smem, sh);
}

}  // namespace linrec
