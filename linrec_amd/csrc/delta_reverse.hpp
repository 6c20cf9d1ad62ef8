// Gated delta rule, the backward's pass against the sequence: dV, dB and the gradient of the state, chunk by chunk (delta_core.hpp).
//
// As the forward's: a workgroup has a (sequence, head), a wave of its first half 16 columns of dS, and the other half loads.
//
// 8 x 4096, 16 heads of 128 x 128 bf16: 430 us for 1.41 GB (276 us at the rate of a copy); without waves that load 560.
#pragma once
#include "delta_scan.hpp"

namespace linrec {

template <typename T, int DK, int WAVES>
struct ReverseShared {
  using U = Inner<T>;
  static constexpr int KEYS = Tile<T, DK>::BYTES, VALUES = Tile<T, 16 * WAVES>::BYTES, SQUARE = triangle_bytes<U>(), GATE_BYTES = 3 * 64 * 4;
  static constexpr bool QUERIES = 2 * KEYS + VALUES + 2 * SQUARE + GATE_BYTES <= 160 * 1024;
  static constexpr int K = 0, Q = K + KEYS, O = Q + (QUERIES ? KEYS : 0), M = O + VALUES, C = M + SQUARE, GATES = C + SQUARE, BYTES = GATES + GATE_BYTES;
  static constexpr bool LOADERS = 2 * BYTES <= 160 * 1024;
  static constexpr int LANES = 64 * WAVES * (LOADERS ? 2 : 1);
};

// CARRY: only what a segment adds to the gradient of the state before it, for delta_segments.hpp.
template <typename T, int DK, int WAVES, bool CARRY>
__global__ __launch_bounds__((ReverseShared<T, DK, WAVES>::LANES)) void delta_reverse_kernel(DeltaArgs a) {
  using U = Inner<T>;
  using Sh = ReverseShared<T, DK, WAVES>;
  using TK = Tile<T, DK>;
  using TV = Tile<T, 16 * WAVES>;
  constexpr int CHAIN = chain_planes<U>(), STAGING = 64 * WAVES, IN = input_planes<T>();
  __shared__ __align__(16) char room[Sh::BYTES * (Sh::LOADERS ? 2 : 1)];
  const linrec_delta_t& p = a.p;
  int64_t pair;
  int cb;
  if (!scan_place(a, a.blocks, &pair, &cb)) return;
  const int64_t place = pair / p.heads;
  const int head = int(pair - place * p.heads), key_head = head / a.shared;
  const Part part = part_of(a, place);
  if (part.count == 0 || (CARRY && part.count == 1)) return;
  const Span span = part.span;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const bool loader = Sh::LOADERS && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= WAVES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - (loader ? WAVES : 0);
  const int c0 = cb * 16 * WAVES, col = c0 + 16 * wave + r;
  const bool mine = col < p.value_dim, kept_column = col < a.columns;  // (of a whole wave)

  auto load = [&](int64_t c, char* smem) __attribute__((always_inline)) {
    const int64_t first = span.first + c * DELTA_CHUNK, block = (span.slot + c) * p.heads + head;
    const int length = int(span.end - first < DELTA_CHUNK ? span.end - first : DELTA_CHUNK), by = wave * 64 + lane;
    Stager<T, DK, STAGING> k, qq;
    Stager<T, 16 * WAVES, STAGING> o;
    TriangleStager<U, true, STAGING> m, cc;
    float gate[(192 + STAGING - 1) / STAGING];
    k.fetch(head_rows<T>(p.k, p.k_stride, span.batch, first, key_head), p.k_stride[1], length, p.key_dim, by);
    if constexpr (Sh::QUERIES) qq.fetch(head_rows<T>(p.q, p.q_stride, span.batch, first, key_head), p.q_stride[1], length, p.key_dim, by);
    o.fetch(head_rows<T>(p.d_o, p.d_o_stride, span.batch, first, head) + c0, p.d_o_stride[1], length, p.value_dim - c0, by);
    m.fetch(a.m_t + block * 4096, by);
    cc.fetch(a.c + block * 4096, by);
#pragma unroll
    for (int i = 0; i < (192 + STAGING - 1) / STAGING; ++i)
      if (i * STAGING + by < 192) gate[i] = a.gates[block * 192 + i * STAGING + by];
    k.put(smem + Sh::K, by);
    if constexpr (Sh::QUERIES) qq.put(smem + Sh::Q, by);
    o.put(smem + Sh::O, by);
    m.put(smem + Sh::M, by);
    cc.put(smem + Sh::C, by);
#pragma unroll
    for (int i = 0; i < (192 + STAGING - 1) / STAGING; ++i)
      if (i * STAGING + by < 192) reinterpret_cast<float*>(smem + Sh::GATES)[i * STAGING + by] = gate[i];
  };

  v4f s[DK / 16];  // dS'
  const int64_t at0 = ((part.n * p.heads + head) * p.key_dim) * int64_t(p.value_dim) + col;
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) s[t] = v4f{0, 0, 0, 0};
  if (loader || CARRY) {
  } else if (a.segment) {
    if (kept_column) load_columns<DK>(a.start + (pair * a.columns + col) * DK, q, s);
  } else if (p.d_state && mine) {
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = row_of_result(t, q) + e;
        if (d < p.key_dim) s[t][e] = p.d_state[at0 + d * int64_t(p.value_dim)];
      }
  }

  const int rows_k = TK::mapped_rows(r, q), rows_s = Tile<U, 32>::mapped_rows(r, q), cols_k = TK::template columns<true>(r, q),
            cols_v = TV::template column_tile<false>(TV::template columns<false>(r, q), wave);
  auto compute = [&](int64_t c, const char* smem) __attribute__((always_inline)) {
    const int64_t first = span.first + c * DELTA_CHUNK, block = (span.slot + c) * p.heads + head;
    const int length = int(span.end - first < DELTA_CHUNK ? span.end - first : DELTA_CHUNK);
    const float* gates = reinterpret_cast<const float*>(smem + Sh::GATES);
    auto four = [&](int kind, int t) __attribute__((always_inline)) { return *reinterpret_cast<const v4f*>(gates + kind * 64 + row_of_result(t, q)); };
    const T* qq = head_rows<T>(p.q, p.q_stride, span.batch, first, key_head);
    Planes<T> sp[DK / 32];
    float un_s;
    split_scaled(s, sp, &un_s);
    if constexpr (!CARRY) {
      float* to = a.d_s + block * a.state + int64_t(col - r) * DK;
#pragma unroll
      for (int b = 0; b < DK / 32; ++b)
        if (kept_column) store_rows(to, b, lane, s[2 * b], s[2 * b + 1]);
    }
    // dO of this wave's columns, a result's layout; fp16 as two bf16
    v4f d_o[4];
    Planes<U, IN> dop[2];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const auto v = TV::template column4<false>(smem + Sh::O, cols_v, TK::mapped_row(t), 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d_o[t][e] = float(v[e]);
        const int i = 4 * (t & 1) + e;
        dop[t >> 1].p[0][i] = U(d_o[t][e]);
        if constexpr (IN == 2) dop[t >> 1].p[1][i] = U(d_o[t][e] - float(dop[t >> 1].p[0][i]));
      }
    }
    v4f x[4];  // dN
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < DK / 32; ++b) {
      Frag<T> f[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = TK::frag(smem + Sh::K, rows_k, TK::mapped_row(t), b);
      if constexpr (std::is_same_v<T, __bf16>) mma_tiles<0, 4>(f, third_plane(s[2 * b], s[2 * b + 1], sp[b]), x);
      mma_tiles<0, 4>(f, sp[b], x);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] *= four(1, t) * un_s;
    mma_triangle<true>(smem + Sh::C, rows_s, dop, x);
    Planes<U, CHAIN> xp[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) xp[b] = split<U, CHAIN>(x[2 * b], x[2 * b + 1]);
    v4f db[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) db[t] = v4f{0, 0, 0, 0};
    mma_triangle<true>(smem + Sh::M, rows_s, xp, db);
    if (!CARRY && kept_column) {
      float* to = a.d_b + block * a.rows + (col - r) * 64;
#pragma unroll
      for (int b = 0; b < 2; ++b) store_rows(to, b, lane, db[2 * b], db[2 * b + 1]);
    }
    const int apart = p.heads * p.value_dim;
    T* d_v = static_cast<T*>(p.d_v) + ((span.batch * p.time + first) * p.heads + head) * int64_t(p.value_dim) + col;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int row = row_of_result(t, q);
      const v4f gamma = four(0, t), beta = four(2, t);
      T* to = d_v + row * int64_t(apart);
#pragma unroll
      for (int e = 0; e < 4; ++e) db[t][e] *= beta[e];
      if constexpr (CARRY) {
      } else if (length == DELTA_CHUNK) {
        if (mine)
#pragma unroll
          for (int e = 0; e < 4; ++e) to[e * apart] = T(db[t][e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (mine && row + e < length) to[e * apart] = T(db[t][e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        db[t][e] *= -gamma[e];
        d_o[t][e] *= gamma[e] * p.scale;
      }
    }
    Planes<T, chain_planes<T>()> vp[2], op[2];
    float un_v, un_o;
    split_scaled(db, vp, &un_v);
    split_scaled(d_o, op, &un_o);
    const float keep = gates[63];
#pragma unroll
    for (int t = 0; t < DK / 16; ++t) {
      auto with_keys = [&](v4f to) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; ++b) to = mma(TK::template column_frag<true>(smem + Sh::K, cols_k, b, t), vp[b], to);
        return to;
      };
      auto with_queries = [&](v4f to) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if constexpr (Sh::QUERIES) {
            to = mma(TK::template column_frag<true>(smem + Sh::Q, cols_k, b, t), op[b], to);
          } else {
            Frag<T> f;
            const int d = row_of_tile(t, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int row = 32 * b + 8 * q + e;
              f[e] = row < length && d < p.key_dim ? qq[row * p.q_stride[1] + d] : T(0.0f);
            }
            to = mma(f, op[b], to);
          }
        }
        return to;
      };
      s[t] *= keep;
      if constexpr (std::is_same_v<T, _Float16>) {
        s[t] += un_v * with_keys(v4f{0, 0, 0, 0});
        s[t] += un_o * with_queries(v4f{0, 0, 0, 0});
      } else {
        s[t] = with_queries(with_keys(s[t]));
      }
    }
  };

  if constexpr (Sh::LOADERS) {
    if (loader && part.begin < part.end) load(part.end - 1, room);
    __syncthreads();
    int turn = 0;
    for (int64_t c = part.end - 1; c >= part.begin; --c, turn ^= 1) {
      if (!loader) compute(c, room + turn * Sh::BYTES);
      else if (c > part.begin) load(c - 1, room + (turn ^ 1) * Sh::BYTES);
      __syncthreads();
    }
  } else {
    for (int64_t c = part.end - 1; c >= part.begin; --c) {
      __syncthreads();
      load(c, room);
      __syncthreads();
      compute(c, room);
    }
  }
  if (loader) return;
  if constexpr (CARRY) {
    if (kept_column) store_columns<DK>(a.carry + (pair * (a.columns + DK) + col) * DK, q, s);
  } else if (p.d_h0 && mine && part.index == 0) {
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = row_of_result(t, q) + e;
        if (d < p.key_dim) p.d_h0[at0 + d * int64_t(p.value_dim)] = s[t][e];
      }
  }
}

}  // namespace linrec
