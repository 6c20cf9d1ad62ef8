// Gated delta rule, the pass along the sequence: N, O and the state, chunk by chunk (delta_core.hpp).
//
// A workgroup has a (sequence, head), or a segment of one (delta_segments.hpp), and 16 columns of the state for each of half of its waves; the
// other half loads what the next chunk needs into LDS meanwhile (a state's chunks follow one another, so nothing else hides those loads: 310 us
// with them, 420 without, when Q S was not taken beside K S; where two chunks do not fit into LDS all waves load first and compute then).
//
// 8 x 4096, 16 heads of 128 x 128 bf16: 325 us with O and 255 with the states, for 0.60 and 1.11 GB (118 and 217 us at the rate of a copy).  A chunk
// is a chain of products by one wave of a SIMD: 216 matrix instructions of 16 cycles, 37 % of its cycles.
#pragma once
#include "delta_core.hpp"

namespace linrec {

enum ScanMode {
  SCAN_OUT,     // the forward: O and the last state
  SCAN_STATES,  // a backward's first pass, which keeps the states before the chunks and N and has no O
  SCAN_CARRY,   // what a segment makes of nothing, and of the unit matrix (where V is zero)
};

template <typename T, int DK, int WAVES, ScanMode MODE>
struct ScanShared {
  static constexpr bool STATES = MODE != SCAN_OUT;
  using U = Inner<T>;
  static constexpr int KEYS = Tile<T, DK>::BYTES, VALUES = Tile<T, 16 * WAVES>::BYTES, SQUARE = triangle_bytes<U>(), GATE_BYTES = 3 * 64 * 4;
  // (fp32 of 256 channels: queries are read from memory where they are used)
  static constexpr bool QUERIES = !STATES && 2 * KEYS + VALUES + 2 * SQUARE + GATE_BYTES <= 160 * 1024;
  static constexpr int K = 0, Q = K + KEYS, V = Q + (QUERIES ? KEYS : 0), M = V + VALUES, C = M + SQUARE, GATES = C + (STATES ? 0 : SQUARE), BYTES = GATES + GATE_BYTES;
  static constexpr bool LOADERS = 2 * BYTES <= 160 * 1024;
  static constexpr int LANES = 64 * WAVES * (LOADERS ? 2 : 1);
};

// Where a lane's part of a state lies that is kept as [columns][DK].
template <int DK>
__device__ __forceinline__ void load_columns(const float* from, int q, v4f (&s)[DK / 16]) {
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) s[t] = *reinterpret_cast<const v4f*>(from + row_of_result(t, q));
}
template <int DK>
__device__ __forceinline__ void store_columns(float* to, int q, const v4f (&s)[DK / 16]) {
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) *reinterpret_cast<v4f*>(to + row_of_result(t, q)) = s[t];
}

template <typename T, int DK, int WAVES, ScanMode MODE>
__global__ __launch_bounds__((ScanShared<T, DK, WAVES, MODE>::LANES)) void delta_scan_kernel(DeltaArgs a) {
  using U = Inner<T>;
  using Sh = ScanShared<T, DK, WAVES, MODE>;
  using TK = Tile<T, DK>;
  using TV = Tile<T, 16 * WAVES>;
  constexpr int CHAIN = chain_planes<U>(), STAGING = 64 * WAVES;
  __shared__ __align__(16) char room[Sh::BYTES * (Sh::LOADERS ? 2 : 1)];
  const linrec_delta_t& p = a.p;
  int64_t pair;
  int cb;
  if (!scan_place(a, MODE == SCAN_CARRY ? a.blocks + DK / (16 * WAVES) : a.blocks, &pair, &cb)) return;
  const int64_t place = pair / p.heads;
  const int head = int(pair - place * p.heads), key_head = head / a.shared;
  const Part part = part_of(a, place);
  if (part.count == 0 || (MODE == SCAN_CARRY && part.count == 1)) return;
  const Span span = part.span;
  const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
  const bool loader = Sh::LOADERS && __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) >= WAVES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - (loader ? WAVES : 0);
  const bool unit = MODE == SCAN_CARRY && cb >= a.blocks;  // columns of the unit matrix
  const int c0 = (unit ? cb - a.blocks : cb) * 16 * WAVES, col = c0 + 16 * wave + r;
  const bool mine = col < p.value_dim, kept_column = col < a.columns;  // (of a whole wave)

  auto load = [&](int64_t c, char* smem) __attribute__((always_inline)) {
    const int64_t first = span.first + c * DELTA_CHUNK, block = (span.slot + c) * p.heads + head;
    const int length = int(span.end - first < DELTA_CHUNK ? span.end - first : DELTA_CHUNK), by = wave * 64 + lane;
    Stager<T, DK, STAGING> k, qq;
    Stager<T, 16 * WAVES, STAGING> v;
    TriangleStager<U, false, STAGING> m, cc;
    float gate[(192 + STAGING - 1) / STAGING];
    k.fetch(head_rows<T>(p.k, p.k_stride, span.batch, first, key_head), p.k_stride[1], length, p.key_dim, by);
    if constexpr (Sh::QUERIES) qq.fetch(head_rows<T>(p.q, p.q_stride, span.batch, first, key_head), p.q_stride[1], length, p.key_dim, by);
    if (!unit) v.fetch(head_rows<T>(p.v, p.v_stride, span.batch, first, head) + c0, p.v_stride[1], length, p.value_dim - c0, by);
    else v.clear();
    m.fetch(a.m + block * 4096, by);
    if constexpr (MODE == SCAN_OUT) cc.fetch(a.c + block * 4096, by);
#pragma unroll
    for (int i = 0; i < (192 + STAGING - 1) / STAGING; ++i)
      if (i * STAGING + by < 192) gate[i] = a.gates[block * 192 + i * STAGING + by];
    k.put(smem + Sh::K, by);
    if constexpr (Sh::QUERIES) qq.put(smem + Sh::Q, by);
    v.put(smem + Sh::V, by);
    m.put(smem + Sh::M, by);
    if constexpr (MODE == SCAN_OUT) cc.put(smem + Sh::C, by);
#pragma unroll
    for (int i = 0; i < (192 + STAGING - 1) / STAGING; ++i)
      if (i * STAGING + by < 192) reinterpret_cast<float*>(smem + Sh::GATES)[i * STAGING + by] = gate[i];
  };

  v4f s[DK / 16];
  const int64_t at0 = ((part.n * p.heads + head) * p.key_dim) * int64_t(p.value_dim) + col;
#pragma unroll
  for (int t = 0; t < DK / 16; ++t) s[t] = v4f{0, 0, 0, 0};
  if (loader) {
  } else if constexpr (MODE == SCAN_CARRY) {
    if (unit)
#pragma unroll
      for (int t = 0; t < DK / 16; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = row_of_result(t, q) + e == col ? 1.0f : 0.0f;
  } else if (a.segment) {
    if (kept_column) load_columns<DK>(a.start + (pair * a.columns + col) * DK, q, s);
  } else if (p.h0 && mine) {
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = row_of_result(t, q) + e;
        if (d < p.key_dim) s[t][e] = p.h0[at0 + d * int64_t(p.value_dim)];
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
    if constexpr (MODE == SCAN_STATES) {
      float* to = a.s + block * a.state + int64_t(col - r) * DK;
#pragma unroll
      for (int b = 0; b < DK / 32; ++b)
        if (kept_column) store_rows(to, b, lane, s[2 * b], s[2 * b + 1]);
    }
    v4f x[4], y[4];  // K S, then beta (V - e^G K S); Q S, then O
#pragma unroll
    for (int t = 0; t < 4; ++t) x[t] = y[t] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < DK / 32; ++b) {
      Frag<T> f[4], g[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        f[t] = TK::frag(smem + Sh::K, rows_k, TK::mapped_row(t), b);
        if constexpr (MODE != SCAN_OUT) {
        } else if constexpr (Sh::QUERIES) {
          g[t] = TK::frag(smem + Sh::Q, rows_k, TK::mapped_row(t), b);
        } else {
          const int from = row_of_tile(t, r);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[t][e] = from < length && 32 * b + 8 * q + e < p.key_dim ? qq[from * p.q_stride[1] + 32 * b + 8 * q + e] : T(0.0f);
        }
      }
      auto with = [&](const auto& planes) __attribute__((always_inline)) {
        mma_tiles<0, 4>(f, planes, x);
        if constexpr (MODE == SCAN_OUT) mma_tiles<0, 4>(g, planes, y);
      };
      if constexpr (std::is_same_v<T, __bf16>) with(third_plane(s[2 * b], s[2 * b + 1], sp[b]));
      with(sp[b]);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const auto v = TV::template column4<false>(smem + Sh::V, cols_v, TK::mapped_row(t), 0);
      const v4f gamma = four(0, t), beta = four(2, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[t][e] = beta[e] * fmaf(-gamma[e] * un_s, x[t][e], float(v[e]));
    }
    Planes<U, CHAIN> xp[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) xp[b] = split<U, CHAIN>(x[2 * b], x[2 * b + 1]);
    v4f nn[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) nn[t] = v4f{0, 0, 0, 0};
    mma_triangle<false>(smem + Sh::M, rows_s, xp, nn);
    if constexpr (MODE == SCAN_CARRY) {
    } else if constexpr (MODE == SCAN_STATES) {
      float* to = a.n + block * a.rows + (col - r) * 64;
#pragma unroll
      for (int b = 0; b < 2; ++b)
        if (kept_column) store_rows(to, b, lane, nn[2 * b], nn[2 * b + 1]);
    } else {
      T* o = static_cast<T*>(p.o) + ((span.batch * p.time + first) * p.heads + head) * int64_t(p.value_dim) + col;
#pragma unroll
      for (int t = 0; t < 4; ++t) y[t] *= four(0, t) * (un_s * p.scale);
      Planes<U, CHAIN> np[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) np[b] = split<U, CHAIN>(nn[2 * b], nn[2 * b + 1]);
      mma_triangle<false>(smem + Sh::C, rows_s, np, y);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int row = row_of_result(t, q);
        T* to = o + row * int64_t(p.heads) * p.value_dim;
        if (length == DELTA_CHUNK) {
          if (mine)
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e * (p.heads * p.value_dim)] = T(y[t][e]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (mine && row + e < length) to[e * (p.heads * p.value_dim)] = T(y[t][e]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) nn[t] *= four(1, t);
    Planes<T, chain_planes<T>()> nt[2];
    float un_n;
    split_scaled(nn, nt, &un_n);
    const float keep = gates[63];
#pragma unroll
    for (int t0 = 0; t0 < DK / 16; t0 += 4) {
      v4f to[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) to[t] = std::is_same_v<T, _Float16> ? v4f{0, 0, 0, 0} : s[t0 + t] * keep;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        Frag<T> f[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) f[t] = TK::template column_frag<true>(smem + Sh::K, cols_k, b, t0 + t);
        mma_tiles<0, 4>(f, nt[b], to);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) s[t0 + t] = std::is_same_v<T, _Float16> ? s[t0 + t] * keep + un_n * to[t] : to[t];
    }
  };

  if constexpr (Sh::LOADERS) {
    if (loader && part.begin < part.end) load(part.begin, room);
    __syncthreads();
    int turn = 0;
    for (int64_t c = part.begin; c < part.end; ++c, turn ^= 1) {
      if (!loader) compute(c, room + turn * Sh::BYTES);
      else if (c + 1 < part.end) load(c + 1, room + (turn ^ 1) * Sh::BYTES);
      __syncthreads();
    }
  } else {
    for (int64_t c = part.begin; c < part.end; ++c) {
      __syncthreads();
      load(c, room);
      __syncthreads();
      compute(c, room);
    }
  }
  if (loader) return;
  if constexpr (MODE == SCAN_CARRY) {
    if (unit || kept_column) store_columns<DK>(a.carry + (pair * (a.columns + DK) + (unit ? a.columns : 0) + col) * DK, q, s);
  } else if (MODE == SCAN_OUT && p.state && mine && part.index == part.count - 1) {
#pragma unroll
    for (int t = 0; t < DK / 16; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = row_of_result(t, q) + e;
        if (d < p.key_dim) p.state[at0 + d * int64_t(p.value_dim)] = s[t][e];
      }
  }
}

}  // namespace linrec
