// What the kernels of the gated delta rule share: the chunk form, fragments of the matrix instructions, tiles in LDS, scratch.
//
// The recurrence S_t = e^{g_t} S_{t-1} + k_t u_t^T, u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t), o_t = scale S_t^T q_t is taken 64
// positions at a time.  With G the sums of g from the chunk's start (inclusive) and S the state before the chunk,
//
//   A_ij = beta_i e^{G_i - G_j} k_i.k_j (i > j)       M = (1 + A)^-1                              delta_prepare.hpp
//   N = M diag(beta) (V - e^G K S)                     the rows u_t of the chunk                   delta_scan.hpp
//   O = scale (e^G Q S + C N), C_ij = e^{G_i - G_j} q_i.k_j (i >= j);   S' = e^{G_63} S + K^T (e^{G_63 - G} N)
//
// and backwards, from dS' behind the chunk,
//
//   dN = scale C^T dO + e^{G_63 - G} K dS',  dB = M^T dN,  dV = beta dB                            delta_reverse.hpp
//   dS = e^{G_63} dS' + Q^T (scale e^G dO) - K^T (e^G dV)
//   the gradients of Q, K and the gates from S, dS', N, dB and dO, chunk by chunk                  delta_gradient.hpp
//
// The columns of S (value channels) are independent of each other in the two passes along the sequence, so a wave owns 16 of them for all
// of the time axis and keeps its key_dim x 16 part of S in accumulators; what it multiplies them with is the same for all waves and
// comes through LDS.
//
// Precision.  States, sums and accumulators are fp32, and so is all that one kernel leaves to another.  An operand of a matrix instruction
// that is not an input is split into bf16 (or, beside fp16 inputs, fp16) numbers, its rounding, the rounding of the rest and so on: three bf16
// carry 24 bits, two fp16 22.  So results in fp32 are as near as sums in fp32 are, 1e-7 to 7e-7, and those in 16 bits are their roundings.  (With M, C, dB and,
// above 64 key channels, the kept S and dS' in two bf16, 16 to 17 bits, states were 2e-6 off, the gradient of beta 4e-6 and that of log_decay 5e-6; with N and S in two where
// O is concerned O was 4e-6 off before its rounding, for 5 of 325 us of 8 x 4096, 16 heads of 128 x 128.)  fp32 inputs take the fp32 instructions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/linrec_delta.h"
#include "layer_common.hpp"

namespace linrec {

constexpr int DELTA_CHUNK = 64;
constexpr float DELTA_LEAST_LOG = -1e4f;  // e^-10000 is zero, and sums of 64 of them keep their digits in fp64

// Type of operands that are computed: T for fp32, bf16 numbers for 16-bit inputs.
template <typename T>
using Inner = std::conditional_t<sizeof(T) == 4, float, __bf16>;
template <typename U>
constexpr int planes_of() {
  return sizeof(U) == 4 ? 1 : 2;
}
// Planes of Inner<T> that hold a T exactly: fp16 has three bits more than bf16.
template <typename T>
constexpr int input_planes() {
  return std::is_same_v<T, _Float16> ? 2 : 1;
}

// e^x; the rounding of x log2(e) is |x| 2^-24 of the result, no more than 2^-25 of one.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// Sum over 16 neighbouring lanes, in each of them.
__device__ __forceinline__ float sum_of_16(float x) {
  auto turned = [&](auto n) __attribute__((always_inline)) {  // lane l has lane l - n of its 16
    return __uint_as_float(unsigned(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(x)), 0x120 + n(), 0xf, 0xf, true)));
  };
  x += turned(std::integral_constant<int, 8>{});
  x += turned(std::integral_constant<int, 4>{});
  x += turned(std::integral_constant<int, 2>{});
  return x + turned(std::integral_constant<int, 1>{});
}

// Eight of the 32 positions that a product sums over at once, for one row (or column): lane 16 q + r holds positions 8 q to 8 q + 7
// of row r.
template <typename U>
using Frag = typename Pack<U, 8>::type;
template <typename U, int N = planes_of<U>()>
struct Planes {
  Frag<U> p[N];
};

// c += a b^T: lane 16 q + r gets rows 4 q to 4 q + 3 of column r.
__device__ __forceinline__ v4f mma(const Frag<__bf16>& a, const Frag<__bf16>& b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(const Frag<_Float16>& a, const Frag<_Float16>& b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma(const Frag<float>& a, const Frag<float>& b, v4f c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}
// MOST: planes whose numbers add up to more than this are left out, the product of two rests where both operands have two.
template <int MOST, typename U, int NA, int NB>
__device__ __forceinline__ v4f mma_up_to(const Planes<U, NA>& a, const Planes<U, NB>& b, v4f c) {
#pragma unroll
  for (int i = NA - 1; i >= 0; --i)
#pragma unroll
    for (int j = NB - 1; j >= 0; --j)
      if (i + j <= MOST) c = mma(a.p[i], b.p[j], c);
  return c;
}
template <typename U, int NA, int NB>
__device__ __forceinline__ v4f mma(const Planes<U, NA>& a, const Planes<U, NB>& b, v4f c) {
  return mma_up_to<(NA > NB ? NA : NB) - 1>(a, b, c);
}
template <typename U, int N>
__device__ __forceinline__ v4f mma(const Frag<U>& a, const Planes<U, N>& b, v4f c) {
#pragma unroll
  for (int j = N - 1; j >= 0; --j) c = mma(a, b.p[j], c);
  return c;
}

// The same for several tiles: one instruction of each before the next of any, whose results it would wait for.  COUNT tiles from FIRST.
template <int FIRST, int COUNT, typename U, int NB, int N>
__device__ __forceinline__ void mma_tiles(const Frag<U> (&a)[N], const Planes<U, NB>& b, v4f* c) {
#pragma unroll
  for (int j = NB - 1; j >= 0; --j)
#pragma unroll
    for (int t = FIRST; t < FIRST + COUNT; ++t) c[t] = mma(a[t], b.p[j], c[t]);
}
template <int FIRST, int COUNT, int MOST = -1, typename U, int NA, int NB, int N>
__device__ __forceinline__ void mma_tiles(const Planes<U, NA> (&a)[N], const Planes<U, NB>& b, v4f* c) {
#pragma unroll
  for (int i = NA - 1; i >= 0; --i)
#pragma unroll
    for (int j = NB - 1; j >= 0; --j)
      if (i + j <= (MOST >= 0 ? MOST : (NA > NB ? NA : NB) - 1))
#pragma unroll
        for (int t = FIRST; t < FIRST + COUNT; ++t) c[t] = mma(a[t].p[i], b.p[j], c[t]);
}

// Results of two products side by side are one operand of the next.  Row r of tile t of an operand whose products' rows are summed
// over next stands for row_of_tile(t, r): then lane 16 q + r holds, of tiles 2 p and 2 p + 1, rows 32 p + 8 q to 32 p + 8 q + 7.
__device__ __forceinline__ int row_of_tile(int t, int r) { return 32 * (t >> 1) + 8 * (r >> 2) + 4 * (t & 1) + (r & 3); }
__device__ __forceinline__ int row_of_result(int t, int q) { return 32 * (t >> 1) + 8 * q + 4 * (t & 1); }  // (the first of four)

template <typename U, int N = planes_of<U>()>
__device__ __forceinline__ Planes<U, N> split(const v4f& lo, const v4f& hi) {
  Planes<U, N> out;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x = e < 4 ? lo[e & 3] : hi[e & 3];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      out.p[k][e] = U(x);
      if (k + 1 < N) x -= float(out.p[k][e]);
    }
  }
  return out;
}
// Planes of an operand in the chain of products of a state.
template <typename U>
constexpr int chain_planes() {
  return std::is_same_v<U, __bf16> ? 3 : planes_of<U>();
}
// The third of them, where two are there.
__device__ __forceinline__ Planes<__bf16, 1> third_plane(const v4f& lo, const v4f& hi, const Planes<__bf16>& f) {
  Planes<__bf16, 1> out;
#pragma unroll
  for (int e = 0; e < 8; ++e) out.p[0][e] = __bf16((e < 4 ? lo[e & 3] : hi[e & 3]) - float(f.p[0][e]) - float(f.p[1][e]));
  return out;
}

// A factor 2^n that brings a column's largest value near 2^13, where two fp16 numbers hold 22 bits of it; 1 for types with the
// exponents of fp32.
template <typename T, int N>
__device__ __forceinline__ float column_factor(const v4f (&x)[N], float* inverse) {
  if constexpr (!std::is_same_v<T, _Float16>) {
    *inverse = 1.0f;
    return 1.0f;
  } else {
    float most = 0.0f;
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[t][e]));
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    int ex = int(__float_as_uint(most) >> 23);
    ex = ex < 14 ? 14 : ex > 253 ? 253 : ex;
    *inverse = __uint_as_float(unsigned(ex - 13) << 23);
    return __uint_as_float(unsigned(267 - ex) << 23);
  }
}
template <typename T, int N, int P>
__device__ __forceinline__ void split_scaled(const v4f (&x)[N], Planes<T, P> (&out)[N / 2], float* inverse) {
  const float f = column_factor<T>(x, inverse);
#pragma unroll
  for (int p = 0; p < N / 2; ++p) {
    if constexpr (std::is_same_v<T, _Float16>) out[p] = split<T, P>(x[2 * p] * f, x[2 * p + 1] * f);
    else out[p] = split<T, P>(x[2 * p], x[2 * p + 1]);
  }
}

// A row-major tile of COLS columns in LDS, in units of 16 bytes; a unit's place is changed by its row, so that eight lanes that read
// a unit of rows 0..3, 8..11 (fragments) and sixteen that read 32 bytes of four rows (transposed ones) spread over the banks.
//
// What a lane reads lies at its view, a place that depends on the lane alone, up to bits that are flipped and bytes that are added
// as the tile or the step says: constants, so that all of a kernel's reads share a few registers of addresses.
template <typename U, int COLS>
struct Tile {
  static constexpr int ROW = COLS * int(sizeof(U)), UNITS = ROW / 16, BYTES = 64 * ROW;
  static constexpr int MASK = UNITS >= 8 ? 7 : UNITS - 1;
  static constexpr int VEC = 16 / int(sizeof(U));
  static constexpr bool HALF = sizeof(U) == 2;
  static_assert(HALF ? UNITS >= 4 : UNITS >= 8, "");

  // (of rows that differ in bits 0, 1 and 3 alone)
  static __device__ __forceinline__ constexpr int flip(int row) { return (((row & 1) << 2) | (row & 2) | ((row >> 3) & 1)) & MASK; }
  static __device__ __forceinline__ int at(int row, int unit) { return row * ROW + ((unit ^ flip(row)) << 4); }

  // 32 columns of a row: row r of tile t of 16 rows, or row row_of_tile(t, r)
  static __device__ __forceinline__ int row_view(int row, int q) { return at(row, HALF ? q : 2 * q); }
  static __device__ __forceinline__ int natural_rows(int r, int q) { return row_view(r, q); }
  static __device__ __forceinline__ int mapped_rows(int r, int q) { return row_view(row_of_tile(0, r), q); }
  static __device__ __forceinline__ constexpr int mapped_row(int t) { return 32 * (t >> 1) + 4 * (t & 1); }
  // columns 32 p + 8 q and up
  static __device__ __forceinline__ Frag<U> frag(const char* tile, int view, int rows, int p) {
    if constexpr (HALF) {
      return *reinterpret_cast<const Frag<U>*>(tile + (view ^ ((p & 1) << 6)) + (rows * ROW + (p >> 1) * 128));
    } else {
      Frag<U> f;
      const v4f a = *reinterpret_cast<const v4f*>(tile + view + (rows * ROW + p * 128));
      const v4f b = *reinterpret_cast<const v4f*>(tile + (view ^ 16) + (rows * ROW + p * 128));
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
      return f;
    }
  }

  // Four rows of a column: lane 16 q + r has rows 8 q and up of column r of a tile of 16 columns, those as they are (natural) or
  // 32 (t / 2) + 8 (r / 4) + 4 (t % 2) + r % 4 (mapped).
  template <bool MAPPED>
  static __device__ __forceinline__ int columns(int r, int q) {
    const int j = HALF ? r & 3 : r >> 2;
    if constexpr (HALF) return at(8 * q + (r >> 2), MAPPED ? j : j >> 1) + (MAPPED ? 0 : (j & 1) * 8);
    else return at(8 * q, MAPPED ? 2 * j : j) + (r & 3) * 4;
  }
  template <bool MAPPED>
  static __device__ __forceinline__ int column_tile(int view, int t) {
    if constexpr (HALF) return MAPPED ? (view ^ (((t >> 1) & 1) << 6)) + ((t >> 2) * 128 + (t & 1) * 8) : (view ^ ((t & 3) << 5)) + (t >> 2) * 128;
    else return (view ^ (MAPPED ? (t & 1) << 4 : (t & 1) << 6)) + (t >> 1) * 128;
  }
  template <bool MAPPED>
  static __device__ __forceinline__ typename Pack<U, 4>::type column4(const char* tile, int view, int rows, int t) {
    typename Pack<U, 4>::type out;
    if constexpr (HALF) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4* lds_t;
      const s4 raw = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(tile + column_tile<MAPPED>(view, t) + rows * ROW));
      __builtin_memcpy(&out, &raw, 8);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = *reinterpret_cast<const U*>(tile + column_tile<MAPPED>(view ^ (flip(e) << 4), t) + (rows + e) * ROW);
    }
    return out;
  }
  // rows 32 p + 8 q and up
  template <bool MAPPED>
  static __device__ __forceinline__ Frag<U> column_frag(const char* tile, int view, int p, int t) {
    const auto a = column4<MAPPED>(tile, view, 32 * p, t), b = column4<MAPPED>(tile, view, 32 * p + 4, t);
    Frag<U> f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = a[e], f[4 + e] = b[e];
    return f;
  }

  // a result's values: rows 4 q and up of column r of a tile of 16 columns
  static __device__ __forceinline__ int points(int r, int q) { return at(4 * q, r / VEC) + r % VEC * int(sizeof(U)); }
  static __device__ __forceinline__ float point(const char* tile, int view, int rows, int e, int t) {
    const int at = (view ^ (flip(e) << 4) ^ (HALF ? (t & 3) << 5 : (t & 1) << 6)) + ((HALF ? t >> 2 : t >> 1) * 128);
    return float(*reinterpret_cast<const U*>(tile + at + (rows + e) * ROW));
  }
};

// f(0) to f(N - 1), constants.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

// A view that a loop's body starts from anew: the places made from it are not all kept in registers outside.
__device__ __forceinline__ int anew(int view) {
  asm volatile("" : "+v"(view));
  return view;
}

// The same, not before `result` is there.
__device__ __forceinline__ int anew_after(int view, v4f& result) {
  asm volatile("" : "+v"(view), "+v"(result));
  return view;
}

// ROWS rows of COLS columns on their way from memory to a tile, by LANES lanes of which this is number `lane`: all loads first, so that
// their latencies are one, and stores to LDS when they are due.
template <typename T, int COLS, int LANES, int ROWS = 64>
struct Stager {
  using L = Tile<T, COLS>;
  using V = typename Slot16<T>::type;
  static constexpr int VEC = L::VEC, STEP = LANES / L::UNITS, N = (ROWS + STEP - 1) / STEP;  // rows side by side, units of a lane
  static_assert(LANES % L::UNITS == 0, "a lane has one column of units");
  V v[N];

  static __device__ __forceinline__ V zero() {
    V z;
#pragma unroll
    for (int e = 0; e < VEC; ++e) z[e] = T(0.0f);
    return z;
  }
  // `back` values down (the same for all lanes), zeros behind them
  static __device__ __forceinline__ V moved(const V& x, int back) {
    uint64_t w[2];
    __builtin_memcpy(w, &x, 16);
    const int bits = back * 8 * int(sizeof(T));
    if (bits >= 64) {
      w[0] = w[1] >> (bits - 64);
      w[1] = 0;
    } else if (bits > 0) {
      w[0] = (w[0] >> bits) | (w[1] << (64 - bits));
      w[1] >>= bits;
    }
    V out;
    __builtin_memcpy(&out, w, 16);
    return out;
  }
  // zeros for rows from `rows` and columns from `cols` (at least one) on
  __device__ __forceinline__ void fetch(const T* from, int64_t stride, int rows, int cols, int lane) {
    typedef T any __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
    const int row = lane / L::UNITS, col = lane % L::UNITS * VEC;
    if (rows >= ROWS && cols >= COLS) {
      const T* p = from + row * stride + col;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (ROWS % STEP == 0 || n * STEP + row < ROWS) v[n] = *reinterpret_cast<const any*>(p + n * STEP * stride);
      return;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = zero();
    if (cols >= VEC) {  // the last columns by a load that ends with the row
      const int at = col <= cols - VEC ? col : cols - VEC;
      const T* p = from + row * stride + at;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (n * STEP + row < rows && col < cols) v[n] = *reinterpret_cast<const any*>(p + n * STEP * stride);
      if (cols < COLS && cols % VEC)
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const V m = moved(v[n], VEC - cols % VEC);
          v[n] = at != col ? m : v[n];
        }
    } else {
      for (int n = 0; n < N; ++n)
        if (n * STEP + row < rows && col == 0)
          for (int e = 0; e < cols; ++e) v[n][e] = from[(n * STEP + row) * stride + e];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = zero();
  }
  __device__ __forceinline__ void put(char* tile, int lane) const {
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (ROWS % STEP == 0 || n * STEP + lane / L::UNITS < ROWS)
        *reinterpret_cast<V*>(tile + L::at(n * STEP + lane / L::UNITS, lane % L::UNITS)) = v[n];
  }
};

// Values of scratch, in fp32, on their way to the planes of a tile of ROWS rows of COLS columns, eight of a row to a lane at a time.
template <typename U, int COLS, int LANES, int ROWS>
struct SplitStager {
  using L = Tile<U, COLS>;
  static constexpr int PLANES = chain_planes<U>(), EIGHTS = COLS / 8, ALL = ROWS * EIGHTS, N = (ALL + LANES - 1) / LANES, BYTES = ROWS * L::ROW;  // (of a plane)
  v4f v[N][2];

  static __device__ __forceinline__ bool has(int n, int lane) { return (n + 1) * LANES <= ALL || n * LANES + lane < ALL; }
  __device__ __forceinline__ void put_at(char* tile, int n, int row, int eighth) const {
    if constexpr (sizeof(U) == 2) {
      const Planes<U, PLANES> f = split<U, PLANES>(v[n][0], v[n][1]);
#pragma unroll
      for (int k = 0; k < PLANES; ++k) *reinterpret_cast<Frag<U>*>(tile + k * BYTES + L::at(row, eighth)) = f.p[k];
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<v4f*>(tile + L::at(row, 2 * eighth + h)) = v[n][h];
    }
  }

  // pieces of store_rows: those of a group of 16 rows from `from_piece` on, of EVERY that it has; load n of N
  template <int EVERY>
  __device__ __forceinline__ void fetch_pieces(int n, const float* from, int from_piece, int lane) {
    const int i = n * LANES + lane, g = i / (16 * EIGHTS), k = (i - g * (16 * EIGHTS)) >> 6;
    if (has(n, lane))
#pragma unroll
      for (int h = 0; h < 2; ++h) v[n][h] = reinterpret_cast<const v4f*>(from)[(g * EVERY + from_piece + 2 * k + h) * 64 + (i & 63)];
  }
  __device__ __forceinline__ void put_pieces(char* tile, int lane) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = n * LANES + lane, g = i / (16 * EIGHTS), k = (i - g * (16 * EIGHTS)) >> 6;
      if (has(n, lane)) put_at(tile, n, 16 * g + (i & 15), 4 * k + ((i >> 4) & 3));
    }
  }
};

// A triangle of a dense 64 x 64 square in LDS without its empty quarter: 64 rows of the 32 columns that are all full, the first ones of a lower and the
// last ones of an upper triangle, and behind them the other 32 columns' rows.
constexpr int TRIANGLE_ROWS = 96;
template <typename U, bool UPPER, int LANES>
struct TriangleStager : SplitStager<U, 32, LANES, TRIANGLE_ROWS> {
  using S = SplitStager<U, 32, LANES, TRIANGLE_ROWS>;
  static_assert(LANES == 256 || LANES == 128, "a load is of one part");
  __device__ __forceinline__ void fetch(const float* from, int lane) {
#pragma unroll
    for (int n = 0; n < S::N; ++n) {
      const int row = n * LANES / 4;  // (of the first lane)
      const float* at = from + (row < 64 ? row * 64 + (UPPER ? 32 : 0) : (UPPER ? row - 64 : row - 32) * 64 + (UPPER ? 0 : 32)) + lane * 8 + (lane >> 2) * 32;
      if (S::has(n, lane))
#pragma unroll
        for (int h = 0; h < 2; ++h) this->v[n][h] = *reinterpret_cast<const v4f*>(at + 4 * h);
    }
  }
  __device__ __forceinline__ void put(char* tile, int lane) const {
#pragma unroll
    for (int n = 0; n < S::N; ++n)
      if (S::has(n, lane)) S::put_at(tile, n, n * LANES / 4 + (lane >> 2), lane & 3);
  }
};
template <typename U>
constexpr int triangle_bytes() {
  return TRIANGLE_ROWS * 32 * int(sizeof(U)) * chain_planes<U>();
}
// to += triangle . by, four tiles of 16 rows (row_of_tile).
template <bool UPPER, typename U, int NB>
__device__ __forceinline__ void mma_triangle(const char* tile, int view, const Planes<U, NB> (&by)[2], v4f (&to)[4]) {
  using L = Tile<U, 32>;
  constexpr int PLANES = chain_planes<U>();
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const bool whole = b == (UPPER ? 1 : 0);  // these 32 columns have all rows
#pragma unroll
    for (int k = PLANES - 1; k >= 0; --k) {
      Frag<U> f[4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (whole || (UPPER ? t < 2 : t >= 2))
          f[t] = L::frag(tile + k * (TRIANGLE_ROWS * L::ROW), view, L::mapped_row(t) + (whole ? 0 : UPPER ? 64 : 32), 0);
#pragma unroll
      for (int j = NB - 1; j >= 0; --j)
        if (k + j < PLANES)
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (whole || (UPPER ? t < 2 : t >= 2)) to[t] = mma(f[t], by[b].p[j], to[t]);
    }
  }
}

// Results that a wave has of 16 columns and 32 rows (columns of scratch), a lane's as it has them: pieces of 1 KB that a wave stores and loads whole (rows of
// their own would be stored 64 bytes at a time).  b: which 32.
__device__ __forceinline__ void store_rows(float* to, int b, int lane, const v4f& lo, const v4f& hi) {
  *reinterpret_cast<v4f*>(to + b * 512 + lane * 4) = lo;
  *reinterpret_cast<v4f*>(to + b * 512 + 256 + lane * 4) = hi;
}

// ---- chunks and scratch ----------------------------------------------------------------------------------------------------------
// A chunk has a slot: those of a sequence follow each other, a packed sequence's start at cu_seqlens[n] / 64 + n (so that no two
// sequences meet, whatever their lengths), a batch item's at n * ceil(time / 64).
struct DeltaArgs {
  linrec_delta_t p;
  int64_t slots;
  int shared;    // value heads of a key head
  int columns;   // value_dim rounded up to 32: rows of the planes of S, dS', N and dB
  int blocks;    // workgroups side by side over the columns
  int64_t pairs; // parts x heads
  int64_t parts; // sequences, or segments of them
  int segment;   // chunks of a segment, 0: sequences are not cut
  // scratch, for every (slot, head); values from one to the next of d_b and n, and of s and d_s:
  int64_t rows, state;
  float* m;      // [64][64] as m_t and c, whose empty quarters are not written
  float* m_t;    // transposed
  float* c;      // C scale, transposed in the backward
  float* gates;  // [3][64]: e^G, e^{G_63 - G}, beta
  double* sums;  // [64]: G
  float* s;      // [columns][DK] in pieces of 16 columns (store_rows), the state before the chunk
  float* d_s;    // the same of dS' behind it
  float* n;      // [columns][64] in such pieces
  float* d_b;
  float* dots;   // [192], sums of the gates' gradients where key_dim comes in turns
  // for every (part, head), where sequences are cut (delta_segments.hpp)
  float* carry;  // [columns + DK][DK]: what a segment makes of nothing, and of the unit matrix
  float* start;  // [columns][DK]: the state that enters a segment
};

struct Span {
  int64_t batch, first, end;  // positions of a sequence in its batch item
  int64_t slot;               // of its first chunk
};
__device__ __forceinline__ int64_t bound_of(const linrec_delta_t& p, int64_t n) {
  const int64_t b = p.cu_seqlens[n];
  return b < 0 ? 0 : b > p.time ? p.time : b;
}
__device__ __forceinline__ Span span_of(const linrec_delta_t& p, int64_t n) {
  if (!p.cu_seqlens) return Span{n, 0, p.time, n * ((p.time + DELTA_CHUNK - 1) / DELTA_CHUNK)};
  const int64_t a = bound_of(p, n), b = bound_of(p, n + 1);
  return Span{0, a, b < a ? a : b, a / DELTA_CHUNK + n};
}
// The first position and the length of the chunk in a slot; a length of zero where there is none.
struct Chunk {
  int64_t batch, first;
  int length;
};
__device__ __forceinline__ Chunk chunk_of(const linrec_delta_t& p, int64_t slot) {
  if (!p.cu_seqlens) {
    const int64_t each = (p.time + DELTA_CHUNK - 1) / DELTA_CHUNK, n = slot / each, first = (slot - n * each) * DELTA_CHUNK;
    return Chunk{n, first, int(p.time - first < DELTA_CHUNK ? p.time - first : DELTA_CHUNK)};
  }
  // the last sequence that starts at or before the slot, 64 bounds at a time
  int lo = 0, hi = int(p.sequences);
  const int lane = threadIdx.x & 63;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + lane * step;
    const bool before = at < hi && bound_of(p, at) / DELTA_CHUNK + at <= slot;
    const int n = __popcll(__ballot(before));
    lo += (n > 0 ? n - 1 : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const Span s = span_of(p, lo);
  const int64_t first = s.first + (slot - s.slot) * DELTA_CHUNK, left = s.end - first;
  if (slot < s.slot || left <= 0) return Chunk{0, 0, 0};
  return Chunk{0, first, int(left < DELTA_CHUNK ? left : DELTA_CHUNK)};
}

// Part of a sequence: all of it, or a segment.  Segments are numbered as slots are: a packed sequence's from slot / segment + n on.
struct Part {
  int64_t n;
  Span span;
  int64_t index, count;  // of the sequence's parts; count is 0 where there is none
  int64_t begin, end;    // chunks
};
__device__ __forceinline__ int64_t chunks_of(const Span& s) { return (s.end - s.first + DELTA_CHUNK - 1) / DELTA_CHUNK; }
__device__ __forceinline__ int64_t first_part(const DeltaArgs& a, int64_t n, const Span& s) {
  if (!a.segment) return n;
  if (a.p.cu_seqlens) return s.slot / a.segment + n;
  return n * ((chunks_of(s) + a.segment - 1) / a.segment);
}
__device__ __forceinline__ int64_t count_of_parts(const DeltaArgs& a, const Span& s) {
  const int64_t chunks = chunks_of(s);
  return a.segment && chunks > a.segment ? (chunks + a.segment - 1) / a.segment : 1;  // (one of nothing hands the state on)
}
__device__ __forceinline__ Part part_of(const DeltaArgs& a, int64_t at) {
  int64_t n = at;
  if (a.segment && !a.p.cu_seqlens) {
    n = at / count_of_parts(a, span_of(a.p, 0));
  } else if (a.segment) {  // the last sequence whose parts start at or before this one, 64 at a time
    int lo = 0, hi = int(a.p.sequences);
    const int lane = threadIdx.x & 63;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, probe = lo + lane * step;
      const bool before = probe < hi && first_part(a, probe, span_of(a.p, probe)) <= at;
      const int found = __popcll(__ballot(before));
      lo += (found > 0 ? found - 1 : 0) * step;
      hi = lo + step < hi ? lo + step : hi;
    }
    n = __builtin_amdgcn_readfirstlane(lo);
  }
  Part part{n, span_of(a.p, n), 0, 0, 0, 0};
  const int64_t chunks = chunks_of(part.span);
  part.count = count_of_parts(a, part.span);
  part.index = at - first_part(a, n, part.span);
  part.begin = part.index * (a.segment ? a.segment : chunks);
  part.end = a.segment && part.begin + a.segment < chunks ? part.begin + a.segment : chunks;
  if (part.index < 0 || part.index >= part.count) part.count = 0;
  return part;
}

template <typename T>
__device__ __forceinline__ const T* head_rows(const void* base, const int64_t (&stride)[3], int64_t batch, int64_t first, int64_t head) {
  return static_cast<const T*>(base) + batch * stride[0] + first * stride[1] + head * stride[2];
}

// Workgroups of one (part, head), which read the same keys and queries, lie on one XCD (workgroups go round the eight in turn).
__device__ __forceinline__ bool scan_place(const DeltaArgs& a, int blocks, int64_t* pair, int* block) {
  const int64_t group = blockIdx.x / unsigned(8 * blocks);
  const int in = int(blockIdx.x - group * unsigned(8 * blocks));
  *block = in >> 3;
  *pair = group * 8 + (in & 7);
  return *pair < a.pairs;
}

}  // namespace linrec
