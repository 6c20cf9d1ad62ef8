// Token embedding, y[n] = scale W[token[n]], and its gradient, d_W[v] = scale * sum of d_y[n] over the n with token[n] == v.
//
// Forward: a wave copies 64 slots of channels of a few rows.  Bound by memory; a row that is looked up again comes from a cache:
// 32768 of 32000 x 1024 bf16 17.6 us (16.3 of the kernel, 134 MB in and out), 32768 of 32000 x 4096 61 us.  Few tokens are bound by
// the launch (64 of 32000 x 4096: 6.4 us, an empty kernel takes 5.7 so timed).
//
// Backward, without atomics on values: the positions are sorted by token (stably, so that each list of positions ascends), the
// gradient is cleared meanwhile, and every list is summed by the wave that finds its start in the sorted tokens.
//   sort   up to SORT_SMALL tokens in one launch: the place of a position is the number of smaller (token, position) pairs, all
//          pairs compared; more are sorted by digits of at most DIGIT_BITS bits from the lowest on, two launches each (counts
//          of blocks; places).  Places are counted, never drawn, so the order is the same in every run.  Every block of
//          the second launch reads all blocks' counts, which grows with the square of the tokens: the gradient of 2^20 tokens of 64
//          channels bf16 takes 150 us, of 2^22 1.1 ms, where d_y is read in 26 and 103 us.  (Every block counting
//          all digits itself, a launch less a digit: 21.6 us each instead of 4.4 and 8.0.  The places adding up the next digit's
//          counts with atomics: 76 us for the gradient of 32768 words where this takes 55.)
//   clear  a few workgroups sort; the others of the same launches write zeros, whole lines front to back, a share in each launch.
//          (Rows of zeros written one by one where a row has no list: 128000 x 333 fp32 58 us for that launch alone.)
//   sums   a list may be as long as all positions, and a wave takes a microsecond for every eight rows it adds up.  Aligned runs of
//          16 sorted positions with one token are summed first, a wave each, then, of many tokens, aligned runs of 16 of those; a
//          long list adds up what is left before, the two kinds of runs, and what is left after, at most 15 of the smaller kinds at
//          each end.  The grouping depends on the tokens alone.  (Runs of 32: 4096 of 1000 x 1024 bf16 26.7 us instead of 23.0,
//          65536 of 256 x 512 45.1 instead of 42.9, 32768 of 32000 x 1024 57.2 instead of 55.0.)
// What bounds it: d_y is read once, the table's gradient written once, rows that have a list twice.  128000 x 333 fp32, 4095 words:
// 45 us for 176 MB (3.9 TB/s), 33 of them the launch that clears.  32000 x 1024 bf16, 32768 words: 55 us for 133 MB, of them 25 for
// the four launches of the sort and the clearing beside it, 11 for the two kinds of runs, 19 for lists; each of the seven launches waits for the one before it.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/linrec_layers.h"
#include "collook_kernel.hpp"  // Held, ld_any, st_any, widen

namespace linrec {

__device__ __forceinline__ int64_t token_at(const linrec_embedding_t& p, int64_t n) {
  return p.token_bytes == 8 ? static_cast<const int64_t*>(p.token)[n] : int64_t(static_cast<const int32_t*>(p.token)[n]);
}
// What a position is sorted by: its token, behind all of them if it has no part in the gradient.
__device__ __forceinline__ int sort_key(const linrec_embedding_t& p, int64_t n) {
  const int64_t v = token_at(p, n);
  return v >= 0 && v < p.vocab && v != p.padding ? int(v) : int(p.vocab);
}

// The channels of a lane of column wave `cw`: the last lanes start early where the channels end and compute, and store, what
// the lane before them does (the same bits).
template <int VEC>
__device__ __forceinline__ int64_t wave_channel(int64_t cw, int lane, int64_t channels) {
  const int64_t c = (cw * 64 + lane) * VEC, last = channels - VEC;
  return c < last ? c : last;
}

// ---- forward ----------------------------------------------------------------------------------
template <typename T, int VEC, int ROWS>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(linrec_embedding_t p, int64_t column_waves) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t row_set = unit / column_waves, cw = unit - row_set * column_waves;
  const int64_t c = wave_channel<VEC>(cw, lane, p.channels), n0 = row_set * ROWS;
  Held<T, VEC> h[ROWS];
  bool there[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int64_t v = n0 + i < p.tokens ? token_at(p, n0 + i) : -1;
    there[i] = v >= 0 && v < p.vocab;
    h[i] = held_zero<T, VEC>();
    if (there[i]) h[i] = ld_any<VEC, false>(static_cast<const T*>(p.weight) + v * p.channels + c);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (n0 + i < p.tokens) {
      Lanes<VEC> v = widen(h[i]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v.v[e] = there[i] ? v.v[e] * p.scale : 0.0f;
      st_any<VEC>(static_cast<T*>(p.y) + (n0 + i) * p.channels + c, v);
    }
  }
}

// ---- clear ------------------------------------------------------------------------------------
// The share of a launch: `first` .. `end` of the gradient's 16-byte slots, and what is left of a slot at its end.
struct Clear {
  int64_t first, end;
  int tail;  // 2-byte words behind the last slot
};
__device__ __forceinline__ void clear_share(const linrec_embedding_t& p, const Clear& c, int64_t block, int64_t blocks) {
  typedef unsigned Slot __attribute__((ext_vector_type(4), aligned(2)));  // (any alignment that a tensor has)
  Slot* to = static_cast<Slot*>(p.d_weight);
  for (int64_t i = c.first + block * blockDim.x + threadIdx.x; i < c.end; i += blocks * blockDim.x) __builtin_nontemporal_store(Slot{0u, 0u, 0u, 0u}, to + i);
  if (block == 0 && int(threadIdx.x) < c.tail) reinterpret_cast<unsigned short*>(to + c.end)[threadIdx.x] = 0;
}

// ---- sort -------------------------------------------------------------------------------------
struct Sorted {
  int* key;
  int* pos;
};

constexpr int SORT_SMALL = 8192;
constexpr int SMALL_TAKE = 32;  // positions a workgroup places

// All pairs: 1024 lanes compare SMALL_TAKE positions with a 32nd of all keys each.
__global__ __launch_bounds__(1024) void sort_small_kernel(linrec_embedding_t p, Sorted out, int blocks, Clear clear) {
  if (int(blockIdx.x) >= blocks) return clear_share(p, clear, blockIdx.x - blocks, gridDim.x - blocks);
  __shared__ alignas(16) int keys[SORT_SMALL];
  __shared__ int counts[32][SMALL_TAKE + 1];
  const int n = int(p.tokens), tid = int(threadIdx.x);
  const int padded = (n + 127) & ~127;
  for (int i = tid; i < padded; i += 1024) keys[i] = i < n ? sort_key(p, i) : 2147483647;
  __syncthreads();
  const int mine = int(blockIdx.x) * SMALL_TAKE + (tid & 31), slice = tid >> 5, per_slice = padded / 32;
  const int key = mine < n ? keys[mine] : 2147483647;
  int count = 0;
  const int first = slice * per_slice;
  for (int j = first; j < first + per_slice; j += 4) {
    const int4 k = *reinterpret_cast<const int4*>(&keys[j]);
    count += (k.x < key || (k.x == key && j < mine)) + (k.y < key || (k.y == key && j + 1 < mine)) +
             (k.z < key || (k.z == key && j + 2 < mine)) + (k.w < key || (k.w == key && j + 3 < mine));
  }
  counts[slice][tid & 31] = count;
  __syncthreads();
  if (tid < SMALL_TAKE && mine < n) {
    int place = 0;
    for (int s = 0; s < 32; ++s) place += counts[s][tid];
    out.key[place] = key;
    out.pos[place] = mine;
  }
}

constexpr int DIGIT_BITS = 9, DIGITS = 1 << DIGIT_BITS;
constexpr int SORT_LANES = 1024, SORT_WAVES = SORT_LANES / 64, SORT_ROUNDS = 2, SORT_BLOCK = SORT_LANES * SORT_ROUNDS;

__device__ __forceinline__ int key_of(const linrec_embedding_t& p, const int* keys, int64_t i) { return keys ? keys[i] : sort_key(p, i); }

__global__ __launch_bounds__(SORT_LANES) void digit_counts_kernel(linrec_embedding_t p, const int* keys, int shift, int* counts, int blocks,
                                                                  Clear clear) {
  if (int(blockIdx.x) >= blocks) return clear_share(p, clear, blockIdx.x - blocks, gridDim.x - blocks);
  __shared__ int bins[DIGITS];
  const int tid = int(threadIdx.x);
  if (tid < DIGITS) bins[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r) {
    const int64_t i = int64_t(blockIdx.x) * SORT_BLOCK + r * SORT_LANES + tid;
    if (i < p.tokens) atomicAdd(&bins[(key_of(p, keys, i) >> shift) & (DIGITS - 1)], 1);
  }
  __syncthreads();
  if (tid < DIGITS) counts[int64_t(blockIdx.x) * DIGITS + tid] = bins[tid];
}

// A position goes behind all of smaller digits, those of its digit in blocks before, in waves before and before it in its wave.
__global__ __launch_bounds__(SORT_LANES) void digit_places_kernel(linrec_embedding_t p, const int* keys, const int* positions, int shift,
                                                                  const int* counts, int blocks, Sorted out, Clear clear) {
  if (int(blockIdx.x) >= blocks) return clear_share(p, clear, blockIdx.x - blocks, gridDim.x - blocks);
  __shared__ int base[DIGITS];
  __shared__ int wave_sums[DIGITS / 64];
  __shared__ int bins[SORT_WAVES][DIGITS];
  const int tid = int(threadIdx.x), lane = tid & 63, wave = tid >> 6;
  // a wave takes 64 * SORT_ROUNDS adjacent positions, in order
  const int64_t first = int64_t(blockIdx.x) * SORT_BLOCK + wave * (64 * SORT_ROUNDS) + lane;
  int key[SORT_ROUNDS], pos[SORT_ROUNDS], rank[SORT_ROUNDS];
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r) {
    const int64_t i = first + r * 64;
    const bool there = i < p.tokens;
    key[r] = there ? key_of(p, keys, i) : 0;
    pos[r] = there ? (positions ? positions[i] : int(i)) : 0;
  }
  for (int i = tid; i < SORT_WAVES * DIGITS; i += SORT_LANES) (&bins[0][0])[i] = 0;
  int all = 0, before = 0;
  if (tid < DIGITS) {
#pragma unroll 8
    for (int b = 0; b < blocks; ++b) {
      const int c = counts[int64_t(b) * DIGITS + tid];
      all += c;
      before += b < int(blockIdx.x) ? c : 0;
    }
  }
  int scan = all;  // over the digits: within waves, then over the waves' sums
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int up = __shfl_up(scan, s);
    if (lane >= s) scan += up;
  }
  if (wave < DIGITS / 64 && lane == 63) wave_sums[wave] = scan;
  __syncthreads();
  if (tid < DIGITS) {
    int lower = 0;
    for (int w = 0; w < wave; ++w) lower += wave_sums[w];
    base[tid] = lower + scan - all + before;
  }
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r) {
    const bool there = first + r * 64 < p.tokens;
    const int digit = (key[r] >> shift) & (DIGITS - 1);
    uint64_t same = __ballot(there);
#pragma unroll
    for (int b = 0; b < DIGIT_BITS; ++b) {
      const uint64_t ones = __ballot(digit >> b & 1);
      same &= (digit >> b & 1) ? ones : ~ones;
    }
    const int ahead = __popcll(same & ((1ull << lane) - 1ull));
    int so_far = 0;
    if (there && ahead == 0) so_far = atomicAdd(&bins[wave][digit], __popcll(same));
    // (the first lane of each digit has asked; the others read what it got)
    so_far = __shfl(so_far, there ? __builtin_ctzll(same) : 0);
    rank[r] = so_far + ahead;
  }
  __syncthreads();
  if (tid < DIGITS) {
    int sum = base[tid];
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const int c = bins[w][tid];
      bins[w][tid] = sum;
      sum += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r) {
    if (first + r * 64 < p.tokens) {
      const int place = bins[wave][(key[r] >> shift) & (DIGITS - 1)] + rank[r];
      out.key[place] = key[r];
      out.pos[place] = pos[r];
    }
  }
}

// ---- sums -------------------------------------------------------------------------------------
constexpr int RUN = 16, RUN2 = RUN * RUN;

template <int VEC>
__device__ __forceinline__ void add_to(Lanes<VEC>& s, const Lanes<VEC>& v) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) s.v[e] += v.v[e];
}
// Adds `count` rows, row(i) their first value for this lane, in order.
template <int VEC, int AT_ONCE = 8, typename Row>
__device__ __forceinline__ void add_rows(Lanes<VEC>& sum, int count, Row&& row) {
  int i = 0;
  for (; i + AT_ONCE <= count; i += AT_ONCE) {
    decltype(ld_any<VEC, false>(row(0))) h[AT_ONCE];
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q) h[q] = ld_any<VEC, false>(row(i + q));
#pragma unroll
    for (int q = 0; q < AT_ONCE; ++q) add_to(sum, widen(h[q]));
  }
  for (; i < count; ++i) add_to(sum, widen(ld_any<VEC, false>(row(i))));
}
template <int VEC>
__device__ __forceinline__ Lanes<VEC> zeros() {
  Lanes<VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = 0.0f;
  return r;
}

// Runs of 16 positions of one token (SECOND: of 16 such sums): a wave each, for 64 slots of channels.
template <typename T, int VEC, bool SECOND>
__global__ __launch_bounds__(256) void run_sums_kernel(linrec_embedding_t p, Sorted sorted, const float* in, float* out, int64_t runs,
                                                       int64_t column_waves) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t run = unit / column_waves, cw = unit - run * column_waves;
  if (run >= runs) return;
  constexpr int LENGTH = SECOND ? RUN2 : RUN;
  const int key = sorted.key[run * LENGTH];
  if (key != sorted.key[run * LENGTH + LENGTH - 1] || key >= int(p.vocab)) return;
  const int64_t c = wave_channel<VEC>(cw, lane, p.channels);
  Lanes<VEC> sum = zeros<VEC>();
  if constexpr (SECOND) {
    add_rows<VEC, 16>(sum, RUN, [&](int i) { return in + (run * RUN + i) * p.channels + c; });
  } else {
    const int pos = sorted.pos[run * RUN + (lane & (RUN - 1))];
    const T* dy = static_cast<const T*>(p.d_y) + c;
    add_rows<VEC, 16>(sum, RUN, [&](int i) { return dy + int64_t(__builtin_amdgcn_readlane(pos, i)) * p.d_y_stride; });
  }
  float* to = out + run * p.channels + c;
#pragma unroll
  for (int e = 0; e < VEC; ++e) to[e] = sum.v[e];
}

// Number of runs of `length` sorted positions from `at` on, at most `most` (up to 64), that hold token v alone (the first position
// does).
__device__ __forceinline__ int whole_runs(const int* keys, int n, int at, int length, int most, int v, int lane) {
  const int64_t i = int64_t(at) + int64_t(lane + 1) * length - 1;
  const uint64_t others = ~__ballot(lane < most && i < n && keys[i < n ? i : 0] == v);
  return others ? __builtin_ctzll(others) : 64;
}

// A wave sums the lists that start among OWN adjacent sorted positions, for 64 slots of channels, and writes their rows.
constexpr int OWN = 8;
template <typename T, int VEC>
__global__ __launch_bounds__(256) void list_sums_kernel(linrec_embedding_t p, Sorted sorted, const float* runs, const float* runs2,
                                                        int64_t column_waves) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t set = unit / column_waves, cw = unit - set * column_waves;
  const int n = int(p.tokens), vocab = int(p.vocab);
  if (set * OWN >= n) return;
  const int first = int(set) * OWN;
  const int64_t c = wave_channel<VEC>(cw, lane, p.channels);
  const T* dy = static_cast<const T*>(p.d_y) + c;
  T* out = static_cast<T*>(p.d_weight) + c;
  // 64 sorted positions; what lies behind them all, or has no part in the gradient, has keys of `vocab` and up
  int base = first, key = 2147483647, pos = 0;
  auto look = [&]() __attribute__((always_inline)) {
    const bool there = base + lane < n;
    key = there ? sorted.key[base + lane] : 2147483647;
    pos = there ? sorted.pos[base + lane] : 0;
  };
  look();
  const int before = first > 0 ? sorted.key[first - 1] : -1;
  const int left = __shfl_up(key, 1);
  const uint64_t starts = __ballot(lane < OWN && key < vocab && key != (lane == 0 ? before : left));
  if (starts == 0) return;
  const int begin = __builtin_ctzll(starts), last = 63 - __builtin_clzll(starts);  // the first and the last list's lanes
  const int last_key = __builtin_amdgcn_readlane(key, last);
  const uint64_t of_last = ~(__ballot(key == last_key) >> last);
  const int end = last + (of_last ? __builtin_ctzll(of_last) : 64 - last);  // of the last list in the window (zeros come in from above)
  const bool longer = end >= 64 || end - last > 24;

  auto store = [&](int v, Lanes<VEC>& sum) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum.v[e] *= p.scale;
    st_any<VEC>(out + int64_t(v) * p.channels, sum);
    sum = zeros<VEC>();
  };
  // Lists that end in the window: their positions one after the other, eight under way at a time, a row of the gradient stored
  // whenever the token changes.
  const int until = longer ? last : end;
  Lanes<VEC> sum = zeros<VEC>();
  int v = __builtin_amdgcn_readlane(key, begin);
  for (int at = begin; at < until; at += 8) {
    Held<T, VEC> h[8];
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (at + q < until) h[q] = ld_any<VEC, false>(dy + int64_t(__builtin_amdgcn_readlane(pos, at + q)) * p.d_y_stride);
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (at + q < until) {
        const int token = __builtin_amdgcn_readlane(key, at + q);
        if (token != v) {
          store(v, sum);
          v = token;
        }
        add_to(sum, widen(h[q]));
      }
  }
  if (until > begin) store(v, sum);
  if (!longer) return;

  // A long list.
  v = last_key;
  int at = first + last;
  for (;;) {
    base = at;
    look();
    const uint64_t others = ~__ballot(key == v);
    const int count = others ? __builtin_ctzll(others) : 64;  // of the list, in the window
    if ((at & (RUN - 1)) != 0 || count < RUN) {  // up to where a run may start, or the end
      const int ahead = RUN - (at & (RUN - 1)), take = count < ahead ? count : ahead;
      add_rows<VEC>(sum, take, [&](int i) { return dy + int64_t(__builtin_amdgcn_readlane(pos, i)) * p.d_y_stride; });
      at += take;
      if (take < ahead) break;
      continue;
    }
    // whole runs from here on: of runs where one of them may start, else as many as come before that
    int length = RUN2, whole = 0;
    if (runs2 && (at & (RUN2 - 1)) == 0) whole = whole_runs(sorted.key, n, at, RUN2, 64, v, lane);
    if (whole == 0) {
      length = RUN;
      whole = whole_runs(sorted.key, n, at, RUN, runs2 ? RUN - (at / RUN & (RUN - 1)) : 64, v, lane);
    }
    const float* rows = (length == RUN2 ? runs2 : runs) + int64_t(at / length) * p.channels + c;
    add_rows<VEC>(sum, whole, [&](int i) { return rows + int64_t(i) * p.channels; });
    at += whole * length;
  }
  store(v, sum);
}

}  // namespace linrec
