// Gated linear recurrence in one launch a pass, and its single-token step.
//
//   log a = -decay sigmoid(gate_a),  decay = scale softplus(rate)
//   h[t] = a h[t-1] + m sigmoid(gate_x) x,  m = sqrt(1 - a^2) = sqrt(-expm1(2 log a))
//
// The shape is that of the look-back segments (collook_kernel.hpp): the scan axis is cut into segments of NW * U positions, a
// workgroup takes one segment of 64 * VEC channels, wave w the run [w*U, w*U + U), and the segments of a channel are chained
// through descriptors in global memory.  The gates are evaluated on the way in, so forward reads three tensors and writes one,
// where coefficients and inputs made by elementwise kernels first are written and read once more each.
//
// Backward, g[t] = d_h[t] + a[t+1] g[t+1] in the opposite direction over the same segments:
//   d_x = g m sx,  d_gate_x = g m x sx (1 - sx)                         (sx, sa: the gates' sigmoids)
//   P = g (log a a h[t-1] - sx x a^2 log a / m),  d_gate_a = P (1 - sa),  d_rate = sigmoid(rate) / softplus(rate) sum P
// (log a and log a / m both go to zero with sigmoid(gate_a), where 1 / m alone does not: every term stays finite.)  h[t-1] is
// not read: the forward saves the value that enters every 64th position in fp32 (4 bytes for 64 positions of a channel), and the
// backward goes on from there with the same operations, so the gradient sees the unrounded values and four tensors are read
// where the saved output would make it five.
//
// The value that enters a segment is always the same chain of multiply-adds over the segments before, whichever of them had
// published what when they were looked at (a window is folded from its farthest segment to its nearest, and a segment's own
// value by the same operation): results are the same bits in every run.
//
// A position at which a packed sequence starts takes the sequence's own initial value instead of what comes from before it, so
// nothing passes from one sequence to the next, not even by 0 * inf.  A segment that holds a start does not wait at all.
//
// A wait is for segments of smaller workgroup number only, and bounded; a lane whose wait runs out walks its channel from the
// sequence's start.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/linrec_layers.h"
#include "collook_kernel.hpp"

namespace linrec {

constexpr int GATED_SAVE = 64;  // positions from one saved value to the next, and of a backward segment

struct GatedArgs {
  linrec_gated_t p;
  TileArgs chain;
  int segments;         // of the scan axis
  int channel_blocks;
};

// ---- arithmetic -------------------------------------------------------------------------------
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ float fast_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * v));
}
// log(1 + exp(v)).  log(w) e / (w - 1) with w = 1 + e rounded is log(1 + e) to a few roundings however small e is.
__device__ __forceinline__ float fast_softplus(float v) {
  const float e = __builtin_amdgcn_exp2f(-LOG2E * fabsf(v));
  const float w = 1.0f + e, d = w - 1.0f;
  const float l = d == 0.0f ? e : LN2 * __builtin_amdgcn_logf(w) * e * __builtin_amdgcn_rcpf(d);
  return (v > 0.0f ? v : 0.0f) + (v != v ? v : l);
}
// 1 - exp(u) for u <= 0: the difference cancels where u is small, the series of seven terms is off by 5e-8 of the result at 1/4.
__device__ __forceinline__ float one_minus_exp(float u, float exp_u) {
  const float s = fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, 1.0f / 720.0f, 1.0f / 120.0f), 1.0f / 24.0f), 1.0f / 6.0f), 0.5f), 1.0f);
  return u > -0.25f ? -u * s : 1.0f - exp_u;
}

struct Gate {
  float sa, sx;   // sigmoids
  float log2_a;   // log a in base 2
  float a;
  float m2;       // 1 - a^2
};
// decay2: the decay rate in base 2
__device__ __forceinline__ Gate gate_of(float ga, float gx, float decay2) {
  Gate g;
  g.sa = fast_sigmoid(ga);
  g.sx = fast_sigmoid(gx);
  g.log2_a = -decay2 * g.sa;
  g.a = __builtin_amdgcn_exp2f(g.log2_a);
  g.m2 = one_minus_exp(2.0f * LN2 * g.log2_a, g.a * g.a);
  return g;
}
__device__ __forceinline__ float taken_in(const Gate& g, float x) { return __builtin_amdgcn_sqrtf(g.m2) * g.sx * x; }

// A product of coefficients that has become too small to be told from zero still passes an infinity on, as the recurrence
// does (the coefficients are never negative).
__device__ __forceinline__ float never_zero(float a) { return a == 0.0f ? __builtin_bit_cast(float, 1u) : a; }

// ---- sequences --------------------------------------------------------------------------------
// Bounds of the packed sequences in scan order: a reversed scan meets the last sequence first.
__device__ __forceinline__ int scan_bound(const linrec_gated_t& p, int64_t j) {
  const int64_t v = p.reverse ? p.time - p.cu_seqlens[p.sequences - j] : p.cu_seqlens[j];
  return int(v < 0 ? 0 : v > p.time ? p.time : v);
}
__device__ __forceinline__ int64_t scan_sequence(const linrec_gated_t& p, int64_t j) { return p.reverse ? p.sequences - 1 - j : j; }
// Number of bounds 0 .. sequences that are at most `pos`.
__device__ __forceinline__ int64_t bounds_up_to(const linrec_gated_t& p, int pos) {
  int64_t lo = 0, hi = p.sequences + 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (scan_bound(p, mid) <= pos) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// Which positions of a segment start and end a sequence.
template <int SEG>
struct SegmentMarks {
  int start[SEG], end[SEG];  // the sequence, where the masks have a bit
  unsigned starts[(SEG + 31) / 32], ends[(SEG + 31) / 32];
};
// (by all lanes of a workgroup; a barrier before the marks are read is the caller's)
template <int SEG, int LANES>
__device__ __forceinline__ void mark_segment(SegmentMarks<SEG>& m, const linrec_gated_t& p, int first) {
  const int tid = int(threadIdx.x);
  if (tid < (SEG + 31) / 32) m.starts[tid] = m.ends[tid] = 0u;
  __syncthreads();
  int64_t j0 = 0;
  if (p.sequences > LANES) {  // few sequences: one look at all of them
    j0 = bounds_up_to(p, first) - 1;
    if (j0 < 0) j0 = 0;
  }
  for (int64_t base = j0; base < p.sequences; base += LANES) {
    if (base > j0 && scan_bound(p, base) >= first + SEG) break;
    const int64_t j = base + tid;
    if (j < p.sequences) {
      const int s0 = scan_bound(p, j) - first, s1 = scan_bound(p, j + 1) - 1 - first;
      if (s0 <= s1) {
        const int n = int(scan_sequence(p, j));
        if (s0 >= 0 && s0 < SEG) {
          m.start[s0] = n;
          atomicOr(&m.starts[s0 >> 5], 1u << (s0 & 31));
        }
        if (s1 >= 0 && s1 < SEG) {
          m.end[s1] = n;
          atomicOr(&m.ends[s1 >> 5], 1u << (s1 & 31));
        }
      }
    }
  }
}
template <int U>
__device__ __forceinline__ unsigned run_bits(const unsigned* mask, int run) {  // of positions run * U .. run * U + U - 1
  static_assert(32 % U == 0, "a run lies in one word");
  const unsigned w = mask[(run * U) >> 5] >> ((run * U) & 31);
  return unsigned(__builtin_amdgcn_readfirstlane(int(U == 32 ? w : w & ((1u << (U & 31)) - 1u))));
}

// Sequences without positions hand `from` (zeros if there is none) on to `to`, for the channels of this block.
template <int NW, typename F>
__device__ __forceinline__ void for_empty_sequences(const linrec_gated_t& p, int wave, int lane, F&& f) {
  for (int64_t base = int64_t(wave) * 64; base < p.sequences; base += 64 * NW) {
    const int64_t j = base + lane;
    uint64_t empty = __ballot(j < p.sequences && scan_bound(p, j < p.sequences ? j : 0) >= scan_bound(p, j < p.sequences ? j + 1 : 0));
    for (; empty; empty &= empty - 1) f(scan_sequence(p, base + __builtin_ctzll(empty)));
  }
}

// ---- the channels of a lane -------------------------------------------------------------------
// Lanes take VEC adjacent channels; the last one starts early where they are not a multiple of VEC and leaves the channels
// that the lane before it has to that one.  Lanes beyond read the last channels and store nothing.
template <int VEC>
struct Channels {
  int base;       // first channel of the block (the same for all lanes)
  unsigned rel;   // first channel of the lane, from there
  int own;        // first of its channels that the lane stores; VEC: none
  bool whole;     // every lane of the block stores all its channels
};
template <int VEC>
__device__ __forceinline__ Channels<VEC> lane_channels(int block, int lane, int channels) {
  Channels<VEC> ch;
  const int c0 = block * 64 * VEC, last = channels - VEC;
  const int want = c0 + lane * VEC, c = want < last ? want : last;
  ch.base = c0 < last ? c0 : last;
  ch.rel = unsigned(c - ch.base);
  ch.own = want - c < VEC ? want - c : VEC;
  ch.whole = c0 + 64 * VEC <= channels;
  return ch;
}
template <int VEC, typename T>
__device__ __forceinline__ void store_channels(T* p, const Lanes<VEC>& v, const Channels<VEC>& ch) {
  if (ch.whole) {
    st_any<VEC>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      if (e >= ch.own) p[e] = T(v.v[e]);
  }
}
template <int VEC>
__device__ __forceinline__ Lanes<VEC> load_floats(const float* p) {
  Lanes<VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = p[e];
  return r;
}
template <int VEC>
__device__ __forceinline__ void store_floats(float* p, const Lanes<VEC>& v, const Channels<VEC>& ch) {
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (e >= ch.own) p[e] = v.v[e];
}
template <typename P>
__device__ __forceinline__ P* plus_bytes(P* p, uint32_t bytes) {
  using C = std::conditional_t<std::is_const_v<P>, const char*, char*>;
  return reinterpret_cast<P*>(reinterpret_cast<C>(p) + bytes);
}

// ---- the chain of segments --------------------------------------------------------------------
// One wave, a channel to a lane: publishes the map (ta, tb) of segment k (in scan order), waits for what enters it and
// publishes what leaves it.  `cut`: a sequence starts inside, so tb leaves whatever enters.  `walk` computes what enters from
// the channel's own data.  mine: this segment's first word of the lane; a segment's words lie `per_segment` from the next one's,
// first words before second words, RPB each.
template <int RPB, typename W>
__device__ __forceinline__ float enter_segment(const TileArgs& ch, uint64_t* mine, long long per_segment, int k, int segments,
                                               uint32_t seq, int lane, float first, float ta, float tb, bool cut, W&& walk) {
  constexpr int LOOK = 4;
  const uint32_t want = (seq << 2) | STATUS_AGGREGATE, done = (seq << 2) | STATUS_INCLUSIVE;
  const bool last = k + 1 >= segments;
  if (!last) {
    if (cut) {
      st_desc(mine + RPB, pack_desc(done, tb));
    } else if (k > 0) {
      st_desc(mine, pack_desc(want, ta));
      st_desc(mine + RPB, pack_desc(want, tb));
    }
  }
  float entering = first;
  if (k > 0) {
    bool found = false;
    for (int polls = 0; polls < ch.spin_limit; ++polls) {
      uint64_t w0[LOOK], w1[LOOK];
#pragma unroll
      for (int q = 0; q < LOOK; ++q) {
        const uint64_t* d = mine - (q < k ? q + 1 : k) * per_segment;  // (beyond segment 0: asked for again, not used)
        w0[q] = ld_desc(d);
        w1[q] = ld_desc(d + RPB);
      }
      int from = -1;
      bool blocked = false;
#pragma unroll
      for (int q = 0; q < LOOK; ++q) {
        const uint32_t f1 = uint32_t(w1[q] >> 32);
        if (from < 0 && !blocked) {
          if (__ballot(f1 != done) == 0) from = q;
          else blocked = __ballot(f1 != done && !(f1 == want && uint32_t(w0[q] >> 32) == want)) != 0;
        }
      }
      if (from >= 0) {
#pragma unroll
        for (int q = LOOK - 1; q >= 0; --q) {
          const float a = __builtin_bit_cast(float, uint32_t(w0[q])), b = __builtin_bit_cast(float, uint32_t(w1[q]));
          if (q == from) entering = b;
          else if (q < from) entering = uint32_t(w1[q] >> 32) == done ? b : fmaf(a, entering, b);
        }
        found = true;
        break;
      }
      __builtin_amdgcn_s_sleep(1);
    }
    if (__builtin_expect(!found, 0)) {
      if (lane == 0) __hip_atomic_fetch_add(&ch.ws->gave_up, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      entering = walk();
    }
  }
  if (!last && !cut) st_desc(mine + RPB, pack_desc(done, fmaf(ta, entering, tb)));
  return entering;
}

// ---- forward ----------------------------------------------------------------------------------
template <typename T, int VEC, int U, int NW, bool PACKED>
__global__ __launch_bounds__(64 * NW) void gated_fwd_kernel(GatedArgs args) {
  constexpr int RPB = 64 * VEC, SEG = NW * U;
  static_assert(VEC <= NW && GATED_SAVE % U == 0, "a wave per channel of a lane looks back; values are saved where runs start");
  __shared__ float sh_a[NW][RPB];
  __shared__ float sh_b[NW][RPB];
  __shared__ float sh_in[RPB];
  __shared__ float sh_decay[RPB];
  __shared__ SegmentMarks<PACKED ? SEG : 1> marks;
  const linrec_gated_t& p = args.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned blocks = unsigned(args.channel_blocks) * unsigned(p.batch);
  const int k = int(blockIdx.x / blocks);
  const unsigned block = blockIdx.x - unsigned(k) * blocks;
  const int batch = int(block / unsigned(args.channel_blocks));
  const int channels = int(p.channels), time = int(p.time);
  const Channels<VEC> ch = lane_channels<VEC>(int(block) - batch * args.channel_blocks, lane, channels);
  const uint32_t seq = args.segments > 1 ? load_seq_through_caches(args.chain.ws) : 0u;

  const uint32_t lane_bytes = ch.rel * uint32_t(sizeof(T));
  const T* x = static_cast<const T*>(p.x) + batch * p.x_stride[0] + ch.base;
  const T* ga = static_cast<const T*>(p.gate_a) + batch * p.gate_a_stride[0] + ch.base;
  const T* gx = static_cast<const T*>(p.gate_x) + batch * p.gate_x_stride[0] + ch.base;
  T* h = static_cast<T*>(p.h) + (int64_t)batch * time * channels + ch.base;
  const int n0 = k * SEG + wave * U;
  auto position = [&](int n) __attribute__((always_inline)) { return int64_t(p.reverse ? time - 1 - n : n); };

  auto segment = [&](auto full_tag) __attribute__((always_inline)) {
    constexpr bool FULL = decltype(full_tag)::value;
    Held<T, VEC> hx[U], ha[U], hg[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (FULL || n0 + u < time) {
        const int64_t l = position(n0 + u);
        hx[u] = ld_any<VEC, true>(plus_bytes(x + l * p.x_stride[1], lane_bytes));
        ha[u] = ld_any<VEC, true>(plus_bytes(ga + l * p.gate_a_stride[1], lane_bytes));
        hg[u] = ld_any<VEC, true>(plus_bytes(gx + l * p.gate_x_stride[1], lane_bytes));
      }
    }
    if (wave < VEC) {  // a channel to a lane
      const float rate = p.rate[ch.base + int(ch.rel) + wave];
      sh_decay[wave * 64 + lane] = LOG2E * p.scale * fast_softplus(rate);
    }
    unsigned starts = 0, ends = 0;
    if constexpr (PACKED) mark_segment<SEG, 64 * NW>(marks, p, k * SEG);
    __syncthreads();
    if constexpr (PACKED) {
      starts = run_bits<U>(marks.starts, wave);
      ends = run_bits<U>(marks.ends, wave);
    }
    auto initial = [&](int u) __attribute__((always_inline)) {
      Lanes<VEC> r;
      if (p.h0) r = load_floats<VEC>(p.h0 + int64_t(__builtin_amdgcn_readfirstlane(marks.start[wave * U + u])) * channels + ch.base + ch.rel);
      else for (int e = 0; e < VEC; ++e) r.v[e] = 0.0f;
      return r;
    };
    Lanes<VEC> decay, ma, mb, a[U], b[U];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      decay.v[e] = sh_decay[e * 64 + lane];
      ma.v[e] = 1.0f;
      mb.v[e] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (FULL || n0 + u < time) {
        const Lanes<VEC> vx = widen(hx[u]), va = widen(ha[u]), vg = widen(hg[u]);
        if constexpr (PACKED) {
          if (starts >> u & 1u) mb = initial(u);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const Gate g = gate_of(va.v[e], vg.v[e], decay.v[e]);
          a[u].v[e] = g.a;
          b[u].v[e] = taken_in(g, vx.v[e]);
          mb.v[e] = fmaf(g.a, mb.v[e], b[u].v[e]);
          ma.v[e] *= g.a;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sh_a[wave][e * 64 + lane] = never_zero(ma.v[e]);
      sh_b[wave][e * 64 + lane] = mb.v[e];
    }
    __syncthreads();
    if (wave < VEC) {
      const int i = wave * 64 + lane;
      const int c = ch.base + int(ch.rel) + wave;
      float ta = sh_a[0][i], tb = sh_b[0][i];
      bool cut = PACKED && run_bits<U>(marks.starts, 0) != 0;
#pragma unroll
      for (int w = 1; w < NW; ++w) {
        if (PACKED && run_bits<U>(marks.starts, w) != 0) {
          tb = sh_b[w][i];
          cut = true;
        } else {
          tb = fmaf(sh_a[w][i], tb, sh_b[w][i]);
          ta = never_zero(ta * sh_a[w][i]);
        }
      }
      const float first = !PACKED && p.h0 ? p.h0[int64_t(batch) * channels + c] : 0.0f;
      const long long per_segment = 2ll * blocks * RPB;
      uint64_t* mine = args.chain.desc + k * per_segment + 2ll * block * RPB + i;
      sh_in[i] = enter_segment<RPB>(args.chain, mine, per_segment, k, args.segments, seq, lane, first, ta, tb, cut, [&] {
        int from = 0;
        float v = first;
        if constexpr (PACKED) {
          const int64_t j = bounds_up_to(p, k * SEG - 1) - 1;
          if (j >= 0) {
            from = scan_bound(p, j);
            if (p.h0 && j < p.sequences) v = p.h0[scan_sequence(p, j) * channels + c];
          }
        }
        const float d2 = sh_decay[i];
        for (int n = from; n < k * SEG; ++n) {
          const int64_t l = position(n), o = int64_t(ch.rel) + wave;
          const Gate g = gate_of(float(ga[l * p.gate_a_stride[1] + o]), float(gx[l * p.gate_x_stride[1] + o]), d2);
          v = fmaf(g.a, v, taken_in(g, float(x[l * p.x_stride[1] + o])));
        }
        return v;
      });
    }
    __syncthreads();
    Lanes<VEC> val;
#pragma unroll
    for (int e = 0; e < VEC; ++e) val.v[e] = sh_in[e * 64 + lane];
    for (int w = 0; w < wave; ++w) {
      const bool cut = PACKED && run_bits<U>(marks.starts, w) != 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float wa = sh_a[w][e * 64 + lane], wb = sh_b[w][e * 64 + lane];
        val.v[e] = cut ? wb : fmaf(wa, val.v[e], wb);
      }
    }
    if (p.saved && n0 % GATED_SAVE == 0 && n0 < time) {
      const int saves = (time + GATED_SAVE - 1) / GATED_SAVE;
      store_floats(p.saved + (int64_t(batch) * saves + n0 / GATED_SAVE) * channels + ch.base + ch.rel, val, ch);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (FULL || n0 + u < time) {
        if constexpr (PACKED) {
          if (starts >> u & 1u) val = initial(u);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) val.v[e] = fmaf(a[u].v[e], val.v[e], b[u].v[e]);
        store_channels(plus_bytes(h + position(n0 + u) * channels, lane_bytes), val, ch);
        if (p.state) {
          if constexpr (PACKED) {
            if (ends >> u & 1u)
              store_floats(p.state + int64_t(__builtin_amdgcn_readfirstlane(marks.end[wave * U + u])) * channels + ch.base + ch.rel, val, ch);
          } else if (n0 + u == time - 1) {
            store_floats(p.state + int64_t(batch) * channels + ch.base + ch.rel, val, ch);
          }
        }
      }
    }
  };
  if ((k + 1) * int64_t(SEG) <= time) segment(std::true_type{});
  else segment(std::false_type{});

  if (PACKED && k == 0 && p.state)
    for_empty_sequences<NW>(p, wave, lane, [&](int64_t n) {
      Lanes<VEC> v;
      for (int e = 0; e < VEC; ++e) v.v[e] = p.h0 ? p.h0[n * channels + ch.base + ch.rel + e] : 0.0f;
      store_floats(p.state + n * channels + ch.base + ch.rel, v, ch);
    });
  // (the look-back waves are past the last barrier: this workgroup touches no descriptor of the launch again)
  if (args.segments > 1 && threadIdx.x == 0) {
    const uint32_t leaf_count = signal_tile_done_begin(args.chain, blockIdx.x);
    signal_tile_done_end(args.chain, blockIdx.x, seq, leaf_count);
  }
}

// ---- backward ---------------------------------------------------------------------------------
template <typename T, int VEC, int U, int NW, bool PACKED>
__global__ __launch_bounds__(64 * NW) void gated_bwd_kernel(GatedArgs args) {
  constexpr int RPB = 64 * VEC, SEG = NW * U;
  static_assert(VEC <= NW && SEG == GATED_SAVE, "a segment starts where a value was saved");
  __shared__ float sh_a[NW][RPB];
  __shared__ float sh_b[NW][RPB];
  __shared__ float sh_g[NW][RPB];
  __shared__ float sh_in[RPB];
  __shared__ float sh_decay[RPB];
  __shared__ SegmentMarks<PACKED ? SEG : 1> marks;
  const linrec_gated_t& p = args.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned blocks = unsigned(args.channel_blocks) * unsigned(p.batch);
  const int kk = int(blockIdx.x / blocks);  // segments from the far end
  const int k = args.segments - 1 - kk;
  const unsigned block = blockIdx.x - unsigned(kk) * blocks;
  const int batch = int(block / unsigned(args.channel_blocks));
  const int channels = int(p.channels), time = int(p.time);
  const Channels<VEC> ch = lane_channels<VEC>(int(block) - batch * args.channel_blocks, lane, channels);
  const uint32_t seq = args.segments > 1 ? load_seq_through_caches(args.chain.ws) : 0u;

  const uint32_t lane_bytes = ch.rel * uint32_t(sizeof(T));
  const T* x = static_cast<const T*>(p.x) + batch * p.x_stride[0] + ch.base;
  const T* ga = static_cast<const T*>(p.gate_a) + batch * p.gate_a_stride[0] + ch.base;
  const T* gx = static_cast<const T*>(p.gate_x) + batch * p.gate_x_stride[0] + ch.base;
  const T* dh = static_cast<const T*>(p.d_h) + batch * p.d_h_stride[0] + ch.base;
  const int64_t dense = (int64_t)batch * time * channels + ch.base;
  T* dx = static_cast<T*>(p.d_x) + dense;
  T* dga = static_cast<T*>(p.d_gate_a) + dense;
  T* dgx = static_cast<T*>(p.d_gate_x) + dense;
  const int n0 = k * SEG + wave * U;
  auto position = [&](int n) __attribute__((always_inline)) { return int64_t(p.reverse ? time - 1 - n : n); };

  auto segment = [&](auto full_tag) __attribute__((always_inline)) {
    constexpr bool FULL = decltype(full_tag)::value;
    Held<T, VEC> hx[U], ha[U], hg[U], hd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (FULL || n0 + u < time) {
        const int64_t l = position(n0 + u);
        hx[u] = ld_any<VEC, true>(plus_bytes(x + l * p.x_stride[1], lane_bytes));
        ha[u] = ld_any<VEC, true>(plus_bytes(ga + l * p.gate_a_stride[1], lane_bytes));
        hg[u] = ld_any<VEC, true>(plus_bytes(gx + l * p.gate_x_stride[1], lane_bytes));
        hd[u] = ld_any<VEC, true>(plus_bytes(dh + l * p.d_h_stride[1], lane_bytes));
      }
    }
    Lanes<VEC> val = load_floats<VEC>(p.saved + (int64_t(batch) * args.segments + k) * channels + ch.base + ch.rel);
    if (wave < VEC) {
      const float rate = p.rate[ch.base + int(ch.rel) + wave];
      sh_decay[wave * 64 + lane] = LOG2E * p.scale * fast_softplus(rate);
    }
    unsigned starts = 0, ends = 0;
    if constexpr (PACKED) mark_segment<SEG, 64 * NW>(marks, p, k * SEG);
    __syncthreads();
    if constexpr (PACKED) {
      starts = run_bits<U>(marks.starts, wave);
      ends = run_bits<U>(marks.ends, wave);
    }
    auto rows_of = [&](const float* t, const int* which, int u) __attribute__((always_inline)) {
      Lanes<VEC> r;
      if (t) r = load_floats<VEC>(t + int64_t(__builtin_amdgcn_readfirstlane(which[wave * U + u])) * channels + ch.base + ch.rel);
      else for (int e = 0; e < VEC; ++e) r.v[e] = 0.0f;
      return r;
    };
    Lanes<VEC> decay, ma, mb, mg, a[U], b[U];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      decay.v[e] = sh_decay[e * 64 + lane];
      ma.v[e] = 1.0f;
      mb.v[e] = mg.v[e] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (FULL || n0 + u < time) {
        const Lanes<VEC> vx = widen(hx[u]), va = widen(ha[u]), vg = widen(hg[u]);
        if constexpr (PACKED) {
          if (starts >> u & 1u) mb = rows_of(p.h0, marks.start, u);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const Gate g = gate_of(va.v[e], vg.v[e], decay.v[e]);
          a[u].v[e] = g.a;
          b[u].v[e] = taken_in(g, vx.v[e]);
          mb.v[e] = fmaf(g.a, mb.v[e], b[u].v[e]);
          ma.v[e] *= g.a;
        }
      }
    }
#pragma unroll
    for (int u = U - 1; u >= 0; --u) {
      if (FULL || n0 + u < time) {
        const Lanes<VEC> vd = widen(hd[u]);
        if constexpr (PACKED) {
          if (ends >> u & 1u) mg = rows_of(p.d_state, marks.end, u);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) mg.v[e] = a[u].v[e] * (mg.v[e] + vd.v[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sh_a[wave][e * 64 + lane] = never_zero(ma.v[e]);
      sh_b[wave][e * 64 + lane] = mb.v[e];
      sh_g[wave][e * 64 + lane] = mg.v[e];
    }
    __syncthreads();
    if (wave < VEC) {
      const int i = wave * 64 + lane;
      const int c = ch.base + int(ch.rel) + wave;
      float ta = sh_a[NW - 1][i], tg = sh_g[NW - 1][i];
      bool cut = PACKED && run_bits<U>(marks.ends, NW - 1) != 0;
#pragma unroll
      for (int w = NW - 2; w >= 0; --w) {
        if (PACKED && run_bits<U>(marks.ends, w) != 0) {
          tg = sh_g[w][i];
          cut = true;
        } else {
          tg = fmaf(sh_a[w][i], tg, sh_g[w][i]);
          ta = never_zero(ta * sh_a[w][i]);
        }
      }
      const float first = !PACKED && p.d_state ? p.d_state[int64_t(batch) * channels + c] : 0.0f;
      const long long per_segment = 2ll * blocks * RPB;
      uint64_t* mine = args.chain.desc + kk * per_segment + 2ll * block * RPB + i;
      sh_in[i] = enter_segment<RPB>(args.chain, mine, per_segment, kk, args.segments, seq, lane, first, ta, tg, cut, [&] {
        int from = time;
        float v = first;
        if constexpr (PACKED) {
          const int64_t j = bounds_up_to(p, (k + 1) * SEG) - 1;  // the sequence of the position after this segment
          if (j >= 0 && j < p.sequences) {
            from = scan_bound(p, j + 1);
            // (a sequence that starts right there ends its own walk at its start: nothing of it enters this segment)
            if (p.d_state) v = p.d_state[scan_sequence(p, j) * channels + c];
          }
        }
        const float d2 = sh_decay[i];
        for (int n = from - 1; n >= (k + 1) * SEG; --n) {
          const int64_t l = position(n), o = int64_t(ch.rel) + wave;
          const float an = __builtin_amdgcn_exp2f(-d2 * fast_sigmoid(float(ga[l * p.gate_a_stride[1] + o])));
          v = an * (v + float(dh[l * p.d_h_stride[1] + o]));
        }
        return v;
      });
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
      const bool cut = PACKED && run_bits<U>(marks.starts, w) != 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float wa = sh_a[w][e * 64 + lane], wb = sh_b[w][e * 64 + lane];
        val.v[e] = cut ? wb : fmaf(wa, val.v[e], wb);
      }
    }
    Lanes<VEC> back, sum;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      back.v[e] = sh_in[e * 64 + lane];
      sum.v[e] = 0.0f;
    }
    for (int w = NW - 1; w > wave; --w) {
      const bool cut = PACKED && run_bits<U>(marks.ends, w) != 0;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float wa = sh_a[w][e * 64 + lane], wg = sh_g[w][e * 64 + lane];
        back.v[e] = cut ? wg : fmaf(wa, back.v[e], wg);
      }
    }
    // the values before each position, in the place of what the position takes in
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (FULL || n0 + u < time) {
        if constexpr (PACKED) {
          if (starts >> u & 1u) val = rows_of(p.h0, marks.start, u);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float before = val.v[e];
          val.v[e] = fmaf(a[u].v[e], before, b[u].v[e]);
          b[u].v[e] = before;
        }
      }
    }
#pragma unroll
    for (int u = U - 1; u >= 0; --u) {
      if (FULL || n0 + u < time) {
        const Lanes<VEC> vx = widen(held_again(hx[u])), va = widen(held_again(ha[u])), vg = widen(held_again(hg[u])),
                         vd = widen(held_again(hd[u]));
        Lanes<VEC> ox, oa, og;
        if constexpr (PACKED) {
          if (ends >> u & 1u) back = rows_of(p.d_state, marks.end, u);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const Gate g = gate_of(va.v[e], vg.v[e], decay.v[e]);
          const float grad = vd.v[e] + back.v[e];
          const float log_a = LN2 * g.log2_a;
          const float inv_m = g.m2 > 0.0f ? __builtin_amdgcn_rsqf(g.m2) : 0.0f;
          const float gmx = grad * (g.m2 * inv_m) * g.sx;
          const float sx_x = g.sx * vx.v[e];
          const float q = grad * log_a * g.a * fmaf(-sx_x * g.a, inv_m, b[u].v[e]);
          ox.v[e] = gmx;
          og.v[e] = gmx * vx.v[e] * (1.0f - g.sx);
          oa.v[e] = q * (1.0f - g.sa);
          sum.v[e] += q;
          back.v[e] = g.a * grad;
        }
        const int64_t o = position(n0 + u) * channels;
        store_channels(plus_bytes(dx + o, lane_bytes), ox, ch);
        store_channels(plus_bytes(dga + o, lane_bytes), oa, ch);
        store_channels(plus_bytes(dgx + o, lane_bytes), og, ch);
        if (p.d_h0) {
          if constexpr (PACKED) {
            if (starts >> u & 1u)
              store_floats(p.d_h0 + int64_t(__builtin_amdgcn_readfirstlane(marks.start[wave * U + u])) * channels + ch.base + ch.rel, back, ch);
          } else if (n0 + u == 0) {
            store_floats(p.d_h0 + int64_t(batch) * channels + ch.base + ch.rel, back, ch);
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) sh_b[wave][e * 64 + lane] = sum.v[e];
    __syncthreads();
    if (wave < VEC) {
      const int i = wave * 64 + lane;
      float s = sh_b[0][i];
#pragma unroll
      for (int w = 1; w < NW; ++w) s += sh_b[w][i];
      if (wave >= ch.own) p.partial[(int64_t(batch) * args.segments + k) * channels + ch.base + int(ch.rel) + wave] = s;
    }
  };
  if ((k + 1) * int64_t(SEG) <= time) segment(std::true_type{});
  else segment(std::false_type{});

  if (PACKED && kk == 0 && p.d_h0)
    for_empty_sequences<NW>(p, wave, lane, [&](int64_t n) {
      Lanes<VEC> v;
      for (int e = 0; e < VEC; ++e) v.v[e] = p.d_state ? p.d_state[n * channels + ch.base + ch.rel + e] : 0.0f;
      store_floats(p.d_h0 + n * channels + ch.base + ch.rel, v, ch);
    });
  if (args.segments > 1 && threadIdx.x == 0) {
    const uint32_t leaf_count = signal_tile_done_begin(args.chain, blockIdx.x);
    signal_tile_done_end(args.chain, blockIdx.x, seq, leaf_count);
  }
}

}  // namespace linrec
