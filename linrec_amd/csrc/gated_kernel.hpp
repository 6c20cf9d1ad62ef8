// Gated linear recurrence in one launch a pass, and its single-token step.
//
//   log a = -decay sigmoid(gate_a),  decay = scale softplus(rate)
//   h[t] = a h[t-1] + m sigmoid(gate_x) x,  m = sqrt(1 - a^2) = sqrt(-expm1(2 log a))
//
// The scan axis is cut into segments of NW * U positions; a workgroup takes one segment of 64 * VEC channels, wave w the run
// [w*U, w*U + U), and the segments of a channel are chained through descriptors in global memory.  The gates are evaluated on the
// way in, so forward reads three tensors and writes one, where coefficients and inputs made by elementwise kernels first are
// written and read once more each.
//
// Backward, g[t] = d_h[t] + a[t+1] g[t+1] in the opposite direction over the same segments:
//   d_x = g m sx,  d_gate_x = g m x sx (1 - sx)                         (sx, sa: the gates' sigmoids)
//   P = g (log a a h[t-1] - sx x a^2 log a / m),  d_gate_a = P (1 - sa),  d_rate = sigmoid(rate) / softplus(rate) sum P
// (log a and log a / m both go to zero with sigmoid(gate_a), where 1 / m alone does not: every term stays finite.)  h[t-1] is
// not read: the forward saves the value that enters every backward segment of 64 positions as 4 bytes, and the backward goes on
// from there with the same operations, so the gradient sees the unrounded values and four tensors are read where the saved output
// would make it five.
//
// What bounds it: memory where channels are many.  8 x 4096 x 2048 in bf16: 122 us forward (537 MB, 4.4 TB/s of the 5.2 TB/s that
// a copy reaches) and 221 us backward (940 MB, 4.2 TB/s); 16 x 2048 x 512 in fp32 out of a projection's rows 57 and 104 us (4.7 and
// 4.5 TB/s).  Without the wait for what enters a segment the former takes 111 and 200 us: the wait is the larger part of the rest,
// the gates' arithmetic the smaller.  With few rows the chain bounds it: 1 x 32768 x 2048 132 and 231 us, 1 x 131072 x 64 49
// and 81 us (floors 103, 181; 13, 23); the former 30 and 35 us less without the wait, 1 x 100001 x 250 22 and 31 of 79 and 129.
//
// Waves and runs: workgroups wait, so that several to a CU have to hide each other's waits, with all that a segment holds in
// registers: at most 128 a lane for sixteen waves to a CU, and as little spilled as can be (32 registers that are cost 7 to 20 %).
// Forward keeps a and the input of 16 positions of two channels, backward a, m and h[t-1] of 8, and the sigmoids in LDS, which
// saves evaluating them twice.  Forward and backward, 8 x 4096 x 2048 and 1 x 100001 x 250 bf16:
//   forward, positions of a wave x waves    16 x 4  123 and 81 us    16 x 8  130 and 76    8 x 4  144 and 105    8 x 8  159 and 100
//   backward                                 8 x 8  222 and 138       8 x 4  222 and 151    4 x 8  299 and 184
// (longer segments make fewer links, more of them hide each other's waits; shorter runs do more links for what is under way; the rows
// of 250 were stored past the caches then, and take 79 and 129 us through them).
//
// The value that enters a segment is always the same chain of multiply-adds over the segments before, whichever of them had
// published what when they were looked at: results are the same bits in every run in which no wait runs out.
//
// A position at which a packed sequence starts takes the sequence's own initial value instead of what comes from before it, so
// nothing passes from one sequence to the next, not even by 0 * inf.  A segment that holds a start publishes what leaves it
// without a wait.
//
// A wait is for segments of smaller workgroup number only, and bounded; a lane whose wait runs out walks its channel from the
// sequence's start, which gives the value by other roundings.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/linrec_layers.h"
#include "collook_kernel.hpp"
#include "gated_chain.hpp"

namespace linrec {

struct GatedArgs {
  linrec_gated_t p;
  TileArgs chain;
  int segments;         // of the scan axis
  int channel_blocks;
  int side;             // segments side by side
  int save;             // positions from one saved value to the next: those of a backward segment
};

// Workgroups go through the segments in sets of `side`, through the blocks of channels within a set and the set's segments within
// a block, so that waits are for smaller numbers.  Sets of a group: its segments run side by side, and what they read is near, 8 x
// 4096 x 2048 bf16 124 and 221 us (one by one 128 and 221), 1 x 32768 x 2048 134 and 247 (154 and 293).  Workgroups are dealt to the
// eight XCDs in turn, so that in sets of eight neighbouring blocks of a segment run on the same one; where rows are not whole lines
// of 128 bytes they write parts of the same lines, which one L2 puts together: 16 x 6250 x 250 bf16 73 and 130 us instead of 81 and
// 144, 4 x 4096 x 1000 43 and 76 instead of 49 and 86 (for whole lines eight are slower: 127 and 235, 136 and 248 above).
struct Place {
  int segment;
  unsigned block;
};
__device__ __forceinline__ Place place_of(const GatedArgs& args, unsigned blocks) {
  const unsigned per_set = blocks * unsigned(args.side), set = blockIdx.x / per_set, in_set = blockIdx.x - set * per_set;
  const unsigned first = set * unsigned(args.side), width = min(unsigned(args.side), unsigned(args.segments) - first);
  const unsigned block = in_set / width;
  return {__builtin_amdgcn_readfirstlane(int(first + in_set - block * width)), unsigned(__builtin_amdgcn_readfirstlane(int(block)))};
}

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
struct Gate {
  float sa, sx;  // sigmoids
  float a;
  float m2;      // 1 - a^2
};
// decay2: the decay rate in base 2.  1 - a^2 = 1 - exp(u), u = 2 log a: the difference cancels where u is small, and six terms of
// the series are off by 4e-8 of the result at u = -1/8 (in l = log2 a: the coefficients are (2 ln 2)^n / n!).
__device__ __forceinline__ Gate gate_of(float ga, float gx, float decay2) {
  constexpr float C1 = 2.0f * LN2, C2 = C1 * C1 / 2.0f, C3 = C2 * C1 / 3.0f, C4 = C3 * C1 / 4.0f, C5 = C4 * C1 / 5.0f, C6 = C5 * C1 / 6.0f;
  Gate g;
  g.sa = fast_sigmoid(ga);
  g.sx = fast_sigmoid(gx);
  const float l = -decay2 * g.sa;
  g.a = __builtin_amdgcn_exp2f(l);
  const float series = -l * fmaf(l, fmaf(l, fmaf(l, fmaf(l, fmaf(l, C6, C5), C4), C3), C2), C1);
  g.m2 = l > -0.125f / C1 ? series : fmaf(-g.a, g.a, 1.0f);
  return g;
}
__device__ __forceinline__ float taken_in(const Gate& g, float x) { return __builtin_amdgcn_sqrtf(g.m2) * g.sx * x; }

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
template <int SEG>
__device__ __forceinline__ bool any_mark(const SegmentMarks<SEG>& m) {  // (the same for all lanes)
  unsigned bits = 0;
#pragma unroll
  for (int i = 0; i < (SEG + 31) / 32; ++i) bits |= m.starts[i] | m.ends[i];
  return __builtin_amdgcn_readfirstlane(int(bits)) != 0;
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
// WHOLE: every lane of the block stores all its channels.  LINES: rows are whole lines of 128 bytes, and stored past the caches (8 x
// 4096 x 2048 bf16 backward 220 us, through them 227); others go through them, where the parts of a line that neighbouring blocks
// and rows write come together (16 x 6250 x 250 bf16 69 and 113 us, past them 74 and 132; 8 x 4096 x 1001 fp32 123 and 233, past them
// 140 and 274).
template <bool LINES, bool WHOLE, int VEC, typename T>
__device__ __forceinline__ void store_channels(T* p, const Lanes<VEC>& v, const Channels<VEC>& ch) {
  auto store = [&]() __attribute__((always_inline)) {
    if constexpr (LINES) {
      st_any<VEC>(p, v);
    } else if constexpr (VEC == 1) {
      *p = T(v.v[0]);
    } else {
      using A = typename AnyPack<T, VEC>::type;
      A q;
#pragma unroll
      for (int e = 0; e < VEC; ++e) q[e] = T(v.v[e]);
      *reinterpret_cast<A*>(p) = q;
    }
  };
  if constexpr (WHOLE) {
    store();
  } else {
    if (ch.own == 0) {
      store();
    } else {
#pragma unroll
      for (int e = 1; e < VEC; ++e)
        if (e >= ch.own) p[e] = T(v.v[e]);
    }
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
// ---- positions of a wave ----------------------------------------------------------------------
// A tensor's positions from the first of a run on, in scan order: a scalar address that goes on by a scalar step, the lane's
// part 32 bits beside it.  (Read as a scalar at each access, or the lane's part is
// added first and every access carries a 64-bit vector address.)
template <typename P>
struct Walk {
  P* at;
  int64_t step;  // elements
  __device__ __forceinline__ Walk(P* tensor, int64_t stride, int n0, int time, bool reverse)
      : at(tensor + int64_t(reverse ? time - 1 - n0 : n0) * stride), step(reverse ? -stride : stride) {}
  __device__ __forceinline__ P* lane(uint32_t bytes) const { return plus_bytes(scalar(at), bytes); }
  __device__ __forceinline__ void next() { at += step; }
  __device__ __forceinline__ void back() { at -= step; }
};

// ---- forward ----------------------------------------------------------------------------------
template <typename T, int VEC, int U, int NW, bool PACKED, bool LINES>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(4))) void gated_fwd_kernel(GatedArgs args) {
  constexpr int RPB = 64 * VEC, SEG = NW * U;
  static_assert(VEC <= NW, "a wave per channel of a lane looks back");
  __shared__ float sh_a[NW][RPB];
  __shared__ float sh_b[NW][RPB];  // the waves' maps, then what enters the waves
  __shared__ float sh_decay[RPB];
  __shared__ SegmentMarks<PACKED ? SEG : 1> marks;
  const linrec_gated_t& p = args.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned blocks = unsigned(args.channel_blocks) * unsigned(p.batch);
  const Place at = place_of(args, blocks);
  const int k = at.segment;
  const unsigned block = at.block;
  const int batch = __builtin_amdgcn_readfirstlane(int(block / unsigned(args.channel_blocks)));
  const int channels = int(p.channels), time = int(p.time);
  const Channels<VEC> ch = lane_channels<VEC>(int(block) - batch * args.channel_blocks, lane, channels);
  const uint32_t seq = args.segments > 1 ? load_seq_through_caches(args.chain.ws) : 0u;
  const bool reverse = p.reverse != 0;

  const uint32_t lane_bytes = ch.rel * uint32_t(sizeof(T));
  const T* x = static_cast<const T*>(p.x) + batch * p.x_stride[0] + ch.base;
  const T* ga = static_cast<const T*>(p.gate_a) + batch * p.gate_a_stride[0] + ch.base;
  const T* gx = static_cast<const T*>(p.gate_x) + batch * p.gate_x_stride[0] + ch.base;
  const int n0 = k * SEG + wave * U;
  const bool full = time - k * SEG >= SEG;

  bool plain = full;
  if constexpr (PACKED) {
    mark_segment<SEG, 64 * NW>(marks, p, k * SEG);
    __syncthreads();
    plain = plain && !any_mark(marks);
  }

  // PLAIN: every position of the segment exists and no sequence starts or ends in it.
  auto segment = [&](auto plain_tag, auto whole_tag) __attribute__((always_inline)) {
    constexpr bool PLAIN = decltype(plain_tag)::value, WHOLE = decltype(whole_tag)::value, CUTS = PACKED && !PLAIN;
    Held<T, VEC> hx[U], ha[U], hg[U];
    {
      Walk<const T> wx(x, p.x_stride[1], n0, time, reverse), wa(ga, p.gate_a_stride[1], n0, time, reverse),
          wg(gx, p.gate_x_stride[1], n0, time, reverse);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (PLAIN || n0 + u < time) {
          hx[u] = ld_any<VEC, true>(wx.lane(lane_bytes));
          ha[u] = ld_any<VEC, true>(wa.lane(lane_bytes));
          hg[u] = ld_any<VEC, true>(wg.lane(lane_bytes));
        }
        wx.next();
        wa.next();
        wg.next();
      }
    }
    if (wave < VEC) {  // a channel to a lane
      const float rate = p.rate[ch.base + int(ch.rel) + wave];
      sh_decay[wave * 64 + lane] = LOG2E * p.scale * fast_softplus(rate);
    }
    __syncthreads();

    unsigned starts = 0, ends = 0;
    if constexpr (CUTS) {
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
      if (PLAIN || n0 + u < time) {
        const Lanes<VEC> vx = widen(hx[u]), va = widen(ha[u]), vg = widen(hg[u]);
        if constexpr (CUTS) {
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
        if constexpr (CUTS) {
          if (starts >> u & 1u) b[u] = mb;  // (whatever is before)
        }
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sh_a[wave][e * 64 + lane] = never_zero(ma.v[e]);
      sh_b[wave][e * 64 + lane] = mb.v[e];
    }
    __syncthreads();
    if (wave < VEC) {  // a channel to a lane
      const int e = wave, i = e * 64 + lane;
      const int c = ch.base + int(ch.rel) + e;
      bool any = false;
      float ta = 1.0f, tb = 0.0f;
      {
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float wa = sh_a[w][i], wb = sh_b[w][i];
          if (CUTS && run_bits<U>(marks.starts, w) != 0) {
            tb = wb;
            any = true;
          } else {
            tb = fmaf(wa, tb, wb);
            ta = never_zero(ta * wa);
          }
        }
      }
      const long long per_segment = 2ll * blocks * RPB;
      uint64_t* words = args.chain.desc + 2ll * block * RPB + e * 64;
      const Chain chain{words, uint32_t(lane) * 8, per_segment, k, args.segments, seq};
      const float first = !PACKED && p.h0 ? p.h0[int64_t(batch) * channels + c] : 0.0f;
      auto walk = [&] {
        int from = 0;
        float w = first;
        if constexpr (PACKED) {
          const int64_t j = bounds_up_to(p, k * SEG - 1) - 1;
          if (j >= 0) {
            from = scan_bound(p, j);
            if (p.h0 && j < p.sequences) w = p.h0[scan_sequence(p, j) * channels + c];
          }
        }
        const float d2 = sh_decay[i];
        for (int n = from; n < k * SEG; ++n) {
          const int64_t l = reverse ? time - 1 - n : n, o = int64_t(ch.rel) + e;
          const Gate g = gate_of(float(ga[l * p.gate_a_stride[1] + o]), float(gx[l * p.gate_x_stride[1] + o]), d2);
          w = fmaf(g.a, w, taken_in(g, float(x[l * p.x_stride[1] + o])));
        }
        return w;
      };
      float v = enter_segment<RPB>(args.chain, chain, lane, first, ta, tb, any, walk);
      {
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float wa = sh_a[w][i], wb = sh_b[w][i];
          sh_b[w][i] = v;
          v = CUTS && run_bits<U>(marks.starts, w) != 0 ? wb : fmaf(wa, v, wb);
        }
      }
    }
    __syncthreads();
    Lanes<VEC> val;
#pragma unroll
    for (int e = 0; e < VEC; ++e) val.v[e] = sh_b[wave][e * 64 + lane];
    if (p.saved && (n0 & (args.save - 1)) == 0 && n0 < time) {
      const int saves = (time + args.save - 1) / args.save;
      store_floats(p.saved + (int64_t(batch) * saves + n0 / args.save) * channels + ch.base + ch.rel, val, ch);
    }
    Walk<T> wh(static_cast<T*>(p.h) + (int64_t)batch * time * channels + ch.base, channels, n0, time, reverse);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (PLAIN || n0 + u < time) {
        if (CUTS && (starts >> u & 1u)) {
          val = b[u];
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) val.v[e] = fmaf(a[u].v[e], val.v[e], b[u].v[e]);
        }
        T* to = wh.lane(lane_bytes);
        wh.next();
        store_channels<LINES, WHOLE>(to, val, ch);
        if (CUTS && p.state && (ends >> u & 1u))
          store_floats(p.state + int64_t(__builtin_amdgcn_readfirstlane(marks.end[wave * U + u])) * channels + ch.base + ch.rel, val, ch);
        if (!PACKED && (!PLAIN || u == U - 1) && n0 + u == time - 1 && p.state)
          store_floats(p.state + int64_t(batch) * channels + ch.base + ch.rel, val, ch);
      }
    }
  };
  if (plain && ch.whole) segment(std::true_type{}, std::true_type{});
  else if (plain) segment(std::true_type{}, std::false_type{});
  else segment(std::false_type{}, std::false_type{});

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
template <typename T, int VEC, int U, int NW, bool PACKED, bool LINES>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(4))) void gated_bwd_kernel(GatedArgs args) {
  constexpr int RPB = 64 * VEC, SEG = NW * U;
  static_assert(2 * VEC <= NW, "a wave per channel of a lane and direction");
  __shared__ float sh_a[NW][RPB];
  __shared__ float sh_b[NW][RPB];  // forward maps, then what enters the waves forward
  __shared__ float sh_g[NW][RPB];  // the same backward
  __shared__ Lanes<VEC> sigmoids[SEG][2][64];
  __shared__ float sh_decay[RPB];
  __shared__ SegmentMarks<PACKED ? SEG : 1> marks;
  const linrec_gated_t& p = args.p;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned blocks = unsigned(args.channel_blocks) * unsigned(p.batch);
  const Place at = place_of(args, blocks);
  const int kk = at.segment;  // from the far end
  const int k = args.segments - 1 - kk;
  const unsigned block = at.block;
  const int batch = __builtin_amdgcn_readfirstlane(int(block / unsigned(args.channel_blocks)));
  const int channels = int(p.channels), time = int(p.time);
  const Channels<VEC> ch = lane_channels<VEC>(int(block) - batch * args.channel_blocks, lane, channels);
  const uint32_t seq = args.segments > 1 ? load_seq_through_caches(args.chain.ws) : 0u;
  const bool reverse = p.reverse != 0;

  const uint32_t lane_bytes = ch.rel * uint32_t(sizeof(T));
  const T* x = static_cast<const T*>(p.x) + batch * p.x_stride[0] + ch.base;
  const T* ga = static_cast<const T*>(p.gate_a) + batch * p.gate_a_stride[0] + ch.base;
  const T* gx = static_cast<const T*>(p.gate_x) + batch * p.gate_x_stride[0] + ch.base;
  const T* dh = static_cast<const T*>(p.d_h) + batch * p.d_h_stride[0] + ch.base;
  const int n0 = k * SEG + wave * U;
  const bool full = time - k * SEG >= SEG;

  bool plain = full;
  if constexpr (PACKED) {
    mark_segment<SEG, 64 * NW>(marks, p, k * SEG);
    __syncthreads();
    plain = plain && !any_mark(marks);
  }

  auto segment = [&](auto plain_tag, auto whole_tag) __attribute__((always_inline)) {
    constexpr bool PLAIN = decltype(plain_tag)::value, WHOLE = decltype(whole_tag)::value, CUTS = PACKED && !PLAIN;
    Held<T, VEC> hx[U], ha[U], hg[U], hd[U];
    {
      Walk<const T> wx(x, p.x_stride[1], n0, time, reverse), wa(ga, p.gate_a_stride[1], n0, time, reverse),
          wg(gx, p.gate_x_stride[1], n0, time, reverse), wd(dh, p.d_h_stride[1], n0, time, reverse);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (PLAIN || n0 + u < time) {
          hx[u] = ld_any<VEC, true>(wx.lane(lane_bytes));
          ha[u] = ld_any<VEC, true>(wa.lane(lane_bytes));
          hg[u] = ld_any<VEC, true>(wg.lane(lane_bytes));
          hd[u] = ld_any<VEC, true>(wd.lane(lane_bytes));
        }
        wx.next();
        wa.next();
        wg.next();
        wd.next();
      }
    }
    if (wave < VEC) {
      const float rate = p.rate[ch.base + int(ch.rel) + wave];
      sh_decay[wave * 64 + lane] = LOG2E * p.scale * fast_softplus(rate);
    }
    __syncthreads();

    unsigned starts = 0, ends = 0;
    if constexpr (CUTS) {
      starts = run_bits<U>(marks.starts, wave);
      ends = run_bits<U>(marks.ends, wave);
    }
    auto rows_of = [&](const float* t, const int* which, int u) __attribute__((always_inline)) {
      Lanes<VEC> r;
      if (t) r = load_floats<VEC>(t + int64_t(__builtin_amdgcn_readfirstlane(which[wave * U + u])) * channels + ch.base + ch.rel);
      else for (int e = 0; e < VEC; ++e) r.v[e] = 0.0f;
      return r;
    };
    // a and m of every position stay in registers until its gradients are made, its sigmoids in LDS
    Lanes<VEC> decay, ma, mb, mg, a[U], b[U], m[U];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      decay.v[e] = sh_decay[e * 64 + lane];
      ma.v[e] = 1.0f;
      mb.v[e] = mg.v[e] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (PLAIN || n0 + u < time) {
        const Lanes<VEC> vx = widen(hx[u]), va = widen(ha[u]), vg = widen(hg[u]);
        if constexpr (CUTS) {
          if (starts >> u & 1u) mb = rows_of(p.h0, marks.start, u);
        }
        Lanes<VEC> sa, sx;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const Gate g = gate_of(va.v[e], vg.v[e], decay.v[e]);
          a[u].v[e] = g.a;
          sa.v[e] = g.sa;
          sx.v[e] = g.sx;
          m[u].v[e] = __builtin_amdgcn_sqrtf(g.m2);
          b[u].v[e] = m[u].v[e] * g.sx * vx.v[e];
          mb.v[e] = fmaf(g.a, mb.v[e], b[u].v[e]);
          ma.v[e] *= g.a;
        }
        sigmoids[wave * U + u][0][lane] = sa;
        sigmoids[wave * U + u][1][lane] = sx;
      }
    }
#pragma unroll
    for (int u = U - 1; u >= 0; --u) {
      if (PLAIN || n0 + u < time) {
        const Lanes<VEC> vd = widen(hd[u]);
        if constexpr (CUTS) {
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
    if (wave >= VEC && wave < 2 * VEC) {  // forward, from the saved value
      const int e = wave - VEC, i = e * 64 + lane;
      float v = p.saved[(int64_t(batch) * args.segments + k) * channels + ch.base + int(ch.rel) + e];
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float wa = sh_a[w][i], wb = sh_b[w][i];
        sh_b[w][i] = v;
        v = CUTS && run_bits<U>(marks.starts, w) != 0 ? wb : fmaf(wa, v, wb);
      }
    }
    if (wave < VEC) {
      const int e = wave, i = e * 64 + lane;
      const int c = ch.base + int(ch.rel) + e;
      bool any = false;
      float ta = 1.0f, tg = 0.0f;
      {
#pragma unroll
        for (int w = NW - 1; w >= 0; --w) {
          const float wa = sh_a[w][i], wg = sh_g[w][i];
          if (CUTS && run_bits<U>(marks.ends, w) != 0) {
            tg = wg;
            any = true;
          } else {
            tg = fmaf(wa, tg, wg);
            ta = never_zero(ta * wa);
          }
        }
      }
      const long long per_segment = 2ll * blocks * RPB;
      uint64_t* words = args.chain.desc + 2ll * block * RPB + e * 64;
      const Chain chain{words, uint32_t(lane) * 8, per_segment, kk, args.segments, seq};
      const float first = !PACKED && p.d_state ? p.d_state[int64_t(batch) * channels + c] : 0.0f;
      auto walk = [&] {
        int from = time;
        float w = first;
        if constexpr (PACKED) {
          const int64_t j = bounds_up_to(p, (k + 1) * SEG) - 1;  // the sequence of the position after this segment
          if (j >= 0 && j < p.sequences) {
            from = scan_bound(p, j + 1);
            // (where that sequence starts right there, nothing of it enters: the segment's last position is an end)
            if (p.d_state) w = p.d_state[scan_sequence(p, j) * channels + c];
          }
        }
        const float d2 = sh_decay[i];
        for (int n = from - 1; n >= (k + 1) * SEG; --n) {
          const int64_t l = reverse ? time - 1 - n : n, o = int64_t(ch.rel) + e;
          const float an = __builtin_amdgcn_exp2f(-d2 * fast_sigmoid(float(ga[l * p.gate_a_stride[1] + o])));
          w = an * (w + float(dh[l * p.d_h_stride[1] + o]));
        }
        return w;
      };
      float v = enter_segment<RPB>(args.chain, chain, lane, first, ta, tg, any, walk);
      {
#pragma unroll
        for (int w = NW - 1; w >= 0; --w) {
          const float wa = sh_a[w][i], wg = sh_g[w][i];
          sh_g[w][i] = v;
          v = CUTS && run_bits<U>(marks.ends, w) != 0 ? wg : fmaf(wa, v, wg);
        }
      }
    }
    __syncthreads();
    Lanes<VEC> val, back, sum, neg_decay;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      neg_decay.v[e] = -LN2 * decay.v[e];
      val.v[e] = sh_b[wave][e * 64 + lane];
      back.v[e] = sh_g[wave][e * 64 + lane];
      sum.v[e] = 0.0f;
    }
    // the value before each position, in the place of what the position takes in
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (PLAIN || n0 + u < time) {
        if constexpr (CUTS) {
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
    const int64_t dense = (int64_t)batch * time * channels + ch.base;
    Walk<T> ox(static_cast<T*>(p.d_x) + dense, channels, n0 + U - 1, time, reverse),
        oa(static_cast<T*>(p.d_gate_a) + dense, channels, n0 + U - 1, time, reverse),
        og(static_cast<T*>(p.d_gate_x) + dense, channels, n0 + U - 1, time, reverse);
#pragma unroll
    for (int u = U - 1; u >= 0; --u) {
      if (PLAIN || n0 + u < time) {
        const Lanes<VEC> vx = widen(held_again(hx[u])), vd = widen(held_again(hd[u]));
        const Lanes<VEC> sa = sigmoids[wave * U + u][0][lane], sx = sigmoids[wave * U + u][1][lane];
        Lanes<VEC> rx, ra, rg;
        if constexpr (CUTS) {
          if (ends >> u & 1u) back = rows_of(p.d_state, marks.end, u);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float av = a[u].v[e], mv = m[u].v[e], sxv = sx.v[e], sav = sa.v[e];
          const float grad = vd.v[e] + back.v[e], back_on = av * grad;
          const float inv_m = __builtin_amdgcn_rcpf(fmaxf(mv, 1e-19f));  // (m is 0 only with log a, which makes the product 0)
          const float sxx = sxv * vx.v[e];
          rx.v[e] = grad * mv * sxv;
          rg.v[e] = grad * mv * fmaf(-sxx, sxv, sxx);
          // P = g log a a (h' - a sx x / m)
          const float q = back_on * (neg_decay.v[e] * sav) * fmaf(-sxx * av, inv_m, b[u].v[e]);
          ra.v[e] = fmaf(-q, sav, q);
          sum.v[e] += q;
          back.v[e] = back_on;
        }
        T* to_x = ox.lane(lane_bytes);
        T* to_a = oa.lane(lane_bytes);
        T* to_g = og.lane(lane_bytes);
        store_channels<LINES, WHOLE>(to_x, rx, ch);
        store_channels<LINES, WHOLE>(to_a, ra, ch);
        store_channels<LINES, WHOLE>(to_g, rg, ch);
        if (CUTS && p.d_h0 && (starts >> u & 1u))
          store_floats(p.d_h0 + int64_t(__builtin_amdgcn_readfirstlane(marks.start[wave * U + u])) * channels + ch.base + ch.rel, back, ch);
        if (!PACKED && u == 0 && n0 == 0 && p.d_h0) store_floats(p.d_h0 + int64_t(batch) * channels + ch.base + ch.rel, back, ch);
      }
      ox.back();
      oa.back();
      og.back();
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) sh_a[wave][e * 64 + lane] = sum.v[e];
    __syncthreads();
    if (wave < VEC) {
      const int i = wave * 64 + lane;
      float s = sh_a[0][i];
#pragma unroll
      for (int w = 1; w < NW; ++w) s += sh_a[w][i];
      if (wave >= ch.own) p.partial[(int64_t(batch) * args.segments + k) * channels + ch.base + int(ch.rel) + wave] = s;
    }
  };
  if (plain && ch.whole) segment(std::true_type{}, std::true_type{});
  else if (plain) segment(std::true_type{}, std::false_type{});
  else segment(std::false_type{}, std::false_type{});

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
