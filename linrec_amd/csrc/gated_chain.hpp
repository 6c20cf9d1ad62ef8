// The chain of segments of the gated linear recurrence (gated_kernel.hpp): how a segment gets the value that enters it.
//
// What enters a segment is a chain of multiply-adds over the maps of the segments before, and every link costs a store and a load
// through memory, 4 to 5 us with the wait between two looks, however many lanes do it side by side.  So the chain goes over blocks
// of GROUP groups of GROUP segments: a segment publishes its map; the last one of a group composes the group's maps and publishes
// that; the last one of a block those of the block's groups; and what enters a segment is what enters its block, which the chain of
// blocks says, taken through the maps of the groups before it in the block and of the segments before it in the group.  LOOK blocks
// are looked at at a time, so the value advances by LOOK * GROUP * GROUP segments a link.  Which of them had published what does not
// matter to the result: the value that leaves a block is the same multiply-add whoever makes it.
//
// Steps that led here, 1 x 100001 x 250 bf16, forward and backward: groups of 8 without blocks over them 119 and 226 us, with blocks 100 and 192; groups
// of 4 / 5 / 6 with blocks 103, 197 / 90, 167 / 96, 187.  1 x 131072 x 64, groups of 4 / 5 / 6 / 8: 66, 125 / 50, 93 / 53, 100 / 59,
// 117 (a link of 4 advances by 64 segments, one of 5 by 100; larger groups take registers that the data needs).  LOOK of 6 instead
// of 4: 8 x 4096 x 2048 130 and 230 us instead of 128 and 221, 50 and 98 here.  The groups before by other waves, while the first
// look at the segments before: no faster here, 240 us instead of 223 for 8 x 4096 x 2048 backward (registers).
//
// Words of a place (a segment's, a group's, a block's): first the factors of the block's channels, then the addends, RPB each, with the
// launch's number; an addend marked `done` leaves the place whatever enters it (a sequence starts inside, or what entered is in it).
// The words of a segment or a group are written once a launch: maps_before takes a place as constant for all lanes of a wave or none,
// and a wave that looks while another one writes sees some lanes' words before and some after.  Those of a block may turn from a
// map to `done`; what leaves blocks is taken lane by lane.
#pragma once
#include <stdint.h>

#include <type_traits>

#include "collook_kernel.hpp"  // descriptors, TileArgs

namespace linrec {

// A product of coefficients that has become too small to be told from zero still passes an infinity on, as the recurrence
// does (the coefficients are never negative).
__device__ __forceinline__ float never_zero(float a) { return a == 0.0f ? __builtin_bit_cast(float, 1u) : a; }

template <typename P>
__device__ __forceinline__ P* plus_bytes(P* p, uint32_t bytes) {
  using C = std::conditional_t<std::is_const_v<P>, const char*, char*>;
  return reinterpret_cast<P*>(reinterpret_cast<C>(p) + bytes);
}

constexpr int LOOK = 4;   // blocks looked at at a time
constexpr int SLEEP = 16;  // between two looks, 64 cycles each (32: 1 x 32768 x 2048 bf16 133 and 234 us instead of 132 and 231; 64: 136 and 244)
constexpr int GROUP = 5;  // segments of a group, groups of a block
// Places of a chain of `segments`: theirs, their groups', their blocks'.
constexpr int64_t chain_places(int64_t segments) { return segments + segments / GROUP + segments / (GROUP * GROUP); }
struct Chain {
  uint64_t* segment_words;  // of segment 0, the wave's (the same for all lanes, as all places are here)
  uint32_t lane_bytes;      // the lane's, from there
  long long per_place;      // from one place's words to the next one's
  int k, segments;
  uint32_t seq;
  __device__ __forceinline__ uint32_t map() const { return (seq << 2) | STATUS_AGGREGATE; }
  __device__ __forceinline__ uint32_t done() const { return (seq << 2) | STATUS_INCLUSIVE; }
};
struct Words {
  uint64_t a, b;
};
template <typename P>
__device__ __forceinline__ P* scalar(P* p) {  // (the same for all lanes, which the compiler need not know)
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<P*>(uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(v)))) |
                              (uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(v >> 32)))) << 32));
}
template <int RPB>
__device__ __forceinline__ Words load_words(const Chain& c, const uint64_t* place) {
  const uint64_t* d = plus_bytes(scalar(place), c.lane_bytes);
  return {ld_desc(d), ld_desc(d + RPB)};
}
template <int RPB>
__device__ __forceinline__ void publish(const Chain& c, uint64_t* place, float a, float b, bool constant) {
  uint64_t* d = plus_bytes(scalar(place), c.lane_bytes);
  if (!constant) st_desc(d, pack_desc(c.map(), a));
  st_desc(d + RPB, pack_desc(constant ? c.done() : c.map(), b));
}
__device__ __forceinline__ float word_value(uint64_t w) { return __builtin_bit_cast(float, uint32_t(w)); }
__device__ __forceinline__ bool is_done(const Chain& c, const Words& w) { return uint32_t(w.b >> 32) == c.done(); }
__device__ __forceinline__ bool is_there(const Chain& c, const Words& w) {
  return is_done(c, w) || (uint32_t(w.b >> 32) == c.map() && uint32_t(w.a >> 32) == c.map());
}
__device__ __forceinline__ float through(const Chain& c, const Words& w, float v) {
  return is_done(c, w) ? word_value(w.b) : fmaf(word_value(w.a), v, word_value(w.b));
}

// The map of the `count` < GROUP places before `place`; a constant one needs nothing of what enters the farthest.
struct Before {
  float a = 1.0f, b = 0.0f;
  bool constant = false, there = true;
};
template <int RPB>
__device__ __forceinline__ Before maps_before(const TileArgs& args, const Chain& c, const uint64_t* place, int count) {
  Before m;
  m.there = count == 0;
  for (int polls = 0; !m.there && polls < args.spin_limit; ++polls) {
    if (polls > 0) __builtin_amdgcn_s_sleep(SLEEP);
    Words w[GROUP - 1];  // the farthest first
#pragma unroll
    for (int q = 0; q < GROUP - 1; ++q)
      if (q < count) w[q] = load_words<RPB>(c, place - (count - q) * c.per_place);
    m.there = true;
#pragma unroll
    for (int q = 0; q < GROUP - 1; ++q)
      if (q < count && __ballot(!is_there(c, w[q])) != 0) m.there = false;
    if (m.there) {
#pragma unroll
      for (int q = 0; q < GROUP - 1; ++q)
        if (q < count) {
          const bool cuts = __ballot(!is_done(c, w[q])) == 0;
          m.b = through(c, w[q], m.b);
          m.a = cuts ? 1.0f : never_zero(m.a * word_value(w[q].a));
          m.constant = m.constant || cuts;
        }
    }
  }
  return m;
}

// One wave, a channel to a lane: publishes the segment's map (ta, tb; cut: a sequence starts inside) and returns what enters it.
// `walk` computes that from the channel's own data.
template <int RPB, typename W>
__device__ __forceinline__ float enter_segment(const TileArgs& args, const Chain& c, int lane, float first, float ta, float tb, bool cut, W&& walk) {
  const int in_group = c.k % GROUP, g = c.k / GROUP, in_block = g % GROUP, s = g / GROUP;
  const bool more = c.k + 1 < c.segments, closes = more && in_group == GROUP - 1, closes_block = closes && in_block == GROUP - 1;
  uint64_t* mine = c.segment_words + c.k * c.per_place;
  uint64_t* of_group = c.segment_words + (c.segments + g) * c.per_place;
  uint64_t* of_block = c.segment_words + (c.segments + c.segments / GROUP + s) * c.per_place;
  if (more && !closes) publish<RPB>(c, mine, ta, tb, cut);
  const Before seg = maps_before<RPB>(args, c, mine, in_group);
  // the maps of the whole group and block, by their last segments
  float whole_a = never_zero(seg.a * ta), whole_b = cut ? tb : fmaf(ta, seg.b, tb);
  bool whole_constant = seg.constant || cut;
  if (seg.there && closes && !closes_block) publish<RPB>(c, of_group, whole_a, whole_b, whole_constant);
  Before grp;
  if (seg.there && !seg.constant) grp = maps_before<RPB>(args, c, of_group, in_block);
  if (!whole_constant) {
    whole_b = fmaf(whole_a, grp.b, whole_b);
    whole_a = never_zero(whole_a * grp.a);
    whole_constant = grp.constant;
  }
  // (the first block never shows a map: who looks beyond it sees it again, and must not take it twice)
  bool known = seg.there && grp.there;
  if (known && closes_block && (s > 0 || whole_constant)) publish<RPB>(c, of_block, whole_a, whole_b, whole_constant);
  float v = first;  // what enters the block
  if (known && s > 0 && !seg.constant && !grp.constant) {
    known = false;
    for (int polls = 0; !known && polls < args.spin_limit; ++polls) {
      if (polls > 0) __builtin_amdgcn_s_sleep(SLEEP);
      Words x[LOOK];
#pragma unroll
      for (int q = 0; q < LOOK; ++q) x[q] = load_words<RPB>(c, of_block - (q < s ? q + 1 : s) * c.per_place);  // (beyond block 0: not used)
      int from = -1;
      bool blocked = false;
#pragma unroll
      for (int q = 0; q < LOOK; ++q) {
        if (from < 0 && !blocked) {
          if (__ballot(!is_done(c, x[q])) == 0) from = q;
          else blocked = __ballot(!is_there(c, x[q])) != 0;
        }
      }
      if (from >= 0) {
#pragma unroll
        for (int q = LOOK - 1; q >= 0; --q) {
          if (q == from) v = word_value(x[q].b);
          else if (q < from) v = through(c, x[q], v);
        }
        known = true;
      }
    }
  }
  if (known) {
    if (closes_block && !whole_constant) st_desc(plus_bytes(scalar(of_block + RPB), c.lane_bytes), pack_desc(c.done(), fmaf(whole_a, v, whole_b)));
    v = grp.constant ? grp.b : in_block == 0 ? v : fmaf(grp.a, v, grp.b);
    v = seg.constant ? seg.b : in_group == 0 ? v : fmaf(seg.a, v, seg.b);
  }
  if (__builtin_expect(!known, 0)) {
    if (lane == 0) __hip_atomic_fetch_add(&args.ws->gave_up, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    v = walk();
    // (whoever looks for what leaves the block, or a group whose map is not there, waits for it: it leaves through this segment)
    if (closes_block || (closes && !seg.there)) st_desc(plus_bytes(scalar((closes_block ? of_block : of_group) + RPB), c.lane_bytes), pack_desc(c.done(), cut ? tb : fmaf(ta, v, tb)));
  }
  return v;
}

}  // namespace linrec
