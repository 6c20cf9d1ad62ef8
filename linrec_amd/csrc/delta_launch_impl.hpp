// See delta_launch.hpp.
#pragma once
#include "delta_gradient.hpp"
#include "delta_launch.hpp"
#include "delta_prepare.hpp"
#include "delta_reverse.hpp"
#include "delta_scan.hpp"
#include "delta_segments.hpp"

namespace linrec {
namespace {

template <typename F>
int with_key_width(int width, F&& f) {
  if (width == 64) return f(std::integral_constant<int, 64>{});
  if (width == 128) return f(std::integral_constant<int, 128>{});
  return f(std::integral_constant<int, 256>{});
}

inline int64_t scan_grid(const DeltaArgs& a, int blocks) { return cdiv(a.pairs, 8) * 8 * blocks; }

template <typename T, bool BWD>
int launch_prepare(const DeltaArgs& a, int key_width) {
  if (a.p.time == 0) return LINREC_OK;
  return with_key_width(key_width, [&](auto dk) {
    return launch_kernel(delta_prepare_kernel<T, dk(), BWD>, a.slots * a.p.heads, 1, 256, a.p.stream, a);
  });
}
template <typename T, ScanMode MODE>
int launch_scan(const DeltaArgs& a, int key_width) {
  return with_key_width(key_width, [&](auto dk) {
    auto go = [&](auto waves) {
      const int blocks = MODE == SCAN_CARRY ? a.blocks + dk() / (16 * waves()) : a.blocks;
      return launch_kernel(delta_scan_kernel<T, dk(), waves(), MODE>, scan_grid(a, blocks), 1, ScanShared<T, dk(), waves(), MODE>::LANES, a.p.stream, a);
    };
    return delta_waves(a.columns) == 4 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 2>{});
  });
}
template <typename T, bool CARRY>
int launch_reverse(const DeltaArgs& a, int key_width) {
  return with_key_width(key_width, [&](auto dk) {
    auto go = [&](auto waves) {
      return launch_kernel(delta_reverse_kernel<T, dk(), waves(), CARRY>, scan_grid(a, a.blocks), 1, ReverseShared<T, dk(), waves()>::LANES, a.p.stream, a);
    };
    return delta_waves(a.columns) == 4 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 2>{});
  });
}
template <bool REVERSE>
int launch_segments(const DeltaArgs& a, int key_width) {
  return with_key_width(key_width, [&](auto dk) {
    return launch_kernel(delta_segments_kernel<dk(), REVERSE>, a.p.sequences * a.p.heads * (a.columns / 16), 1, 256, a.p.stream, a);
  });
}
// The states that enter the segments.
template <typename T>
int launch_entries(const DeltaArgs& a, int key_width) {
  if (!a.segment) return LINREC_OK;
  if (const int rc = launch_scan<T, SCAN_CARRY>(a, key_width)) return rc;
  return launch_segments<false>(a, key_width);
}

}  // namespace

template <typename T>
int delta_forward(const DeltaArgs& a, int key_width) {
  if (const int rc = launch_prepare<T, false>(a, key_width)) return rc;
  if (const int rc = launch_entries<T>(a, key_width)) return rc;
  return launch_scan<T, SCAN_OUT>(a, key_width);
}

template <typename T>
int delta_backward(const DeltaArgs& a, int key_width) {
  if (const int rc = launch_prepare<T, true>(a, key_width)) return rc;
  if (const int rc = launch_entries<T>(a, key_width)) return rc;
  if (a.p.time > 0)
    if (const int rc = launch_scan<T, SCAN_STATES>(a, key_width)) return rc;
  if (a.segment) {
    if (const int rc = launch_reverse<T, true>(a, key_width)) return rc;
    if (const int rc = launch_segments<true>(a, key_width)) return rc;
  }
  const int rc = launch_reverse<T, false>(a, key_width);
  if (rc || a.p.time == 0) return rc;
  const int64_t grid = a.slots * a.p.key_heads;
  if (key_width == 64) return launch_kernel(delta_gradient_kernel<T, 64, false>, grid, 1, GRADIENT_LANES, a.p.stream, a);
  if (key_width == 128) return launch_kernel(delta_gradient_kernel<T, 128, false>, grid, 1, GRADIENT_LANES, a.p.stream, a);
  return launch_kernel(delta_gradient_kernel<T, 128, true>, grid, 1, GRADIENT_LANES, a.p.stream, a);
}

}  // namespace linrec
