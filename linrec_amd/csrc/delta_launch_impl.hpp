// See delta_launch.hpp.
#pragma once
#include "delta_gradient.hpp"
#include "delta_launch.hpp"
#include "delta_prepare.hpp"
#include "delta_reverse.hpp"
#include "delta_scan.hpp"

namespace linrec {
namespace {

template <typename F>
int with_key_width(int width, F&& f) {
  if (width == 64) return f(std::integral_constant<int, 64>{});
  if (width == 128) return f(std::integral_constant<int, 128>{});
  return f(std::integral_constant<int, 256>{});
}

inline int64_t scan_grid(const DeltaArgs& a) { return cdiv(a.pairs, 8) * 8 * a.blocks; }

template <typename T, bool BWD>
int launch_prepare(const DeltaArgs& a, int key_width) {
  if (a.p.time == 0) return LINREC_OK;
  return with_key_width(key_width, [&](auto dk) {
    return launch_kernel(delta_prepare_kernel<T, dk(), BWD>, a.slots * a.p.heads, 1, 256, a.p.stream, a);
  });
}
template <typename T, bool STATES>
int launch_scan(const DeltaArgs& a, int key_width) {
  return with_key_width(key_width, [&](auto dk) {
    auto go = [&](auto waves) {
      return launch_kernel(delta_scan_kernel<T, dk(), waves(), STATES>, scan_grid(a), 1, ScanShared<T, dk(), waves(), STATES>::LANES, a.p.stream, a);
    };
    return delta_waves(a.columns) == 4 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 2>{});
  });
}

}  // namespace

template <typename T>
int delta_forward(const DeltaArgs& a, int key_width) {
  if (const int rc = launch_prepare<T, false>(a, key_width)) return rc;
  return launch_scan<T, false>(a, key_width);
}

template <typename T>
int delta_backward(const DeltaArgs& a, int key_width) {
  if (const int rc = launch_prepare<T, true>(a, key_width)) return rc;
  if (a.p.time > 0)
    if (const int rc = launch_scan<T, true>(a, key_width)) return rc;
  const int rc = with_key_width(key_width, [&](auto dk) {
    auto go = [&](auto waves) {
      return launch_kernel(delta_reverse_kernel<T, dk(), waves()>, scan_grid(a), 1, ReverseShared<T, dk(), waves()>::LANES, a.p.stream, a);
    };
    return delta_waves(a.columns) == 4 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 2>{});
  });
  if (rc || a.p.time == 0) return rc;
  const int64_t grid = a.slots * a.p.key_heads;
  if (key_width == 64) return launch_kernel(delta_gradient_kernel<T, 64, false>, grid, 1, GRADIENT_LANES, a.p.stream, a);
  if (key_width == 128) return launch_kernel(delta_gradient_kernel<T, 128, false>, grid, 1, GRADIENT_LANES, a.p.stream, a);
  return launch_kernel(delta_gradient_kernel<T, 128, true>, grid, 1, GRADIENT_LANES, a.p.stream, a);
}

}  // namespace linrec
