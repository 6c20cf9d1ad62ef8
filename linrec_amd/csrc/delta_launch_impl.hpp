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
int launch_prepare(const DeltaArgs& a) {
  if (a.p.time == 0) return LINREC_OK;
  return launch_kernel(delta_prepare_kernel<T, BWD>, a.slots * a.p.heads, 1, 256, a.p.stream, a);
}
template <typename T, bool STATES>
int launch_scan(const DeltaArgs& a, int key_width) {
  return with_key_width(key_width, [&](auto dk) {
    if (delta_waves(a.columns) == 4) return launch_kernel(delta_scan_kernel<T, dk(), 4, STATES>, scan_grid(a), 1, 256, a.p.stream, a);
    return launch_kernel(delta_scan_kernel<T, dk(), 2, STATES>, scan_grid(a), 1, 128, a.p.stream, a);
  });
}

}  // namespace

template <typename T>
int delta_forward(const DeltaArgs& a, int key_width) {
  if (const int rc = launch_prepare<T, false>(a)) return rc;
  return launch_scan<T, false>(a, key_width);
}

template <typename T>
int delta_backward(const DeltaArgs& a, int key_width) {
  if (const int rc = launch_prepare<T, true>(a)) return rc;
  if (a.p.time > 0)
    if (const int rc = launch_scan<T, true>(a, key_width)) return rc;
  const int rc = with_key_width(key_width, [&](auto dk) {
    if (delta_waves(a.columns) == 4) return launch_kernel(delta_reverse_kernel<T, dk(), 4>, scan_grid(a), 1, 256, a.p.stream, a);
    return launch_kernel(delta_reverse_kernel<T, dk(), 2>, scan_grid(a), 1, 128, a.p.stream, a);
  });
  if (rc || a.p.time == 0) return rc;
  const int64_t grid = a.slots * a.p.key_heads;
  if (key_width == 64) return launch_kernel(delta_gradient_kernel<T, 64, false>, grid, 1, 256, a.p.stream, a);
  if (key_width == 128) return launch_kernel(delta_gradient_kernel<T, 128, false>, grid, 1, 256, a.p.stream, a);
  return launch_kernel(delta_gradient_kernel<T, 128, true>, grid, 1, 256, a.p.stream, a);
}

}  // namespace linrec
