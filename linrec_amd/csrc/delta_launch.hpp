// Launches of the gated delta rule's chunk kernels for one storage type; a translation unit for each (delta_f32.hip, delta_f16.hip,
// delta_bf16.hip).
#pragma once
#include "delta_core.hpp"

namespace linrec {

template <typename T>
int delta_forward(const DeltaArgs& a, int key_width);
template <typename T>
int delta_backward(const DeltaArgs& a, int key_width);

// key_dim as the kernels have it
inline int delta_key_width(int key_dim) { return key_dim <= 64 ? 64 : key_dim <= 128 ? 128 : 256; }
// waves of a workgroup of the passes along the sequence, 16 columns each; two where four would have no columns for half of them (8 x 4096
// bf16, 16 heads of 64 x 32, forward and backward: 1095 us with two, 1210 with four; 4 x 4096, 16 heads of 128 x 32: 1067 and 1114)
inline int delta_waves(int columns) { return columns > 32 ? 4 : 2; }

}  // namespace linrec
