// Chunk kernels of the gated delta rule for f32 inputs.
#include "delta_launch_impl.hpp"

namespace linrec {
template int delta_forward<float>(const DeltaArgs&, int);
template int delta_backward<float>(const DeltaArgs&, int);
}  // namespace linrec
