// Chunk kernels of the gated delta rule for f16 inputs.
#include "delta_launch_impl.hpp"

namespace linrec {
template int delta_forward<_Float16>(const DeltaArgs&, int);
template int delta_backward<_Float16>(const DeltaArgs&, int);
}  // namespace linrec
