// Chunk kernels of the gated delta rule for bf16 inputs.
#include "delta_launch_impl.hpp"

namespace linrec {
template int delta_forward<__bf16>(const DeltaArgs&, int);
template int delta_backward<__bf16>(const DeltaArgs&, int);
}  // namespace linrec
