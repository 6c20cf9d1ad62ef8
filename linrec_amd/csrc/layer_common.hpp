// What the layer operators (gated.hip, group_norm.hip, embedding.hip) share: storage types, and the launch helper.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/linrec_layers.h"
#include "memio.hpp"

namespace linrec {

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Calls f with a value of the storage type's C++ type.
template <typename F>
int with_dtype(int dtype, F&& f) {
  switch (dtype) {
    case LINREC_DTYPE_F32: return f(float{});
    case LINREC_DTYPE_F16: return f(_Float16{});
    case LINREC_DTYPE_BF16: return f(__bf16{});
  }
  return LINREC_E_UNSUPPORTED;
}

// Launches `kernel`; grids beyond what the runtime takes are refused.
template <typename... P, typename... A>
int launch_kernel(void (*kernel)(P...), int64_t gx, int64_t gy, int block, void* stream, A&&... args) {
  if (gx <= 0 || gy <= 0) return LINREC_OK;
  if (gx > 2147483647LL || gy > 65535) return LINREC_E_TOO_LARGE;
  hipLaunchKernelGGL(kernel, dim3(unsigned(gx), unsigned(gy)), dim3(unsigned(block)), 0, static_cast<hipStream_t>(stream),
                     static_cast<P>(args)...);
  return int(hipGetLastError());
}

}  // namespace linrec
