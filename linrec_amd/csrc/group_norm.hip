// Group norm with an activation, channels last: a workgroup per (batch, group).
#include "layer_common.hpp"

namespace linrec {
namespace {

__device__ __forceinline__ float act_value(int act, float z) {
  switch (act) {
    case LINREC_ACT_RELU: return z < 0.0f ? 0.0f : z;  // (NaN stays)
    case LINREC_ACT_SILU: return z / (1.0f + expf(-z));
    case LINREC_ACT_GELU: return 0.5f * z * erfcf(-z * 0.70710678118654752f);
  }
  return z;
}
__device__ __forceinline__ float act_slope(int act, float z) {
  switch (act) {
    case LINREC_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case LINREC_ACT_SILU: {
      const float s = 1.0f / (1.0f + expf(-z));
      return s * (1.0f + z * (1.0f - s));
    }
    case LINREC_ACT_GELU: return 0.5f * erfcf(-z * 0.70710678118654752f) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
  }
  return 1.0f;
}
__device__ __forceinline__ float param(const void* p, int dtype, int64_t c, float none) {
  if (!p) return none;
  switch (dtype) {
    case LINREC_DTYPE_F16: return float(static_cast<const _Float16*>(p)[c]);
    case LINREC_DTYPE_BF16: return float(static_cast<const __bf16*>(p)[c]);
  }
  return static_cast<const float*>(p)[c];
}
__device__ __forceinline__ void set_param(void* p, int dtype, int64_t c, float v) {
  switch (dtype) {
    case LINREC_DTYPE_F16: static_cast<_Float16*>(p)[c] = _Float16(v); return;
    case LINREC_DTYPE_BF16: static_cast<__bf16*>(p)[c] = __bf16(v); return;
  }
  static_cast<float*>(p)[c] = v;
}
// Sum over the 256 lanes of a workgroup, the same in all of them.
__device__ float block_sum(float v) {
  __shared__ float sh[256];
  __syncthreads();
  sh[threadIdx.x] = v;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (int(threadIdx.x) < o) sh[threadIdx.x] += sh[threadIdx.x + o];
    __syncthreads();
  }
  return sh[0];
}

template <typename T>
__global__ void norm_fwd_kernel(linrec_group_norm_t p) {
  const int64_t n = blockIdx.x / p.groups, g = blockIdx.x % p.groups, cg = p.channels / p.groups, count = cg * p.positions;
  const T* x = static_cast<const T*>(p.x) + n * p.x_stride[0];
  float s = 0.0f;
  for (int64_t i = threadIdx.x; i < count; i += 256) s += float(x[(i / cg) * p.x_stride[1] + g * cg + i % cg]);
  const float mean = block_sum(s) / float(count);
  s = 0.0f;
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const float d = float(x[(i / cg) * p.x_stride[1] + g * cg + i % cg]) - mean;
    s += d * d;
  }
  const float rstd = rsqrtf(block_sum(s) / float(count) + p.eps);
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const int64_t c = g * cg + i % cg;
    const float z = (float(x[(i / cg) * p.x_stride[1] + c]) - mean) * rstd * param(p.weight, p.weight_dtype, c, 1.0f) +
                    param(p.bias, p.weight_dtype, c, 0.0f);
    static_cast<T*>(p.y)[(n * p.positions + i / cg) * p.channels + c] = T(act_value(p.act, z));
  }
  if (threadIdx.x == 0) {
    p.mean[n * p.groups + g] = mean;
    p.rstd[n * p.groups + g] = rstd;
  }
}

template <typename T>
__global__ void norm_bwd_kernel(linrec_group_norm_t p) {
  const int64_t n = blockIdx.x / p.groups, g = blockIdx.x % p.groups, cg = p.channels / p.groups, count = cg * p.positions;
  const T* x = static_cast<const T*>(p.x) + n * p.x_stride[0];
  const T* dy = static_cast<const T*>(p.d_y) + n * p.d_y_stride[0];
  const float mean = p.mean[n * p.groups + g], rstd = p.rstd[n * p.groups + g];
  float s1 = 0.0f, s2 = 0.0f;
  auto at = [&](int64_t i, float& xh, float& ew) {
    const int64_t c = g * cg + i % cg;
    const float w = param(p.weight, p.weight_dtype, c, 1.0f);
    xh = (float(x[(i / cg) * p.x_stride[1] + c]) - mean) * rstd;
    ew = float(dy[(i / cg) * p.d_y_stride[1] + c]) * act_slope(p.act, xh * w + param(p.bias, p.weight_dtype, c, 0.0f)) * w;
  };
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    float xh, ew;
    at(i, xh, ew);
    s1 += ew;
    s2 += ew * xh;
  }
  s1 = block_sum(s1) / float(count);
  s2 = block_sum(s2) / float(count);
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    float xh, ew;
    at(i, xh, ew);
    static_cast<T*>(p.d_x)[(n * p.positions + i / cg) * p.channels + g * cg + i % cg] = T(rstd * (ew - s1 - xh * s2));
  }
}

template <typename T>
__global__ void norm_params_kernel(linrec_group_norm_t p) {
  const int64_t c = blockIdx.x, cg = p.channels / p.groups, g = c / cg;
  const float w = param(p.weight, p.weight_dtype, c, 1.0f), b = param(p.bias, p.weight_dtype, c, 0.0f);
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t i = threadIdx.x; i < p.batch * p.positions; i += 256) {
    const int64_t n = i / p.positions, q = i % p.positions;
    const float xh = (float(static_cast<const T*>(p.x)[n * p.x_stride[0] + q * p.x_stride[1] + c]) - p.mean[n * p.groups + g]) *
                     p.rstd[n * p.groups + g];
    const float e = float(static_cast<const T*>(p.d_y)[n * p.d_y_stride[0] + q * p.d_y_stride[1] + c]) * act_slope(p.act, xh * w + b);
    s1 += e;
    s2 += e * xh;
  }
  s1 = block_sum(s1);
  s2 = block_sum(s2);
  if (threadIdx.x == 0) {
    set_param(p.d_bias, p.weight_dtype, c, s1);
    set_param(p.d_weight, p.weight_dtype, c, s2);
  }
}

int check_norm(const linrec_group_norm_t* p) {
  if (!p || p->batch < 0 || p->positions < 0 || p->channels < 0 || p->groups < 1 || p->channels % p->groups) return LINREC_E_INVALID;
  if (p->act < LINREC_ACT_NONE || p->act > LINREC_ACT_GELU || !p->weight != !p->bias) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16 || p->weight_dtype < LINREC_DTYPE_F32 || p->weight_dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->batch > 0 && p->positions > 0 && p->channels > 0 && (!p->x || !p->mean || !p->rstd)) return LINREC_E_INVALID;
  return LINREC_OK;
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

int64_t linrec_group_norm_partial_floats(int, int64_t, int64_t, int64_t, int64_t, int) { return 0; }

int linrec_group_norm_fwd(const linrec_group_norm_t* p) {
  if (const int rc = check_norm(p)) return rc;
  if (p->batch == 0 || p->positions == 0 || p->channels == 0) return LINREC_OK;
  if (!p->y) return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) { return launch_kernel(norm_fwd_kernel<decltype(t)>, p->batch * p->groups, 1, 256, p->stream, *p); });
}

int linrec_group_norm_bwd(const linrec_group_norm_t* p) {
  if (const int rc = check_norm(p)) return rc;
  if (p->channels == 0) return LINREC_OK;
  if (p->weight && (!p->d_weight || !p->d_bias)) return LINREC_E_INVALID;
  if (p->batch > 0 && p->positions > 0 && (!p->d_y || !p->d_x)) return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) {
    if (p->positions > 0 && p->channels > 0)
      if (const int rc = launch_kernel(norm_bwd_kernel<decltype(t)>, p->batch * p->groups, 1, 256, p->stream, *p)) return rc;
    return p->weight ? launch_kernel(norm_params_kernel<decltype(t)>, p->channels, 1, 256, p->stream, *p) : LINREC_OK;
  });
}

}  // extern "C"
