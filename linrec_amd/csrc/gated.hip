// Gated linear recurrence: a lane walks one channel of one sequence.
#include "layer_common.hpp"

namespace linrec {
namespace {

struct Gates {
  float sig_a, sig_x, log_a, a, m2;  // m2 = 1 - a^2
};
__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + __expf(-v)); }
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))); }
__device__ __forceinline__ Gates gates(float ga, float gx, float decay) {
  Gates g;
  g.sig_a = sigmoid(ga);
  g.sig_x = sigmoid(gx);
  g.log_a = -decay * g.sig_a;
  g.a = expf(g.log_a);
  g.m2 = -expm1f(2.0f * g.log_a);
  return g;
}

struct Span {
  int64_t batch, first, count;
};
__device__ Span sequence_span(const linrec_gated_t& p, int64_t n) {
  if (!p.cu_seqlens) return {n, 0, p.time};
  int64_t lo = p.cu_seqlens[n], hi = p.cu_seqlens[n + 1];
  lo = lo < 0 ? 0 : lo;
  hi = hi > p.time ? p.time : hi;
  return {0, lo, hi > lo ? hi - lo : 0};
}

template <typename T>
__global__ void gated_fwd_kernel(linrec_gated_t p) {
  const int64_t c = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t n = blockIdx.y;
  if (c >= p.channels) return;
  const Span s = sequence_span(p, n);
  const float decay = p.scale * softplus(p.rate[c]);
  float h = p.h0 ? p.h0[n * p.channels + c] : 0.0f;
  for (int64_t i = 0; i < s.count; ++i) {
    const int64_t t = s.first + (p.reverse ? s.count - 1 - i : i);
    const float x = float(static_cast<const T*>(p.x)[s.batch * p.x_stride[0] + t * p.x_stride[1] + c]);
    const float ga = float(static_cast<const T*>(p.gate_a)[s.batch * p.gate_a_stride[0] + t * p.gate_a_stride[1] + c]);
    const float gx = float(static_cast<const T*>(p.gate_x)[s.batch * p.gate_x_stride[0] + t * p.gate_x_stride[1] + c]);
    const Gates g = gates(ga, gx, decay);
    const int64_t o = (s.batch * p.time + t) * p.channels + c;
    if (p.saved) p.saved[o] = h;
    h = fmaf(g.a, h, sqrtf(g.m2) * g.sig_x * x);
    static_cast<T*>(p.h)[o] = T(h);
  }
  if (p.state) p.state[n * p.channels + c] = h;
}

template <typename T>
__global__ void gated_bwd_kernel(linrec_gated_t p) {
  const int64_t c = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (c >= p.channels) return;
  const float rate = p.rate[c], sp = softplus(rate), decay = p.scale * sp;
  float sum = 0.0f;
  for (int64_t n = 0; n < p.sequences; ++n) {
    const Span s = sequence_span(p, n);
    float carry = p.d_state ? p.d_state[n * p.channels + c] : 0.0f;
    for (int64_t i = s.count - 1; i >= 0; --i) {
      const int64_t t = s.first + (p.reverse ? s.count - 1 - i : i);
      const float x = float(static_cast<const T*>(p.x)[s.batch * p.x_stride[0] + t * p.x_stride[1] + c]);
      const float ga = float(static_cast<const T*>(p.gate_a)[s.batch * p.gate_a_stride[0] + t * p.gate_a_stride[1] + c]);
      const float gx = float(static_cast<const T*>(p.gate_x)[s.batch * p.gate_x_stride[0] + t * p.gate_x_stride[1] + c]);
      const float dh = float(static_cast<const T*>(p.d_h)[s.batch * p.d_h_stride[0] + t * p.d_h_stride[1] + c]);
      const Gates g = gates(ga, gx, decay);
      const int64_t o = (s.batch * p.time + t) * p.channels + c;
      const float m = sqrtf(g.m2);
      const float grad = dh + carry;
      const float through_m = g.m2 > 0.0f ? g.log_a / m : 0.0f;
      const float q = grad * (g.log_a * g.a * p.saved[o] - g.sig_x * x * g.a * g.a * through_m);
      static_cast<T*>(p.d_x)[o] = T(grad * m * g.sig_x);
      static_cast<T*>(p.d_gate_a)[o] = T(q * (1.0f - g.sig_a));
      static_cast<T*>(p.d_gate_x)[o] = T(grad * m * x * g.sig_x * (1.0f - g.sig_x));
      sum += q;
      carry = grad * g.a;
    }
    if (p.d_h0) p.d_h0[n * p.channels + c] = carry;
  }
  p.d_rate[c] = sp > 0.0f ? sum * (sigmoid(rate) / sp) : sum;
}

template <typename T>
__global__ void gated_step_kernel(linrec_gated_step_t p) {
  const int64_t c = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t n = blockIdx.y;
  if (c >= p.channels) return;
  const int64_t slot = p.slots ? p.slots[n] : n;
  if (slot < 0 || slot >= p.slots_total) {
    static_cast<T*>(p.h)[n * p.channels + c] = T(0.0f);
    return;
  }
  const float x = float(static_cast<const T*>(p.x)[n * p.x_stride + c]);
  const Gates g = gates(float(static_cast<const T*>(p.gate_a)[n * p.gate_a_stride + c]),
                        float(static_cast<const T*>(p.gate_x)[n * p.gate_x_stride + c]), p.scale * softplus(p.rate[c]));
  float* s = p.state + slot * p.state_stride + c;
  const float h = fmaf(g.a, *s, sqrtf(g.m2) * g.sig_x * x);
  *s = h;
  static_cast<T*>(p.h)[n * p.channels + c] = T(h);
}

int check_gated(const linrec_gated_t* p) {
  if (!p || p->batch < 0 || p->time < 0 || p->channels < 0 || p->sequences < 0) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->cu_seqlens ? p->batch != 1 : p->sequences != p->batch) return LINREC_E_INVALID;
  if (p->time > 2147483647LL - 4096 || p->channels > 2147483647LL - 4096) return LINREC_E_TOO_LARGE;
  if (p->channels > 0 && p->batch > 0 && p->time > 0 && (!p->x || !p->gate_a || !p->gate_x || !p->rate)) return LINREC_E_INVALID;
  return LINREC_OK;
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

int64_t linrec_gated_saved_floats(int64_t batch, int64_t time, int64_t channels) { return batch * time * channels; }
int64_t linrec_gated_partial_floats(int64_t, int64_t, int64_t) { return 0; }
size_t linrec_gated_workspace_bytes(int, int64_t, int64_t, int64_t, int) { return 0; }

int linrec_gated_fwd(const linrec_gated_t* p) {
  if (const int rc = check_gated(p)) return rc;
  if (p->sequences == 0 || p->channels == 0 || p->batch == 0) return LINREC_OK;
  if (p->time > 0 && !p->h) return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) {
    return launch_kernel(gated_fwd_kernel<decltype(t)>, cdiv(p->channels, 64), p->sequences, 64, p->stream, *p);
  });
}

int linrec_gated_bwd(const linrec_gated_t* p) {
  if (const int rc = check_gated(p)) return rc;
  if (p->channels == 0) return LINREC_OK;
  if (!p->d_rate || !p->rate || (p->batch > 0 && p->time > 0 && (!p->saved || !p->d_h || !p->d_x || !p->d_gate_a || !p->d_gate_x)))
    return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) {
    return launch_kernel(gated_bwd_kernel<decltype(t)>, cdiv(p->channels, 64), 1, 64, p->stream, *p);
  });
}

int linrec_gated_step(const linrec_gated_step_t* p) {
  if (!p || p->batch < 0 || p->channels < 0 || p->slots_total < 0) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->batch == 0 || p->channels == 0) return LINREC_OK;
  if (!p->x || !p->gate_a || !p->gate_x || !p->rate || !p->h || (!p->state && p->slots_total > 0)) return LINREC_E_INVALID;
  if (!p->slots && p->slots_total < p->batch) return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) {
    return launch_kernel(gated_step_kernel<decltype(t)>, cdiv(p->channels, 256), p->batch, 256, p->stream, *p);
  });
}

}  // extern "C"
