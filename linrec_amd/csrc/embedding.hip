// Token embedding and its gradient: a workgroup per row looked up, and per row of the table.
#include "layer_common.hpp"

namespace linrec {
namespace {

__device__ __forceinline__ int64_t token_at(const linrec_embedding_t& p, int64_t n) {
  return p.token_bytes == 8 ? static_cast<const int64_t*>(p.token)[n] : int64_t(static_cast<const int32_t*>(p.token)[n]);
}

template <typename T>
__global__ void embedding_fwd_kernel(linrec_embedding_t p) {
  const int64_t n = blockIdx.x, v = token_at(p, n);
  const bool there = v >= 0 && v < p.vocab;
  for (int64_t c = threadIdx.x; c < p.channels; c += 256)
    static_cast<T*>(p.y)[n * p.channels + c] = there ? T(p.scale * float(static_cast<const T*>(p.weight)[v * p.channels + c])) : T(0.0f);
}

template <typename T>
__global__ void embedding_bwd_kernel(linrec_embedding_t p) {
  const int64_t v = blockIdx.x;
  for (int64_t c = threadIdx.x; c < p.channels; c += 256) {
    float s = 0.0f;
    if (v != p.padding)
      for (int64_t n = 0; n < p.tokens; ++n)
        if (token_at(p, n) == v) s += float(static_cast<const T*>(p.d_y)[n * p.d_y_stride + c]);
    static_cast<T*>(p.d_weight)[v * p.channels + c] = T(s * p.scale);
  }
}

int check_embedding(const linrec_embedding_t* p) {
  if (!p || p->tokens < 0 || p->vocab < 0 || p->channels < 0 || (p->token_bytes != 4 && p->token_bytes != 8)) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->tokens > 2147483647LL - 4096 || p->vocab > 2147483647LL - 4096) return LINREC_E_TOO_LARGE;
  if (p->tokens > 0 && p->channels > 0 && !p->token) return LINREC_E_INVALID;
  return LINREC_OK;
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

size_t linrec_embedding_scratch_bytes(int64_t, int64_t, int64_t) { return 0; }

int linrec_embedding_fwd(const linrec_embedding_t* p) {
  if (const int rc = check_embedding(p)) return rc;
  if (p->tokens == 0 || p->channels == 0) return LINREC_OK;
  if (!p->y || (p->vocab > 0 && !p->weight)) return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) { return launch_kernel(embedding_fwd_kernel<decltype(t)>, p->tokens, 1, 256, p->stream, *p); });
}

int linrec_embedding_bwd(const linrec_embedding_t* p) {
  if (const int rc = check_embedding(p)) return rc;
  if (p->vocab == 0 || p->channels == 0) return LINREC_OK;
  if (!p->d_weight || (p->tokens > 0 && !p->d_y)) return LINREC_E_INVALID;
  return with_dtype(p->dtype, [&](auto t) { return launch_kernel(embedding_bwd_kernel<decltype(t)>, p->vocab, 1, 256, p->stream, *p); });
}

}  // extern "C"
