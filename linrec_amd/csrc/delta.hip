// C ABI of the gated delta rule, and its single-token step.
#include "delta_launch.hpp"

namespace linrec {
namespace {

int check_delta(const linrec_delta_t* p) {
  if (!p || p->batch < 0 || p->time < 0 || p->sequences < 0) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->key_heads < 1 || p->heads < 1 || p->heads % p->key_heads || p->key_dim < 1 || p->value_dim < 1) return LINREC_E_INVALID;
  if (p->key_dim > LINREC_DELTA_KEY_DIM_MAX) return LINREC_E_UNSUPPORTED;
  if (p->cu_seqlens ? p->batch != 1 : p->sequences != p->batch) return LINREC_E_INVALID;
  if (p->time > 2147483647LL - 4096 || p->batch > 2147483647LL || p->sequences > 2147483647LL - 64) return LINREC_E_TOO_LARGE;
  if (p->value_dim > (1 << 20) || int64_t(p->heads) * p->value_dim > LINREC_DELTA_ROW_MAX) return LINREC_E_TOO_LARGE;
  return LINREC_OK;
}

size_t aligned(size_t n) { return (n + 255) & ~size_t(255); }

// Chunks of a segment, 0 where sequences are not cut.
//
// A workgroup of a pass is taken to fill a CU (the passes that keep states or carry segments leave room for a second one up to 64 key channels, in 16 bits, and
// are counted as more rounds than they are), so `w` of them take ceil(w / 256) rounds, each as long as its chunks are many.  Cut into n segments a pass becomes
// two, the first with the columns of the unit matrix as well, and what goes from segment to segment: about half a chunk's time for
// each, and two chunks' for two launches more.  What counts is n at which a pass's rounds are about to grow, and the most that leaves four
// chunks to a segment (1 x 2048 with 8 heads of 64 x 64, forward and backward: 198 us with 4, 231 with 8, 332 not cut; with 2, which is not taken, 179).
// 1 x 8192 with 128 x 128 bf16, forward and backward, cut and not: 16 heads (8 segments) 892 and 1741 us, 32 heads (4) 1554 and 2004; 48 heads,
// where two segments take longer (2544 and 2304), are not cut.
//
// Packed sequences are taken for as many of the mean length, since their bounds are not on the host: a long one among many short ones is not cut (one of 16384
// positions with 4 heads of 128 x 128 bf16 beside 7 of 64: 191 us forward, beside 15: 928).
int segment_of(const DeltaArgs& a, int width) {
  constexpr int64_t CUS = 256, LEAST = 4;
  const linrec_delta_t& p = a.p;
  if (p.sequences == 0 || p.time == 0) return 0;
  const int64_t side = p.sequences * p.heads, one = side * a.blocks, both = side * (a.blocks + width / (16 * delta_waves(a.columns)));
  const int64_t chunks = cdiv(a.slots, p.sequences);  // of a sequence (of packed ones the mean)
  int64_t best = 2 * chunks * cdiv(one, CUS), segments = 0;  // (times in half chunks)
  auto look = [&](int64_t n) {
    if (n > chunks / LEAST) n = chunks / LEAST;
    if (n < 2) return;
    const int64_t time = 2 * cdiv(chunks, n) * (cdiv(both * n, CUS) + cdiv(one * n, CUS)) + n + 4;
    if (time < best) best = time, segments = n;
  };
  for (int64_t rounds = 1; rounds <= 4; ++rounds) {
    look(CUS * rounds / both);
    look(CUS * rounds / one);
  }
  return segments ? int(cdiv(chunks, segments)) : 0;
}

// Sizes, and scratch parts from `base` on; returns the bytes of scratch.
size_t lay_out(const linrec_delta_t& p, bool bwd, char* base, DeltaArgs* a) {
  a->p = p;
  a->shared = p.heads / p.key_heads;
  a->columns = int(cdiv(p.value_dim, 32) * 32);
  a->blocks = int(cdiv(a->columns, 16 * delta_waves(a->columns)));
  a->slots = p.cu_seqlens ? p.time / DELTA_CHUNK + p.sequences : p.batch * cdiv(p.time, DELTA_CHUNK);
  const int width = delta_key_width(p.key_dim);
  a->segment = segment_of(*a, width);
  a->parts = !a->segment ? p.sequences : p.cu_seqlens ? a->slots / a->segment + p.sequences : p.batch * cdiv(cdiv(p.time, DELTA_CHUNK), a->segment);
  a->pairs = a->parts * p.heads;
  const size_t blocks = size_t(a->slots) * size_t(p.heads);
  size_t at = 0;
  auto part = [&](size_t bytes_of_block) {
    char* to = base + at;
    at += aligned(blocks * bytes_of_block);
    return to;
  };
  a->rows = int64_t(a->columns) * 64;
  a->state = int64_t(a->columns) * width;
  auto floats = [&](size_t of_block) { return reinterpret_cast<float*>(part(of_block * 4)); };
  a->m = floats(4096);
  a->c = floats(4096);
  a->gates = floats(192);
  if (bwd) {
    a->sums = reinterpret_cast<double*>(part(64 * 8));
    a->m_t = floats(4096);
    a->s = floats(a->state);
    a->d_s = floats(a->state);
    a->n = floats(a->rows);
    a->d_b = floats(a->rows);
    a->dots = floats(192);
  }
  if (a->segment) {
    a->carry = reinterpret_cast<float*>(base + at);
    at += aligned(size_t(a->pairs) * size_t(a->columns + width) * size_t(width) * 4);
    a->start = reinterpret_cast<float*>(base + at);
    at += aligned(size_t(a->pairs) * size_t(a->columns) * size_t(width) * 4);
  }
  return at;
}

int check_scratch(const linrec_delta_t* p, size_t need) {
  if (need && (!p->scratch || (reinterpret_cast<uintptr_t>(p->scratch) & 15u) || p->scratch_bytes < need)) return LINREC_E_WORKSPACE;
  return LINREC_OK;
}

// One position.  A workgroup has 64 columns of a head's state, a lane four of them in every 16th row, all in registers: the state
// is read once and written once, which is all the time it takes.  S^T k and S^T q are summed together, o follows from them as
// e^g S^T q + (q.k) u.
constexpr int STEP_ROWS = 16, STEP_COLUMNS = 64;

template <typename T, int ITER>
__global__ __launch_bounds__(256) void delta_step_kernel(linrec_delta_step_t p, int blocks) {
  __shared__ float sh_k[ITER * STEP_ROWS], sh_q[ITER * STEP_ROWS];
  __shared__ float sh_sum[4][9][16];
  const int64_t item = blockIdx.x / unsigned(blocks);
  const int cb = int(blockIdx.x - item * unsigned(blocks));
  const int64_t n = item / p.heads;
  const int head = int(item - n * p.heads), key_head = head / (p.heads / p.key_heads);
  const int wave = threadIdx.x >> 6, cl = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int col = cb * STEP_COLUMNS + 4 * cl;
  const int own = p.value_dim - col < 4 ? p.value_dim - col : 4;  // columns of this lane, none of some
  T* o = static_cast<T*>(p.o) + item * int64_t(p.value_dim) + col;
  const int64_t slot = p.slots ? p.slots[n] : n;
  if (slot < 0 || slot >= p.slots_total) {
    if (group == 0)
      for (int e = 0; e < own; ++e) o[e] = T(0.0f);
    return;
  }
  float* state = p.state + slot * p.state_stride + head * int64_t(p.key_dim) * p.value_dim + col;
  v4f s[ITER];
  typedef float any4 __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int row = i * STEP_ROWS + group;
    s[i] = v4f{0, 0, 0, 0};
    if (row < p.key_dim) {
      const float* from = state + int64_t(row) * p.value_dim;
      if (own == 4) s[i] = *reinterpret_cast<const any4*>(from);
      else
        for (int e = 0; e < own; ++e) s[i][e] = from[e];
    }
  }
  const T* k = static_cast<const T*>(p.k) + n * p.k_stride[0] + key_head * p.k_stride[1];
  const T* q = static_cast<const T*>(p.q) + n * p.q_stride[0] + key_head * p.q_stride[1];
  for (int d = threadIdx.x; d < ITER * STEP_ROWS; d += 256) {
    sh_k[d] = d < p.key_dim ? float(k[d]) : 0.0f;
    sh_q[d] = d < p.key_dim ? float(q[d]) : 0.0f;
  }
  float g = p.log_decay[n * p.log_decay_stride[0] + head * p.log_decay_stride[1]];
  const float beta = p.beta[n * p.beta_stride[0] + head * p.beta_stride[1]];
  const T* v = static_cast<const T*>(p.v) + n * p.v_stride[0] + head * p.v_stride[1] + col;
  float vv[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) vv[e] = e < own ? float(v[e]) : 0.0f;
  if (g < DELTA_LEAST_LOG) g = DELTA_LEAST_LOG;
  const float keep = expf(g);
  __syncthreads();
  float sums[9];
#pragma unroll
  for (int e = 0; e < 9; ++e) sums[e] = 0.0f;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const float kd = sh_k[i * STEP_ROWS + group], qd = sh_q[i * STEP_ROWS + group];
    s[i] *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sums[e] = fmaf(kd, s[i][e], sums[e]);
      sums[4 + e] = fmaf(qd, s[i][e], sums[4 + e]);
    }
    sums[8] = fmaf(qd, kd, sums[8]);
  }
#pragma unroll
  for (int e = 0; e < 9; ++e) {
    sums[e] += __shfl_xor(sums[e], 16);
    sums[e] += __shfl_xor(sums[e], 32);
    if ((threadIdx.x & 63) < 16) sh_sum[wave][e][cl] = sums[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 9; ++e) sums[e] = (sh_sum[0][e][cl] + sh_sum[1][e][cl]) + (sh_sum[2][e][cl] + sh_sum[3][e][cl]);
  v4f u;
#pragma unroll
  for (int e = 0; e < 4; ++e) u[e] = beta * (vv[e] - sums[e]);
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int row = i * STEP_ROWS + group;
    const float kd = sh_k[row];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = fmaf(kd, u[e], s[i][e]);
    if (row < p.key_dim) {
      float* to = state + int64_t(row) * p.value_dim;
      if (own == 4) *reinterpret_cast<any4*>(to) = s[i];
      else
        for (int e = 0; e < own; ++e) to[e] = s[i][e];
    }
  }
  if (group == 0)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < own) o[e] = T(p.scale * fmaf(sums[8], u[e], sums[4 + e]));
}

}  // namespace
}  // namespace linrec

using namespace linrec;

extern "C" {

size_t linrec_delta_scratch_bytes(const linrec_delta_t* p, int is_bwd) {
  if (check_delta(p)) return 0;
  DeltaArgs a{};
  return lay_out(*p, is_bwd != 0, nullptr, &a);
}

int linrec_delta_fwd(const linrec_delta_t* p) {
  if (const int rc = check_delta(p)) return rc;
  if (p->sequences == 0) return LINREC_OK;
  if (p->time > 0 && (!p->q || !p->k || !p->v || !p->log_decay || !p->beta || !p->o)) return LINREC_E_INVALID;
  DeltaArgs a{};
  if (const int rc = check_scratch(p, lay_out(*p, false, static_cast<char*>(p->scratch), &a))) return rc;
  const int width = delta_key_width(p->key_dim);
  return with_dtype(p->dtype, [&](auto t) { return delta_forward<decltype(t)>(a, width); });
}

int linrec_delta_bwd(const linrec_delta_t* p) {
  if (const int rc = check_delta(p)) return rc;
  if (p->sequences == 0) return LINREC_OK;
  if (p->time > 0 && (!p->q || !p->k || !p->v || !p->log_decay || !p->beta || !p->d_o || !p->d_q || !p->d_k || !p->d_v || !p->d_log_decay || !p->d_beta))
    return LINREC_E_INVALID;
  DeltaArgs a{};
  if (const int rc = check_scratch(p, lay_out(*p, true, static_cast<char*>(p->scratch), &a))) return rc;
  const int width = delta_key_width(p->key_dim);
  return with_dtype(p->dtype, [&](auto t) { return delta_backward<decltype(t)>(a, width); });
}

int linrec_delta_step(const linrec_delta_step_t* p) {
  if (!p || p->batch < 0 || p->slots_total < 0) return LINREC_E_INVALID;
  if (p->dtype < LINREC_DTYPE_F32 || p->dtype > LINREC_DTYPE_BF16) return LINREC_E_UNSUPPORTED;
  if (p->key_heads < 1 || p->heads < 1 || p->heads % p->key_heads || p->key_dim < 1 || p->value_dim < 1) return LINREC_E_INVALID;
  if (p->key_dim > LINREC_DELTA_KEY_DIM_MAX) return LINREC_E_UNSUPPORTED;
  if (p->value_dim > (1 << 20)) return LINREC_E_TOO_LARGE;
  if (p->batch == 0) return LINREC_OK;
  if (!p->q || !p->k || !p->v || !p->log_decay || !p->beta || !p->o || (!p->state && p->slots_total > 0)) return LINREC_E_INVALID;
  if (!p->slots && p->slots_total < p->batch) return LINREC_E_INVALID;
  const int64_t blocks = cdiv(p->value_dim, STEP_COLUMNS);
  return with_dtype(p->dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto kernel) { return launch_kernel(kernel, p->batch * p->heads * blocks, 1, 256, p->stream, *p, int(blocks)); };
    return p->key_dim <= 64 ? launch(delta_step_kernel<T, 4>) : p->key_dim <= 128 ? launch(delta_step_kernel<T, 8>) : launch(delta_step_kernel<T, 16>);
  });
}

}  // extern "C"
