/*
 * linrec_delta -- C ABI of the gated delta rule, a linear recurrence whose state is a matrix, and of its single-token step.
 *
 * The conventions are those of linrec_layers.h: device pointers, sizes and strides in elements, a HIP stream handle passed as
 * void*; every call only enqueues work on its stream, none synchronises, allocates or frees.  0 on success, a negative
 * LINREC_E_* code for a rejected call, a positive hipError_t from a launch.  LINREC_DTYPE_* is the storage type of q, k, v, o
 * and their gradients; what is declared float* is fp32 whatever the storage type.  Outputs must not alias inputs unless said
 * otherwise.
 */
#ifndef LINREC_DELTA_H_
#define LINREC_DELTA_H_

#include <stddef.h>
#include <stdint.h>

#include "linrec_layers.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LINREC_DELTA_KEY_DIM_MAX 256
#define LINREC_DELTA_ROW_MAX (1 << 28) /* heads x value_dim, of linrec_delta_t */

/*
 * Gated delta rule.  Every value head has a state S of key_dim x value_dim, and at a position
 *
 *   S <- exp(log_decay) S,   S <- S + k (beta (v - S^T k))^T,   o = scale S^T q
 *
 * q and k are (batch, time, key_heads, key_dim), v and o (batch, time, heads, value_dim), log_decay and beta
 * (batch, time, heads); `heads` is a multiple of key_heads, and heads / key_heads neighbouring value heads share a key head.
 * The last dimension of q, k, v and d_o has unit stride, the others are strided as given (batch, time, head); o and the
 * gradients are dense.  h0 (sequences, heads, key_dim, value_dim) is S before the first position (zeros if NULL), `state` S
 * behind the last.  Packed sequences (cu_seqlens) are as in linrec_gated_t.
 *
 * A log_decay below -10000 counts as -10000 (whose exponential is zero).
 */
typedef struct linrec_delta {
  int32_t dtype, key_heads, heads, key_dim, value_dim;
  float scale;
  int64_t batch, time, sequences;
  const int32_t* cu_seqlens; /* NULL: not packed */
  const void* q;
  const void* k;
  const void* v;
  int64_t q_stride[3], k_stride[3], v_stride[3]; /* batch, time, head */
  const float* log_decay;
  const float* beta;
  int64_t log_decay_stride[3], beta_stride[3]; /* batch, time, head */
  const float* h0;
  void* o;      /* forward */
  float* state; /* forward, or NULL */
  const void* d_o;
  int64_t d_o_stride[3]; /* batch, time, head */
  const float* d_state; /* as `state`, or NULL */
  void* d_q;
  void* d_k;
  void* d_v;
  float* d_log_decay;
  float* d_beta;
  float* d_h0;   /* as h0, or NULL */
  void* scratch; /* linrec_delta_scratch_bytes(), 16-byte aligned, any contents */
  uint64_t scratch_bytes;
  void* stream;
} linrec_delta_t;

/* of a block whose sizes are filled in; nothing else of it is read */
size_t linrec_delta_scratch_bytes(const linrec_delta_t* args, int is_bwd);
int linrec_delta_fwd(const linrec_delta_t* args);
int linrec_delta_bwd(const linrec_delta_t* args);

/*
 * One position of the rule for every row of a batch, the states updated in place: q and k are (batch, key_heads, key_dim), v
 * and o (batch, heads, value_dim), log_decay and beta (batch, heads).  Row n uses row slots[n] of `state` (row n if slots is
 * NULL), whose rows are state_stride apart, each dense (heads, key_dim, value_dim).  A row whose slot is negative or beyond
 * the last of `slots_total` rows takes no part: its o is zero and no state is touched.  No two rows may name the same slot.
 */
typedef struct linrec_delta_step {
  int32_t dtype, key_heads, heads, key_dim, value_dim;
  float scale;
  int64_t batch, slots_total;
  const void* q;
  const void* k;
  const void* v;
  int64_t q_stride[2], k_stride[2], v_stride[2]; /* row, head */
  const float* log_decay;
  const float* beta;
  int64_t log_decay_stride[2], beta_stride[2]; /* row, head */
  const int32_t* slots;
  float* state;
  int64_t state_stride;
  void* o; /* dense */
  void* stream;
} linrec_delta_step_t;
int linrec_delta_step(const linrec_delta_step_t* args);

#ifdef __cplusplus
}
#endif
#endif /* LINREC_DELTA_H_ */
