/*
 * linrec_layers -- C ABI of the layer operators around the scan (linrec_hip.h): the gated linear recurrence and its
 * single-token step, group norm with an activation, and the token embedding with its gradient.
 *
 * The conventions are those of linrec_hip.h: device pointers, sizes and strides in elements, a HIP stream handle passed as
 * void*; every call only enqueues work on its stream, none synchronises, allocates or frees.  0 on success, a negative
 * LINREC_E_* code for a rejected call, a positive hipError_t from a launch.  Arguments come in one block of memory, which a
 * binding may keep and reuse.  LINREC_DTYPE_* is the storage type of the activations; what is declared float* is fp32
 * whatever the storage type, and all arithmetic is fp32.  Outputs must not alias inputs unless said otherwise.
 */
#ifndef LINREC_LAYERS_H_
#define LINREC_LAYERS_H_

#include <stddef.h>
#include <stdint.h>

#include "linrec_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Gated linear recurrence over (batch, time, channels) activations:
 *
 *   log a[t] = -scale * softplus(rate) * sigmoid(gate_a[t])
 *   h[t]     = a[t] * h[t-1] + sqrt(1 - a[t]^2) * sigmoid(gate_x[t]) * x[t]
 *
 * h[-1] is h0 (zeros if NULL); `reverse` runs from the last position to the first.  Channels have unit stride; x, gate_a,
 * gate_x and d_h have a batch and a time stride each (chunks of one projection need no copy), h and the gradients are dense.
 * Packed sequences: batch is 1, cu_seqlens holds sequences + 1 ascending bounds in [0, time], the first 0 and the last
 * `time`; sequence n runs over the positions from cu_seqlens[n] up to cu_seqlens[n + 1] (a reversed one starts at the far
 * end), row n of h0 enters it and row n of `state` is what leaves it.  An empty sequence hands h0 on.  Otherwise
 * sequences = batch.
 */
typedef struct linrec_gated {
  int32_t dtype;
  int32_t reverse;
  float scale;
  int32_t reserved;
  int64_t batch, time, channels, sequences;
  const int32_t* cu_seqlens; /* NULL: not packed */
  const void* x;
  const void* gate_a;
  const void* gate_x;
  int64_t x_stride[2], gate_a_stride[2], gate_x_stride[2]; /* batch, time */
  const float* rate; /* (channels) */
  const float* h0;   /* (sequences, channels) or NULL */
  void* h;           /* forward: (batch, time, channels) */
  float* state;      /* forward: (sequences, channels), the last value of every sequence; or NULL */
  float* saved;      /* linrec_gated_saved_floats() of them: written by a forward whose gradient will be asked for (NULL
                        otherwise), read by the backward */
  const void* d_h;
  int64_t d_h_stride[2];
  const float* d_state; /* (sequences, channels) or NULL */
  void* d_x;
  void* d_gate_a;
  void* d_gate_x;
  float* d_rate;  /* (channels) */
  float* d_h0;    /* (sequences, channels) or NULL */
  float* partial; /* backward: scratch of linrec_gated_partial_floats() */
  void* workspace; /* as in linrec_hip.h (the same one may serve both): linrec_gated_workspace_bytes() */
  uint64_t workspace_bytes;
  void* stream;
} linrec_gated_t;

int64_t linrec_gated_saved_floats(int dtype, int64_t batch, int64_t time, int64_t channels);
int64_t linrec_gated_partial_floats(int dtype, int64_t batch, int64_t time, int64_t channels);
size_t linrec_gated_workspace_bytes(int dtype, int64_t batch, int64_t time, int64_t channels, int is_bwd);
int linrec_gated_fwd(const linrec_gated_t* args);
int linrec_gated_bwd(const linrec_gated_t* args);

/*
 * One position of the recurrence for every row of a batch, the states updated in place: row n of the dense
 * (batch, channels) activations uses row slots[n] of `state` (row n if slots is NULL).  A row whose slot is negative or
 * beyond the last of `slots_total` rows takes no part: its h is zero and no state is touched.  No two rows may name the
 * same slot.
 */
typedef struct linrec_gated_step {
  int32_t dtype;
  float scale;
  int64_t batch, channels, slots_total;
  int64_t x_stride, gate_a_stride, gate_x_stride; /* rows */
  int64_t state_stride;
  const void* x;
  const void* gate_a;
  const void* gate_x;
  const float* rate;
  const int32_t* slots;
  float* state;
  void* h;
  void* stream;
} linrec_gated_step_t;
int linrec_gated_step(const linrec_gated_step_t* args);

/*
 * Group norm with an activation, channels last: x is (batch, positions, channels), channels of unit stride; the channels are
 * cut into `groups` equal runs and mean and variance are taken over all positions and channels of a run.
 *
 *   z = (x - mean) / sqrt(var + eps) * weight + bias,   y = act(z)
 *
 * weight and bias (channels), both or none, are of type weight_dtype.  mean and rstd (batch, groups) are written by the
 * forward and read by the backward.
 */
#define LINREC_ACT_NONE 0
#define LINREC_ACT_RELU 1
#define LINREC_ACT_SILU 2 /* z * sigmoid(z) */
#define LINREC_ACT_GELU 3 /* z * (1 + erf(z / sqrt 2)) / 2 */
typedef struct linrec_group_norm {
  int32_t dtype, weight_dtype, act;
  float eps;
  int64_t batch, positions, channels, groups;
  const void* x;
  int64_t x_stride[2]; /* batch, position */
  const void* weight;
  const void* bias;
  void* y;     /* forward: dense */
  float* mean; /* (batch, groups) */
  float* rstd;
  const void* d_y;
  int64_t d_y_stride[2];
  void* d_x;      /* backward: dense */
  void* d_weight; /* of weight_dtype, NULL if there is no weight */
  void* d_bias;
  float* partial; /* scratch of linrec_group_norm_partial_floats() */
  void* stream;
} linrec_group_norm_t;
int64_t linrec_group_norm_partial_floats(int dtype, int64_t batch, int64_t positions, int64_t channels, int64_t groups, int is_bwd);
int linrec_group_norm_fwd(const linrec_group_norm_t* args);
int linrec_group_norm_bwd(const linrec_group_norm_t* args);

/*
 * Embedding: y[n] = scale * weight[token[n]], and its gradient d_weight[v] = scale * sum of d_y[n] over the n with
 * token[n] == v, in an order that depends on the tokens alone.  Tokens are int32 or int64 (token_bytes 4 or 8).  A token outside [0, vocab) gives
 * a row of zeros and no gradient; `padding` (negative: none) names a token that is looked up but gets no gradient.
 * weight, y, d_y and d_weight are of type dtype; d_y has a row stride, the others are dense.
 */
typedef struct linrec_embedding {
  int32_t dtype, token_bytes;
  float scale;
  int32_t reserved;
  int64_t tokens, vocab, channels, padding;
  const void* token;
  const void* weight;
  void* y;
  const void* d_y;
  int64_t d_y_stride;
  void* d_weight;
  void* scratch; /* backward: linrec_embedding_scratch_bytes(), 16-byte aligned, any contents */
  uint64_t scratch_bytes;
  void* stream;
} linrec_embedding_t;
size_t linrec_embedding_scratch_bytes(int64_t tokens, int64_t vocab, int64_t channels);
int linrec_embedding_fwd(const linrec_embedding_t* args);
int linrec_embedding_bwd(const linrec_embedding_t* args);

#ifdef __cplusplus
}
#endif
#endif /* LINREC_LAYERS_H_ */
