/*
 * purin_ops.h -- C ABI of the training-step operators around the projection layer.
 *
 * A model that is trained through the projection layer of purin_cp.h looks token
 * rows up in a table, sends tokens to experts by projected gates, takes a loss
 * over a vocabulary and clips its gradients.  These entry points are those four
 * operators and their gradients; none has a counterpart in PURIN.
 *
 * Conventions.  As in purin_cp.h: array arguments are DEVICE pointers on
 * `device`, row-major; strides count elements between rows, whose own elements
 * are adjacent; all work is enqueued on the caller's stream; nothing allocates,
 * synchronises or copies to the host; the caller owns every buffer and the
 * workspace whose size the matching *_workspace_size call reports (256-byte
 * aligned).  Every function returns a PurinStatus and leaves a message for
 * purin_cp_last_error().  Results do not depend on scheduling: no floating-point
 * atomics are used, so the same inputs give the same bits (of a norm: at the same
 * addresses modulo 16, by which its sums are ordered).
 */
#ifndef PURIN_OPS_H
#define PURIN_OPS_H

#include "purin_cp.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types.  The first two have PurinDtype's values. */
typedef enum PurinOpsDtype {
  PURIN_OPS_FLOAT64 = 0,
  PURIN_OPS_FLOAT32 = 1,
  PURIN_OPS_BFLOAT16 = 2,
  PURIN_OPS_FLOAT16 = 3
} PurinOpsDtype;

/* ---- embedding -----------------------------------------------------------------
 * out[i] = scale * table[ids[i]].  An id outside [0, vocab), or equal to `padding`,
 * gives a zero row and no gradient.
 * grad_table[v] = scale * sum of grad_out[i] over the i with ids[i] = v, in the order
 * of i, summed in 32 bits (64 for double); every row of grad_table is written. */
typedef struct PurinEmbeddingArgs {
  int32_t device;
  int32_t dtype;      /* PurinOpsDtype of table, out, grad_out, grad_table     */
  int32_t ids_64bit;  /* 1: ids are int64, 0: int32                            */
  int64_t tokens;
  int64_t vocab;
  int64_t dim;
  double scale;
  int64_t padding;    /* an id without a row; negative: none                   */
  const void* ids;    /* (tokens)                                              */
  const void* table;  /* (vocab, dim), forward                                 */
  int64_t table_stride;
  void* out;          /* (tokens, dim) contiguous, forward                     */
  const void* grad_out; /* (tokens, dim), backward                             */
  int64_t grad_out_stride;
  void* grad_table;   /* (vocab, dim) contiguous, backward                     */
} PurinEmbeddingArgs;

int32_t purin_embedding_forward(const PurinEmbeddingArgs* args, void* stream);
int32_t purin_embedding_backward_workspace_size(const PurinEmbeddingArgs* args, size_t* bytes);
int32_t purin_embedding_backward(const PurinEmbeddingArgs* args, void* workspace,
                                 size_t workspace_bytes, void* stream);

/* ---- tokens to experts and back ------------------------------------------------
 * Slot j = t * slots + k of token t names expert experts[j]; a value outside
 * [0, num_experts) drops the slot.  purin_route sorts the slots by expert, stably,
 * the dropped ones last: offsets[e]..offsets[e + 1] are expert e's sorted rows,
 * position[j] the sorted row of slot j, source its inverse. */
typedef struct PurinRouteArgs {
  int32_t device;
  int32_t experts_64bit; /* 1: int64, 0: int32                                 */
  int64_t tokens;
  int64_t slots;
  int64_t num_experts;
  const void* experts;   /* (tokens, slots)                                    */
  int32_t* offsets;      /* (num_experts + 1)                                  */
  int32_t* position;     /* (tokens, slots)                                    */
  int32_t* source;       /* (tokens * slots)                                   */
} PurinRouteArgs;

int32_t purin_route_workspace_size(const PurinRouteArgs* args, size_t* bytes);
int32_t purin_route(const PurinRouteArgs* args, void* workspace, size_t workspace_bytes,
                    void* stream);

/* Rows moved by a routing.  Token rows are (tokens, dim), sorted rows
 * (tokens * slots, dim); a sorted row r is dropped if r >= offsets[num_experts].  A
 * position outside [0, tokens * slots) is neither read nor written.
 *   spread: sorted[position[t,k]] = token_rows[t], dropped rows zero
 *   gather: token_out[t] = sum over kept k of weights[t,k] * sorted_rows[position[t,k]]
 *           (weights null: 1), summed in 32 bits (64 for double), k ascending
 *   combine_backward: grad_sorted[position[t,k]] = weights[t,k] * token_rows[t], dropped
 *           rows zero; grad_weights[t,k] = <token_rows[t], sorted_rows[position[t,k]]>,
 *           0 for dropped slots */
typedef struct PurinRouteRowsArgs {
  int32_t device;
  int32_t dtype;          /* PurinOpsDtype of the rows                          */
  int32_t weights_dtype;  /* PURIN_OPS_FLOAT64 or PURIN_OPS_FLOAT32             */
  int64_t tokens;
  int64_t slots;
  int64_t num_experts;
  int64_t dim;
  const int32_t* offsets;
  const int32_t* position;
  const void* token_rows;  /* spread, combine_backward                          */
  int64_t token_stride;
  const void* sorted_rows; /* gather, combine_backward                          */
  int64_t sorted_stride;
  const void* weights;     /* (tokens, slots) contiguous                        */
  void* token_out;         /* gather, (tokens, dim) contiguous                  */
  void* sorted_out;        /* spread, combine_backward; contiguous; may be null in
                              combine_backward                                  */
  void* grad_weights;      /* combine_backward, (tokens, slots); may be null     */
} PurinRouteRowsArgs;

int32_t purin_route_spread(const PurinRouteRowsArgs* args, void* stream);
int32_t purin_route_gather(const PurinRouteRowsArgs* args, void* stream);
int32_t purin_route_combine_backward(const PurinRouteRowsArgs* args, void* stream);

/* ---- linear layer and softmax cross entropy ------------------------------------
 * z = hidden weight^T, lse[i] = log sum_v exp z[i,v], loss[i] = lse[i] - z[i, targets[i]].
 * A target equal to `ignore` or outside [0, vocab) gives loss 0 and no gradient.
 * The logits are made in pieces and not kept; the backward makes them again. */
typedef struct PurinLossArgs {
  int32_t device;
  int32_t dtype;         /* PURIN_OPS_BFLOAT16 or PURIN_OPS_FLOAT32            */
  int32_t targets_64bit;
  int64_t tokens;
  int64_t vocab;
  int64_t dim;
  int64_t ignore;
  const void* hidden;    /* (tokens, dim)                                      */
  int64_t hidden_stride;
  const void* weight;    /* (vocab, dim)                                       */
  int64_t weight_stride;
  const void* targets;   /* (tokens)                                           */
  float* softmax;        /* (tokens, 2), 8-byte aligned: a row's softmax is
                            exp2(z log2 e - first) / second; the forward writes it, the
                            backward reads it                                  */
  float* loss;           /* (tokens), forward                                  */
  float* sum;            /* one value: the sum of the losses, forward; may be null */
  float* mean;           /* one value: the mean over targets that count (0 if none),
                            forward; may be null                               */
  float* count;          /* one value: how many targets count (at least 1), forward;
                            may be null                                        */
  const float* grad_loss;  /* backward: one value (grad_stride 0) or one per token */
  int64_t grad_stride;
  const float* divisor;    /* backward: the gradients are divided by it; may be null */
  void* grad_hidden;     /* (tokens, dim) contiguous, may be null              */
  void* grad_weight;     /* (vocab, dim) contiguous, may be null               */
} PurinLossArgs;

int32_t purin_loss_workspace_size(const PurinLossArgs* args, int32_t backward, size_t* bytes);
int32_t purin_loss_forward(const PurinLossArgs* args, void* workspace, size_t workspace_bytes,
                           void* stream);
int32_t purin_loss_backward(const PurinLossArgs* args, void* workspace, size_t workspace_bytes,
                            void* stream);

/* ---- gradient norm and clipping ------------------------------------------------
 * norm = sqrt(sum of x^2 over all tensors); out = x * min(1, max_norm / (norm + eps)).
 * Each tensor is contiguous; in and out may be the same pointer but may not overlap
 * otherwise.  `norm` is one float (or double). */
typedef struct PurinGradient {
  const void* in;
  void* out;          /* clip only                                             */
  int64_t values;
  int32_t dtype;      /* PurinOpsDtype of in and out                           */
  int32_t reserved;
} PurinGradient;

typedef struct PurinGradientsArgs {
  int32_t device;
  int32_t norm_dtype;           /* PURIN_OPS_FLOAT64 or PURIN_OPS_FLOAT32      */
  int64_t tensors;
  const PurinGradient* list;    /* HOST pointer, `tensors` entries             */
  int32_t clip;                 /* 0: only the norm                            */
  double max_norm;
  double eps;
  void* norm;                   /* one value                                   */
} PurinGradientsArgs;

int32_t purin_gradients_workspace_size(const PurinGradientsArgs* args, size_t* bytes);
int32_t purin_gradients(const PurinGradientsArgs* args, void* workspace, size_t workspace_bytes,
                        void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PURIN_OPS_H */
