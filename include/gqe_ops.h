/* gqe_ops.h — operators on plain device tensors, next to the conjunctive-query path of gqe.h: the softmax cross entropy of query
 * embeddings over every row of an entity table with its gradients, the global gradient norm with clipping, layer normalisation
 * with its backward pass, and the query side of relation chains (the reference trains with one sampled negative per query,
 * netquery/model.py:112-127; these train against the whole table).
 *
 * Conventions: as in gqe.h — plain C types, borrowed device pointers, all work enqueued on the caller's hipStream_t, no hidden
 * synchronisation, 0 on success or a negative gqe_status.  The calls need no gqe_ctx and keep no state: every buffer they use is an
 * argument, so calls on different streams (with workspaces of their own) and from different threads are independent, and a call can
 * be captured into a HIP graph (kernels only; the workspace then belongs to that graph, and the first call of a kind, which loads its
 * kernels, comes before).  `device` is the HIP device of the pointers and the stream; it need not be the current one.  Results and
 * workspaces share no memory with inputs or with one another (what is scaled or added to in place apart).  gqe_ops_last_error() is the text of the calling thread's last refusal.
 * Rows are `dim` elements with unit stride; row strides are in elements.  Results do not depend on the order of atomics (there are
 * none): the same call on the same inputs gives the same bits. */
#ifndef GQE_OPS_H
#define GQE_OPS_H

#include <stdint.h>

#include "gqe.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum { GQE_F32 = 0, GQE_BF16 = 1 } gqe_dtype;

const char* gqe_ops_last_error(void);

/* ---- softmax cross entropy over a whole table ------------------------------------------------------------------------------
 * z_bv = scale * q_b . t_v, t_v = table row v, divided by its length if normalize (a zero row stays zero: what the encoder does
 * with the rows it reads, encoders.py:40-43);   lse_b = log sum_v exp z_bv;   loss_b = lse_b - z_b,target(b).
 * Gradients are those of sum_b weight_b loss_b.  The logits are never kept.  target[b] < 0 ignores query b: loss 0, no gradient
 * (lse is still given); target[b] >= n_rows gives loss NaN and no gradient.
 * phase: what the call computes, any sum of
 *   GQE_XENT_LOSS    loss, lse, stat                                (always part of GQE_XENT_DQ)
 *   GQE_XENT_DQ      dq; weight NULL = all ones
 *   GQE_XENT_DTABLE  dtable.  Without LOSS / DQ the call reads `stat` as an earlier call with the same q, table, target, scale and
 *                    normalize wrote it — the backward call of an autograd node, whose weights are known only then
 * dim <= 256; n_queries may be 0 (dtable is then zeroed, or left if accumulate). */
enum { GQE_XENT_LOSS = 1, GQE_XENT_DQ = 2, GQE_XENT_DTABLE = 4 };
typedef struct {
  int32_t device;
  int32_t phase;
  int32_t dtype;            /* gqe_dtype of q, table, dq and dtable                                         */
  int32_t dim;
  int64_t n_queries, n_rows;
  const void* q;
  int64_t q_stride;
  const void* table;
  int64_t table_stride;
  const int32_t* target;    /* [n_queries]                                                                  */
  const float* weight;      /* [n_queries] or NULL                                                          */
  float scale;              /* finite; logits = scale * product                                             */
  int32_t normalize;
  float* loss;              /* [n_queries] or NULL                                                          */
  float* lse;               /* [n_queries] or NULL                                                          */
  float* stat;              /* [n_queries][2]: log2 of the sum, log2 of the share of the rows != target     */
  void* dq;
  int64_t dq_stride;
  int32_t dq_f32;           /* dq is float32 whatever dtype says                                            */
  int32_t accumulate;       /* dtable += (float32 only) instead of =                                        */
  void* dtable;
  int64_t dtable_stride;
  void* workspace;          /* gqe_softmax_xent_workspace bytes, 256-byte aligned                           */
  int64_t workspace_bytes;
  void* stream;
} gqe_xent_args;
int64_t gqe_softmax_xent_workspace(const gqe_xent_args* args);   /* from phase, dtype, dim, n_queries, n_rows and whether stat is given; negative: refused */
int gqe_softmax_xent(const gqe_xent_args* args);

/* ---- global gradient norm and clipping --------------------------------------------------------------------------------------
 * norm = sqrt(sum over all tensors of g^2), summed in 64 bits; with max_norm >= 0 every tensor is multiplied in place by
 * min(1, max_norm / (norm + 1e-6)) — torch.nn.utils.clip_grad_norm_.  A factor of 1 writes nothing.  A norm that is not finite
 * multiplies by what the formula gives (0 or NaN).  max_norm < 0: the norm alone.  Tensors are contiguous; numel 0 is allowed. */
typedef struct {
  void* data;
  int64_t numel;
  int32_t dtype;            /* gqe_dtype */
  int32_t reserved;
} gqe_tensor;
int64_t gqe_clip_grads_workspace(const gqe_tensor* tensors, int32_t n_tensors);
int gqe_clip_grads(int32_t device, const gqe_tensor* tensors, int32_t n_tensors, float max_norm, float* norm, void* workspace,
                   int64_t workspace_bytes, void* stream);

/* ---- layer normalisation ----------------------------------------------------------------------------------------------------
 * y = (x - mean) * rstd * weight + bias, mean / rstd = 1 / sqrt(var + eps) per row (biased variance), kept in float32 for the backward
 * pass:  g = dy * weight, xhat = (x - mean) * rstd;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat));  dweight = sum_rows dy * xhat,
 * dbias = sum_rows dy.  weight / bias / dweight / dbias are float32; x, y, dy, dx have dtype; weight and bias may be NULL (1 and 0),
 * dweight and dbias NULL (not computed), accumulate: += into dweight / dbias.  1 <= dim <= 16384; n_rows may be 0. */
typedef struct {
  int32_t device;
  int32_t dtype;
  int32_t dim;
  int32_t accumulate;
  int64_t n_rows;
  const void* x;
  int64_t x_stride;
  const float* weight;
  const float* bias;
  float eps;
  int32_t reserved;
  void* y;                  /* forward */
  int64_t y_stride;
  float* mean;              /* [n_rows]: written by the forward call, read by the backward call */
  float* rstd;
  const void* dy;           /* backward */
  int64_t dy_stride;
  void* dx;                 /* or NULL */
  int64_t dx_stride;
  float* dweight;
  float* dbias;
  void* workspace;          /* gqe_layer_norm_workspace bytes (backward with dweight or dbias; 0 for few rows) */
  int64_t workspace_bytes;
  void* stream;
} gqe_layer_norm_args;
int64_t gqe_layer_norm_workspace(const gqe_layer_norm_args* args);
int gqe_layer_norm_forward(const gqe_layer_norm_args* args);
int gqe_layer_norm_backward(const gqe_layer_norm_args* args);

/* ---- the query side of a relation chain -------------------------------------------------------------------------------------
 * q_b = (w / |w|) r_1 .. r_k element by element, w = table row rows[b]: the bilinear-diag score of a chain (decoders.py:228-233) is q_b . t
 * for every target t, so this is what gqe_softmax_xent scores against a whole table.  A row outside 0 .. n_rows - 1 gives NaN and no
 * gradient.  Backward: ADDS into dtable and drel[j] (which may name one relation more than once).  float32; n <= 65536; workspace of the
 * backward call: 8 n dim bytes. */
typedef struct {
  int32_t device;
  int32_t dim;
  int64_t n;
  const int32_t* rows;      /* [n] */
  const float* table;
  int64_t table_stride, n_rows;
  int32_t n_rels;           /* 0 .. 3 */
  int32_t reserved;
  const float* rel[3];
  float* q;                 /* forward */
  int64_t q_stride;
  const float* dq;          /* backward */
  int64_t dq_stride;
  float* dtable;
  int64_t dtable_stride;
  float* drel[3];
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} gqe_chain_args;
int gqe_chain_rows_forward(const gqe_chain_args* args);
int gqe_chain_rows_backward(const gqe_chain_args* args);

#ifdef __cplusplus
}
#endif
#endif /* GQE_OPS_H */
