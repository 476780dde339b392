/*
 * rwkvq_train.h -- C ABI of the operators a training step runs around the
 * packed products of rwkvq.h, in the same library (librwkvq_hip.so):
 *
 *   rq_linear*           <- the dense nn.Linear products the stock quantizer leaves unpacked
 *                           (tmix r/k/v/o and the low-rank tanh / sigmoid branches,
 *                           rwkv_metal/lora/finetune.py:40-42,
 *                           rwkv_metal/model/rwkv7_x070.py:108-111,142-182) and the dense FFN
 *                           with its relu^2 (rwkv7_x070.py:215-221), with their bias, activation
 *                           and residual in the product's output stage, and their gradients
 *   rq_embed*            <- nn.Embedding of a table that is trained (rwkv7_x070.py:302) with a
 *                           factor on its rows, and the table's gradient
 *   rq_grad_norm, rq_clip_grads
 *                        <- optim.clip_grad_norm of the fine-tune loop
 *                           (rwkv_metal/lora/finetune.py:108-205)
 *
 * Conventions, return codes and rq_last_error() are those of rwkvq.h: device
 * pointers owned by the caller, nothing allocated, work enqueued on `stream`
 * without synchronisation, row-major contiguous tensors, pointers 16-byte
 * aligned unless an entry point says otherwise.  Workspaces need no
 * initialisation; calls that overlap in time need separate ones.  Every
 * result is deterministic: the same inputs give the same bits.
 */
#ifndef RWKVQ_TRAIN_H
#define RWKVQ_TRAIN_H

#include "rwkvq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* relu2 is relu(v)^2; gelu is v * Phi(v) with the normal distribution's Phi;
 * silu is v * sigmoid(v). */
typedef enum {
    RQ_ACT_NONE = 0,
    RQ_ACT_RELU = 1,
    RQ_ACT_RELU2 = 2,
    RQ_ACT_SILU = 3,
    RQ_ACT_GELU = 4,
    RQ_ACT_SIGMOID = 5,
    RQ_ACT_TANH = 6
} rq_act;

/* What the backward pass takes act'(v) from: nothing (act'(v) = 1), the output
 * y, or a tensor of slopes act'(v) that the forward pass wrote. */
enum { RQ_SLOPE_NONE = 0, RQ_SLOPE_Y = 1, RQ_SLOPE_F16 = 2, RQ_SLOPE_F32 = 3 };

/* The form of the slope for operands of type dt: RQ_SLOPE_Y where y alone gives
 * it (relu, and relu2 of bf16 or fp32, with no residual added), float16 for the
 * other activations of bf16 operands, whose slopes are bounded and keep three
 * bits more than in bf16, float32 otherwise.  RQ_EINVAL for an unknown act or dt. */
int rq_linear_slope(rq_act act, rq_dtype dt, int has_residual);

/* Bytes of workspace of rq_linear, rq_linear_dx and rq_linear_dw (0: none, the
 * pointer may be NULL) for x [m, k], w [n, k], operands of type dt; or a
 * negative return code.  op: 0 rq_linear, 1 rq_linear_dx, 2 rq_linear_dw,
 * 3 rq_linear_dpre. */
int64_t rq_linear_workspace_bytes(int op, int64_t m, int64_t n, int64_t k, rq_dtype dt);

/* y[m, n] = act(x[m, k] . w[n, k]^T + bias[n]) + residual[m, n].
 * x, w and bias (or NULL) in dt; residual (or NULL) and y in y_dt, which is dt
 * or RQ_F32.  One pass: v is accumulated in fp32 (bf16 and f16 operands on the
 * 16-bit matrix instructions, fp32 ones on the fp32 instruction) and rounded
 * once, into y.  slope: NULL, or where the backward pass wants
 * it [m, n] float16 or float32 as rq_linear_slope says.  k == 0 gives act(bias) +
 * residual. */
int rq_linear(const void* x, const void* w, const void* bias, rq_dtype dt, const void* residual,
              rq_dtype y_dt, int64_t m, int64_t n, int64_t k, rq_act act, void* y, void* slope,
              void* workspace, int64_t workspace_bytes, void* stream);

/* g = dy * act'(v) [m, n] in dt and db[n] = sum over m of g, in dt, from the
 * unrounded g.  Either output may be NULL.  dy in y_dt.  slope: y (in y_dt) for
 * RQ_SLOPE_Y, the forward's slopes for RQ_SLOPE_F16 / RQ_SLOPE_F32, NULL for
 * RQ_SLOPE_NONE. */
int rq_linear_dpre(const void* dy, rq_dtype y_dt, const void* slope, int slope_kind, rq_act act,
                   rq_dtype dt, int64_t m, int64_t n, void* g, void* db, void* workspace,
                   int64_t workspace_bytes, void* stream);

/* dx[m, k] = g[m, n] . w[n, k] and dw[n, k] = g[m, n]^T . x[m, k], everything
 * in dt, accumulated in fp32. */
int rq_linear_dx(const void* g, const void* w, rq_dtype dt, int64_t m, int64_t n, int64_t k,
                 void* dx, void* workspace, int64_t workspace_bytes, void* stream);
int rq_linear_dw(const void* g, const void* x, rq_dtype dt, int64_t m, int64_t n, int64_t k,
                 void* dw, void* workspace, int64_t workspace_bytes, void* stream);

/* out[i, :] = scale * table[idx[i], :], i < n, table [vocab, dim] and out in
 * dt, rounded once.  idx: int32 (idx_bytes 4) or int64 (8).  An index outside
 * [0, vocab) gives a row of NaN and reads nothing outside the table.  table,
 * out and idx need the alignment of their elements only. */
int rq_embed(const void* idx, int idx_bytes, int64_t n, const void* table, rq_dtype dt,
             int64_t vocab, int64_t dim, float scale, void* out, void* stream);

/* The table's gradient: dtable[v, :] = scale * sum of dout[i, :] over the i
 * with idx[i] == v, every row written (0 where no index points, and for
 * padding_idx; -1: none).  Indices outside [0, vocab) are left out.  dout [n,
 * dim] and dtable in dt.  The rows of one token are added in fp32, in an order
 * that depends on the sizes only.  n and vocab below 2^31. */
int64_t rq_embed_grad_workspace_bytes(int64_t n, int64_t vocab, int64_t dim);
int rq_embed_grad(const void* idx, int idx_bytes, int64_t n, const void* dout, rq_dtype dt,
                  int64_t vocab, int64_t dim, float scale, int64_t padding_idx, void* dtable,
                  void* workspace, int64_t workspace_bytes, void* stream);

/* One tensor of a gradient list: n elements of type dt at g; out is where
 * rq_clip_grads writes (g itself: in place).  g and out need the alignment of
 * their elements only. */
typedef struct {
    const void* g;
    void* out;
    int64_t n;
    int32_t dt;
    int32_t pad;
} rq_grad;

/* norm[0] = sqrt(sum of squares of every element of every tensor), fp32.  The
 * squares are added in fp64, so no finite gradient overflows the sum.  grads is
 * a host array of `count` entries, read before the call returns; the fields
 * `out` are not used.  rq_clip_grads also writes out = g * c, rounded once, c =
 * min(max_norm / (norm + eps), 1) in fp32; a NaN norm gives a NaN c.  Where c
 * is 1, tensors given in place are not touched. */
int64_t rq_grad_norm_workspace_bytes(const rq_grad* grads, int64_t count);
int rq_grad_norm(const rq_grad* grads, int64_t count, float* norm, void* workspace,
                 int64_t workspace_bytes, void* stream);
int rq_clip_grads(const rq_grad* grads, int64_t count, float max_norm, float eps, float* norm,
                  void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
