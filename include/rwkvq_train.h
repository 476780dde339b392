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

/* relu2 is relu(v)^2, whose slope 2 relu(v) of a NaN is NaN, relu's is 1; gelu is v * Phi(v) with the normal distribution's Phi;
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
enum { RQ_SLOPE_NONE = 0, RQ_SLOPE_Y = 1, RQ_SLOPE_BOUND16 = 2, RQ_SLOPE_F32 = 3, RQ_SLOPE_WIDE16 = 4 };

/* The form of the slope for operands of type dt.  RQ_SLOPE_Y where y alone gives
 * it: relu, and relu2 of fp32, with no residual added.  For bf16 operands 16 bits
 * that keep three bits more than bf16 where float16 is normal and bf16's elsewhere:
 * RQ_SLOPE_BOUND16 of slopes s below 2: the float16 bits of s, or where |s| < 2^-14 its
 * sign and 0x4000 + the bf16 bits of |s| (a 0 may have either);
 * RQ_SLOPE_WIDE16 of relu2, whose slope 2 v is not bounded but has no sign: the
 * float16 bits of a slope in [2^-14, 2^15), else 0x8000 + its bf16 bits.  float32
 * otherwise.
 * RQ_EINVAL for an unknown act or dt. */
int rq_linear_slope(rq_act act, rq_dtype dt, int has_residual);

/* Bytes of workspace of rq_linear for these sizes (0: none, the pointer may be
 * NULL), or a negative return code. */
int64_t rq_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, rq_dtype dt);

/* y[m, n] = act(x[m, k] . w[n, k]^T + bias[n]) + residual[m, n].
 * x, w and bias (or NULL) in dt; residual (or NULL) and y in y_dt, which is dt
 * or RQ_F32.  One pass: v is accumulated in fp32 (bf16 and f16 operands on the
 * 16-bit matrix instructions, fp32 ones on the fp32 instruction) and rounded
 * once, into y.  slope: NULL, or where the backward pass wants
 * it [m, n] in the 16 or 32 bits that rq_linear_slope says.  k == 0 gives act(bias) +
 * residual. */
int rq_linear(const void* x, const void* w, const void* bias, rq_dtype dt, const void* residual,
              rq_dtype y_dt, int64_t m, int64_t n, int64_t k, rq_act act, void* y, void* slope,
              void* workspace, int64_t workspace_bytes, void* stream);

/* The gradients of rq_linear's x, w and bias: with g = dy * act'(v) [m, n]
 *   dx[m, k] = g . w      dw[n, k] = g^T . x      db[n] = sum over m of g
 * in dt, each written only where its pointer is not NULL (x and w may be NULL where
 * no wanted gradient reads them).  dy is in y_dt (dt or RQ_F32).  slope: y (in y_dt) for
 * RQ_SLOPE_Y, what rq_linear wrote for the kinds it writes, NULL for RQ_SLOPE_NONE.
 * g is rounded to dt once for the two products (dy itself is g where the slope is 1 and
 * the types are equal) and added up unrounded for db; all sums are fp32.
 * rq_linear_backward_workspace_bytes: for the gradients wanted (has_*). */
int64_t rq_linear_backward_workspace_bytes(int64_t m, int64_t n, int64_t k, rq_dtype dt, rq_dtype y_dt,
                                           int slope_kind, int has_dx, int has_dw, int has_db);
int rq_linear_backward(const void* dy, rq_dtype y_dt, const void* slope, int slope_kind, rq_act act,
                       const void* x, const void* w, rq_dtype dt, int64_t m, int64_t n, int64_t k,
                       void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes,
                       void* stream);

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
 * that depends on the sizes only.  n below 2^31, vocab at most 2^30. */
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
 * is 1, tensors given in place are not touched.  An entry listed again (the same g,
 * out, n and dt: tied weights) counts again in the norm and is scaled once.  An entry
 * may read what another one writes, which then runs after it; RQ_EINVAL where that
 * has no order (an entry that does both, or a g that overlaps its own out without being it) and
 * where two outputs overlap otherwise. */
int64_t rq_grad_norm_workspace_bytes(const rq_grad* grads, int64_t count);
int rq_grad_norm(const rq_grad* grads, int64_t count, float* norm, void* workspace,
                 int64_t workspace_bytes, void* stream);
int rq_clip_grads(const rq_grad* grads, int64_t count, float max_norm, float eps, float* norm,
                  void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
