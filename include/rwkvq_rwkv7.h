/*
 * rwkvq_rwkv7.h -- C ABI of what an RWKV-7 block and its token choice run
 * between the products of rwkvq.h, in the same library (librwkvq_hip.so):
 *
 *   rq_wkv7, rq_wkv7_backward  <- the time mixing's recurrence over a sequence and its
 *                                 gradients (rwkv_metal/kernel/wkv7.py:67-107,109-214,
 *                                 called at rwkv_metal/model/rwkv7_x070.py:184-187)
 *   rq_wkv7_step               <- its form for one token (rwkv7_x070.py:174-182)
 *   rq_sample                  <- the token chosen from the head's logits
 *
 * Conventions, return codes and rq_last_error() are those of rwkvq.h: device
 * pointers owned by the caller, nothing allocated, work enqueued on `stream`
 * without synchronisation, row-major contiguous tensors, pointers 16-byte
 * aligned unless an entry point says otherwise.  Workspaces need no
 * initialisation; calls that overlap in time need separate ones.  Every
 * result is deterministic: the same inputs give the same bits.
 */
#ifndef RWKVQ_RWKV7_H
#define RWKVQ_RWKV7_H

#include "rwkvq.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RQ_WKV7_HEAD 64  /* channels of a head: 64 values, 64 keys */
#define RQ_WKV7_CHUNK 16 /* tokens between two stored states */

/* The recurrence of every head, with its state S [64 values, 64 keys] in fp32:
 *
 *     d_t = exp(-exp(w_t))
 *     S_t = S_{t-1} diag(d_t) + (S_{t-1} a_t) b_t^T + v_t k_t^T
 *     y_t = S_t r_t
 *
 * r, w, k, v, a, b: [batch, time, heads, 64] of dt; y the same of y_dt (dt or
 * RQ_F32).  A token with w = -inf, k = 0 and b = 0 (and finite r, v, a) leaves the state as it was.
 * Tokens are taken in chunks of 16: a NaN or an infinity may reach the y before it in its own chunk.
 *
 * cu_seqlens NULL: `seqs` is batch, every row of the batch a sequence.  Else
 * batch is 1 and sequence n has the tokens cu_seqlens[n] .. cu_seqlens[n + 1] - 1 of
 * `time` (seqs + 1 values on the device, not decreasing; an empty sequence keeps its
 * state).  Values outside [0, time] are read as the nearest inside, a
 * sequence that would end before it starts as empty; y is 0 before the first sequence
 * and behind the last.  Where the boundaries decrease, tokens may be in several
 * sequences or in none: what is written for them is undefined.
 *
 * state: [seqs, heads, 64, 64] before the first token, NULL for 0; state_out the same
 * after the last, or NULL; the two may be one buffer.  states [rq_wkv7_chunks(), heads, 64, 64] and
 * sa [rq_wkv7_chunks(), heads, 16, 64], both or neither: what rq_wkv7_backward reads
 * (every 16th state, and S_{t-1} a_t of every token).
 *
 * At most 2^21 heads of sequences (seqs * heads), and where states are kept 2^23 heads of chunks. */
int64_t rq_wkv7_chunks(int64_t batch, int64_t time, int64_t seqs, int has_cu_seqlens);
int64_t rq_wkv7_workspace_bytes(int64_t batch, int64_t time, int64_t heads, int64_t seqs, int has_cu_seqlens);
int rq_wkv7(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
            rq_dtype dt, int64_t batch, int64_t time, int64_t heads, const int32_t* cu_seqlens, int64_t seqs,
            const float* state, void* y, rq_dtype y_dt, float* state_out, float* states, float* sa, void* workspace,
            int64_t workspace_bytes, void* stream);

/* The gradients of rq_wkv7's inputs from dy (of y_dt) and dstate_out (fp32, NULL for
 * 0).  dr .. db are of dt, dstate is fp32; each may be NULL.  states and sa are those
 * that rq_wkv7 wrote. */
int64_t rq_wkv7_backward_workspace_bytes(int64_t batch, int64_t time, int64_t heads, int64_t seqs,
                                         int has_cu_seqlens);
int rq_wkv7_backward(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                     rq_dtype dt, int64_t batch, int64_t time, int64_t heads, const int32_t* cu_seqlens,
                     int64_t seqs, const float* states, const float* sa, const void* dy, rq_dtype y_dt,
                     const float* dstate_out, void* dr, void* dw, void* dk, void* dv, void* da, void* db,
                     float* dstate, void* workspace, int64_t workspace_bytes, void* stream);

/* One token of every sequence: r .. b and y [batch, heads, 64], state and state_out
 * [batch, heads, 64, 64] (they may be one buffer; state NULL for 0).  Otherwise what is written must
 * not overlap what is read: there is no order between the heads. */
int rq_wkv7_step(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                 rq_dtype dt, int64_t batch, int64_t heads, const float* state, void* y, rq_dtype y_dt,
                 float* state_out, void* stream);

/* token[i] from the logits [rows, vocab] of dt (at most 2^21 rows, vocab at most 2^20, no alignment of the rows) and
 * u[i] in [0, 1), in this order, with e_j = exp((l_j - max l) / temperature):
 *   1. the top_k largest stay (0: all);
 *   2. of these, from the largest, those before whom less than top_p of their sum lies (1: all);
 *   3. of these, those with e_j >= min_p;
 *   4. the first by index at which the running sum of what stays exceeds u times the whole.
 * Equal logits rank by index.  A temperature of 0 takes the largest logit.  logprob[i] (or NULL) is the log of the
 * token's share of what stays.  -inf logits never come; +inf ones share everything.  A row with a NaN, or of
 * -inf alone, gives token -1 and a NaN.  The sums are exact, of terms of float64 rounded to 2^-36
 * (2^-33 past 2^17 logits); a token whose e_j is below half of that never comes.
 *
 * temperature, top_k, top_p, min_p: one for each row, or NULL for the value behind it.  Values on the
 * device are not checked: a temperature that is not above 0 is 0, top_k below 1 is 0, a top_p of 0 or less keeps the
 * largest alone and one that is not below 1 all, min_p is moved into [0, 1] (NaN: 0), u into [0, 1) (NaN: 0).
 * u, temperature, top_p and min_p are 4-byte aligned, top_k and token 8-byte. */
int rq_sample(const void* logits, rq_dtype dt, int64_t rows, int64_t vocab, const float* u,
              const float* temperature, float temperature_all, const int64_t* top_k, int64_t top_k_all,
              const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* token,
              float* logprob, void* stream);

#ifdef __cplusplus
}
#endif
#endif
