// rq_rwkv7_abi.cpp -- the extern "C" boundary of the recurrence and the sampler
// (include/rwkvq_rwkv7.h): argument checks, then the launchers.
#include <hip/hip_runtime.h>

#include <initializer_list>

#include "../../include/rwkvq_rwkv7.h"
#include "rq_error.h"
#include "rq_sample.h"
#include "rq_wkv7.h"

using rq::aligned16;
using rq::fail;
using rq::ok;
using rq::valid_dt;

namespace {

// A grid holds fewer than 2^32 threads: up to 1024 for each head of a sequence or segment in the scan, 4 x 256 in the
// joins, 256 in a decode step.  A chunk's state is 16 KB: 2^23 of them and the tensors they belong to are more than the
// card's memory.
constexpr int64_t kMaxHeadsOfSeqs = 1 << 21, kMaxHeadsOfChunks = 1 << 23, kMaxTokens = 1ll << 31;

int check_shape(const char* what, int64_t batch, int64_t time, int64_t heads, bool packed, int64_t seqs) {
    if (batch < 0 || time < 0 || heads < 0 || seqs < 0)
        return fail(RQ_EINVAL, "%s: negative size (batch=%lld time=%lld heads=%lld seqs=%lld)", what, (long long)batch,
                    (long long)time, (long long)heads, (long long)seqs);
    if (packed ? batch != 1 : seqs != batch)
        return fail(RQ_EINVAL, packed ? "%s: packed sequences take a batch of 1 (got %lld)" : "%s: seqs must be the batch (%lld)",
                    what, (long long)batch);
    if (batch >= kMaxTokens || time >= kMaxTokens || heads >= kMaxTokens || seqs >= kMaxTokens)
        return fail(RQ_EINVAL, "%s: a size is 2^31 or more", what);
    if (seqs * heads > kMaxHeadsOfSeqs)
        return fail(RQ_EINVAL, "%s: more than %lld heads of sequences", what, (long long)kMaxHeadsOfSeqs);
    return RQ_OK;
}

int check_types(const char* what, int dt, int y_dt) {
    if (!valid_dt(dt)) return fail(RQ_EINVAL, "%s: unsupported dtype", what);
    if (!valid_dt(y_dt) || (y_dt != dt && y_dt != RQ_F32))
        return fail(RQ_EINVAL, "%s: y must have the inputs' dtype or fp32", what);
    return RQ_OK;
}

int check_ptrs(const char* what, std::initializer_list<const void*> needed, std::initializer_list<const void*> others) {
    for (const void* p : needed)
        if (!p) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    for (auto list : {needed, others})
        for (const void* p : list)
            if (!aligned16(p)) return fail(RQ_EALIGN, "%s: pointers must be 16-byte aligned", what);
    return RQ_OK;
}

int check_cu(const char* what, const int32_t* cu) {
    return ((uintptr_t)cu & 3u) ? fail(RQ_EALIGN, "%s: cu_seqlens must be 4-byte aligned", what) : RQ_OK;
}

int check_chunks(const char* what, const rq::WkvShape& s) {
    if (s.heads && rq::wkv_chunks(s) > kMaxHeadsOfChunks / s.heads)
        return fail(RQ_EINVAL, "%s: more than %lld heads of chunks", what, (long long)kMaxHeadsOfChunks);
    return RQ_OK;
}

// any pointer stands for "packed" where only sizes count
const int32_t kPacked = 0;

// The segments of a scan with their workspace, whose bytes are a multiple of 16.
rq::WkvSegments segments(const rq::WkvShape& shape, bool backward, void* workspace) {
    rq::WkvSegments g = rq::wkv_segments(shape, backward);
    g.ends = (float*)workspace;
    g.begins = g.ends ? g.ends + 2 * g.slots * shape.heads * RQ_WKV7_HEAD * RQ_WKV7_HEAD : nullptr;
    return g;
}

}  // namespace

extern "C" {

int64_t rq_wkv7_chunks(int64_t batch, int64_t time, int64_t seqs, int has_cu_seqlens) {
    if (int rc = check_shape("rq_wkv7_chunks", batch, time, 0, has_cu_seqlens, seqs)) return rc;
    ok();
    return rq::wkv_chunks({has_cu_seqlens ? &kPacked : nullptr, batch, time, 0, seqs});
}

int64_t rq_wkv7_workspace_bytes(int64_t batch, int64_t time, int64_t heads, int64_t seqs, int has_cu_seqlens) {
    if (int rc = check_shape("rq_wkv7_workspace_bytes", batch, time, heads, has_cu_seqlens, seqs)) return rc;
    ok();
    const rq::WkvShape shape{has_cu_seqlens ? &kPacked : nullptr, batch, time, heads, seqs};
    return 4 * rq::wkv_segment_floats(rq::wkv_segments(shape, false), heads);
}

int rq_wkv7(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b, rq_dtype dt,
            int64_t batch, int64_t time, int64_t heads, const int32_t* cu_seqlens, int64_t seqs, const float* state,
            void* y, rq_dtype y_dt, float* state_out, float* states, float* sa, void* workspace, int64_t workspace_bytes,
            void* stream) {
    const char* what = "rq_wkv7";
    if (int rc = check_types(what, dt, y_dt)) return rc;
    if (int rc = check_shape(what, batch, time, heads, cu_seqlens, seqs)) return rc;
    if (!states != !sa) return fail(RQ_EINVAL, "%s: states and sa are kept together", what);
    const rq::WkvShape shape{cu_seqlens, batch, time, heads, seqs};
    if (states)
        if (int rc = check_chunks(what, shape)) return rc;
    if (heads == 0 || (batch * time == 0 && seqs == 0)) return ok();
    if (batch * time > 0)
        if (int rc = check_ptrs(what, {r, w, k, v, a, b, y}, {})) return rc;
    if (int rc = check_ptrs(what, {}, {state, state_out, states, sa, workspace})) return rc;
    if (int rc = check_cu(what, cu_seqlens)) return rc;
    const rq::WkvSegments seg = segments(shape, false, workspace);
    const int64_t need = 4 * rq::wkv_segment_floats(seg, heads);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(RQ_EINVAL, "%s: needs a workspace of %lld bytes", what, (long long)need);
    if (seqs == 0) return fail(RQ_EINVAL, "%s: tokens but no sequence", what);
    return rq::launch_status(
        rq::launch_wkv_scan({shape, {r, w, k, v, a, b, dt}, false, v, dt, y, y_dt, state, state_out, states, sa, seg, {}},
                            (hipStream_t)stream),
        what);
}

int64_t rq_wkv7_backward_workspace_bytes(int64_t batch, int64_t time, int64_t heads, int64_t seqs, int has_cu_seqlens) {
    const char* what = "rq_wkv7_backward_workspace_bytes";
    if (int rc = check_shape(what, batch, time, heads, has_cu_seqlens, seqs)) return rc;
    const rq::WkvShape shape{has_cu_seqlens ? &kPacked : nullptr, batch, time, heads, seqs};
    if (int rc = check_chunks(what, shape)) return rc;
    ok();
    return 4 * rq::wkv_segment_floats(rq::wkv_segments(shape, true), heads);
}

int rq_wkv7_backward(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b,
                     rq_dtype dt, int64_t batch, int64_t time, int64_t heads, const int32_t* cu_seqlens, int64_t seqs,
                     const float* states, const float* sa, const void* dy, rq_dtype y_dt, const float* dstate_out,
                     void* dr, void* dw, void* dk, void* dv, void* da, void* db, float* dstate, void* workspace,
                     int64_t workspace_bytes, void* stream) {
    const char* what = "rq_wkv7_backward";
    if (int rc = check_types(what, dt, y_dt)) return rc;
    if (int rc = check_shape(what, batch, time, heads, cu_seqlens, seqs)) return rc;
    const rq::WkvShape shape{cu_seqlens, batch, time, heads, seqs};
    if (int rc = check_chunks(what, shape)) return rc;
    if (heads == 0 || (batch * time == 0 && seqs == 0)) return ok();
    if (batch * time > 0) {
        if (int rc = check_ptrs(what, {r, w, k, v, a, b, states, sa, dy}, {dr, dw, dk, dv, da, db})) return rc;
        if (cu_seqlens && seqs == 0) return fail(RQ_EINVAL, "%s: tokens but no sequence", what);
    }
    if (int rc = check_ptrs(what, {}, {dstate_out, dstate, workspace})) return rc;
    if (int rc = check_cu(what, cu_seqlens)) return rc;
    const rq::WkvSegments seg = segments(shape, true, workspace);
    const int64_t need = 4 * rq::wkv_segment_floats(seg, heads);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(RQ_EINVAL, "%s: needs a workspace of %lld bytes", what, (long long)need);
    return rq::launch_status(
        rq::launch_wkv_scan({shape, {r, w, k, v, a, b, dt}, true, dy, y_dt, dv, dt, dstate_out, dstate, nullptr, nullptr, seg,
                             {states, sa, dr, dw, dk, da, db}},
                            (hipStream_t)stream),
        what);
}

int rq_wkv7_step(const void* r, const void* w, const void* k, const void* v, const void* a, const void* b, rq_dtype dt,
                 int64_t batch, int64_t heads, const float* state, void* y, rq_dtype y_dt, float* state_out,
                 void* stream) {
    const char* what = "rq_wkv7_step";
    if (int rc = check_types(what, dt, y_dt)) return rc;
    if (int rc = check_shape(what, batch, 1, heads, false, batch)) return rc;
    if (batch * heads == 0) return ok();
    if (int rc = check_ptrs(what, {r, w, k, v, a, b, y}, {state, state_out})) return rc;
    return rq::launch_status(
        rq::launch_wkv_step({{r, w, k, v, a, b, dt}, batch * heads, state, y, y_dt, state_out}, (hipStream_t)stream), what);
}

int rq_sample(const void* logits, rq_dtype dt, int64_t rows, int64_t vocab, const float* u, const float* temperature,
              float temperature_all, const int64_t* top_k, int64_t top_k_all, const float* top_p, float top_p_all,
              const float* min_p, float min_p_all, int64_t* token, float* logprob, void* stream) {
    const char* what = "rq_sample";
    if (!valid_dt(dt)) return fail(RQ_EINVAL, "%s: unsupported dtype", what);
    if (rows < 0 || vocab < 0) return fail(RQ_EINVAL, "%s: negative size (rows=%lld vocab=%lld)", what, (long long)rows, (long long)vocab);
    if (vocab > rq::kSampleMaxVocab) return fail(RQ_EINVAL, "%s: a vocabulary of more than %lld", what, (long long)rq::kSampleMaxVocab);
    if (rows > (1 << 21)) return fail(RQ_EINVAL, "%s: more than %d rows", what, 1 << 21);
    if (rows > 0 && vocab == 0) return fail(RQ_EINVAL, "%s: rows without a logit", what);
    if (!temperature && !(temperature_all >= 0.f)) return fail(RQ_EINVAL, "%s: a temperature is 0 or more", what);
    if (!top_k && top_k_all < 0) return fail(RQ_EINVAL, "%s: top_k is 0 or more", what);
    if (!top_p && !(top_p_all > 0.f && top_p_all <= 1.f)) return fail(RQ_EINVAL, "%s: top_p lies in (0, 1]", what);
    if (!min_p && !(min_p_all >= 0.f && min_p_all <= 1.f)) return fail(RQ_EINVAL, "%s: min_p lies in [0, 1]", what);
    if (rows == 0) return ok();
    if (!logits || !u || !token) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    const uintptr_t fours = (uintptr_t)u | (uintptr_t)temperature | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)logprob;
    if (((uintptr_t)logits & (dt == RQ_F32 ? 3u : 1u)) || (fours & 3u) || (((uintptr_t)top_k | (uintptr_t)token) & 7u))
        return fail(RQ_EALIGN, "%s: pointers must be aligned to their elements", what);
    return rq::launch_status(
        rq::launch_sample({logits, dt, rows, vocab, u, temperature, top_k, top_p, min_p, temperature_all, top_k_all,
                           top_p_all, min_p_all, token, logprob},
                          (hipStream_t)stream),
        what);
}

}  // extern "C"
