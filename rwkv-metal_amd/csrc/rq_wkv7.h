// rq_wkv7.h -- the recurrence's arguments, shared by its kernels and the entry
// points.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/rwkvq_rwkv7.h"

namespace rq {

// Where the tokens of a sequence lie, and the chunks of 16 that they fall into.
struct WkvShape {
    const int32_t* cu;  // or NULL: every row of the batch is a sequence
    int64_t batch, time, heads, seqs;
};

struct WkvInputs {
    const void *r, *w, *k, *v, *a, *b;
    int dt;
};

// One pass over the tokens, forwards or backwards in time.
struct WkvScan {
    WkvShape shape;
    WkvInputs in;
    bool reverse;
    const void* x;        // v, or dy backwards
    int x_dt;
    void* y;              // y, or dv backwards; or NULL
    int y_dt;
    const float* state;   // where the pass begins, or NULL for 0
    float* state_out;     // where it ends, or NULL
    float* states;        // [chunks, heads, 64, 64]: the state with which the pass enters each chunk, or NULL
    float* sa;            // [chunks, heads, 16, 64]: S a of every token (its gradient backwards), or NULL
};

// dr, dw, dk, da and db of every chunk from what the two passes stored.
struct WkvGrads {
    WkvShape shape;
    WkvInputs in;
    const void* dy;
    int dy_dt;
    const float *states, *sa, *dstates, *dz;
    void *dr, *dw, *dk, *da, *db;  // each may be NULL
};

struct WkvStep {
    WkvInputs in;
    int64_t rows;  // batch * heads
    const float* state;
    void* y;
    int y_dt;
    float* state_out;
};

inline int64_t wkv_chunks(const WkvShape& s) {
    // sequence n of a packed batch begins at chunk cu[n] / 16 + n: its ceil(len / 16) chunks
    // end before the next one's, whatever the lengths
    return s.cu ? s.time / RQ_WKV7_CHUNK + s.seqs : s.batch * ((s.time + RQ_WKV7_CHUNK - 1) / RQ_WKV7_CHUNK);
}

hipError_t launch_wkv_scan(const WkvScan& a, hipStream_t stream);
hipError_t launch_wkv_grads(const WkvGrads& a, hipStream_t stream);
hipError_t launch_wkv_step(const WkvStep& a, hipStream_t stream);
// 0 in the rows of a packed batch that belong to no sequence; NULL tensors are left out.
hipError_t launch_wkv_rest(const WkvShape& s, int dt, void* const* tensors, int n, hipStream_t stream);

}  // namespace rq
