// rq_wkv7.h -- the recurrence's arguments, shared by its kernels and the entry
// points.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

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

// A scan whose heads are too few for the GPU's 256 CUs takes each sequence in segments, all at
// once: first every segment's end from a state of 0 and from the identity (what it adds
// and how it maps a state), then the state at each segment's beginning, then the segments as
// sequences of their own.
struct WkvSegments {
    int64_t chunks;  // of a segment, 0: the sequences are taken whole
    int64_t slots;   // segments, and the unused places of a packed batch
    float* ends;     // [slots, heads, 128, 64]: 64 rows from 0, 64 from the identity
    float* begins;   // [slots, heads, 64, 64]
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
    WkvSegments seg;
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

// The segments that take the least time by what was measured: a chunk of a block takes kScanUs, one
// of a segment's end kEndsUs, a step from segment to segment kJoinUs, the further launches kMoreUs.
inline WkvSegments wkv_segments(const WkvShape& s) {
    constexpr double kScanUs = 2.4, kEndsUs = 2.7, kJoinUs = 0.6, kMoreUs = 12, kCus = 256;
    WkvSegments best{0, 0, nullptr, nullptr};
    if (s.seqs == 0 || s.heads == 0 || s.time == 0) return best;
    const int64_t all = wkv_chunks(s);
    const int64_t row = (s.time + RQ_WKV7_CHUNK - 1) / RQ_WKV7_CHUNK;
    // of a packed batch the lengths are not known here: one sequence may be this long
    const int64_t longest = s.cu ? std::min<int64_t>(row, 4 * row / s.seqs + 1) : row;
    const double share = (double)all * s.heads / kCus;
    double least = kScanUs * std::max((double)longest, share);
    for (int64_t chunks = 8; chunks < longest; chunks += chunks < 32 ? 4 : chunks / 8) {
        const double us = (kScanUs + kEndsUs) * std::max((double)chunks, share) +
                          kJoinUs * ((longest + chunks - 1) / chunks) + kMoreUs;
        if (us < least) {
            least = us;
            best.chunks = chunks;
        }
    }
    if (best.chunks) {
        const int64_t per = (row + best.chunks - 1) / best.chunks;
        best.slots = s.cu ? s.time / (RQ_WKV7_CHUNK * best.chunks) + s.seqs : s.batch * per;
    }
    return best;
}

inline int64_t wkv_segment_floats(const WkvSegments& g, int64_t heads) {
    return 3 * g.slots * heads * RQ_WKV7_HEAD * RQ_WKV7_HEAD;
}

hipError_t launch_wkv_scan(const WkvScan& a, hipStream_t stream);
hipError_t launch_wkv_grads(const WkvGrads& a, hipStream_t stream);
hipError_t launch_wkv_step(const WkvStep& a, hipStream_t stream);
// 0 in the rows of a packed batch that belong to no sequence; NULL tensors are left out.
hipError_t launch_wkv_rest(const WkvShape& s, int dt, void* const* tensors, int n, hipStream_t stream);

}  // namespace rq
