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

// Of the backward pass: what the forward one stored, and where the gradients go (each may be NULL).
struct WkvGrads {
    const float *states, *sa;
    void *dr, *dw, *dk, *da, *db;
};

// One pass over the tokens, forwards or backwards in time.  Rows of a packed batch that belong to no sequence become 0.
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
    float* states;        // forwards, [chunks, heads, 64, 64]: the state with which the pass enters each chunk, or NULL
    float* sa;            // forwards, [chunks, heads, 16, 64]: S a of every token, or NULL
    WkvSegments seg;
    WkvGrads grads;       // backwards
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

// The segments that take the least time by what was measured: a chunk of a block's scan takes kScanUs (kBackUs with
// the gradients), one of a segment's end kEndsUs, and as much as two chunks to begin; a step from segment to segment
// kJoinUs, the further launches kMoreUs.  A block has a CU to itself, and one block more than there are CUs is a
// whole turn more: 12 heads of 8192 tokens took 93 us forwards in 264 blocks of 24 chunks, 73 us in 252 of 25.
inline WkvSegments wkv_segments(const WkvShape& s, bool backward) {
    constexpr double kScanUs = 2.4, kBackUs = 7, kEndsUs = 2.7, kJoinUs = 0.8, kMoreUs = 12;
    constexpr int64_t kCus = 256, kBegin = 2;
    WkvSegments best{0, 0, nullptr, nullptr};
    if (s.seqs == 0 || s.heads == 0 || s.time == 0) return best;
    const int64_t all = wkv_chunks(s);
    const int64_t row = (s.time + RQ_WKV7_CHUNK - 1) / RQ_WKV7_CHUNK;
    // of a packed batch the lengths are not known here: one sequence may be this long
    const int64_t longest = s.cu ? std::min<int64_t>(row, 4 * row / s.seqs + 1) : row;
    const auto slots = [&](int64_t chunks) {
        return s.cu ? s.time / (RQ_WKV7_CHUNK * chunks) + s.seqs : s.batch * ((row + chunks - 1) / chunks);
    };
    // chunks, one after another, of the CU that has most
    const auto turns = [&](int64_t chunks, int64_t n) {
        const int64_t blocks = n * s.heads;
        const double share = (double)(all + kBegin * n) * s.heads / kCus;
        if (s.cu) return std::max((double)(chunks + kBegin), share + (blocks > kCus ? 0.5 * chunks : 0));
        return (double)(chunks + kBegin) * ((blocks + kCus - 1) / kCus);
    };
    const double scan = backward ? kBackUs : kScanUs;
    double least = scan * turns(longest, s.seqs);
    for (int64_t chunks = 4; chunks < longest; chunks += chunks < 64 ? 1 : chunks / 32) {
        const double us = (scan + kEndsUs) * turns(chunks, slots(chunks)) +
                          kJoinUs * ((longest + chunks - 1) / chunks) + kMoreUs;
        if (us < least) {
            least = us;
            best.chunks = chunks;
        }
    }
    if (best.chunks) best.slots = slots(best.chunks);
    return best;
}

inline int64_t wkv_segment_floats(const WkvSegments& g, int64_t heads) {
    return 3 * g.slots * heads * RQ_WKV7_HEAD * RQ_WKV7_HEAD;
}

hipError_t launch_wkv_scan(const WkvScan& a, hipStream_t stream);
hipError_t launch_wkv_step(const WkvStep& a, hipStream_t stream);

}  // namespace rq
