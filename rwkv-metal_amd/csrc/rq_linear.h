// rq_linear.h -- the dense products' arguments, shared by their kernels and
// the entry points.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/rwkvq_train.h"

namespace rq {

// C[i, j] = sum over c of A(i, c) B(j, c), i < m, j < n, c < k, followed by the
// output stage y = act(C + bias[j]) + residual[i, j].  A(i, c) is a[i * lda + c],
// or a[c * lda + i] where a_t is set; B likewise.  Rows of y have n elements.
struct DenseArgs {
    const void* a;
    const void* b;
    int64_t lda, ldb;
    int64_t m, n, k;
    int dt;                // of a, b and bias
    bool a_t, b_t;
    const void* bias;      // [n] or NULL
    const void* residual;  // [m, n] of y_dt, or NULL
    int act;
    void* y;
    int y_dt;
    void* slope;           // [m, n]: act'(C + bias), or NULL
    int slope_kind;        // RQ_SLOPE_BOUND16, _F32 or _WIDE16 where slope is set
};

// Of m, n and k.  Offsets from a tile's first element stay in 32 bits: 256 rows of 2
// bytes or 128 of 4 an element, this long, are 2^31 bytes.
constexpr int kDenseMaxSide = 1 << 22;

hipError_t launch_dense(const DenseArgs& a, void* workspace, hipStream_t stream);
int64_t dense_workspace_bytes(const DenseArgs& a);  // of a's sizes, type and orders

// g = dy * act'(v) and db = its column sums, the start of rq_linear_backward.
struct DpreArgs {
    const void* dy;
    int y_dt;
    const void* slope;
    int slope_kind;
    int act;
    int dt;
    int64_t m, n;
    void* g;   // or NULL
    void* db;  // or NULL
};

hipError_t launch_dpre(const DpreArgs& a, void* workspace, hipStream_t stream);
int64_t dpre_workspace_bytes(int64_t m, int64_t n);

}  // namespace rq
