// rq_train_abi.cpp -- the extern "C" boundary of the dense products
// (include/rwkvq_train.h): argument checks, then the launchers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <initializer_list>

#include "../../include/rwkvq_train.h"
#include "rq_error.h"
#include "rq_linear.h"

using rq::aligned16;
using rq::fail;
using rq::ok;
using rq::valid_dt;

namespace {

int check_sizes(const char* what, int64_t m, int64_t n, int64_t k, int dt) {
    if (!valid_dt(dt)) return fail(RQ_EINVAL, "%s: unsupported dtype", what);
    if (m < 0 || n < 0 || k < 0)
        return fail(RQ_EINVAL, "%s: negative size (m=%lld n=%lld k=%lld)", what, (long long)m, (long long)n, (long long)k);
    if (m > rq::kDenseMaxSide || n > rq::kDenseMaxSide || k > rq::kDenseMaxSide)
        return fail(RQ_EINVAL, "%s: a size is more than %d", what, rq::kDenseMaxSide);
    return RQ_OK;
}

int check_ptrs(const char* what, std::initializer_list<const void*> needed, std::initializer_list<const void*> all) {
    for (const void* p : needed)
        if (!p) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    for (const void* p : all)
        if (!aligned16(p)) return fail(RQ_EALIGN, "%s: pointers must be 16-byte aligned", what);
    return RQ_OK;
}

rq::DenseArgs forward_args(const void* x, const void* w, int64_t m, int64_t n, int64_t k, int dt) {
    return {x, w, k, k, m, n, k, dt, false, false, nullptr, nullptr, RQ_ACT_NONE, nullptr, dt, nullptr, 0};
}
rq::DenseArgs dx_args(const void* g, const void* w, int64_t m, int64_t n, int64_t k, int dt, void* dx) {
    return {g, w, n, k, m, k, n, dt, false, true, nullptr, nullptr, RQ_ACT_NONE, dx, dt, nullptr, 0};
}
rq::DenseArgs dw_args(const void* g, const void* x, int64_t m, int64_t n, int64_t k, int dt, void* dw) {
    return {g, x, n, k, n, k, m, dt, true, true, nullptr, nullptr, RQ_ACT_NONE, dw, dt, nullptr, 0};
}

// Where rq_linear_backward keeps what in its workspace.
struct Backward {
    bool own_g;                 // g is not dy itself
    int64_t g, sums, products;  // bytes of g, of the partial column sums, of the products' partial sums
    int64_t bytes() const { return g + sums + products; }
};

int64_t lines(int64_t bytes) { return (bytes + 15) & ~15ll; }

Backward backward_of(int64_t m, int64_t n, int64_t k, int dt, int y_dt, int kind, bool has_dx, bool has_dw, bool has_db) {
    Backward b{};
    b.own_g = (has_dx || has_dw) && (kind != RQ_SLOPE_NONE || y_dt != dt);
    b.g = b.own_g ? lines(m * n * (dt == RQ_F32 ? 4 : 2)) : 0;
    b.sums = has_db ? lines(rq::dpre_workspace_bytes(m, n)) : 0;
    if (has_dx) b.products = rq::dense_workspace_bytes(dx_args(nullptr, nullptr, m, n, k, dt, nullptr));
    if (has_dw) b.products = std::max(b.products, rq::dense_workspace_bytes(dw_args(nullptr, nullptr, m, n, k, dt, nullptr)));
    return b;
}

int check_backward(const char* what, int64_t m, int64_t n, int64_t k, int dt, int y_dt, int kind) {
    if (int rc = check_sizes(what, m, n, k, dt)) return rc;
    if (!valid_dt(y_dt) || (y_dt != dt && y_dt != RQ_F32))
        return fail(RQ_EINVAL, "%s: dy must have the operands' dtype or fp32", what);
    if (kind < RQ_SLOPE_NONE || kind > RQ_SLOPE_WIDE16) return fail(RQ_EINVAL, "%s: unknown slope kind %d", what, kind);
    return RQ_OK;
}

}  // namespace

extern "C" {

int rq_linear_slope(rq_act act, rq_dtype dt, int has_residual) {
    if ((int)act < 0 || act > RQ_ACT_TANH) return fail(RQ_EINVAL, "rq_linear_slope: unknown activation %d", (int)act);
    if (!valid_dt(dt)) return fail(RQ_EINVAL, "rq_linear_slope: unsupported dtype");
    ok();
    if (act == RQ_ACT_NONE) return RQ_SLOPE_NONE;
    // 2 sqrt(y) for relu2 of 16-bit types would carry half of y's rounding error
    // into every gradient, and y = v^2 underflows in f16 where v does not
    if (!has_residual && (act == RQ_ACT_RELU || (act == RQ_ACT_RELU2 && dt == RQ_F32))) return RQ_SLOPE_Y;
    if (dt != RQ_BF16) return RQ_SLOPE_F32;
    return act == RQ_ACT_RELU2 ? RQ_SLOPE_WIDE16 : RQ_SLOPE_BOUND16;
}

int64_t rq_linear_workspace_bytes(int64_t m, int64_t n, int64_t k, rq_dtype dt) {
    if (int rc = check_sizes("rq_linear_workspace_bytes", m, n, k, dt)) return rc;
    ok();
    return rq::dense_workspace_bytes(forward_args(nullptr, nullptr, m, n, k, dt));
}

int rq_linear(const void* x, const void* w, const void* bias, rq_dtype dt, const void* residual, rq_dtype y_dt,
              int64_t m, int64_t n, int64_t k, rq_act act, void* y, void* slope, void* workspace,
              int64_t workspace_bytes, void* stream) {
    const char* what = "rq_linear";
    if (int rc = check_sizes(what, m, n, k, dt)) return rc;
    if (!valid_dt(y_dt) || (y_dt != dt && y_dt != RQ_F32))
        return fail(RQ_EINVAL, "%s: y must have the operands' dtype or fp32", what);
    const int kind = rq_linear_slope(act, dt, residual != nullptr);
    if (kind < 0) return kind;
    if (m == 0 || n == 0) return ok();
    if (int rc = check_ptrs(what, {y}, {x, w, bias, residual, y, slope, workspace})) return rc;
    if (k > 0 && (!x || !w)) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    if (slope && kind < RQ_SLOPE_BOUND16)
        return fail(RQ_EINVAL, "%s: this activation keeps no slopes (rq_linear_slope)", what);
    rq::DenseArgs g = forward_args(x, w, m, n, k, dt);
    g.bias = bias;
    g.residual = residual;
    g.act = act;
    g.y = y;
    g.y_dt = y_dt;
    g.slope = slope;
    g.slope_kind = kind;
    const int64_t need = rq::dense_workspace_bytes(g);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(RQ_EINVAL, "%s: needs a workspace of %lld bytes", what, (long long)need);
    return rq::launch_status(rq::launch_dense(g, workspace, (hipStream_t)stream), what);
}

int64_t rq_linear_backward_workspace_bytes(int64_t m, int64_t n, int64_t k, rq_dtype dt, rq_dtype y_dt,
                                           int slope_kind, int has_dx, int has_dw, int has_db) {
    if (int rc = check_backward("rq_linear_backward_workspace_bytes", m, n, k, dt, y_dt, slope_kind)) return rc;
    ok();
    return backward_of(m, n, k, dt, y_dt, slope_kind, has_dx, has_dw, has_db).bytes();
}

int rq_linear_backward(const void* dy, rq_dtype y_dt, const void* slope, int slope_kind, rq_act act, const void* x,
                       const void* w, rq_dtype dt, int64_t m, int64_t n, int64_t k, void* dx, void* dw, void* db,
                       void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "rq_linear_backward";
    if (int rc = check_backward(what, m, n, k, dt, y_dt, slope_kind)) return rc;
    if ((int)act < 0 || act > RQ_ACT_TANH) return fail(RQ_EINVAL, "%s: unknown activation %d", what, (int)act);
    if (slope_kind == RQ_SLOPE_Y && act != RQ_ACT_RELU && act != RQ_ACT_RELU2)
        return fail(RQ_EINVAL, "%s: y does not give the slope of activation %d", what, (int)act);
    // gradients without an element have nothing to write
    if (m == 0 || k == 0) dx = nullptr;
    if (n == 0 || k == 0) dw = nullptr;
    if (n == 0) db = nullptr;
    if (!dx && !dw && !db) return ok();
    if (int rc = check_ptrs(what, {}, {dy, slope, x, w, dx, dw, db, workspace})) return rc;
    const bool some = m > 0 && n > 0;
    if (some && (!dy || (slope_kind != RQ_SLOPE_NONE && !slope) || (dx && !w) || (dw && !x)))
        return fail(RQ_EINVAL, "%s: NULL pointer", what);
    const Backward b = backward_of(m, n, k, dt, y_dt, slope_kind, dx, dw, db);
    if (b.bytes() > 0 && (!workspace || workspace_bytes < b.bytes()))
        return fail(RQ_EINVAL, "%s: needs a workspace of %lld bytes", what, (long long)b.bytes());
    hipStream_t s = (hipStream_t)stream;
    uint8_t* const ws = (uint8_t*)workspace;
    const void* g = b.own_g ? ws : dy;
    hipError_t e = hipSuccess;
    if (b.own_g || db) {
        const rq::DpreArgs a{dy, y_dt, slope, slope_kind, act, dt, m, n, b.own_g ? ws : nullptr, db};
        e = rq::launch_dpre(a, ws + b.g, s);
    }
    if (e == hipSuccess && dx) e = rq::launch_dense(dx_args(g, w, m, n, k, dt, dx), ws + b.g + b.sums, s);
    if (e == hipSuccess && dw) e = rq::launch_dense(dw_args(g, x, m, n, k, dt, dw), ws + b.g + b.sums, s);
    return rq::launch_status(e, what);
}

}  // extern "C"
