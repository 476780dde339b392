// rq_train_abi.cpp -- the extern "C" boundary of the dense products
// (include/rwkvq_train.h): argument checks, then the launchers.
#include <hip/hip_runtime.h>

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
    // grids count tiles of 64 rows in y, and offsets inside a tile stay in 32 bits
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

int run_dense(const char* what, const rq::DenseArgs& g, void* workspace, int64_t bytes, void* stream) {
    const int64_t need = rq::dense_workspace_bytes(g);
    if (need > 0 && (!workspace || bytes < need))
        return fail(RQ_EINVAL, "%s: needs a workspace of %lld bytes", what, (long long)need);
    return rq::launch_status(rq::launch_dense(g, workspace, (hipStream_t)stream), what);
}

}  // namespace

extern "C" {

int rq_linear_slope(rq_act act, rq_dtype dt, int has_residual) {
    if ((int)act < 0 || act > RQ_ACT_TANH) return fail(RQ_EINVAL, "rq_linear_slope: unknown activation %d", (int)act);
    if (!valid_dt(dt)) return fail(RQ_EINVAL, "rq_linear_slope: unsupported dtype");
    ok();
    if (act == RQ_ACT_NONE) return RQ_SLOPE_NONE;
    // relu2 in f16: y = v^2 underflows where v does not
    if (!has_residual && (act == RQ_ACT_RELU || (act == RQ_ACT_RELU2 && dt != RQ_F16))) return RQ_SLOPE_Y;
    // the slope 2 v of relu2 is not bounded by float16's range
    return dt == RQ_BF16 && act != RQ_ACT_RELU2 ? RQ_SLOPE_F16 : RQ_SLOPE_F32;
}

int64_t rq_linear_workspace_bytes(int op, int64_t m, int64_t n, int64_t k, rq_dtype dt) {
    const char* what = "rq_linear_workspace_bytes";
    if (int rc = check_sizes(what, m, n, k, dt)) return rc;
    ok();
    switch (op) {
        case 0: return rq::dense_workspace_bytes(forward_args(nullptr, nullptr, m, n, k, dt));
        case 1: return rq::dense_workspace_bytes(dx_args(nullptr, nullptr, m, n, k, dt, nullptr));
        case 2: return rq::dense_workspace_bytes(dw_args(nullptr, nullptr, m, n, k, dt, nullptr));
        case 3: return rq::dpre_workspace_bytes(m, n);
        default: return fail(RQ_EINVAL, "%s: unknown op %d", what, op);
    }
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
    if (slope && kind != RQ_SLOPE_F16 && kind != RQ_SLOPE_F32)
        return fail(RQ_EINVAL, "%s: this activation keeps no slopes (rq_linear_slope)", what);
    rq::DenseArgs g = forward_args(x, w, m, n, k, dt);
    g.bias = bias;
    g.residual = residual;
    g.act = act;
    g.y = y;
    g.y_dt = y_dt;
    g.slope = slope;
    g.slope_kind = kind;
    return run_dense(what, g, workspace, workspace_bytes, stream);
}

int rq_linear_dpre(const void* dy, rq_dtype y_dt, const void* slope, int slope_kind, rq_act act, rq_dtype dt,
                   int64_t m, int64_t n, void* g, void* db, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "rq_linear_dpre";
    if (int rc = check_sizes(what, m, n, 0, dt)) return rc;
    if (!valid_dt(y_dt) || (y_dt != dt && y_dt != RQ_F32))
        return fail(RQ_EINVAL, "%s: dy must have the operands' dtype or fp32", what);
    if ((int)act < 0 || act > RQ_ACT_TANH) return fail(RQ_EINVAL, "%s: unknown activation %d", what, (int)act);
    if (slope_kind < RQ_SLOPE_NONE || slope_kind > RQ_SLOPE_F32 ||
        (slope_kind == RQ_SLOPE_Y && act != RQ_ACT_RELU && act != RQ_ACT_RELU2))
        return fail(RQ_EINVAL, "%s: slope kind %d does not give the slope of activation %d", what, slope_kind, (int)act);
    if (n == 0 || (!g && !db)) return ok();
    if (int rc = check_ptrs(what, {}, {dy, slope, g, db, workspace})) return rc;
    if (m > 0 && (!dy || (slope_kind != RQ_SLOPE_NONE && !slope))) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    const int64_t need = rq::dpre_workspace_bytes(m, n);
    if (db && need > 0 && (!workspace || workspace_bytes < need))
        return fail(RQ_EINVAL, "%s: needs a workspace of %lld bytes", what, (long long)need);
    const rq::DpreArgs a{dy, y_dt, slope, slope_kind, act, dt, m, n, g, db};
    return rq::launch_status(rq::launch_dpre(a, workspace, (hipStream_t)stream), what);
}

int rq_linear_dx(const void* g, const void* w, rq_dtype dt, int64_t m, int64_t n, int64_t k, void* dx,
                 void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "rq_linear_dx";
    if (int rc = check_sizes(what, m, n, k, dt)) return rc;
    if (m == 0 || k == 0) return ok();
    if (int rc = check_ptrs(what, {dx}, {g, w, dx, workspace})) return rc;
    if (n > 0 && (!g || !w)) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    return run_dense(what, dx_args(g, w, m, n, k, dt, dx), workspace, workspace_bytes, stream);
}

int rq_linear_dw(const void* g, const void* x, rq_dtype dt, int64_t m, int64_t n, int64_t k, void* dw,
                 void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "rq_linear_dw";
    if (int rc = check_sizes(what, m, n, k, dt)) return rc;
    if (n == 0 || k == 0) return ok();
    if (int rc = check_ptrs(what, {dw}, {g, x, dw, workspace})) return rc;
    if (m > 0 && (!g || !x)) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    return run_dense(what, dw_args(g, x, m, n, k, dt, dw), workspace, workspace_bytes, stream);
}

}  // extern "C"
