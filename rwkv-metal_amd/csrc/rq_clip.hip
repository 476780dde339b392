// rq_clip.hip -- the 2-norm over a list of gradient tensors and their scaling
// by min(max_norm / (norm + eps), 1).
//
// norm = sqrt(sum over all tensors and elements of g^2); out = T(g * c).
// Memory bound: the norm reads S bytes, the scaling reads them again and writes
// S (the factor is known only after the last element has been read).  1.2 GB of
// bf16: 225 us (5.4 TB/s) and 434 (5.6); twice the blocks or twice the chunk
// change nothing.  288 adapters of 28 MB: three launches of 4 - 7 us and three of
// 5 - 10.
//
// A launch takes its tensors' descriptors as kernel arguments (no table to
// upload, nothing to keep alive, capturable), kClipTensors at most; longer
// lists take more launches.  Work is cut into chunks of kChunkBytes of one
// tensor, dealt to the blocks in turn.  Every block of a norm launch adds the
// squares of its chunks in fp64 -- no finite fp32 value's square overflows or
// vanishes there, and at one conversion and one fma an element the fp64 units
// keep up with the memory -- and stores one partial sum.  The partial sums are
// added up by every block of the scaling launches, in the same order each time,
// so that neither an atomic nor a launch of its own stands between the two.
#include <algorithm>
#include <utility>
#include <vector>

#include "rq_common.h"
#include "rq_error.h"
#include "rq_vec.h"
#include "../../include/rwkvq_train.h"

namespace {

constexpr int kBlock = 256;
constexpr int kChunkBytes = 16 * 1024;  // 4 loads of 16 bytes a thread in flight
constexpr int kClipTensors = 128;       // 28 bytes each: under 4 KB of kernel arguments
constexpr int kNormBlocks = 1024;       // blocks (and partial sums) of a norm launch at most
constexpr int kSumInPlace = 4096;       // partial sums that every scaling block adds up itself

struct ClipList {
    const void* g[kClipTensors];
    void* out[kClipTensors];
    uint64_t n_dt[kClipTensors];       // elements * 4 + dtype
    uint32_t first[kClipTensors + 1];  // the tensor's first chunk in the launch
    int count;
};

struct Piece {
    const uint8_t* g;
    uint8_t* out;
    int64_t n;  // elements of this chunk
    int dt;
};

RQ_DEV Piece piece_of(const ClipList& l, uint32_t chunk) {
    int lo = 0, hi = l.count - 1;  // the last tensor whose first chunk is <= chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    Piece p;
    p.dt = (int)(l.n_dt[lo] & 3);
    const int64_t n = (int64_t)(l.n_dt[lo] >> 2);
    const int per = p.dt == RQ_F32 ? kChunkBytes / 4 : kChunkBytes / 2;
    const int64_t at = (int64_t)(chunk - l.first[lo]) * per;
    p.n = n - at < per ? n - at : per;
    const int64_t b = at * (p.dt == RQ_F32 ? 4 : 2);
    p.g = (const uint8_t*)l.g[lo] + b;
    p.out = (uint8_t*)l.out[lo] + b;
    return p;
}

constexpr int kLoads = kChunkBytes / 16 / kBlock;

// The thread's vectors of a chunk, all their loads in flight; 16 bytes at any
// element alignment, so that a view behind an odd-sized one runs the same path.
RQ_DEV void load_chunk(const Piece& p, int nv, Bytes16 (&v)[kLoads]) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int k = threadIdx.x + i * kBlock;
        v[i] = k < nv ? ((const Bytes16*)p.g)[k] : Bytes16{{0u, 0u, 0u, 0u}};
    }
}

template <int DT>
RQ_DEV double chunk_squares(const Piece& p) {
    constexpr int E = kVec<DT>;
    double s = 0.0;
    const int nv = (int)(p.n / E);
    Bytes16 v[kLoads];
    load_chunk(p, nv, v);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        float f[E];
        unpack_vec<DT>(v[i], f);
#pragma unroll
        for (int j = 0; j < E; ++j) s = __builtin_fma((double)f[j], (double)f[j], s);
    }
    for (int64_t i = (int64_t)nv * E + threadIdx.x; i < p.n; i += kBlock) {
        const double f = load_dt(p.g, DT, i);
        s = __builtin_fma(f, f, s);
    }
    return s;
}

template <int DT>
RQ_DEV void chunk_scale(const Piece& p, float c) {
    constexpr int E = kVec<DT>;
    const int nv = (int)(p.n / E);
    Bytes16 v[kLoads];
    load_chunk(p, nv, v);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int k = threadIdx.x + i * kBlock;
        if (k >= nv) break;
        float f[E];
        unpack_vec<DT>(v[i], f);
#pragma unroll
        for (int j = 0; j < E; ++j) f[j] *= c;
        store_vec<DT>(p.out + (int64_t)k * 16, f);
    }
    for (int64_t i = (int64_t)nv * E + threadIdx.x; i < p.n; i += kBlock)
        store_dt(p.out, DT, i, load_dt(p.g, DT, i) * c);
}

// The block's sum of one double a thread, in thread order of the halvings; valid in every thread.
RQ_DEV double block_sum(double s) {
    __shared__ double red[kBlock / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kBlock / 64; ++w) t += red[w];
    return t;
}

__global__ __launch_bounds__(kBlock) void grad_squares_kernel(const ClipList l, uint32_t chunks,
                                                              double* __restrict__ part) {
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const Piece p = piece_of(l, c);
        switch (p.dt) {
            case RQ_BF16: s += chunk_squares<RQ_BF16>(p); break;
            case RQ_F16: s += chunk_squares<RQ_F16>(p); break;
            default: s += chunk_squares<RQ_F32>(p); break;
        }
    }
    const double t = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = t;
}

// sqrt of the sum of the partial sums, in one order for every caller.
RQ_DEV float norm_of(const double* __restrict__ part, int parts) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += kBlock) s += part[i];
    return (float)sqrt(block_sum(s));
}

__global__ __launch_bounds__(kBlock) void grad_norm_kernel(const double* __restrict__ part,
                                                           int parts, float* __restrict__ norm) {
    const float v = norm_of(part, parts);
    if (threadIdx.x == 0) norm[0] = v;
}

__global__ __launch_bounds__(kBlock) void grad_scale_kernel(const ClipList l, uint32_t chunks,
                                                            const double* __restrict__ part,
                                                            int parts, float max_norm, float eps,
                                                            float* norm, bool known) {
    float v;
    if (known) {
        v = norm[0];
    } else {
        v = norm_of(part, parts);
        if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = v;
    }
    const float q = max_norm / (v + eps);
    const float c = q >= 1.f ? 1.f : q;  // NaN stays
    for (uint32_t b = blockIdx.x; b < chunks; b += gridDim.x) {
        // last chunks first: the norm pass read them last, so of lists larger
        // than the 256 MB cache these are the ones still in it
        const Piece p = piece_of(l, chunks - 1 - b);
        if (c == 1.f && p.g == p.out) continue;
        switch (p.dt) {
            case RQ_BF16: chunk_scale<RQ_BF16>(p, c); break;
            case RQ_F16: chunk_scale<RQ_F16>(p, c); break;
            default: chunk_scale<RQ_F32>(p, c); break;
        }
    }
}

int64_t chunks_of(const rq_grad& t) {
    const int64_t per = t.dt == RQ_F32 ? kChunkBytes / 4 : kChunkBytes / 2;
    return (t.n + per - 1) / per;
}

// Calls f(list, chunks) for each launch over grads, in order; empty tensors
// take no place.  A tensor of more than 2^31 chunks' worth is refused by the checks.
template <class F>
void for_lists(const rq_grad* grads, int64_t count, F&& f) {
    ClipList l;
    l.count = 0;
    uint32_t chunks = 0;
    auto flush = [&] {
        if (l.count == 0) return;
        l.first[l.count] = chunks;
        f(l, chunks);
        l.count = 0;
        chunks = 0;
    };
    for (int64_t i = 0; i < count; ++i) {
        const int64_t c = chunks_of(grads[i]);
        if (c == 0) continue;
        if (l.count == kClipTensors || (int64_t)chunks + c > INT32_MAX) flush();
        l.g[l.count] = grads[i].g;
        l.out[l.count] = grads[i].out;
        l.n_dt[l.count] = (uint64_t)grads[i].n * 4 + grads[i].dt;
        l.first[l.count++] = chunks;
        chunks += (uint32_t)c;
    }
    flush();
}

int check_list(const char* what, const rq_grad* grads, int64_t count, bool outs) {
    using rq::fail;
    if (count < 0) return fail(RQ_EINVAL, "%s: negative count", what);
    if (count > 0 && !grads) return fail(RQ_EINVAL, "%s: NULL list", what);
    for (int64_t i = 0; i < count; ++i) {
        const rq_grad& t = grads[i];
        if (!rq::valid_dt(t.dt)) return fail(RQ_EINVAL, "%s: tensor %lld has an unsupported dtype", what, (long long)i);
        if (t.n < 0) return fail(RQ_EINVAL, "%s: tensor %lld has a negative size", what, (long long)i);
        if (chunks_of(t) > INT32_MAX)
            return fail(RQ_EINVAL, "%s: tensor %lld has more than 2^43 bytes", what, (long long)i);
        if (t.n > 0 && (!t.g || (outs && !t.out)))
            return fail(RQ_EINVAL, "%s: NULL pointer (tensor %lld)", what, (long long)i);
        const uintptr_t m = t.dt == RQ_F32 ? 3 : 1;
        if (t.n > 0 && (((uintptr_t)t.g | (outs ? (uintptr_t)t.out : 0)) & m))
            return fail(RQ_EALIGN, "%s: tensor %lld is not aligned to its elements", what, (long long)i);
    }
    return RQ_OK;
}

int64_t partials(const rq_grad* grads, int64_t count) {
    int64_t parts = 0;
    for_lists(grads, count, [&](const ClipList&, uint32_t chunks) {
        parts += std::min<int64_t>(chunks, kNormBlocks);
    });
    return parts;
}

int check_work(const char* what, const float* norm, const void* workspace, int64_t bytes, int64_t parts) {
    if (!norm) return rq::fail(RQ_EINVAL, "%s: NULL norm", what);
    if ((uintptr_t)norm & 3) return rq::fail(RQ_EALIGN, "%s: norm must be 4-byte aligned", what);
    if (parts > INT32_MAX) return rq::fail(RQ_EINVAL, "%s: too many tensors", what);
    if (parts > 0 && (!workspace || bytes < parts * 8))
        return rq::fail(RQ_EINVAL, "%s: needs a workspace of %lld bytes", what, (long long)(parts * 8));
    if ((uintptr_t)workspace & 15) return rq::fail(RQ_EALIGN, "%s: the workspace must be 16-byte aligned", what);
    return RQ_OK;
}

// What a list's scaling launches may run side by side.  Blocks of one launch run in
// any order, so an output must not be written twice, and not before another
// tensor that shares its memory has been read.
struct Scaling {
    bool as_listed = true;       // every entry once, all together
    std::vector<rq_grad> early;  // otherwise: entries without repeats whose outputs no other entry reads,
    std::vector<rq_grad> late;   // and then those that others read
};

int64_t bytes_of(const rq_grad& t) { return t.n * (t.dt == RQ_F32 ? 4 : 2); }

// The outputs by address, each with the entry that writes it.  The same tensor listed
// again is one output; other outputs that share memory have no sound order.
int order_scaling(const char* what, const rq_grad* grads, int64_t count, Scaling& plan) {
    struct Span {
        uintptr_t b, e;
        int64_t i;
    };
    const auto out_of = [&](int64_t i) {
        const uintptr_t b = (uintptr_t)grads[i].out;
        return Span{b, b + (uintptr_t)bytes_of(grads[i]), i};
    };
    // Most lists need no order: outputs in ascending order, and gradients that are
    // scaled in place or lie outside all outputs.
    bool sorted = true;
    uintptr_t end = 0, out_lo = UINTPTR_MAX, g_lo = UINTPTR_MAX, g_hi = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (grads[i].n == 0) continue;
        const Span o = out_of(i);
        sorted = sorted && o.b >= end;
        end = std::max(end, o.e);
        out_lo = std::min(out_lo, o.b);
        if (grads[i].g == grads[i].out) continue;
        g_lo = std::min(g_lo, (uintptr_t)grads[i].g);
        g_hi = std::max(g_hi, (uintptr_t)grads[i].g + (uintptr_t)bytes_of(grads[i]));
    }
    const bool apart = g_lo >= end || g_hi <= out_lo;  // also where every entry is in place
    if (sorted && apart) return RQ_OK;

    std::vector<Span> outs;
    outs.reserve((size_t)count);
    for (int64_t i = 0; i < count; ++i)
        if (grads[i].n > 0) outs.push_back(out_of(i));
    const auto before = [](const Span& a, const Span& b) { return a.b != b.b ? a.b < b.b : a.i < b.i; };
    // gradients are often allocated from the last parameter to the first; 288 tensors in no order sort in 7 us
    if (!sorted && outs.front().b > outs.back().b) std::reverse(outs.begin(), outs.end());
    if (!std::is_sorted(outs.begin(), outs.end(), before)) std::sort(outs.begin(), outs.end(), before);
    std::vector<uint8_t> again;  // entries that repeat another one
    size_t kept = 0;
    for (const Span& o : outs) {
        if (kept > 0 && o.b < outs[kept - 1].e) {
            const rq_grad &t = grads[o.i], &u = grads[outs[kept - 1].i];
            if (t.out != u.out || t.g != u.g || t.n != u.n || t.dt != u.dt)
                return rq::fail(RQ_EINVAL, "%s: the outputs of tensors %lld and %lld overlap", what,
                                (long long)outs[kept - 1].i, (long long)o.i);
            if (again.empty()) again.assign((size_t)count, 0);
            again[o.i] = 1;
        } else {
            outs[kept++] = o;
        }
    }
    outs.resize(kept);

    std::vector<uint8_t> late;  // entries whose output another entry reads
    if (!apart) {
        std::vector<std::pair<int64_t, int64_t>> reads;  // (entry, the entry whose output it reads)
        auto o = outs.begin();  // the first output that ends past the gradient: mostly the last one's or the next
        for (int64_t i = 0; i < count; ++i) {
            if (grads[i].n == 0 || grads[i].g == grads[i].out) continue;  // in place: no other output is there
            const uintptr_t b = (uintptr_t)grads[i].g, e = b + (uintptr_t)bytes_of(grads[i]);
            const bool here = (o == outs.begin() || o[-1].e <= b) && (o == outs.end() || b < o->e);
            const bool next = !here && o != outs.end() && o->e <= b && (o + 1 == outs.end() || b < o[1].e);
            if (next) ++o;
            else if (!here)
                o = std::upper_bound(outs.begin(), outs.end(), b, [](uintptr_t at, const Span& s) { return at < s.e; });
            for (auto w = o; w != outs.end() && w->b < e; ++w) {
                if (late.empty()) late.assign((size_t)count, 0);
                late[w->i] = 1;
                reads.emplace_back(i, w->i);
            }
        }
        for (const auto& [reader, writer] : reads)
            if (late[reader])
                return rq::fail(RQ_EINVAL, "%s: tensor %lld and the output of tensor %lld overlap", what,
                                (long long)reader, (long long)writer);
    }
    if (again.empty() && late.empty()) return RQ_OK;
    plan.as_listed = false;
    for (int64_t i = 0; i < count; ++i) {
        if (!again.empty() && again[i]) continue;
        (!late.empty() && late[i] ? plan.late : plan.early).push_back(grads[i]);
    }
    return RQ_OK;
}

hipError_t launch_squares(const rq_grad* grads, int64_t count, double* part, hipStream_t s) {
    int64_t at = 0;
    for_lists(grads, count, [&](const ClipList& l, uint32_t chunks) {
        const int blocks = (int)std::min<int64_t>(chunks, kNormBlocks);
        grad_squares_kernel<<<blocks, kBlock, 0, s>>>(l, chunks, part + at);
        at += blocks;
    });
    return hipGetLastError();
}

}  // namespace

extern "C" {

int64_t rq_grad_norm_workspace_bytes(const rq_grad* grads, int64_t count) {
    if (int rc = check_list("rq_grad_norm_workspace_bytes", grads, count, false)) return rc;
    rq::ok();
    return partials(grads, count) * 8;
}

int rq_grad_norm(const rq_grad* grads, int64_t count, float* norm, void* workspace,
                 int64_t workspace_bytes, void* stream) {
    if (int rc = check_list("rq_grad_norm", grads, count, false)) return rc;
    const int64_t parts = partials(grads, count);
    if (int rc = check_work("rq_grad_norm", norm, workspace, workspace_bytes, parts)) return rc;
    hipStream_t s = (hipStream_t)stream;
    hipError_t e = launch_squares(grads, count, (double*)workspace, s);
    if (e == hipSuccess) {
        grad_norm_kernel<<<1, kBlock, 0, s>>>((const double*)workspace, (int)parts, norm);
        e = hipGetLastError();
    }
    return rq::launch_status(e, "rq_grad_norm");
}

int rq_clip_grads(const rq_grad* grads, int64_t count, float max_norm, float eps, float* norm,
                  void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check_list("rq_clip_grads", grads, count, true)) return rc;
    if (!(max_norm >= 0.f) || !(eps >= 0.f))
        return rq::fail(RQ_EINVAL, "rq_clip_grads: max_norm and eps must not be negative");
    Scaling plan;
    try {  // host memory for lists whose entries share theirs
        if (int rc = order_scaling("rq_clip_grads", grads, count, plan)) return rc;
    } catch (...) {
        return rq::fail(RQ_ELAUNCH, "rq_clip_grads: out of host memory");
    }
    const int64_t parts = partials(grads, count);
    if (int rc = check_work("rq_clip_grads", norm, workspace, workspace_bytes, parts)) return rc;
    hipStream_t s = (hipStream_t)stream;
    const double* part = (const double*)workspace;
    hipError_t e = launch_squares(grads, count, (double*)workspace, s);
    // every scaling block adds up the partial sums itself, unless they are many (or none)
    const bool known = parts == 0 || parts > kSumInPlace;
    if (e == hipSuccess && known) grad_norm_kernel<<<1, kBlock, 0, s>>>(part, (int)parts, norm);
    if (e == hipSuccess) {
        float* first = norm;  // one block of the first launch writes it
        const auto scale = [&](const ClipList& l, uint32_t chunks) {
            const int blocks = (int)std::min<int64_t>(chunks, 2 * kNormBlocks);
            grad_scale_kernel<<<blocks, kBlock, 0, s>>>(l, chunks, part, (int)parts, max_norm, eps, first, known);
            if (!known) first = nullptr;
        };
        if (plan.as_listed) {
            for_lists(grads, count, scale);
        } else {
            for_lists(plan.early.data(), (int64_t)plan.early.size(), scale);
            for_lists(plan.late.data(), (int64_t)plan.late.size(), scale);
        }
        e = hipGetLastError();
    }
    return rq::launch_status(e, "rq_clip_grads");
}

}  // extern "C"
