// rq_embed.hip -- lookup of a dense embedding table with a factor on its rows,
// and the table's gradient by sorted tokens.
//
//   out[i, :]    = T(scale * table[idx[i], :])
//   dtable[v, :] = T(scale * sum over i with idx[i] == v of dout[i, :])
//
// Both are memory bound: the lookup moves 2 n D elements, the gradient reads n D
// and writes vocab D, nearly all of them zeros for a step's 4096 tokens against
// a vocabulary of 65536.
//
// The gradient takes three launches and no atomic on a sum, so that it gives the
// same bits on every run:
//   1. embed_sort_kernel: a stable counting sort of the tokens in ONE launch.
//      Block b of nb owns the tokens with id % nb == b (frequent ids are
//      neighbours in most vocabularies: a range of ids to a block would give one
//      block most of the tokens) and scans all n indices twice; wave w always
//      reads the w-th part of them in order, so that the counts (wave, id) of the
//      first scan give every wave its own places and the second scan needs no
//      barrier.  The rows of the block's ids that do not occur are cleared here.
//   2. embed_sum_kernel: equal shares of the sorted tokens, whatever their
//      distribution.  A token whose places lie in one share is written; the sum
//      of one that continues in a neighbouring share goes to a fp32 partial row.
//   3. embed_join_kernel: adds the partial rows of each such token in order.
// 4096 tokens against a [65536, 2048] bf16 table: 46 us (5.8 TB/s of cleared rows
// once the scan is through; a fill reaches 6.9), 13 and 4; the lookup 9.5.  30011
// tokens against [5003, 517] fp32: 24 (the scan of every index by every block), 22
// and 5.5.
#include <algorithm>

#include "rq_common.h"
#include "rq_error.h"
#include "rq_vec.h"
#include "../../include/rwkvq_train.h"

namespace {

RQ_DEV int64_t index_at(const void* idx, bool wide, int64_t i) {
    return wide ? ((const int64_t*)idx)[i] : (int64_t)((const int32_t*)idx)[i];
}

// ------------------------------------------------------------------ lookup

constexpr int kBlock = 256;
constexpr int kRowLoads = 4;  // 16-byte loads a lane has in flight
constexpr int64_t kLookupRows = 1 << 25;  // of one launch: a grid holds fewer than 2^32 threads, 64 of them a row

// A wave takes kRowLoads * 64 vectors of one row.
template <int DT>
__global__ __launch_bounds__(kBlock) void embed_kernel(const void* __restrict__ idx, bool wide,
                                                       int64_t n, const uint8_t* __restrict__ table,
                                                       int64_t vocab, int64_t dim, float scale,
                                                       uint8_t* __restrict__ out) {
    constexpr int V = kVec<DT>;
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
    if (i >= n) return;
    const int64_t c0 = ((int64_t)blockIdx.y * kRowLoads * 64 + lane) * V;
    const int64_t v = index_at(idx, wide, i);
    const bool in = v >= 0 && v < vocab;
    const uint8_t* src = table + (in ? v : 0) * dim * kSize<DT>;
    uint8_t* dst = out + i * dim * kSize<DT>;
    float f[kRowLoads][V];
    if (in) {
#pragma unroll
        for (int k = 0; k < kRowLoads; ++k)
            if (c0 + (int64_t)k * 64 * V < dim) load_cols<DT>(src, c0 + (int64_t)k * 64 * V, dim, f[k]);
    }
#pragma unroll
    for (int k = 0; k < kRowLoads; ++k) {
        const int64_t c = c0 + (int64_t)k * 64 * V;
        if (c >= dim) break;
#pragma unroll
        for (int j = 0; j < V; ++j) f[k][j] = in ? f[k][j] * scale : __builtin_nanf("");
        store_cols<DT>(dst, c, dim, f[k]);
    }
}

// ---------------------------------------------------------------- gradient

constexpr int kSortWaves = 16;
constexpr int kSortBlock = 64 * kSortWaves;
constexpr int kMinSortBlocks = 256;  // one for each CU; a power of two
constexpr int kMaxIds = 512;         // ids of one block: 16 waves * 512 counters of LDS, 32 KB
constexpr int kScan = 16;            // index loads of a lane in flight
constexpr int64_t kMaxVocab = 1 << 30;  // 2^21 sort blocks of 1024 threads: a grid holds fewer than 2^32
constexpr int kMaxShares = 1024;
constexpr int kMaxDim = 65535 * 256;  // blockIdx.y counts columns by 256 and more

struct SortPlan {
    int nb, ids;     // blocks, ids of a block
    int share;       // sorted tokens of one share, a multiple of 8
    int shares;
};

SortPlan sort_plan(int64_t n, int64_t vocab) {
    SortPlan p;
    p.nb = kMinSortBlocks;
    while ((vocab + p.nb - 1) / p.nb > kMaxIds) p.nb *= 2;
    p.ids = (int)((vocab + p.nb - 1) / p.nb);
    p.share = (int)((n + 8ll * kMaxShares - 1) / (8ll * kMaxShares)) * 8;
    if (p.share < 8) p.share = 8;
    p.shares = (int)((n + p.share - 1) / p.share);
    return p;
}

struct Work {
    int32_t* order;   // [n] position of the k-th token in sorted order
    int32_t* token;   // [n] its id
    int32_t* count;   // [1] tokens that take part
    float* part;      // [shares][2][part_ld(dim)] sums that continue from the share before / into the next
};

// Rows of whole 16-byte lines, also where the width is odd.
__host__ RQ_DEV int64_t part_ld(int64_t dim) { return (dim + 3) & ~3ll; }

size_t align16(size_t b) { return (b + 15) & ~(size_t)15; }

size_t work_bytes(int64_t n, int64_t dim, const SortPlan& p) {
    return 16 + 2 * align16((size_t)n * 4) + (size_t)p.shares * 2 * part_ld(dim) * 4;
}

Work work_of(void* ws, int64_t n) {
    Work w;
    uint8_t* b = (uint8_t*)ws;
    w.count = (int32_t*)b;
    w.order = (int32_t*)(b + 16);
    w.token = (int32_t*)(b + 16 + align16((size_t)n * 4));
    w.part = (float*)(b + 16 + 2 * align16((size_t)n * 4));
    return w;
}

template <int DT>
__global__ __launch_bounds__(kSortBlock) void embed_sort_kernel(const void* __restrict__ idx,
                                                                bool wide, int64_t n, int64_t vocab,
                                                                int64_t dim, int64_t padding, int nb_shift,
                                                                int ids, Work ws,
                                                                uint8_t* __restrict__ dtable) {
    __shared__ int32_t cnt[kSortWaves][kMaxIds];  // counts, then the next place, of (wave, id)
    __shared__ int32_t less[kSortWaves];          // tokens of lower blocks that the wave saw
    __shared__ int32_t wsum[kSortWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t me = blockIdx.x, mask = gridDim.x - 1;
    for (int i = tid; i < kSortWaves * kMaxIds; i += kSortBlock) (&cnt[0][0])[i] = 0;
    __syncthreads();

    const int64_t part = ((n + kSortWaves - 1) / kSortWaves + 63) & ~63ll;
    const int64_t lo = wave * part, hi = lo + part < n ? lo + part : n;
    // the ids of kScan * 64 places from i on, -1 where nothing takes part
    int32_t v[kScan];
    auto fetch = [&](int64_t i) {
        int64_t f[kScan];
#pragma unroll
        for (int k = 0; k < kScan; ++k) {
            const int64_t at = i + k * 64 + lane;
            f[k] = at < hi ? index_at(idx, wide, at) : -1;
        }
#pragma unroll
        for (int k = 0; k < kScan; ++k) v[k] = f[k] < 0 || f[k] >= vocab || f[k] == padding ? -1 : (int32_t)f[k];
    };
    int32_t below = 0;
    for (int64_t i = lo; i < hi; i += kScan * 64) {
        fetch(i);
#pragma unroll
        for (int k = 0; k < kScan; ++k) {
            const int32_t o = v[k] & mask;
            below += v[k] >= 0 && o < me;
            if (v[k] >= 0 && o == me) atomicAdd(&cnt[wave][v[k] >> nb_shift], 1);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o);
    if (lane == 0) less[wave] = below;
    __syncthreads();

    // places: all tokens of lower blocks, then this block's ids in order, each
    // id's waves in order.  Thread t scans id t.
    int32_t mine = 0;
    if (tid < ids)
        for (int w = 0; w < kSortWaves; ++w) mine += cnt[w][tid];
    int32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int32_t u = __shfl_up(incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    int32_t at = incl - mine, total = 0;
    for (int w = 0; w < kSortWaves; ++w) {
        at += less[w] + (w < wave ? wsum[w] : 0);
        total += less[w] + wsum[w];
    }
    if (me == mask && tid == 0) ws.count[0] = total;
    // the counts become each wave's first places; which ids do not occur is kept beside them
    __shared__ uint8_t absent[kMaxIds];
    if (tid < ids) {
        absent[tid] = mine == 0;
        for (int w = 0; w < kSortWaves; ++w) {
            const int32_t c = cnt[w][tid];
            cnt[w][tid] = at;
            at += c;
        }
    }
    __syncthreads();

    // clear the rows of absent ids, a wave to a row
    constexpr int V = kVec<DT>;
    float zero[V];
#pragma unroll
    for (int j = 0; j < V; ++j) zero[j] = 0.f;
    for (int s = wave; s < ids; s += kSortWaves) {
        const int64_t row = ((int64_t)s << nb_shift) + me;
        if (!absent[s] || row >= vocab) continue;
        uint8_t* dst = dtable + row * dim * kSize<DT>;
        for (int64_t c = lane * V; c < dim; c += 64 * V) store_cols<DT>(dst, c, dim, zero);
    }

    // the second scan: every wave places its own tokens in order
    volatile int32_t* next = cnt[wave];
    for (int64_t i = lo; i < hi; i += kScan * 64) {
        if (part > kScan * 64) fetch(i);  // else they are still there
#pragma unroll
        for (int k = 0; k < kScan; ++k) {
            const bool own = v[k] >= 0 && (v[k] & mask) == me;
            const int id = own ? (int)(v[k] >> nb_shift) : -1;
            uint64_t todo = __ballot(own);
            while (todo) {  // the distinct ids among these 64 places, lowest lane first
                const int lead = __ffsll((unsigned long long)todo) - 1;
                const int key = __shfl(id, lead);
                const uint64_t same = __ballot(id == key);
                const int32_t base = next[key];
                if (id == key) {
                    const int32_t place = base + __popcll(same & ((1ull << lane) - 1));
                    ws.order[place] = (int32_t)(i + k * 64 + lane);
                    ws.token[place] = v[k];
                }
                __builtin_amdgcn_wave_barrier();
                if (lane == lead) next[key] = base + __popcll(same);
                __builtin_amdgcn_wave_barrier();
                todo &= ~same;
            }
        }
    }
}

template <int V>
RQ_DEV void store_part(float* row, int64_t c, int64_t dim, const float* f) {
#pragma unroll
    for (int h = 0; h < V; h += 4)  // the row's padding takes what is past its end
        if (c + h < dim) *(f32x4_t*)(row + c + h) = f32x4_t{f[h], f[h + 1], f[h + 2], f[h + 3]};
}

// A wave takes a share of the sorted tokens and 64 vectors of columns (blockIdx.y).
template <int DT>
__global__ __launch_bounds__(kBlock) void embed_sum_kernel(const int32_t* __restrict__ count,
                                                           const int32_t* __restrict__ order,
                                                           const int32_t* __restrict__ token,
                                                           float* __restrict__ part, int share, int64_t dim,
                                                           const uint8_t* __restrict__ dout,
                                                           float scale, uint8_t* __restrict__ dtable) {
    constexpr int V = kVec<DT>;
    // the same for all lanes: tokens and rows are scalar loads, run ends scalar branches
    const int64_t s = (int64_t)blockIdx.x * (kBlock / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = count[0];
    const int64_t b = s * share;
    if (b >= n) return;
    const int64_t e = b + share < n ? b + share : n;
    const int64_t c = ((int64_t)blockIdx.y * 64 + (threadIdx.x & 63)) * V;
    const bool in = c < dim;
    bool open = b > 0 && token[b - 1] == token[b];  // the run began in an earlier share
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    int32_t id = token[b];
    for (int64_t i = b; i < e; i += 8) {
        float f[8][V];
        int32_t ids[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            ids[k] = -1;
            if (i + k < e) {
                ids[k] = token[i + k];
                const uint8_t* row = dout + (int64_t)order[i + k] * dim * kSize<DT>;
                if (in) load_cols<DT>(row, c, dim, f[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (ids[k] < 0) break;
            if (ids[k] != id) {  // the run of `id` ends inside the share
                if (in) {
                    if (open) {
                        store_part<V>(part + (s * 2) * part_ld(dim), c, dim, acc);
                    } else {
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[j] *= scale;
                        store_cols<DT>(dtable + (int64_t)id * dim * kSize<DT>, c, dim, acc);
                    }
                }
#pragma unroll
                for (int j = 0; j < V; ++j) acc[j] = 0.f;
                id = ids[k];
                open = false;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] += f[k][j];
        }
    }
    if (!in) return;
    const bool goes_on = e < n && token[e] == id;
    if (open || goes_on) {
        store_part<V>(part + (s * 2 + (open ? 0 : 1)) * part_ld(dim), c, dim, acc);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] *= scale;
        store_cols<DT>(dtable + (int64_t)id * dim * kSize<DT>, c, dim, acc);
    }
}

// Share blockIdx.x: the token whose run begins in it and goes on in the next.
// The four waves take a quarter of the partial rows each, in order.
template <int DT>
__global__ __launch_bounds__(kBlock) void embed_join_kernel(Work ws, int share, int64_t dim, float scale,
                                                            uint8_t* __restrict__ dtable) {
    constexpr int W = kBlock / 64;
    __shared__ f32x4_t red[W][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t s = blockIdx.x, ld = part_ld(dim);
    const int n = ws.count[0];
    const int64_t b = s * share, e = b + share;
    if (e >= n) return;
    const int32_t id = ws.token[e - 1];
    if (ws.token[e] != id) return;                                   // nothing goes on
    if (b > 0 && ws.token[b] == id && ws.token[b - 1] == id) return;  // it began earlier
    // the run's last share: the next one does not begin with its id (64 looked at together)
    int64_t last = s + 1;
    for (;;) {
        const int64_t at = (last + 1 + lane) * share;
        const uint64_t other = __ballot(at >= n || ws.token[at < n ? at : 0] != id);
        if (other) {
            last += __ffsll((unsigned long long)other) - 1;
            break;
        }
        last += 64;
    }
    const int64_t rows = last - s + 1;  // partial rows: this share's second, the others' first
    const int64_t q = (rows + W - 1) / W;
    const int64_t r0 = wave * q, r1 = r0 + q < rows ? r0 + q : rows;
    const int64_t c = ((int64_t)blockIdx.y * 64 + lane) * 4;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    if (c < dim) {
        for (int64_t r = r0; r < r1; r += 8) {
            f32x4_t f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t x = r + k;
                f[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (x < r1) f[k] = *(const f32x4_t*)(ws.part + ((s + x) * 2 + (x == 0 ? 1 : 0)) * ld + c);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) acc += f[k];
        }
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave == 0) {
        f32x4_t v = red[0][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < dim) store_dt(dtable + (int64_t)id * dim * kSize<DT>, DT, c + e, v[e] * scale);
    }
}

int check_embed(const char* what, const void* idx, int idx_bytes, int64_t n, const void* a, rq_dtype dt,
                int64_t vocab, int64_t dim, const void* b, bool need_b) {
    using rq::fail;
    if (idx_bytes != 4 && idx_bytes != 8)
        return fail(RQ_EINVAL, "%s: indices must have 4 or 8 bytes (got %d)", what, idx_bytes);
    if (!rq::valid_dt(dt)) return fail(RQ_EINVAL, "%s: unsupported dtype", what);
    if (n < 0 || vocab < 0 || dim < 0)
        return fail(RQ_EINVAL, "%s: negative size (n=%lld vocab=%lld dim=%lld)", what, (long long)n,
                    (long long)vocab, (long long)dim);
    if (dim > kMaxDim) return fail(RQ_EINVAL, "%s: dim is more than %d", what, kMaxDim);
    const uintptr_t m = dt == RQ_F32 ? 3 : 1;
    if (n > 0 && dim > 0) {
        if (!idx || !a) return fail(RQ_EINVAL, "%s: NULL pointer", what);
        if (((uintptr_t)idx & (idx_bytes - 1)) || ((uintptr_t)a & m))
            return fail(RQ_EALIGN, "%s: a pointer is not aligned to its elements", what);
    }
    if (need_b && !b) return fail(RQ_EINVAL, "%s: NULL pointer", what);
    if ((uintptr_t)b & m) return fail(RQ_EALIGN, "%s: a pointer is not aligned to its elements", what);
    return RQ_OK;
}

}  // namespace

extern "C" {

int rq_embed(const void* idx, int idx_bytes, int64_t n, const void* table, rq_dtype dt, int64_t vocab,
             int64_t dim, float scale, void* out, void* stream) {
    const bool some = n > 0 && dim > 0;
    // an empty table has no row to read: every index is outside it
    if (int rc = check_embed("rq_embed", idx, idx_bytes, n, vocab > 0 ? table : out, dt, vocab, dim, out, some))
        return rc;
    if (!some) return rq::ok();
    const int64_t per = (int64_t)kRowLoads * 64 * (dt == RQ_F32 ? 4 : 8);
    const int64_t segs = (dim + per - 1) / per;
    const bool wide = idx_bytes == 8;
    hipError_t e = hipSuccess;
    for (int64_t i = 0; i < n && e == hipSuccess; i += kLookupRows) {
        const int64_t count = std::min(n - i, kLookupRows), blocks = (count + kBlock / 64 - 1) / (kBlock / 64);
        RQ_DISPATCH_DT(dt, DT, embed_kernel<DT><<<dim3((unsigned)blocks, (unsigned)segs), kBlock, 0, (hipStream_t)stream>>>(
                                   (const uint8_t*)idx + i * idx_bytes, wide, count, (const uint8_t*)table, vocab, dim,
                                   scale, (uint8_t*)out + i * dim * kSize<DT>));
        e = hipGetLastError();
    }
    return rq::launch_status(e, "rq_embed");
}

int64_t rq_embed_grad_workspace_bytes(int64_t n, int64_t vocab, int64_t dim) {
    if (n < 0 || vocab < 0 || dim < 0)
        return rq::fail(RQ_EINVAL, "rq_embed_grad_workspace_bytes: negative size");
    if (n > INT32_MAX || vocab > kMaxVocab || dim > kMaxDim)
        return rq::fail(RQ_EINVAL, "rq_embed_grad_workspace_bytes: n must be below 2^31, vocab at most 2^30, dim at most %d",
                        kMaxDim);
    rq::ok();
    return vocab == 0 || dim == 0 ? 0 : (int64_t)work_bytes(n, dim, sort_plan(n, vocab));
}

int rq_embed_grad(const void* idx, int idx_bytes, int64_t n, const void* dout, rq_dtype dt, int64_t vocab,
                  int64_t dim, float scale, int64_t padding_idx, void* dtable, void* workspace,
                  int64_t workspace_bytes, void* stream) {
    if (int rc = check_embed("rq_embed_grad", idx, idx_bytes, n, dout, dt, vocab, dim, dtable, vocab > 0 && dim > 0))
        return rc;
    if (n > INT32_MAX || vocab > kMaxVocab)
        return rq::fail(RQ_EINVAL, "rq_embed_grad: n must be below 2^31, vocab at most 2^30");
    if (vocab == 0 || dim == 0) return rq::ok();
    const SortPlan p = sort_plan(n, vocab);
    if (!workspace || workspace_bytes < (int64_t)work_bytes(n, dim, p))
        return rq::fail(RQ_EINVAL, "rq_embed_grad: needs a workspace of %lld bytes", (long long)work_bytes(n, dim, p));
    if (!rq::aligned16(workspace)) return rq::fail(RQ_EALIGN, "rq_embed_grad: the workspace must be 16-byte aligned");
    const Work ws = work_of(workspace, n);
    const bool wide = idx_bytes == 8;
    hipStream_t s = (hipStream_t)stream;
    const int per = 64 * (dt == RQ_F32 ? 4 : 8);
    const int tiles = (int)((dim + per - 1) / per), jtiles = (int)((dim + 255) / 256);
    const unsigned sums = (p.shares + kBlock / 64 - 1) / (kBlock / 64);
    RQ_DISPATCH_DT(dt, DT, {
        embed_sort_kernel<DT><<<p.nb, kSortBlock, 0, s>>>(idx, wide, n, vocab, dim, padding_idx,
                                                          __builtin_ctz(p.nb), p.ids, ws, (uint8_t*)dtable);
        if (n > 0)
            embed_sum_kernel<DT><<<dim3(sums, tiles), kBlock, 0, s>>>(
                ws.count, ws.order, ws.token, ws.part, p.share, dim, (const uint8_t*)dout, scale, (uint8_t*)dtable);
        if (p.shares > 1)
            embed_join_kernel<DT><<<dim3(p.shares - 1, jtiles), kBlock, 0, s>>>(ws, p.share, dim, scale,
                                                                                (uint8_t*)dtable);
    });
    return rq::launch_status(hipGetLastError(), "rq_embed_grad");
}

}  // extern "C"
