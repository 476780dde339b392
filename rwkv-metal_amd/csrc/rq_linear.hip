// rq_linear.hip -- dense products with bias, activation and residual in the
// output stage, and the products of their backward pass.
//
//   forward  y = act(x w^T + bias) + residual     A = x [m, k],   B = w [n, k]
//   dx       dx = g w                             A = g [m, n],   B = w transposed
//   dw       dw = g^T x                           A = g and B = x, both transposed
//
// v = x w^T + bias stays in the fp32 accumulators: activation, slope and residual
// are applied there and the result is rounded once.
#include "rq_act.h"
#include "rq_common.h"
#include "rq_linear.h"

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------ output stage

// y and slope of the four outputs (i, j) .. (i, j + 3) whose sums are v.
RQ_DEV void store_out(const rq::DenseArgs& g, int64_t i, int64_t j, const f32x4_t& v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (j + e >= g.n) break;
        const int64_t at = i * g.n + j + e;
        float u = v[e];
        if (g.bias) u += load_dt(g.bias, g.dt, j + e);
        if (g.slope) {
            const float s = act_slope(g.act, u);
            if (g.slope_kind == RQ_SLOPE_F16) ((uint16_t*)g.slope)[at] = (uint16_t)f32_to_f16_bits(s);
            else ((float*)g.slope)[at] = s;
        }
        float y = act_value(g.act, u);
        if (g.residual) y += load_dt(g.residual, g.y_dt, at);
        store_dt(g.y, g.y_dt, at, y);
    }
}

// ------------------------------------------------------------- plain tiles

// 64 x 64 outputs a block, a stage of 32 (16-bit) or 16 (fp32) contraction
// elements staged through LDS element by element with every index checked:
// any size, alignment and order.  Wave w computes 32 x 32 of them from four
// MFMA tiles.  The weights' side is the MFMA's first operand, so that a lane
// holds four neighbouring outputs of a row.
template <int DT>
struct Mma;
template <>
struct Mma<RQ_BF16> {
    typedef uint16_t elem;
    static constexpr int KS = 32;  // contraction elements of one instruction, 8 a lane
    static constexpr int E = 8;
    static RQ_DEV f32x4_t run(const elem* a, const elem* b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8_t*)a, *(const bf16x8_t*)b, c, 0, 0, 0);
    }
};
template <>
struct Mma<RQ_F16> {
    typedef uint16_t elem;
    static constexpr int KS = 32;
    static constexpr int E = 8;
    static RQ_DEV f32x4_t run(const elem* a, const elem* b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const f16x8_t*)a, *(const f16x8_t*)b, c, 0, 0, 0);
    }
};
template <>
struct Mma<RQ_F32> {
    typedef float elem;
    static constexpr int KS = 4;  // one a lane
    static constexpr int E = 1;
    static RQ_DEV f32x4_t run(const elem* a, const elem* b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(*a, *b, c, 0, 0, 0);
    }
};

constexpr int kBlock = 256;

template <int DT>
__global__ __launch_bounds__(kBlock) void dense_plain(const rq::DenseArgs g) {
    typedef Mma<DT> M;
    typedef typename M::elem elem;
    constexpr int BK = DT == RQ_F32 ? 16 : 32;
    constexpr int P = BK + 16 / (int)sizeof(elem);  // padded row
    __shared__ __attribute__((aligned(16))) elem as[64 * P];
    __shared__ __attribute__((aligned(16))) elem bs[64 * P];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t i0 = (int64_t)blockIdx.y * 64, j0 = (int64_t)blockIdx.x * 64;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    f32x4_t acc[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) acc[a][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto stage = [&](elem* s, const void* p, int64_t ld, bool t, int64_t r0, int64_t rows, int64_t c0) {
        for (int e = tid; e < 64 * BK; e += kBlock) {
            // neighbouring threads along the contiguous direction
            const int r = t ? e % 64 : e / BK, c = t ? e / 64 : e % BK;
            const bool in = r0 + r < rows && c0 + c < g.k;
            const int64_t at = t ? (c0 + c) * ld + r0 + r : (r0 + r) * ld + c0 + c;
            s[r * P + c] = in ? ((const elem*)p)[at] : (elem)0;
        }
    };
    for (int64_t c0 = 0; c0 < g.k; c0 += BK) {
        __syncthreads();
        stage(as, g.a, g.lda, g.a_t, i0, g.m, c0);
        stage(bs, g.b, g.ldb, g.b_t, j0, g.n, c0);
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < BK; ks += M::KS) {
            const int o = ks + (lane >> 4) * M::E;
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    acc[a][b] = M::run(bs + (wj + 16 * b + (lane & 15)) * P + o,
                                       as + (wi + 16 * a + (lane & 15)) * P + o, acc[a][b]);
        }
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t i = i0 + wi + 16 * a + (lane & 15);
            if (i < g.m) store_out(g, i, j0 + wj + 16 * b + 4 * (lane >> 4), acc[a][b]);
        }
}

}  // namespace

namespace rq {

int64_t dense_workspace_bytes(int64_t, int64_t, int64_t, int, bool, bool) { return 0; }

hipError_t launch_dense(const DenseArgs& a, void*, hipStream_t stream) {
    const dim3 grid((unsigned)((a.n + 63) / 64), (unsigned)((a.m + 63) / 64));
    RQ_DISPATCH_DT(a.dt, DT, dense_plain<DT><<<grid, kBlock, 0, stream>>>(a));
    return hipGetLastError();
}

}  // namespace rq
