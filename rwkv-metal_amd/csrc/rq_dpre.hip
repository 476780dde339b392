// rq_dpre.hip -- the start of the dense products' backward pass: the gradient of
// the sums in front of the activation, and the bias gradient.
//
//   g[i, j] = T(dy[i, j] * act'(v[i, j]))       db[j] = T(sum over i of dy act'(v))
//
// g is rounded to the operands' type T because the 16-bit matrix instructions of
// the two products take it so: their results are off by 1.41 roundings of T instead of
// one (bf16 0.0024 against 0.0017 of their norm).  g in two parts of T would
// double both products, which take 227 of the 420 us of a 4096 x 2048 x 8192 step;
// float32 operands keep all of g.  db adds the unrounded products.
// Memory bound: dy and the slopes in, g out, one pass; the column sums ride along
// in registers, from the unrounded products.  [4096, 8192] bf16 with 16-bit slopes,
// 201 MB: 46 us, 4.4 TB/s (a copy reaches 5.1; blocks that walked down the rows of
// one column tile instead of along the columns took 51).
#include "rq_act.h"
#include "rq_linear.h"
#include "rq_vec.h"

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kRows = 8;                  // rows of one wave, all their loads in flight together
constexpr int kPart = kRows * kWaves;     // rows of one partial column sum
constexpr int kCols = 64 * 8;             // columns of a wave

// Elements [c, c + 8) of a row of `n`, 0 past its end.
template <int DT>
RQ_DEV void load8(const uint8_t* row, int64_t c, int64_t n, float* f) {
#pragma unroll
    for (int h = 0; h < 8; h += kVec<DT>) load_cols<DT>(row, c + h, n, f + h);
}

template <int DT>
RQ_DEV void store8(uint8_t* row, int64_t c, int64_t n, const float* f) {
#pragma unroll
    for (int h = 0; h < 8; h += kVec<DT>) store_cols<DT>(row, c + h, n, f + h);
}

// KIND: RQ_SLOPE_*.  SDT: the type the slopes (or y) are held in, -1 where act'(v) is 1.
// Neighbouring blocks take neighbouring columns of the same rows.
template <int DT, int YDT, int KIND, int SDT>
__global__ __launch_bounds__(kBlock) void dpre_kernel(const rq::DpreArgs a, uint32_t ctiles,
                                                      float* __restrict__ part) {
    __shared__ float red[kWaves][kCols];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t rtile = blockIdx.x / ctiles, ctile = blockIdx.x % ctiles;
    const int64_t c = (int64_t)ctile * kCols + lane * 8;
    const int64_t r0 = (int64_t)rtile * kPart + wave * kRows;
    const bool in = c < a.n;
    const uint8_t* dy = (const uint8_t*)a.dy;
    const uint8_t* sl = (const uint8_t*)a.slope;
    float f[kRows][8], s[SDT >= 0 ? kRows : 1][8];
    if (in) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (r0 + r >= a.m) break;
            load8<YDT>(dy + (r0 + r) * a.n * kSize<YDT>, c, a.n, f[r]);
            if constexpr (SDT >= 0) load8<SDT>(sl + (r0 + r) * a.n * kSize<SDT>, c, a.n, s[r]);
            if constexpr (KIND == RQ_SLOPE_BOUND16 || KIND == RQ_SLOPE_WIDE16) {  // read as bf16, which keeps the bits
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t b = __float_as_uint(s[r][j]) >> 16;
                    s[r][j] = KIND == RQ_SLOPE_WIDE16 ? wide16_value(b) : bound16_value(b);
                }
            }
        }
    }
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j] = 0.f;
    if (in) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (r0 + r >= a.m) break;
            if constexpr (SDT >= 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j) f[r][j] *= KIND == RQ_SLOPE_Y ? act_slope_of_y(a.act, s[r][j]) : s[r][j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += f[r][j];
            if (a.g) store8<DT>((uint8_t*)a.g + (r0 + r) * a.n * kSize<DT>, c, a.n, f[r]);
        }
    }
    if (!part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[wave][lane * 8 + j] = sum[j];
    __syncthreads();
    for (int j = threadIdx.x; j < kCols; j += kBlock) {
        const int64_t col = (int64_t)ctile * kCols + j;
        if (col >= a.n) break;
        float v = red[0][j];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += red[w][j];
        part[(int64_t)rtile * a.n + col] = v;
    }
}

// db[j] = the partial sums of column j in order: 64 columns a block, a wave to
// a quarter of them.
__global__ __launch_bounds__(kBlock) void colsum_kernel(const float* __restrict__ part, int64_t parts,
                                                        int64_t n, void* __restrict__ db, int dt) {
    __shared__ float red[kWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    const int64_t q = (parts + kWaves - 1) / kWaves;
    const int64_t r0 = wave * q, r1 = r0 + q < parts ? r0 + q : parts;
    float acc = 0.f;
    if (c < n) {
        for (int64_t r = r0; r < r1; r += 8) {
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = r + k < r1 ? part[(r + k) * n + c] : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc += f[k];
        }
    }
    red[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < n) {
        float v = red[0][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += red[w][lane];
        store_dt(db, dt, c, v);
    }
}

template <int DT, int YDT>
void launch_as(const rq::DpreArgs& a, float* part, int64_t parts, hipStream_t s) {
    const uint32_t ct = (uint32_t)((a.n + kCols - 1) / kCols);
    const uint32_t grid = (uint32_t)parts * ct;
    switch (a.slope_kind) {
        case RQ_SLOPE_Y: dpre_kernel<DT, YDT, RQ_SLOPE_Y, YDT><<<grid, kBlock, 0, s>>>(a, ct, part); break;
        case RQ_SLOPE_BOUND16: dpre_kernel<DT, YDT, RQ_SLOPE_BOUND16, RQ_BF16><<<grid, kBlock, 0, s>>>(a, ct, part); break;
        case RQ_SLOPE_F32: dpre_kernel<DT, YDT, RQ_SLOPE_F32, RQ_F32><<<grid, kBlock, 0, s>>>(a, ct, part); break;
        case RQ_SLOPE_WIDE16: dpre_kernel<DT, YDT, RQ_SLOPE_WIDE16, RQ_BF16><<<grid, kBlock, 0, s>>>(a, ct, part); break;
        default: dpre_kernel<DT, YDT, RQ_SLOPE_NONE, -1><<<grid, kBlock, 0, s>>>(a, ct, part); break;
    }
}

}  // namespace

namespace rq {

int64_t dpre_workspace_bytes(int64_t m, int64_t n) { return (m + kPart - 1) / kPart * n * 4; }

hipError_t launch_dpre(const DpreArgs& a, void* workspace, hipStream_t stream) {
    const int64_t parts = (a.m + kPart - 1) / kPart;
    float* part = a.db ? (float*)workspace : nullptr;
    if (parts > 0) {
        if (parts * ((a.n + kCols - 1) / kCols) * kBlock > UINT32_MAX) return hipErrorInvalidConfiguration;
        RQ_DISPATCH_DT(a.dt, DT, {
            if (a.y_dt == DT) launch_as<DT, DT>(a, part, parts, stream);
            else launch_as<DT, RQ_F32>(a, part, parts, stream);
        });
    }
    if (a.db) colsum_kernel<<<(unsigned)((a.n + 63) / 64), kBlock, 0, stream>>>(part, parts, a.n, a.db, a.dt);
    return hipGetLastError();
}

}  // namespace rq
