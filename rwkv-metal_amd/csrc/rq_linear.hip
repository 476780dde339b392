// rq_linear.hip -- dense products with bias, activation and residual in the
// output stage, and the products of their backward pass.
//
//   forward  y = act(x w^T + bias) + residual     A = x [m, k],   B = w [n, k]
//   dx       dx = g w                             A = g [m, n],   B = w transposed
//   dw       dw = g^T x                           A = g and B = x, both transposed
//
// v = x w^T + bias stays in the fp32 accumulators: activation, slope and residual
// are applied there and the result is rounded once.
#include <algorithm>

#include "rq_act.h"
#include "rq_common.h"
#include "rq_linear.h"
#include "rq_vec.h"

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_p;

// Row stride of the partial sums of a split contraction.
__host__ RQ_DEV int64_t part_ld(int64_t n) { return (n + 3) & ~3ll; }

template <int N_>
struct Count {
    static constexpr int N = N_;
};

// ------------------------------------------------------------ output stage

// Four or eight neighbouring elements at any element-aligned address: rows of odd
// width take the same wide accesses (global memory allows them unaligned).
struct __attribute__((packed, aligned(2))) Bytes8 {
    uint32_t w[2];
};

RQ_DEV f32x4_t load4(const void* p, int dt, int64_t at) {
    if (dt == RQ_F32) {
        float f[4];
        load_vec<RQ_F32>((const uint8_t*)p + at * 4, f);
        return f32x4_t{f[0], f[1], f[2], f[3]};
    }
    const Bytes8 v = *(const Bytes8*)((const uint16_t*)p + at);
    if (dt == RQ_BF16)
        return f32x4_t{__uint_as_float(v.w[0] << 16), __uint_as_float(v.w[0] & 0xffff0000u),
                       __uint_as_float(v.w[1] << 16), __uint_as_float(v.w[1] & 0xffff0000u)};
    return f32x4_t{f16_bits_to_f32(v.w[0] & 0xffffu), f16_bits_to_f32(v.w[0] >> 16),
                   f16_bits_to_f32(v.w[1] & 0xffffu), f16_bits_to_f32(v.w[1] >> 16)};
}

RQ_DEV void store4(void* p, int dt, int64_t at, const f32x4_t& v) {
    if (dt == RQ_F32) {
        const float f[4] = {v[0], v[1], v[2], v[3]};
        store_vec<RQ_F32>((uint8_t*)p + at * 4, f);
    } else {
        Bytes8 b;
        if (dt == RQ_BF16) {
            b.w[0] = pack_bf16x2(v[0], v[1]);
            b.w[1] = pack_bf16x2(v[2], v[3]);
        } else {
            b.w[0] = f32_to_f16_bits(v[0]) | (f32_to_f16_bits(v[1]) << 16);
            b.w[1] = f32_to_f16_bits(v[2]) | (f32_to_f16_bits(v[3]) << 16);
        }
        *(Bytes8*)((uint16_t*)p + at) = b;
    }
}

// y and slope of the four outputs (i, j) .. (i, j + 3) whose sums are v.
RQ_DEV void store_out(const rq::DenseArgs& g, int64_t i, int64_t j, f32x4_t v) {
    const int64_t at = i * g.n + j;
    if (j >= g.n) return;
    const bool whole = j + 4 <= g.n;
    if (g.bias) {
        if (whole) {
            v += load4(g.bias, g.dt, j);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < g.n) v[e] += load_dt(g.bias, g.dt, j + e);
        }
    }
    if (g.slope) {
        const f32x4_t s = act_slope4(g.act, v);
        if (g.slope_kind != RQ_SLOPE_F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < g.n) ((uint16_t*)g.slope)[at + e] = (uint16_t)slope16_bits(g.act, s[e]);
        } else if (whole) {
            store4(g.slope, RQ_F32, at, s);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j + e < g.n) ((float*)g.slope)[at + e] = s[e];
        }
    }
    v = act_value4(g.act, v);
    if (whole) {
        if (g.residual) v += load4(g.residual, g.y_dt, at);
        store4(g.y, g.y_dt, at, v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (j + e >= g.n) break;
            if (g.residual) v[e] += load_dt(g.residual, g.y_dt, at + e);
            store_dt(g.y, g.y_dt, at + e, v[e]);
        }
    }
}

// ------------------------------------------------------------------- tiles

// BM x BN outputs a block of four waves, WM x WN of them a wave, in stages of 128
// bytes of contraction (64 16-bit elements, 32 fp32 ones) with two stages in LDS.
//
// A stage is two MFMA steps ks.  Its fragments are read one step ahead into a
// second set of registers, so all reads of stage s are done in the middle of its
// products.  There stands the only barrier of a stage: behind it stage s + 1 has
// been written by every wave and stage s will not be read again, so stage s + 2
// goes from registers (loaded one stage earlier) into its place, and the first
// fragments of stage s + 1 are read, under the products of the second step.
//
// LDS: rows of 128 bytes whose 16-byte chunks are XORed with a key of the row. An
// operand with a contiguous contraction has an output a row, and eight lanes
// reading one chunk of eight rows hit all banks.  A transposed operand keeps its
// memory order: blocks of 128 bytes of outputs, a contraction element a row.  Its
// 16-bit fragments come from the transposing read: 32 lanes take 32 bytes each of
// rows 0 - 3 and 8 - 11 at a time, eight different eighths of the 256 bytes of
// banks by the key ((row % 4) ^ (row / 8 % 2)) * 2 (without its second term
// SQ_LDS_BANK_CONFLICT counts half of all LDS cycles).  32-bit ones come from
// single-word reads.
//
// The first MFMA operand is B, so that a lane holds four neighbouring outputs of a row.
constexpr int kBlock = 256;

template <int DT>
RQ_DEV f32x4_t mma(const u32x4_t& a, const u32x4_t& b, f32x4_t c) {
    if constexpr (DT == RQ_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                       __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else if constexpr (DT == RQ_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a),
                                                      __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    } else {  // 16 contraction elements, four a lane: element e of every lane in one instruction
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
        return c;
    }
}

// One operand's side of a tile: R rows (outputs) of 128 bytes of contraction.
template <int DT, bool T, int R>
struct Side {
    static constexpr int ES = kSize<DT>;
    static constexpr int E = kVec<DT>;        // elements of a 16-byte chunk
    static constexpr int BK = 128 / ES;       // contraction elements of a stage
    static constexpr int LD = R * 8 / kBlock; // chunks a thread stages
    static constexpr int BYTES = R * 128;

    static RQ_DEV int key(int row) {
        if constexpr (!T) return row & 7;
        else if constexpr (ES == 2) return ((row & 3) ^ (row >> 3 & 1)) << 1;
        else return row & 4;
    }

    const uint8_t* p;   // the stage's first element of the tile
    int64_t step;       // bytes from stage to stage
    uint32_t off[LD];   // of this thread's chunks, rows clamped to the last one inside
    int rows;           // outputs of the tile inside the matrix
    int64_t ld;
    bool cut;           // a transposed tile whose last chunk is cut: every stage is checked
    bool wide;          // rows hold 16 bytes at least

    RQ_DEV void init(const void* base, int64_t ld_, int64_t r0, int64_t all, int64_t k0) {
        ld = ld_;
        rows = (int)(all - r0 < R ? all - r0 : R);
        p = (const uint8_t*)base + (T ? k0 * ld + r0 : r0 * ld + k0) * ES;
        step = (T ? BK * ld : (int64_t)BK) * ES;
        cut = T && rows < R && rows % E != 0;
        wide = (T ? all : ld) >= E;
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            int r, c;
            place(i, r, c);
            if constexpr (T) off[i] = (uint32_t)(c * ld * ES) + (r < rows ? r : 0) * ES;
            else off[i] = (uint32_t)((r < rows ? r : rows - 1) * ld * ES) + c * ES;
        }
    }
    // chunk i of this thread: its first row (output) and contraction element
    static RQ_DEV void place(int i, int& r, int& c) {
        const int q = threadIdx.x + kBlock * i;
        if constexpr (T) {
            c = (q >> 3) % BK;
            r = q / (8 * BK) * BK + ((q & 7) ^ key(c)) * E;
        } else {
            r = q >> 3;
            c = ((q & 7) ^ key(r)) * E;
        }
    }
    // the chunks of the next stage, of which `left` contraction elements are inside
    RQ_DEV void load(u32x4_t* v, int64_t left) {
        if (left >= BK && !cut) {
#pragma unroll
            for (int i = 0; i < LD; ++i) {
                const Bytes16 b = *(const Bytes16*)(p + off[i]);
                v[i] = u32x4_t{b.w[0], b.w[1], b.w[2], b.w[3]};
            }
        } else {
            checked(v, left);
        }
        p += step;
    }
    // A chunk cut by the end of its row: the row's last 16 bytes, shifted down.
    RQ_DEV void checked(u32x4_t* v, int64_t left) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            int r, c;
            place(i, r, c);
            v[i] = u32x4_t{0u, 0u, 0u, 0u};
            const int64_t in64 = T ? (c < left ? rows - r : 0) : (r < rows ? left - c : 0);
            const int in = in64 < E ? (int)in64 : E;
            if (in <= 0) continue;
            if (wide) {
                const Bytes16 b = *(const Bytes16*)(p + off[i] - (E - in) * ES);
                v[i] = down(u32x4_t{b.w[0], b.w[1], b.w[2], b.w[3]}, E - in);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (e >= in) break;
                    if constexpr (ES == 4) v[i][e] = ((const uint32_t*)(p + off[i]))[e];
                    else v[i][e >> 1] |= (uint32_t)((const uint16_t*)(p + off[i]))[e] << (16 * (e & 1));
                }
            }
        }
    }
    // 128 bits shifted down by n < E elements, zeros from above
    static RQ_DEV u32x4_t down(u32x4_t v, int n) {
        if constexpr (ES == 2) {
            if (n & 1)
                v = u32x4_t{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16),
                            __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
            n >>= 1;
        }
        if (n & 1) v = u32x4_t{v[1], v[2], v[3], 0u};
        if (n & 2) v = u32x4_t{v[2], v[3], 0u, 0u};
        return v;
    }
    static RQ_DEV void put(uint8_t* lds, const u32x4_t* v) {
#pragma unroll
        for (int i = 0; i < LD; ++i) *(u32x4_t*)(lds + (threadIdx.x + kBlock * i) * 16) = v[i];
    }
    // fragment t (16 outputs from r0 + 16 t on) of step ks; r0 is a multiple of W
    template <int W>
    static RQ_DEV u32x4_t frag(const uint8_t* lds, int r0, int t, int ks) {
        const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
        if constexpr (!T) {
            return *(const u32x4_t*)(lds + (r0 + lr) * 128 + (((ks * 4 + lg) ^ (lr & 7)) << 4) + 16 * 128 * t);
        } else {
            // the block of BK outputs, and where in it
            const int in = (W % BK ? r0 % BK : 0) + 16 * t;
            const uint8_t* l = lds + r0 / BK * (BK * 128) + in / BK * (BK * 128);
            if constexpr (ES == 2) {
                const int col = in % BK + 4 * (lr & 3);
                const int at = (8 * lg + (lr >> 2)) * 128 + (((col >> 3) ^ key(8 * lg + (lr >> 2))) << 4) + (lr & 1) * 8;
                s16x4_t h[2];
#pragma unroll
                for (int v = 0; v < 2; ++v)
                    h[v] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_p)(l + at + (32 * ks + 4 * v) * 128));
                return __builtin_bit_cast(u32x4_t, s16x8_t{h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1],
                                                           h[1][2], h[1][3]});
            } else {
                const int col = in % BK + lr;
                const int at = 4 * lg * 128 + (((col >> 2) ^ key(4 * lg)) << 4) + (lr & 3) * 4;
                u32x4_t v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = *(const uint32_t*)(l + at + (16 * ks + e) * 128);
                return v;
            }
        }
    }
};

// Rows of a wave's tile that its part of LDS takes at a time in the output stage.
template <int WM, int WN>
constexpr int kOutRows = WM * WN > 4096 ? 8192 / WN : WM;

// Eight neighbouring elements of type DT, or fp32.
template <int DT>
RQ_DEV void load8(const void* p, bool f32, int64_t at, f32x4_t& lo, f32x4_t& hi) {
    float f[8];
    if (DT == RQ_F32 || f32) {
        load_vec<RQ_F32>((const uint8_t*)p + at * 4, f);
        load_vec<RQ_F32>((const uint8_t*)p + at * 4 + 16, f + 4);
    } else {
        load_vec<DT>((const uint8_t*)p + at * 2, f);
    }
    lo = f32x4_t{f[0], f[1], f[2], f[3]};
    hi = f32x4_t{f[4], f[5], f[6], f[7]};
}

template <int DT>
RQ_DEV void store8(void* p, bool f32, int64_t at, const f32x4_t& lo, const f32x4_t& hi) {
    const float f[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    if (DT == RQ_F32 || f32) {
        store_vec<RQ_F32>((uint8_t*)p + at * 4, f);
        store_vec<RQ_F32>((uint8_t*)p + at * 4 + 16, f + 4);
    } else {
        store_vec<DT>((uint8_t*)p + at * 2, f);
    }
}

// `rows` rows of a wave's tile from LDS (row r at own + r * P) to row i0 + r, columns
// j .. j + 7 of this lane (all inside); every 64 / LPR-th row from r0 on is this lane's.
// BATCH rows at a time, their loads together: one wave to a SIMD runs this in
// the large tiles, and every wait is felt.
template <int DT, int ACT, int P, int LPR, int BATCH>
RQ_DEV void out_rows(const rq::DenseArgs& g, const float* own, int64_t i0, int64_t j, int rows) {
    constexpr int STEP = 64 / LPR;
    const int r0 = (threadIdx.x & 63) / LPR;
    const bool y32 = g.y_dt == RQ_F32, res = g.residual != nullptr, slope = g.slope != nullptr;
    f32x4_t blo = {0.f, 0.f, 0.f, 0.f}, bhi = blo;
    if (g.bias) load8<DT>(g.bias, false, j, blo, bhi);
    const float* src = own + r0 * P + ((threadIdx.x & 63) % LPR) * 8;
    int64_t at = (i0 + r0) * g.n + j;
    const int64_t step = STEP * g.n;
    for (int r = r0; r < rows; r += BATCH * STEP) {
        f32x4_t lo[BATCH], hi[BATCH], rl[BATCH], rh[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            // rows of LDS are there for the whole tile, rows of memory are not
            lo[u] = ((const f32x4_t*)(src + u * STEP * P))[0];
            hi[u] = ((const f32x4_t*)(src + u * STEP * P))[1];
            if (res && r + u * STEP < rows) load8<DT>(g.residual, y32, at + u * step, rl[u], rh[u]);
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            if (r + u * STEP >= rows) break;
            lo[u] += blo;
            hi[u] += bhi;
            if (ACT != RQ_ACT_NONE && slope) {
                f32x4_t sl, sh;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sl[e] = act_slope(ACT, lo[u][e]);
                    sh[e] = act_slope(ACT, hi[u][e]);
                }
                if (DT == RQ_BF16 && g.slope_kind != RQ_SLOPE_F32) {
                    u32x4_t w;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[e] = slope16_pair(ACT, sl[2 * e], sl[2 * e + 1]);
                        w[e + 2] = slope16_pair(ACT, sh[2 * e], sh[2 * e + 1]);
                    }
                    *(Bytes16*)((uint16_t*)g.slope + at + u * step) = Bytes16{{w[0], w[1], w[2], w[3]}};
                } else {
                    store8<RQ_F32>(g.slope, true, at + u * step, sl, sh);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lo[u][e] = act_value(ACT, lo[u][e]);
                hi[u][e] = act_value(ACT, hi[u][e]);
            }
            if (res) {
                lo[u] += rl[u];
                hi[u] += rh[u];
            }
            store8<DT>(g.y, y32, at + u * step, lo[u], hi[u]);
        }
        src += BATCH * STEP * P;
        at += BATCH * step;
    }
}

// The output stage of a wave's tile at (i0, j0), through its own part of LDS: eight
// neighbouring outputs a lane, whole rows of the tile a store.
template <int DT, int MT, int NT>
RQ_DEV void tile_out(const rq::DenseArgs& g, const f32x4_t (&acc)[MT][NT], float* own, int64_t i0, int64_t j0,
                     float* part) {
    constexpr int WM = MT * 16, WN = NT * 16;
    constexpr int ROWS = kOutRows<WM, WN>, P = WN + 4, LPR = WN / 8;
    // four rows together: the same with a residual, tanh 181 us instead of 171 (4096 x 2048 x 8192 with slopes)
    constexpr int BATCH = 2;
    static_assert(ROWS % (BATCH * (64 / LPR)) == 0, "rows of LDS are read in whole batches");
    static_assert(WM / ROWS <= 2, "");
    const int lane = threadIdx.x & 63;
    auto put = [&](auto half) {
        constexpr int p0 = decltype(half)::N * (ROWS / 16);
#pragma unroll
        for (int p = 0; p < ROWS / 16; ++p)
#pragma unroll
            for (int q = 0; q < NT; ++q)
                *(f32x4_t*)(own + (16 * p + (lane & 15)) * P + 16 * q + 4 * (lane >> 4)) = acc[p0 + p][q];
    };
#pragma unroll 1
    for (int h = 0; h < WM / ROWS; ++h) {  // one copy of the code below for both halves
        if (h == 0) put(Count<0>{});
        else put(Count<WM / ROWS - 1>{});
        __builtin_amdgcn_wave_barrier();
        const int64_t ib = i0 + h * ROWS;
        const int rows = (int)(g.m - ib < ROWS ? g.m - ib : ROWS);
        const int64_t j = j0 + lane % LPR * 8;
        if (part) {  // rows of whole 16-byte lines
            const int64_t ld = part_ld(g.n);
            float* o = part + ((int64_t)blockIdx.y * g.m + ib) * ld + j;
            if (j < ld) {
#pragma unroll 4
                for (int r = lane / LPR; r < rows; r += 64 / LPR) {
                    const float* v = own + r * P + lane % LPR * 8;
                    *(f32x4_t*)(o + r * ld) = *(const f32x4_t*)v;
                    if (j + 4 < ld) *(f32x4_t*)(o + r * ld + 4) = *(const f32x4_t*)(v + 4);
                }
            }
        } else if (j + 8 > g.n) {  // the lane at the end of rows that are not whole eights
            for (int r = lane / LPR; r < rows && j < g.n; r += 64 / LPR) {
                const float* v = own + r * P + lane % LPR * 8;
                store_out(g, ib + r, j, *(const f32x4_t*)v);
                store_out(g, ib + r, j + 4, *(const f32x4_t*)(v + 4));
            }
        } else {
            switch (g.act) {
#define RQ_OUT(A) \
    case A: out_rows<DT, A, P, LPR, BATCH>(g, own, ib, j, rows); break;
                RQ_OUT(RQ_ACT_NONE)
                RQ_OUT(RQ_ACT_RELU)
                RQ_OUT(RQ_ACT_RELU2)
                RQ_OUT(RQ_ACT_SILU)
                RQ_OUT(RQ_ACT_GELU)
                RQ_OUT(RQ_ACT_SIGMOID)
                RQ_OUT(RQ_ACT_TANH)
#undef RQ_OUT
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The tile of a block.  Blocks b, b + 8, .. run on one XCD: each gets a run of
// neighbouring tiles, columns of kTall tiles at a time, so that its L2 holds the
// rows and columns they share.
constexpr int kTall = 8;
RQ_DEV void tile_of(int64_t b, int64_t tiles, int64_t ti, int64_t tj, int64_t& i, int64_t& j) {
    const int64_t x = b & 7, per = tiles >> 3, more = tiles & 7;
    int64_t t = x * per + (x < more ? x : more) + (b >> 3);
    const int64_t band = t / (kTall * tj), r = t - band * kTall * tj;
    const int64_t high = ti - band * kTall < kTall ? ti - band * kTall : kTall;
    i = band * kTall + r % high;
    j = r / high;
}

template <int DT, bool AT, bool BT, int BM, int BN, int WM, int WN, int NB = 2>
constexpr int kTileLds = std::max(NB * (Side<DT, AT, BM>::BYTES + Side<DT, BT, BN>::BYTES),
                                  kBlock / 64 * kOutRows<WM, WN> * (WN + 4) * 4);

template <int DT, bool AT, bool BT, int BM, int BN, int WM, int WN, int OCC>
__global__ __launch_bounds__(kBlock, OCC) void dense_tile(const rq::DenseArgs g, int64_t kper, float* part) {
    typedef Side<DT, AT, BM> SA;
    typedef Side<DT, BT, BN> SB;
    constexpr int MT = WM / 16, NT = WN / 16;
    static_assert((BM / WM) * (BN / WN) == kBlock / 64, "");
    constexpr int STAGE = SA::BYTES + SB::BYTES;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = (wave / (BN / WN)) * WM, wn = (wave % (BN / WN)) * WN;
    const int64_t ti = (g.m + BM - 1) / BM, tj = (g.n + BN - 1) / BN;
    int64_t i0, j0;
    tile_of(blockIdx.x, ti * tj, ti, tj, i0, j0);
    i0 *= BM;
    j0 *= BN;
    const int64_t k0 = (int64_t)blockIdx.y * kper;
    const int64_t k1 = k0 + kper < g.k ? k0 + kper : g.k;
    const int stages = (int)((k1 - k0 + SA::BK - 1) / SA::BK);
    SA a;
    SB b;
    a.init(g.a, g.lda, i0, g.m, k0);
    b.init(g.b, g.ldb, j0, g.n, k0);

    f32x4_t acc[MT][NT];
#pragma unroll
    for (int p = 0; p < MT; ++p)
#pragma unroll
        for (int q = 0; q < NT; ++q) acc[p][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};

    u32x4_t va[SA::LD], vb[SB::LD];      // a stage on its way to LDS
    u32x4_t fa[2][MT], fb[2][NT];
    auto load = [&](int s) {
        const int64_t left = k1 - k0 - (int64_t)s * SA::BK;
        a.load(va, left);
        b.load(vb, left);
    };
    auto put = [&](int s) {
        SA::put(lds + (s & 1) * STAGE, va);
        SB::put(lds + (s & 1) * STAGE + SA::BYTES, vb);
    };
    auto read = [&](int s, int ks) {
        const uint8_t* l = lds + (s & 1) * STAGE;
#pragma unroll
        for (int p = 0; p < MT; ++p) fa[ks][p] = SA::template frag<WM>(l, wm, p, ks);
#pragma unroll
        for (int q = 0; q < NT; ++q) fb[ks][q] = SB::template frag<WN>(l + SA::BYTES, wn, q, ks);
    };
    auto products = [&](int ks) {
#pragma unroll
        for (int p = 0; p < MT; ++p)
#pragma unroll
            for (int q = 0; q < NT; ++q) acc[p][q] = mma<DT>(fb[ks][q], fa[ks][p], acc[p][q]);
    };

    if (stages > 0) {
        load(0);
        put(0);
        if (stages > 1) {
            load(1);
            put(1);
        }
        if (stages > 2) load(2);
        __syncthreads();
        read(0, 0);
        for (int s = 0; s < stages; ++s) {
            read(s, 1);
            products(0);
            __syncthreads();  // stage s is read, stage s + 1 is written
            if (s + 2 < stages) {
                put(s);       // stage s + 2
                if (s + 3 < stages) load(s + 3);
            }
            if (s + 1 < stages) read(s + 1, 0);
            products(1);
        }
    }

    __syncthreads();
    tile_out<DT, MT, NT>(g, acc, (float*)lds + wave * kOutRows<WM, WN> * (WN + 4), i0 + wm, j0 + wn, part);
}

// ---------------------------------------------------- tiles, straight to LDS

// The same tiles with stages that go from global memory to LDS without passing
// registers (1 KB a wave and instruction, lane l's 16 bytes at 16 l), for operands
// whose rows are whole 16-byte lines.  LDS places are those of Side: the
// XOR is applied to the address each lane reads from.  Every share of the
// contraction holds at least one whole stage: the loop fetches whole stages only.
__device__ const uint4 kZero16 = {0u, 0u, 0u, 0u};

template <int KS_, bool FETCH_>
struct Step {
    static constexpr int KS = KS_;
    static constexpr bool FETCH = FETCH_;
};

// m0 is written for the loads and named as clobbered; that it is a register the
// compiler reserves, which it warns of, is why it has to be named.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int DT, bool T, int R>
struct Direct : Side<DT, T, R> {
    typedef Side<DT, T, R> S;
    // chunk i of a wave to LDS at `lds` (the wave's first byte of it)
    RQ_DEV void fetch(uint32_t lds, int i) const {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :: "s"(lds), "v"(this->off[i]), "s"(this->p) : "memory", "m0");
    }
    // the same of a stage `left` contraction elements long: what is past them comes from a line of zeros
    RQ_DEV void fetch_part(uint32_t lds, int i, int left) const {
        int r, c;
        S::place(i, r, c);
        const uint8_t* q = c < left ? this->p + this->off[i] : (const uint8_t*)&kZero16;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                     :: "s"(lds), "v"(q) : "memory", "m0");
    }
};
#pragma clang diagnostic pop

// mma with its sums in the accumulation registers, where the 256 x 256 tile's fill
// all 256: left to itself the compiler moves them between the two files, up to
// eight moves a product (8192^3 bf16: forward 955 us with its moves, 741 without;
// dw 2272 against 759).
template <int DT>
RQ_DEV void mma_acc(const u32x4_t& a, const u32x4_t& b, f32x4_t& c) {
    if constexpr (DT == RQ_BF16) asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

// NB stages fit LDS: a stage is fetched NB - 1 stages ahead of its products.  bf16,
// forward / dx / dw: 256 x 256 tiles 8192^3 741 / 750 / 759 us (1483 - 1449 TFLOP/s; a
// product's stage of 2048 matrix cycles takes 1.02 us where the card is cool, and a
// round of tiles 12 us beside its stages); two 128 x 128 blocks a CU 921 / 980 /
// 993.  64 x 64 tiles of 4 stages, 333 x 2560 x 2560: 12.3 us (6 stages 12.8, 2 20.9).
template <int DT, bool AT, bool BT, int BM, int BN, int WM, int WN, int OCC, int NB>
__global__ __launch_bounds__(kBlock, OCC) void dense_direct(const rq::DenseArgs g, int64_t kper, float* part) {
    typedef Direct<DT, AT, BM> SA;
    typedef Direct<DT, BT, BN> SB;
    constexpr int MT = WM / 16, NT = WN / 16, BK = SA::BK;
    constexpr int STAGE = SA::BYTES + SB::BYTES;
    constexpr int LD = SA::LD + SB::LD;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave / (BN / WN)) * WM, wn = (wave % (BN / WN)) * WN;
    const int64_t ti = (g.m + BM - 1) / BM, tj = (g.n + BN - 1) / BN;
    int64_t i0, j0;
    tile_of(blockIdx.x, ti * tj, ti, tj, i0, j0);
    i0 *= BM;
    j0 *= BN;
    const int64_t k0 = (int64_t)blockIdx.y * kper;
    const int64_t k1 = k0 + kper < g.k ? k0 + kper : g.k;
    const int stages = (int)((k1 - k0 + BK - 1) / BK);
    // a stage that is not whole comes first (the order of a contraction is free),
    // so that the loop has whole ones only
    const int whole = (int)((k1 - k0) / BK), rest = (int)((k1 - k0) % BK);
    SA a;
    SB b;
    a.init(g.a, g.lda, i0, g.m, k0);
    b.init(g.b, g.ldb, j0, g.n, k0);

    f32x4_t acc[MT][NT];
#pragma unroll
    for (int p = 0; p < MT; ++p)
#pragma unroll
        for (int q = 0; q < NT; ++q) acc[p][q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    u32x4_t fa[2][MT], fb[2][NT];

    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds + wave * 1024;
    // load i of the next stage, into buffer u
    auto fetch = [&](int u, int i) {
        const uint32_t at = base + u * STAGE;
        if (i < SA::LD) a.fetch(at + i * (kBlock * 16), i);
        else b.fetch(at + SA::BYTES + (i - SA::LD) * (kBlock * 16), i - SA::LD);
    };
    auto next = [&] {
        a.p += a.step;
        b.p += b.step;
    };
    auto read = [&](int u, int ks, int i) {  // fragment i of step ks
        const uint8_t* l = lds + u * STAGE;
        if (i < NT) fb[ks][i] = SB::template frag<WN>(l + SA::BYTES, wn, i, ks);
        else fa[ks][i - NT] = SA::template frag<WM>(l, wm, i - NT, ks);
    };
    constexpr int FR = MT + NT;
    // The products of step KS, row by row of fragments, between them the reads of the
    // other step's fragments from buffer u and, FETCH, the next stage's loads into buffer v.
    auto products = [&](auto step, int u, int v) {
        constexpr int KS = decltype(step)::KS;
        constexpr bool FETCH = decltype(step)::FETCH;
        constexpr int N = MT * NT, EACH = N / FR > 1 ? N / FR / 2 : 1;  // products between two reads
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int p = x / NT, q = x % NT;
            if constexpr (MT * NT == 64) mma_acc<DT>(fb[KS][q], fa[KS][p], acc[p][q]);
            else acc[p][q] = mma<DT>(fb[KS][q], fa[KS][p], acc[p][q]);
            if (x % EACH == 0) {  // behind the first product: it waits for its own operands only
                const int i = x / EACH;
                if (FETCH && i < LD) fetch(v, i);
                if (i < FR) read(u, 1 - KS, i);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // own loads but the last STAGES' have landed, own reads are done; then everybody's
    auto sync = [&](auto stages_left) {
        constexpr int V = decltype(stages_left)::N * LD;
        static_assert(V < 64, "vmcnt");
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(V) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };

    if (stages > 0) {
        // Past the last stage the loads below and in the loop repeat it and the
        // reads take what is there: nothing uses either, and every pass is the
        // same code with the same counts.
        int ahead = 0;  // stages fetched
        auto move = [&] {
            if (++ahead < stages) next();
        };
        if (rest) {
            const uint8_t *pa = a.p, *pb = b.p;
            a.p += whole * a.step;
            b.p += whole * b.step;
#pragma unroll
            for (int i = 0; i < SA::LD; ++i) a.fetch_part(base + i * (kBlock * 16), i, rest);
#pragma unroll
            for (int i = 0; i < SB::LD; ++i) b.fetch_part(base + SA::BYTES + i * (kBlock * 16), i, rest);
            a.p = pa;
            b.p = pb;
            ++ahead;
        } else {
#pragma unroll
            for (int i = 0; i < LD; ++i) fetch(0, i);
            move();
        }
#pragma unroll
        for (int v = 1; v < NB; ++v) {
#pragma unroll
            for (int i = 0; i < LD; ++i) fetch(v, i);
            move();
        }
        sync(Count<NB - 1>{});
#pragma unroll
        for (int i = 0; i < FR; ++i) read(0, 0, i);
        int u = 0;
        for (int s = 0; s < stages; ++s) {
            products(Step<0, false>{}, u, 0);
            sync(Count<NB - 2>{});
            const int v = u;
            u = u + 1 < NB ? u + 1 : 0;
            products(Step<1, true>{}, u, v);
            move();
        }
        sync(Count<0>{});
        if constexpr (MT * NT == 64) {
            // the compiler knows no latency of the last products: a wait, and every sum
            // passes through an asm behind it, so that none is read before
            asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
            for (int p = 0; p < MT; ++p)
#pragma unroll
                for (int q = 0; q < NT; ++q) asm volatile("" : "+a"(acc[p][q]));
        }
    }
    tile_out<DT, MT, NT>(g, acc, (float*)lds + wave * kOutRows<WM, WN> * (WN + 4), i0 + wm, j0 + wn, part);
}

// ---------------------------------------------------------------- few rows

// Products of a few rows (decode): 16 weight rows and MT * 16 rows of A a block, whose
// W waves take equal shares of the contraction.  Bound by reading the weights once: they go
// from memory straight into the matrix instruction's first operand (a lane has 16
// bytes of a row, four lanes 64 contiguous ones), kAhead steps in flight, and A's
// rows, which every block reads, come from the caches.  The waves' sums are added
// in order through LDS.  5 rows against [8192, 2048] bf16: 8.1 us, 4.2 TB/s.
constexpr int kAhead = 8;

template <int DT, int MT, int W>
__global__ __launch_bounds__(64 * W) void dense_few(const rq::DenseArgs g) {
    constexpr int ES = kSize<DT>, E = kVec<DT>, SK = 4 * E;
    __shared__ f32x4_t red[W][MT][64];
    const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t j0 = (int64_t)blockIdx.x * 16;
    const int whole = (int)(g.k / SK), rest = (int)(g.k % SK);
    const int per = (whole + W - 1) / W;
    const int s0 = wave * per, s1 = s0 + per < whole ? s0 + per : whole;
    const uint8_t* b = (const uint8_t*)g.b + ((j0 + lr < g.n ? j0 + lr : g.n - 1) * g.ldb + lg * E) * ES;
    const uint8_t* a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        a[t] = (const uint8_t*)g.a + ((16 * t + lr < g.m ? 16 * t + lr : g.m - 1) * g.lda + lg * E) * ES;
    f32x4_t acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto chunk = [](const uint8_t* p) {
        const Bytes16 v = *(const Bytes16*)p;
        return u32x4_t{v.w[0], v.w[1], v.w[2], v.w[3]};
    };
    auto steps = [&](int s, auto count) {
        constexpr int N = decltype(count)::N;
        u32x4_t fb[N], fa[N][MT];
#pragma unroll
        for (int u = 0; u < N; ++u) fb[u] = chunk(b + (int64_t)(s + u) * SK * ES);
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) fa[u][t] = chunk(a[t] + (int64_t)(s + u) * SK * ES);
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = mma<DT>(fb[u], fa[u][t], acc[t]);
    };
    int s = s0;
    for (; s + kAhead <= s1; s += kAhead) steps(s, Count<kAhead>{});
    for (; s + 2 <= s1; s += 2) steps(s, Count<2>{});
    if (s < s1) steps(s, Count<1>{});
    if (rest && wave == W - 1) {  // the last, partial step, element by element
        auto cut = [&](const uint8_t* p) {
            u32x4_t v = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (lg * E + e >= rest) break;
                if constexpr (ES == 4) v[e] = ((const uint32_t*)p)[e];
                else v[e >> 1] |= (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1));
            }
            return v;
        };
        const u32x4_t fb = cut(b + (int64_t)whole * SK * ES);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = mma<DT>(fb, cut(a[t] + (int64_t)whole * SK * ES), acc[t]);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) red[wave][t][lane] = acc[t];
    __syncthreads();
    if (wave < MT) {
        f32x4_t v = red[0][wave][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += red[w][wave][lane];
        const int64_t i = 16 * wave + lr;
        if (i < g.m) store_out(g, i, j0 + 4 * lg, v);
    }
}

// The output stage of a product whose contraction was split: the partial sums of
// four outputs in order, then store_out.
__global__ __launch_bounds__(kBlock) void dense_join(const rq::DenseArgs g, const float* __restrict__ part,
                                                     int splits) {
    const int64_t ld = part_ld(g.n), quads = ld / 4;
    const int64_t q = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    const int64_t i = q / quads, j = (q - i * quads) * 4;
    if (i >= g.m) return;
    const float* p = part + i * ld + j;
    f32x4_t v = *(const f32x4_t*)p;
    for (int s = 1; s < splits; ++s) v += *(const f32x4_t*)(p + s * g.m * ld);
    store_out(g, i, j, v);
}

enum Form { kDirect256, kDirect128, kDeep128, kDirect128x64, kDirect64, kDeep64, kTile128, kTile64, kFew };

struct Plan {
    Form form;
    int splits;
    int64_t kper;  // contraction elements of a share
};

// What a product costs in each form, in us: a start, and for every tile on the
// fullest of 256 CUs an amount of its own and an amount a stage, which is less where
// several tiles of a CU run together, and more (`turned`) with two transposed
// operands, half of that with one; a split adds its partial sums' traffic and a
// launch.  The numbers are least squares over 2600 timings on an MI355X (operands
// beyond the L2 caches): 100 sizes of m 1 - 4096, k and n 64 - 8192 in all three
// orders, every form with up to 16 shares.  The fit is 12 % off (odd widths 21 %,
// fp32 7 %), and what it chooses 2 % slower than the best of each size (4 %, 1 %).
struct Cost {
    int bm, bn, together;
    float tile, turned, stage[4];  // stage: of 1 .. `together` tiles running together, all of them
};
constexpr float kStart = 3.f, kJoin = 2.9f, kJoinBytes = 6e6f;  // us, us, bytes a us
constexpr Cost kCost[kFew] = {
    {256, 256, 1, 7.2f, 1.21f, {1.02f}},
    {128, 128, 2, 1.9f, 1.13f, {0.47f, 0.68f}},
    {128, 128, 1, 2.6f, 1.33f, {0.36f}},
    {128, 64, 2, 1.5f, 1.29f, {0.23f, 0.40f}},
    {64, 64, 4, 0.7f, 1.06f, {0.34f, 0.41f, 0.46f, 0.48f}},
    {64, 64, 2, 1.2f, 1.36f, {0.17f, 0.25f}},
    {128, 128, 2, 2.1f, 2.44f, {0.79f, 0.83f}},  // the staged tiles on rows of odd width
    {64, 64, 2, 0.34f, 1.87f, {0.45f, 0.46f}},
};
// fp32, 32 elements a stage: bound by the fp32 matrix instruction
constexpr Cost kCost32[2] = {
    {128, 128, 2, 2.6f, 1.11f, {2.1f, 3.9f}},
    {64, 64, 2, 0.9f, 1.21f, {0.65f, 1.0f}},
};

float cost_of(const Cost& c, const rq::DenseArgs& a, int bk, int splits) {
    const int64_t tiles = ((a.m + c.bm - 1) / c.bm) * ((a.n + c.bn - 1) / c.bn) * splits;
    const float stages = (float)((a.k / splits + bk - 1) / bk);
    const int64_t most = (tiles + 255) / 256;  // on one CU
    const int rest = (int)(most % c.together);
    const float all = (float)(most / c.together) * c.stage[c.together - 1] + (rest ? c.stage[rest - 1] : 0.f);
    float t = kStart + most * c.tile + stages * all * (1.f + (c.turned - 1.f) * (a.a_t + a.b_t) / 2);
    if (splits > 1) t += kJoin + (float)a.m * a.n * splits * 8.f / kJoinBytes;
    return t;
}

// kFew: 1024 weights of 256 blocks' rows
float cost_few(const rq::DenseArgs& a) {
    const int mt = a.m <= 16 ? 1 : a.m <= 32 ? 2 : 4;
    const float blocks = (float)((a.n + 15) / 16), k = (float)a.k * (a.dt == RQ_F32 ? 4 : 2) / 2048.f;
    const float per = a.dt == RQ_F32 ? 1.34f * mt : a.k % 8 ? 2.25f + 0.53f * mt : 0.33f + 0.61f * mt;
    return 3.9f + per * std::max(1.f, blocks / 256.f) * k;
}

Plan plan_of(const rq::DenseArgs& a) {
    const bool f32 = a.dt == RQ_F32;
    const int bk = f32 ? 32 : 64;
    // rows of whole 16-byte lines, and a whole stage in the contraction
    const bool direct = !f32 && (a.lda | a.ldb) % 8 == 0 && a.k >= 64;
    Plan p{kTile64, 1, a.k};
    float best = 1e30f;
    if (!a.a_t && !a.b_t && a.m <= 64) {
        p.form = kFew;
        best = cost_few(a);
    }
    for (int f = direct ? kDirect256 : kTile128; f <= (direct ? kDeep64 : kTile64); ++f) {
        const Cost& c = f32 ? kCost32[f - kTile128] : kCost[f];
        for (int splits = 1; splits <= 32; splits *= 2) {
            const int64_t per = ((a.k + splits - 1) / splits + bk - 1) / bk * bk;
            // shares of two stages at least, and a whole one in the last
            if (splits > 1 && (per < 2 * bk || a.k - (splits - 1) * per < bk)) break;
            const float t = cost_of(c, a, bk, splits);
            if (t < best) {
                best = t;
                p = {(Form)f, splits, splits > 1 ? per : a.k};
            }
        }
    }
    return p;
}

template <class K>
hipError_t launch_lds(K* kernel, const rq::DenseArgs& a, const Plan& p, int bm, int bn, int lds, float* part,
                      hipStream_t s) {
    const int64_t tiles = ((a.m + bm - 1) / bm) * ((a.n + bn - 1) / bn);
    if (tiles * kBlock > UINT32_MAX) return hipErrorInvalidConfiguration;  // threads of a grid dimension
    kernel<<<dim3((unsigned)tiles, (unsigned)p.splits), kBlock, lds, s>>>(a, p.kper, part);
    return hipGetLastError();
}

// More than 64 KB of LDS has to be asked for.  Asked on every launch: a record of
// which device has been asked would have to be kept for each kernel.
template <class K>
hipError_t allow_lds(K* kernel, int lds) {
    return lds <= 64 * 1024 ? hipSuccess
                            : hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <int DT, bool AT, bool BT, int BM, int BN, int WM, int WN, int OCC, int NB>
hipError_t launch_tile(const rq::DenseArgs& a, const Plan& p, float* part, hipStream_t s) {
    constexpr int lds = kTileLds<DT, AT, BT, BM, BN, WM, WN, NB ? NB : 2>;
    if constexpr (NB > 0) {
        auto* kernel = dense_direct<DT, AT, BT, BM, BN, WM, WN, OCC, NB>;
        if (hipError_t e = allow_lds(kernel, lds); e != hipSuccess) return e;
        return launch_lds(kernel, a, p, BM, BN, lds, part, s);
    } else {
        auto* kernel = dense_tile<DT, AT, BT, BM, BN, WM, WN, OCC>;
        if (hipError_t e = allow_lds(kernel, lds); e != hipSuccess) return e;
        return launch_lds(kernel, a, p, BM, BN, lds, part, s);
    }
}

template <int DT>
hipError_t launch_few(const rq::DenseArgs& a, hipStream_t s) {
    const unsigned blocks = (unsigned)((a.n + 15) / 16);
    if (a.m <= 16) dense_few<DT, 1, 8><<<blocks, 512, 0, s>>>(a);
    else if (a.m <= 32) dense_few<DT, 2, 8><<<blocks, 512, 0, s>>>(a);
    else dense_few<DT, 4, 8><<<blocks, 512, 0, s>>>(a);
    return hipGetLastError();
}

template <int DT, bool AT, bool BT>
hipError_t launch_as(const rq::DenseArgs& a, const Plan& p, float* part, hipStream_t s) {
    if constexpr (DT != RQ_F32) {
        if (p.form == kDirect256) return launch_tile<DT, AT, BT, 256, 256, 128, 128, 1, 2>(a, p, part, s);
        if (p.form == kDirect128) return launch_tile<DT, AT, BT, 128, 128, 64, 64, 2, 2>(a, p, part, s);
        if (p.form == kDeep128) return launch_tile<DT, AT, BT, 128, 128, 64, 64, 2, 4>(a, p, part, s);
        if (p.form == kDirect128x64) return launch_tile<DT, AT, BT, 128, 64, 64, 32, 2, 3>(a, p, part, s);
        if (p.form == kDeep64) return launch_tile<DT, AT, BT, 64, 64, 32, 32, 2, 4>(a, p, part, s);
        if (p.form == kDirect64) return launch_tile<DT, AT, BT, 64, 64, 32, 32, 4, 2>(a, p, part, s);
    }
    if constexpr (!AT && !BT) {
        if (p.form == kFew) return launch_few<DT>(a, s);
    }
    if (p.form == kTile64) return launch_tile<DT, AT, BT, 64, 64, 32, 32, 2, 0>(a, p, part, s);
    return launch_tile<DT, AT, BT, 128, 128, 64, 64, 2, 0>(a, p, part, s);
}

}  // namespace

namespace rq {

int64_t dense_workspace_bytes(const DenseArgs& a) {
    const Plan p = plan_of(a);
    return p.splits > 1 ? p.splits * a.m * part_ld(a.n) * 4 : 0;
}

hipError_t launch_dense(const DenseArgs& a, void* workspace, hipStream_t stream) {
    const Plan p = plan_of(a);
    float* part = p.splits > 1 ? (float*)workspace : nullptr;
    hipError_t e = hipErrorInvalidValue;
    RQ_DISPATCH_DT(a.dt, DT, {
        e = a.a_t ? launch_as<DT, true, true>(a, p, part, stream)
                  : a.b_t ? launch_as<DT, false, true>(a, p, part, stream) : launch_as<DT, false, false>(a, p, part, stream);
    });
    if (e == hipSuccess && part) {
        const int64_t quads = a.m * (part_ld(a.n) / 4);
        dense_join<<<(unsigned)((quads + kBlock - 1) / kBlock), kBlock, 0, stream>>>(a, part, p.splits);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace rq
