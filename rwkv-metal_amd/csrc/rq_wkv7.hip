// rq_wkv7.hip -- the recurrence of RWKV-7's time mixing: over a sequence, its
// gradients, and one token.
//
//   d_t = exp(-exp(w_t)),  S_t = S_{t-1} diag(d_t) + (S_{t-1} a_t) b_t^T + v_t k_t^T,  y_t = S_t r_t
//
// The tokens are taken in chunks of 16.  With the running sums L of log d within a
// chunk (Lx without the token's own) and
//   A~ = a e^Lx   R~ = r e^L   B~ = b e^-L   K~ = k e^-L   B^ = b e^(Lend - L)   K^ = k e^(Lend - L)
//   Mab = strict(A~ B~^T)  Mak = strict(A~ K~^T)  Mrb = incl(R~ B~^T)  Mrk = incl(R~ K~^T)
// (strict: below the diagonal, incl: with it) a chunk is
//   SA = (1 - Mab)^-1 (A~ S^T + Mak V)      the rows S_{t-1} a_t
//   Y  = R~ S^T + Mrb SA + Mrk V
//   S' = S diag(e^Lend) + SA^T B^ + V^T K^
// and its adjoint, from dY and dS' backwards in time, has the same form:
//   dZ = (1 - Mab)^-T (B^ dS'^T + Mrb^T dY)
//   dV = K^ dS'^T + Mak^T dZ + Mrk^T dY
//   dS = dS' diag(e^Lend) + dZ^T A~ + dY^T R~
// so that one kernel runs both, the second with its tokens in reverse order.
// The other gradients take one chunk each and nothing of the others but the states:
//   dr = e^L (dY S + dMrb B~ + dMrk K~)             dMrb = incl(dY SA^T), dMrk = incl(dY V^T)
//   da = e^Lx (dZ S + dMab B~ + dMak K~)            dMab = strict(dZ SA^T), dMak = strict(dZ V^T)
//   db = e^-L (e^Lend SA dS' + dMrb^T R~ + dMab^T A~), dk alike with V, dMrk, dMak
//   dlog d_i = e^Lend sum_v S dS' + sum_{s<i} b_s e^(Lend-L_s) (SA dS')_s (and k, V)
//            + sum_{t>=i} r_t e^L_t (dY S)_t + sum_{t>i} a_t e^Lx_t (dZ S)_t
//            + sum_{s<i<=t} r_t e^(L_t-L_s) (dMrb_ts b_s + dMrk_ts k_s) + sum_{s<i<t} a_t e^(Lx_t-L_s) (dMab_ts b_s + dMak_ts k_s)
//
// All products are fp32 MFMAs (v_mfma_f32_16x16x4_f32): the state lives in fp32 and feeds itself for thousands of
// tokens, and the gradients of 16-bit tensors are rounded once, where they are stored.
//
// e^-L overflows where the decays of a chunk are strong.  Below 2^-32 over one
// chunk (RWKV-7's own decays reach 2^-14) a chunk's pair matrices are formed by VALU from
// e^(L_t - L_s), whose exponents are sums of the terms between s and t and never
// positive; that also serves decays of 0.
#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "rq_common.h"
#include "rq_error.h"
#include "rq_wkv7.h"

namespace {

using namespace rq;

constexpr int kHead = RQ_WKV7_HEAD;
constexpr int kChunk = RQ_WKV7_CHUNK;
constexpr int kRow = kHead + 4;  // LDS row of a [16, 64] array: lanes 16 rows apart meet in no bank
constexpr float kStrong = -32.f;  // log2 of the weakest product of decays that e^-L stands for
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLog2Log2e = 0.5287663729448977f;  // log2(log2 e)

RQ_DEV f32x4_t mfma4(float a, float b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Four steps of a contraction: lane (m = lane & 15, g = lane >> 4) holds A[m][4g + i] in
// a[i] and B[4g + i][m] in b[i]; c[i] is C[4g + i][m].  A result is the next product's B as it lies.
RQ_DEV f32x4_t mma16(const f32x4_t& a, const f32x4_t& b, f32x4_t c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = mfma4(a[i], b[i], c);
    return c;
}

// The same in all lanes, and known to be: branches on it are scalar.  MFMAs do not heed the execution mask, so that
// one in a branch that lanes are masked out of instead of jumping over it would still write.
RQ_DEV int wave_index() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

RQ_DEV float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// log2 of the decay: -exp(w) log2 e.
RQ_DEV float log2_decay(float w) { return -exp2_hw(fmaf(w, kLog2e, kLog2Log2e)); }

template <int CTRL>
RQ_DEV float dpp(float x) {  // 0 where the row of 16 lanes ends
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int kRowShl = 0x100, kRowShr = 0x110, kRowBcast = 0x150;

// Over the 16 lanes of a row, in time: forwards lane m is token m, backwards 15 - m.
template <bool REV>
RQ_DEV float upto(float x) {  // the sum of the tokens up to and with the lane's own
    constexpr int C = REV ? kRowShl : kRowShr;
    x += dpp<C + 1>(x);
    x += dpp<C + 2>(x);
    x += dpp<C + 4>(x);
    x += dpp<C + 8>(x);
    return x;
}
template <bool REV>
RQ_DEV float before(float x) {  // the previous token's value, 0 for the first
    return dpp<(REV ? kRowShl : kRowShr) + 1>(x);
}
template <bool REV>
RQ_DEV float before_or_one(float x) {  // 1 for the first
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(1.f), __float_as_int(x),
                                                      (REV ? kRowShl : kRowShr) + 1, 0xf, 0xf, false));
}
template <bool REV>
RQ_DEV float of_last(float x) {  // the last token's value
    return dpp<kRowBcast + (REV ? 0 : 15)>(x);
}

struct Span {
    int64_t start, len, chunk0;  // first token (row of the flattened batch), tokens, first chunk
    RQ_DEV int64_t chunks() const { return (len + kChunk - 1) / kChunk; }
};

// A boundary, the same in all lanes: addresses that follow from it are scalar.
RQ_DEV int64_t boundary(const WkvShape& s, int64_t n) {
    const int32_t v = __builtin_amdgcn_readfirstlane(s.cu[n]);
    return v < 0 ? 0 : (v > s.time ? s.time : v);
}

RQ_DEV Span span_of(const WkvShape& s, int64_t n) {
    if (!s.cu) return {n * s.time, s.time, n * ((s.time + kChunk - 1) / kChunk)};
    const int64_t from = boundary(s, n), to = boundary(s, n + 1);
    return {from, to > from ? to - from : 0, from / kChunk + n};
}

// ------------------------------------------------------- operands of a chunk

// The 16 channels from `ch` of a token's head, as they are stored.
template <int DT>
struct Raw {
    uint4 v[DT == RQ_F32 ? 4 : 2];
};
template <int DT>
RQ_DEV Raw<DT> load_raw(const void* p, int64_t at, bool there) {
    Raw<DT> r;
    const uint4* q = (const uint4*)((const uint8_t*)p + at * (DT == RQ_F32 ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (DT == RQ_F32 ? 4 : 2); ++i) r.v[i] = there ? q[i] : make_uint4(0, 0, 0, 0);
    return r;
}
template <int DT>
RQ_DEV void unpack_raw(const Raw<DT>& r, float* f) {
#pragma unroll
    for (int i = 0; i < (DT == RQ_F32 ? 4 : 2); ++i) {
        const uint32_t u[4] = {r.v[i].x, r.v[i].y, r.v[i].z, r.v[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == RQ_F32) {
                f[4 * i + j] = __uint_as_float(u[j]);
            } else {
                f[8 * i + 2 * j] = dt_traits<DT>::to_f32((uint16_t)(u[j] & 0xffffu));
                f[8 * i + 2 * j + 1] = dt_traits<DT>::to_f32((uint16_t)(u[j] >> 16));
            }
        }
    }
}

// What the block's waves hand on: the arrays of three chunks and the matrices of two.  Backwards
// the tensors change places: to_sa is B^, to_y K^, from_sa A~, from_x R~, and the matrices are transposed.
typedef float Rows[kChunk][kRow];
struct Arrays {
    Rows to_sa;    // A~
    Rows to_y;     // R~
    Rows from_sa;  // B^
    Rows from_x;   // K^
    Rows x;        // V
    float decay[kHead];  // e^Lend
};
struct Matrices {  // [lane] as A operands
    f32x4_t inv[64];   // (1 - Mab)^-1
    f32x4_t sa_x[64];  // Mak
    f32x4_t y_sa[64];  // Mrb
    f32x4_t y_x[64];   // Mrk
};
struct ScanLds {
    Arrays arrays[3];
    Rows inverse[2][2];  // B~ and K~
    Matrices matrices[2];
    Rows y[2];
    int strong[3][4];    // whether a wave's channels hold strong decays
};
// For the gradients of a chunk; rows of tokens are [15 - token].
struct GradRows {
    Rows d[4];   // dS', [value / 16][value % 16][key]
    Rows dz, v, sa;
    Rows io[5];  // log2 d, r, a, b and k; then, each in its place, dw, dr, da, db and dk
    float pairs[4][kChunk][kChunk + 4];  // dMab, dMak, dMrb and dMrk
};
struct ScanGradLds : ScanLds {
    GradRows grads;
};

// X^T of X = (1 - M)^-1 from m[i] = M^T[4g + i][lane & 15], nonzero above the diagonal:
// rows from the last, X^T[s] = e_s + sum over u > s of M^T[s, u] X^T[u], four at a time.
RQ_DEV f32x4_t unit_inverse(const f32x4_t& m, int lane) {
    const int g = lane >> 4, col = lane & 15;
    f32x4_t x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = 4 * g + i == col ? 1.f : 0.f;
#define RQ_STEP(U, I, V) x[I] = fmaf(dpp<kRowBcast + U>(mm[I]), V, x[I])
#define RQ_BLOCK(G)                                                                        \
    {                                                                                      \
        f32x4_t mm;                                                                        \
        _Pragma("unroll") for (int i = 0; i < 4; ++i) mm[i] = g == G ? m[i] : 0.f;         \
        RQ_STEP(4 * G + 3, 0, x[3]);                                                       \
        RQ_STEP(4 * G + 3, 1, x[3]);                                                       \
        RQ_STEP(4 * G + 3, 2, x[3]);                                                       \
        RQ_STEP(4 * G + 2, 0, x[2]);                                                       \
        RQ_STEP(4 * G + 2, 1, x[2]);                                                       \
        RQ_STEP(4 * G + 1, 0, x[1]);                                                       \
        if constexpr (G > 0) {                                                             \
            f32x4_t rows;                                                                  \
            _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                \
                rows[i] = __shfl(x[i], 16 * G + col);                                      \
                mm[i] = g < G ? m[i] : 0.f;                                                \
            }                                                                              \
            _Pragma("unroll") for (int i = 0; i < 4; ++i) {                                \
                RQ_STEP(4 * G + 3, i, rows[3]);                                            \
                RQ_STEP(4 * G + 2, i, rows[2]);                                            \
                RQ_STEP(4 * G + 1, i, rows[1]);                                            \
                RQ_STEP(4 * G + 0, i, rows[0]);                                            \
            }                                                                              \
        }                                                                                  \
    }
    RQ_BLOCK(3)
    RQ_BLOCK(2)
    RQ_BLOCK(1)
    RQ_BLOCK(0)
#undef RQ_BLOCK
#undef RQ_STEP
    return x;
}

// One pair matrix of a chunk whose decays are too strong for e^-L: entry (t, s) is the sum over
// the channels of late_t early_s e^(log d between them), the later token's own decay among them
// unless `strict`.  Rows are the source's tokens, columns the target's, as mma16 leaves them.
template <bool REV>
__device__ __attribute__((noinline)) f32x4_t strong_pairs(const float* late, const float* early, const float* g2,
                                                          bool strict, int lane) {
    const int g = lane >> 4, m = lane & 15;
    f32x4_t out = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < kChunk; ++s) {
        float sum = 0.f;
        const bool after = REV ? m < s : m > s;
        for (int c = 0; c < 16; ++c) {
            const float e = __shfl(early[c], 16 * g + s);
            float between = upto<REV>(after ? g2[c] : 0.f);
            if (strict) between = before<REV>(between);
            sum += late[c] * e * exp2_hw(between);
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if constexpr (REV) {  // the rows are the later tokens
            for (int i = 0; i < 4; ++i) {
                const float x = __shfl(sum, 4 * g + i);
                if (m == s) out[i] = x;
            }
        } else {
            for (int i = 0; i < 4; ++i)
                if (4 * g + i == s) out[i] = sum;
        }
    }
    return out;
}

// Four contiguous values as they are stored.
template <int DT>
struct __attribute__((aligned(DT == RQ_F32 ? 16 : 8))) Raw4 {
    uint32_t v[DT == RQ_F32 ? 4 : 2];
};
template <int DT>
RQ_DEV Raw4<DT> load_raw4(const void* p, int64_t at) {
    return *(const Raw4<DT>*)((const uint8_t*)p + at * (DT == RQ_F32 ? 4 : 2));
}
template <int DT>
RQ_DEV f32x4_t unpack_raw4(const Raw4<DT>& r) {
    f32x4_t f;
    if constexpr (DT == RQ_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f[2 * i] = dt_traits<DT>::to_f32((uint16_t)(r.v[i] & 0xffffu));
            f[2 * i + 1] = dt_traits<DT>::to_f32((uint16_t)(r.v[i] >> 16));
        }
    }
    return f;
}

template <int DT>
RQ_DEV void store4(void* p, int64_t at, f32x4_t f) {
    Raw4<DT> r;
    if constexpr (DT == RQ_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.v[i] = __float_as_uint(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            r.v[i] = dt_traits<DT>::from_f32(f[2 * i]) | ((uint32_t)dt_traits<DT>::from_f32(f[2 * i + 1]) << 16);
    }
    *(Raw4<DT>*)((uint8_t*)p + at * (DT == RQ_F32 ? 4 : 2)) = r;
}

// A producer wave's share of the arrays: 16 channels of the chunk's 16 tokens.  Lane (m, g): token m,
// four channels.
template <int DT, int XDT, bool REV>
struct Elementwise {
    int lane, wave;
    bool there;
    Raw4<DT> r, w, k, a, b;
    Raw4<XDT> x;

    // `row`: the flattened row of the lane's token and head, or any that exists.  A load under a
    // condition would be waited for where the condition ends.
    RQ_DEV void load(const WkvInputs& in, const void* of_x, int64_t row, bool exists) {
        there = exists;
        const int64_t at = row * kHead + 16 * wave + 4 * (lane >> 4);
        r = load_raw4<DT>(in.r, at);
        w = load_raw4<DT>(in.w, at);
        k = load_raw4<DT>(in.k, at);
        a = load_raw4<DT>(in.a, at);
        b = load_raw4<DT>(in.b, at);
        x = load_raw4<XDT>(of_x, at);
    }
    RQ_DEV void run(Arrays& to, Rows* inverse, int& strong_flag) const {
        const int m = lane & 15, c = 16 * wave + 4 * (lane >> 4);
        const f32x4_t zero = {0.f, 0.f, 0.f, 0.f}, fw = unpack_raw4<DT>(w);
        const f32x4_t fr = there ? unpack_raw4<DT>(r) : zero, fk = there ? unpack_raw4<DT>(k) : zero,
                      fa = there ? unpack_raw4<DT>(a) : zero, fb = there ? unpack_raw4<DT>(b) : zero;
        f32x4_t l, g2, el, ex, il, hat;
        bool strong = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            g2[i] = there ? log2_decay(fw[i]) : 0.f;
            l[i] = upto<REV>(g2[i]);
            strong |= !(of_last<REV>(l[i]) >= kStrong);
        }
        strong = __any(strong);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            el[i] = exp2_hw(l[i]);
            ex[i] = before_or_one<REV>(el[i]);
            il[i] = exp2_hw(-l[i]);
            hat[i] = of_last<REV>(el[i]) * il[i];
        }
        if (strong) {
#pragma unroll
            for (int i = 0; i < 4; ++i) hat[i] = exp2_hw(before<!REV>(upto<!REV>(g2[i])));
        }
        *(f32x4_t*)&(REV ? to.from_sa : to.to_sa)[m][c] = fa * ex;
        *(f32x4_t*)&(REV ? to.from_x : to.to_y)[m][c] = fr * el;
        *(f32x4_t*)&(REV ? to.to_sa : to.from_sa)[m][c] = fb * hat;
        *(f32x4_t*)&(REV ? to.to_y : to.from_x)[m][c] = fk * hat;
        *(f32x4_t*)&to.x[m][c] = there ? unpack_raw4<XDT>(x) : zero;
        *(f32x4_t*)&inverse[0][m][c] = fb * il;
        *(f32x4_t*)&inverse[1][m][c] = fk * il;
        if (m == (REV ? 0 : 15)) *(f32x4_t*)&to.decay[c] = el;
        if (lane == 0) strong_flag = strong;
    }
};

// Wave `pair` of four forms one of Mab, Mak / Mrb, Mrb / Mak, Mrk from the arrays: an entry is a product
// of a row of the later tensor and one of the earlier one.  Lane (m, g): token m, a quarter of the channels.
template <int DT, bool REV>
RQ_DEV void form_matrix(const WkvInputs& in, const Arrays& from, const Rows* inverse, bool strong, Matrices& to, int lane,
                        int pair, int64_t row, bool exists) {
    const int m = lane & 15, g = lane >> 4;
    const bool is_a = pair == 0 || pair == (REV ? 2 : 1), is_b = pair == 0 || pair == (REV ? 1 : 2);
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
    if (!strong) {
        const Rows& late = is_a ? (REV ? from.from_sa : from.to_sa) : (REV ? from.from_x : from.to_y);
        const Rows& early = inverse[is_b ? 0 : 1];
        f32x4_t l[4], e[4], other = x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            l[j] = *(const f32x4_t*)&late[m][16 * g + 4 * j];
            e[j] = *(const f32x4_t*)&early[m][16 * g + 4 * j];
        }
        // two sums: a product of this shape waits for the one before only where they share the sum
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            x = REV ? mma16(l[j], e[j], x) : mma16(e[j], l[j], x);
            other = REV ? mma16(l[j + 1], e[j + 1], other) : mma16(e[j + 1], l[j + 1], other);
        }
        x += other;
    } else {
        float late[16], early[16], g2[16];
        const int64_t at = row * kHead + 16 * g;
        unpack_raw<DT>(load_raw<DT>(is_a ? in.a : in.r, at, exists), late);
        unpack_raw<DT>(load_raw<DT>(is_b ? in.b : in.k, at, exists), early);
        unpack_raw<DT>(load_raw<DT>(in.w, at, exists), g2);
        for (int i = 0; i < 16; ++i) g2[i] = exists ? log2_decay(g2[i]) : 0.f;
        x = strong_pairs<REV>(late, early, g2, is_a, lane);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (is_a ? 4 * g + i < m : 4 * g + i <= m) ? x[i] : 0.f;
    if (pair == 0) to.inv[lane] = unit_inverse(x, lane);
    if (pair == 1) to.sa_x[lane] = x;
    if (pair == 2) to.y_sa[lane] = x;
    if (pair == 3) to.y_x[lane] = x;
}

// ----------------------------------------------------------- the gradients

// Over a lane's four tokens and the four lanes of its key: lane (m, g) holds tokens 4g + i.
RQ_DEV float groups_before(float x, int g) {  // the sum over the groups before the lane's own
    float a = __shfl_up(x, 16), b = __shfl_up(x, 32), c = __shfl_up(x, 48);
    return (g > 0 ? a : 0.f) + (g > 1 ? b : 0.f) + (g > 2 ? c : 0.f);
}
RQ_DEV float groups_after(float x, int g) {
    float a = __shfl_down(x, 16), b = __shfl_down(x, 32), c = __shfl_down(x, 48);
    return (g < 3 ? a : 0.f) + (g < 2 ? b : 0.f) + (g < 1 ? c : 0.f);
}
RQ_DEV float over_groups(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// A product over the 64 values: lane (m, g) holds values 16q + 4g + i of row m of A and of column m of B.
RQ_DEV f32x4_t mma64(const f32x4_t* a, const f32x4_t* b, f32x4_t c) {
#pragma unroll
    for (int q = 0; q < 4; ++q) c = mma16(a[q], b[q], c);
    return c;
}
// Row m of a chunk's tokens.
struct TokenRow {
    f32x4_t v[4];
    RQ_DEV TokenRow(const Rows& from, int lane) {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = *(const f32x4_t*)&from[kChunk - 1 - (lane & 15)][16 * q + 4 * (lane >> 4)];
    }
};

// x of the token `t` (the same in all lanes) and the lane's key, from tokens 4g + i
RQ_DEV float at_token(const f32x4_t& x, int t, int m) {
    const float own = (t & 3) == 0 ? x[0] : (t & 3) == 1 ? x[1] : (t & 3) == 2 ? x[2] : x[3];
    return __shfl(own, 16 * (t >> 2) + m);
}

RQ_DEV float of_lane(float x, int lane) {  // the same in all lanes
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// A wave's accesses of LDS before it are done before those behind it, for all its lanes: the machine keeps their order, and
// this has the compiler keep it too, which takes a lane's addresses for its own.
RQ_DEV void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One of dMab, dMak, dMrb and dMrk, by wave: [target][source].
RQ_DEV void pair_grads(const Rows& dy, GradRows& lds, int lane, int wave) {
    const TokenRow source(wave & 1 ? lds.v : lds.sa, lane), target(wave < 2 ? lds.dz : dy, lane);
    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
    *(f32x4_t*)&lds.pairs[wave][lane & 15][4 * (lane >> 4)] = mma64(source.v, target.v, zero);
}

// A chunk's dr, dw, dk, da and db for the 16 keys of a wave, s[q][i] = S[value 16q + 4g + i][key].  In products over the
// values a lane holds rows of tokens (A) and columns of keys (B); the results, tokens 4g + i of key lane & 15, are
// where the gradients are formed.  The pair matrices are the same for all keys: each wave forms one of the four.
RQ_DEV void chunk_grads(const f32x4_t* s, const Rows& dy_rows, GradRows& lds, int lane, int wave) {
    const int g = lane >> 4, m = lane & 15, key = 16 * wave + m;
    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
    f32x4_t gr, ga, gb, gk;
    float through = 0.f;  // sum over the values of S dS' of this key
    pair_grads(dy_rows, lds, lane, wave);
    {
        const TokenRow dy(dy_rows, lane), dz(lds.dz, lane), sa(lds.sa, lane), v(lds.v, lane);
        f32x4_t d[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                d[q][i] = lds.d[q][4 * g + i][key];
                through = fmaf(s[q][i], d[q][i], through);
            }
        }
        gr = mma64(dy.v, s, zero);
        ga = mma64(dz.v, s, zero);
        gb = mma64(sa.v, d, zero);
        gk = mma64(v.v, d, zero);
    }
    __syncthreads();
    f32x4_t g2, r, a, b, k, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = kChunk - 1 - (4 * g + i);
        g2[i] = lds.io[0][at][key];
        r[i] = lds.io[1][at][key];
        a[i] = lds.io[2][at][key];
        b[i] = lds.io[3][at][key];
        k[i] = lds.io[4][at][key];
        l[i] = i ? l[i - 1] + g2[i] : g2[i];
    }
    const float off = groups_before(l[3], g);
    l += off;
    const float end = __shfl(l[3], 48 + m);
    const bool strong = __any(!(end >= kStrong));
    through = over_groups(through);
    f32x4_t own_b, own_k;  // a token's own pair passes no decay: it stays out of the sums below
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        own_b[i] = lds.pairs[2][4 * g + i][4 * g + i];
        own_k[i] = lds.pairs[3][4 * g + i][4 * g + i];
    }
    f32x4_t to_end, el, ex;  // e^(Lend - L), e^L, e^Lx
    {
        float after = groups_after((g2[0] + g2[1]) + (g2[2] + g2[3]), g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            el[i] = exp2_hw(l[i]);
            ex[i] = i ? el[i - 1] : exp2_hw(off);
        }
#pragma unroll
        for (int i = 3; i >= 0; --i) {
            to_end[i] = exp2_hw(after);
            after += g2[i];
        }
    }
    gb *= to_end;
    gk *= to_end;
    gr *= el;
    ga *= ex;
    const f32x4_t enters = b * gb + k * gk, leaves_r = r * gr, leaves_a = a * ga;  // what each token adds to, and takes from, the state
    // of the pairs of tokens s < t: their parts of dr, da, db and dk, and of each token's decay those that pass it (s < i <= t;
    // of a, that reads the state before its own decay, s < i < t).  Only these: a difference of sums over all pairs
    // would leave the rounding of pairs that lie to one side of the token, which may be any number of times larger.
    f32x4_t pr = zero, pa = zero, pb = zero, pk = zero, cross = zero;
    if (strong) {
        // pair by pair, from the sums of the terms between the two tokens
#pragma unroll 1
        for (int src = 0; src < kChunk - 1; ++src) {
            const float bs = at_token(b, src, m), ks = at_token(k, src, m);
            const float of_m[4] = {lds.pairs[0][m][src], lds.pairs[1][m][src], lds.pairs[2][m][src], lds.pairs[3][m][src]};
            float e = 0.f;
#pragma unroll 1
            for (int t = src + 1; t < kChunk; ++t) {
                const float h = exp2_hw(e);
                e += at_token(g2, t, m);
                const float f = exp2_hw(e), rt = at_token(r, t, m) * f, at_ = at_token(a, t, m) * h;
                const float m0 = of_lane(of_m[0], t), m1 = of_lane(of_m[1], t), m2 = of_lane(of_m[2], t), m3 = of_lane(of_m[3], t);
                const float of_a = m0 * bs + m1 * ks, of_r = m2 * bs + m3 * ks;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int own = 4 * g + i;
                    pr[i] += own == t ? of_r * f : 0.f;
                    pa[i] += own == t ? of_a * h : 0.f;
                    pb[i] += own == src ? m0 * at_ + m2 * rt : 0.f;
                    pk[i] += own == src ? m1 * at_ + m3 * rt : 0.f;
                    cross[i] += own > src && own <= t ? of_r * rt : 0.f;
                    cross[i] += own > src && own < t ? of_a * at_ : 0.f;  // a's decays end before t
                }
            }
        }
    } else {
        // between groups of four tokens by products, a step's contraction over the four of one group
        f32x4_t il;
#pragma unroll
        for (int i = 0; i < 4; ++i) il[i] = exp2_hw(-l[i]);
        const f32x4_t rt = r * el, at = a * ex, bt = b * il, kt = k * il;  // R~, A~, B~, K~
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // to the lanes of the contraction; the wave's own keys
            const int row = kChunk - 1 - (4 * g + i);
            lds.io[1][row][key] = rt[i];
            lds.io[2][row][key] = at[i];
            lds.io[3][row][key] = bt[i];
            lds.io[4][row][key] = kt[i];
        }
        wave_lds_order();
        f32x4_t of_r[3], of_a[3];  // of the sources of group 0, 1, 2; for the targets of later groups only
#pragma unroll
        for (int o = 0; o < 3; ++o) {
            const int row = kChunk - 1 - (4 * o + g);
            const float b_ = lds.io[3][row][key], k_ = lds.io[4][row][key];
            of_a[o] = mfma4(lds.pairs[0][m][4 * o + g], b_, zero);
            of_r[o] = mfma4(lds.pairs[2][m][4 * o + g], b_, zero);
            of_a[o] = mfma4(lds.pairs[1][m][4 * o + g], k_, of_a[o]);
            of_r[o] = mfma4(lds.pairs[3][m][4 * o + g], k_, of_r[o]);
        }
#pragma unroll
        for (int o = 1; o < 4; ++o) {  // the targets of group o, for the sources of earlier ones
            const int row = kChunk - 1 - (4 * o + g), t = 4 * o + g;
            const float r_ = lds.io[1][row][key], a_ = lds.io[2][row][key];
            const bool earlier = m < 4 * o;
            pb = mfma4(earlier ? lds.pairs[0][t][m] : 0.f, a_, pb);
            pk = mfma4(earlier ? lds.pairs[1][t][m] : 0.f, a_, pk);
            pb = mfma4(earlier ? lds.pairs[2][t][m] : 0.f, r_, pb);
            pk = mfma4(earlier ? lds.pairs[3][t][m] : 0.f, r_, pk);
        }
        float over[2] = {0.f, 0.f};  // what the pairs with the lane's group as target and group 0, groups 0 and 1 as source add to a decay between
#pragma unroll
        for (int o = 0; o < 3; ++o) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = rt[i] * of_r[o][i] + at[i] * of_a[o][i];
                if (o == 0) over[0] += x;
                if (o < 2) over[1] += x;
                pr[i] += o < g ? of_r[o][i] : 0.f;
                pa[i] += o < g ? of_a[o][i] : 0.f;
            }
        }
        {
            const float from2 = __shfl(over[0], 32 + m), from3 = __shfl(over[0], 48 + m), both = __shfl(over[1], 48 + m);
            cross += g == 1 ? from2 + from3 : g == 2 ? both : 0.f;
        }
        pr *= el;
        pa *= ex;
        pb *= il;
        pk *= il;
        float behind = 0.f, ahead = 0.f;
#pragma unroll
        for (int i = 3; i >= 0; --i) {  // of an earlier group's sources, read in this one
            behind += r[i] * pr[i];
            cross[i] += behind;
            behind += a[i] * pa[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // of this group's sources, read in a later one
            cross[i] += ahead;
            ahead += b[i] * pb[i] + k[i] * pk[i];
        }
        // within the group
        float d[4];
#pragma unroll
        for (int i = 1; i < 4; ++i) d[i] = exp2_hw(g2[i]);
#pragma unroll
        for (int t = 1; t < 4; ++t) {
            f32x4_t pairs[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) pairs[j] = *(const f32x4_t*)&lds.pairs[j][4 * g + t][4 * g];
            float h = 1.f;  // the decays between the two
#pragma unroll
            for (int s = t - 1; s >= 0; --s) {
                const float f = h * d[t], rf = r[t] * f, ah = a[t] * h;
                const float to_r = pairs[2][s] * b[s] + pairs[3][s] * k[s], to_a = pairs[0][s] * b[s] + pairs[1][s] * k[s];
                pr[t] += to_r * f;
                pa[t] += to_a * h;
                pb[s] += pairs[0][s] * ah + pairs[2][s] * rf;
                pk[s] += pairs[1][s] * ah + pairs[3][s] * rf;
#pragma unroll
                for (int i = s + 1; i <= t; ++i) cross[i] += i < t ? to_r * rf + to_a * ah : to_r * rf;
                if (s > 0) h *= d[s];
            }
        }
    }
    gr += pr + own_b * b + own_k * k;
    ga += pa;
    gb += pb + own_b * r;
    gk += pk + own_k * r;
    // the state's own way through the chunk, what entered before and what leaves at or behind
    const float whole = exp2_hw(end) * through;
    float into = groups_before((enters[0] + enters[1]) + (enters[2] + enters[3]), g);
    float out_of = groups_after((leaves_r[0] + leaves_a[0]) + (leaves_r[1] + leaves_a[1]) +
                                    (leaves_r[2] + leaves_a[2]) + (leaves_r[3] + leaves_a[3]), g);
    f32x4_t gw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        gw[i] = cross[i] + whole + into;
        into += enters[i];
    }
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        gw[i] += out_of + leaves_r[i];
        out_of += leaves_r[i] + leaves_a[i];
        // d log d / dw = -exp(w), inf where the decay, and with it what passes it, is 0
        gw[i] = gw[i] == 0.f ? 0.f : gw[i] * (g2[i] * kLn2);
    }
    wave_lds_order();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = kChunk - 1 - (4 * g + i);
        lds.io[0][at][key] = gw[i];
        lds.io[1][at][key] = gr[i];
        lds.io[2][at][key] = ga[i];
        lds.io[3][at][key] = gb[i];
        lds.io[4][at][key] = gk[i];
    }
}

// A producer wave's share of what the gradients of a chunk read and give: 16 channels of its 16 tokens, as in
// Elementwise.
template <int DT>
struct GradTensors {
    bool there;
    Raw4<DT> w, r, a, b, k, v;
    f32x4_t sa;

    // `sa_row`: of the lane's token, which is there also for tokens that are not
    RQ_DEV void load(const WkvScan& p, int64_t row, bool exists, int64_t sa_row, int lane, int wave) {
        there = exists;
        const int c = 16 * wave + 4 * (lane >> 4);
        const int64_t at = row * kHead + c;
        w = load_raw4<DT>(p.in.w, at);
        r = load_raw4<DT>(p.in.r, at);
        a = load_raw4<DT>(p.in.a, at);
        b = load_raw4<DT>(p.in.b, at);
        k = load_raw4<DT>(p.in.k, at);
        v = load_raw4<DT>(p.in.v, at);
        sa = *(const f32x4_t*)(p.grads.sa + sa_row * kHead + c);
    }
    RQ_DEV void put(GradRows& lds, int lane, int wave) const {
        const int m = lane & 15, c = 16 * wave + 4 * (lane >> 4);
        const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
        f32x4_t g2 = unpack_raw4<DT>(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) g2[i] = there ? log2_decay(g2[i]) : 0.f;
        *(f32x4_t*)&lds.io[0][m][c] = g2;
        *(f32x4_t*)&lds.io[1][m][c] = there ? unpack_raw4<DT>(r) : zero;
        *(f32x4_t*)&lds.io[2][m][c] = there ? unpack_raw4<DT>(a) : zero;
        *(f32x4_t*)&lds.io[3][m][c] = there ? unpack_raw4<DT>(b) : zero;
        *(f32x4_t*)&lds.io[4][m][c] = there ? unpack_raw4<DT>(k) : zero;
        *(f32x4_t*)&lds.v[m][c] = there ? unpack_raw4<DT>(v) : zero;
        *(f32x4_t*)&lds.sa[m][c] = sa;
    }
};
template <int DT>
RQ_DEV void store_grads(const WkvGrads& to, const GradRows& lds, int64_t row, int lane, int wave) {
    const int m = lane & 15, c = 16 * wave + 4 * (lane >> 4);
    const int64_t at = row * kHead + c;
    if (to.dw) store4<DT>(to.dw, at, *(const f32x4_t*)&lds.io[0][m][c]);
    if (to.dr) store4<DT>(to.dr, at, *(const f32x4_t*)&lds.io[1][m][c]);
    if (to.da) store4<DT>(to.da, at, *(const f32x4_t*)&lds.io[2][m][c]);
    if (to.db) store4<DT>(to.db, at, *(const f32x4_t*)&lds.io[3][m][c]);
    if (to.dk) store4<DT>(to.dk, at, *(const f32x4_t*)&lds.io[4][m][c]);
}

// ------------------------------------------------------------------ the scan

// A segment of a sequence: which, and its chunks in processing order.
struct Segment {
    int64_t seq, index, first, end;
    bool last;
};

RQ_DEV Segment segment_of(const WkvShape& s, const WkvSegments& g, int64_t slot, Span& span) {
    int64_t seq = slot, index = 0;
    if (g.chunks && s.cu) {
        // as the chunks' places (WkvShape), in units of a segment: the last sequence that begins here or before
        const int64_t tokens = g.chunks * kChunk;
        int64_t lo = 0, hi = s.seqs;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (boundary(s, mid) / tokens + mid <= slot) lo = mid;
            else hi = mid;
        }
        seq = lo;
        index = slot - (boundary(s, lo) / tokens + lo);
    } else if (g.chunks) {
        const int64_t per = ((s.time + kChunk - 1) / kChunk + g.chunks - 1) / g.chunks;
        seq = slot / per;
        index = slot % per;
    }
    span = span_of(s, seq);
    const int64_t n = span.chunks();
    if (!g.chunks) return {seq, 0, 0, n, true};
    // an empty sequence has one segment, without a chunk; places behind the last segment begin behind the end
    const int64_t first = index * g.chunks;
    return {seq, index, first, std::min(first + g.chunks, n), first + g.chunks >= n};
}
RQ_DEV bool unused(const Segment& s) { return s.index < 0 || (s.index > 0 && s.first >= s.end); }

// 0 in the tokens outside [cu[0], cu[seqs]): each block takes its share of them, without a launch of their own (3 us).
template <int DT>
RQ_DEV void clear_rest(const WkvShape& s, std::initializer_list<void*> tensors) {
    const int64_t first = boundary(s, 0), last = boundary(s, s.seqs), behind = last > first ? last : first;
    const int64_t rows = first + (s.time - behind), vecs = s.heads * kHead * (DT == RQ_F32 ? 4 : 2) / 16;
    for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
        const int64_t t = i < first ? i : behind + (i - first);
        for (void* p : tensors) {
            if (!p) continue;
            uint4* at = (uint4*)p + t * vecs;
            for (int64_t x = threadIdx.x; x < vecs; x += blockDim.x) at[x] = make_uint4(0, 0, 0, 0);
        }
    }
}

// Four waves form the arrays of chunk c + 2, load chunk c + 3 and store the y of chunk c - 1, four others form
// the matrices of chunk c + 1, while four scan waves, each with 16 of the 64 values, take chunk c.  A scan wave
// holds its state transposed, acc[q][i] = S[value lane & 15][key 16q + 4g + i]: the layout in which a product's
// result comes and in which the next takes it.  It reads nothing from memory: on this machine loads and
// stores are waited for in their order, and a load behind a store waits for the store too.
// What bounds it: of a chunk's 2.35 us (2.9 us with the states written for the backward pass) the scan wave's 80 fp32
// MFMAs and the matrix wave's 16 keep a SIMD's matrix core busy for 42 %, its three waves' other instructions take 16 % of its
// issue, a CU's LDS is busy for 19 %; the rest is the way from one product to the next.  Backwards 6.9 us a chunk: 39, 23 and 27
// %.  32 heads of 8 x 512 tokens take 93 us forwards, 226 backwards, at 2.2 TB/s of HBM.  Of one sequence of 2047
// tokens: 100 us in eight segments, 290 us whole.
//
// ENDS: only where a segment ends, from a state of 0 (four scan waves) and, without x, from the identity (four more).
//
// Backwards (GRADS) the scan waves also form the other gradients of their chunk, from its dS' and dZ in LDS.  That takes more
// than the 168 registers of twelve waves: there are eight, four for the arrays and the matrices.  A chunk has three phases, with
// a barrier behind each: the scan; the pair matrices, one a wave, and the products over the values; the pairs.  The next
// chunk's matrices are formed in the third: in the second they shared the matrix cores, 7.3 us a chunk against 6.9, and of
// strong decays the two pairwise loops came one after the other (4.9 ms against 6.0 for 8 x 512 tokens of 32 heads, with
// the forward pass).  The first four waves have time left: what the gradients need but the state, and the
// gradients on their way to memory, pass through them and LDS, in whole rows.  In an earlier form, of two phases and 6.4 us a chunk,
// the scan waves' own loads and stores of single 16-bit numbers took 7.4 us, four waves of their own for chunk c - 1
// 8.9 us, and a kernel of its own behind the scan, dS' and dZ through memory, 145 + 100 us for 8 x 512 tokens against 205.
template <bool REV, bool ENDS>
constexpr int kScanThreads = (ENDS ? 16 : REV ? 8 : 12) * 64;

template <int DT, int XDT, int YDT, bool REV, bool ENDS>
__global__ __launch_bounds__((kScanThreads<REV, ENDS>)) void wkv7_scan_kernel(WkvScan p) {
    constexpr bool GRADS = REV && !ENDS;
    __shared__ std::conditional_t<GRADS, ScanGradLds, ScanLds> lds;
    const int lane = threadIdx.x & 63, wave = wave_index();
    const int g = lane >> 4, m = lane & 15;
    const int64_t H = p.shape.heads, slot = blockIdx.x / H, head = blockIdx.x % H;
    if (!ENDS && p.shape.cu) {
        if constexpr (GRADS) clear_rest<YDT>(p.shape, {p.grads.dr, p.grads.dw, p.grads.dk, p.y, p.grads.da, p.grads.db});
        else clear_rest<YDT>(p.shape, {p.y});
    }
    Span span;
    const Segment seg = segment_of(p.shape, p.seg, slot, span);
    if (unused(seg) || (ENDS && seg.last)) return;
    const int64_t n = span.chunks(), first = seg.first, end = seg.end;
    // the chunk's token of index i, i in processing order
    const auto token = [&](int64_t c, int i) { return REV ? kChunk * (n - 1 - c) + (kChunk - 1 - i) : kChunk * c + i; };
    const auto exists = [&](int64_t c) { return token(c, m) < span.len; };
    const auto row = [&](int64_t c) { return (span.start + (exists(c) ? token(c, m) : 0)) * H + head; };  // where n > 0
    const auto odd = [&](int64_t c) { return (int)(c - first) & 1; };

    const auto matrix = [&](int64_t c, int ring) {
        if (c >= end) return;
        const int* f = lds.strong[ring];
        const bool strong = __builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3]);
        form_matrix<DT, REV>(p.in, lds.arrays[ring], lds.inverse[odd(c)], strong, lds.matrices[odd(c)], lane, wave & 3, row(c),
                             exists(c));
    };
    if (wave < 4) {
        Elementwise<DT, XDT, REV> el{lane, wave};
        const auto load = [&](int64_t c) {
            if (c < end) el.load(p.in, p.x, row(c), exists(c));
        };
        const auto arrays = [&](int64_t c, int ring) {
            if (c < end) el.run(lds.arrays[ring], lds.inverse[odd(c)], lds.strong[ring][wave]);
        };
        const auto store_y = [&](int64_t c) {
            if (ENDS || c < first || !p.y || !exists(c)) return;
            const int at = 16 * wave + 4 * g;
            store4<YDT>(p.y, row(c) * kHead + at, *(const f32x4_t*)&lds.y[odd(c)][m][at]);
        };
        GradTensors<DT> of_grads;
        const auto load_of_grads = [&](int64_t c) {
            if (c < end)
                of_grads.load(p, row(c), exists(c),
                              ((span.chunk0 + n - 1 - c) * H + head) * kChunk + (kChunk - 1 - m), lane, wave);
        };
        const auto store_of_grads = [&](int64_t c) {
            if constexpr (GRADS) {
                if (c >= first && exists(c)) store_grads<DT>(p.grads, lds.grads, row(c), lane, wave);
            }
        };
        load(first);
        if (GRADS) load_of_grads(first);
        arrays(first, 0);
        load(first + 1);
        __syncthreads();
        if (GRADS) matrix(first, 0);
        arrays(first + 1, 1);
        load(first + 2);
        __syncthreads();
        int next = 1, ring = 2;  // of chunks c + 1 and c + 2
        for (int64_t c = first; c < end; ++c) {
            if constexpr (GRADS) {
                store_of_grads(c - 1);
                of_grads.put(lds.grads, lane, wave);
                load_of_grads(c + 1);
            }
            arrays(c + 2, ring);
            if (!GRADS) store_y(c - 1);
            load(c + 3);
            __syncthreads();
            if (GRADS) {
                store_y(c);
                __syncthreads();
                matrix(c + 1, next);
                __syncthreads();
            }
            next = ring;
            ring = ring == 2 ? 0 : ring + 1;
        }
        if (GRADS) store_of_grads(end - 1);
        else store_y(end - 1);
        return;
    }
    if (!GRADS && wave < 8) {
        __syncthreads();
        matrix(first, 0);
        __syncthreads();
        int ring = 1;  // of chunk c + 1
        for (int64_t c = first; c < end; ++c) {
            matrix(c + 1, ring);
            ring = ring == 2 ? 0 : ring + 1;
            __syncthreads();
        }
        return;
    }
    const bool map = ENDS && wave >= 12;
    const int value = 16 * (wave & 3) + m;
    f32x4_t acc[4];
    {
        const float* from = ENDS ? nullptr
                            : p.seg.chunks && !(seg.index == 0 && seg.last)
                                ? p.seg.begins + ((slot * H + head) * kHead + value) * kHead
                            : p.state ? p.state + ((seg.seq * H + head) * kHead + value) * kHead
                                        : nullptr;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            acc[q] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (from) acc[q] = *(const f32x4_t*)(from + 16 * q + 4 * g);
            if (map) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[q][i] = 16 * q + 4 * g + i == value ? 1.f : 0.f;
            }
        }
    }
    __syncthreads();
    __syncthreads();
    int ring = 0;
    for (int64_t c = first; c < end; ++c) {
        const Arrays& b = lds.arrays[ring];
        const Matrices& mat = lds.matrices[odd(c)];
        ring = ring == 2 ? 0 : ring + 1;
        const int64_t chunk = (span.chunk0 + (REV ? n - 1 - c : c)) * H + head;
        f32x4_t s[4];  // of the gradients: keys 16 (wave & 3) + m
        if constexpr (GRADS) {
            const float* from = p.grads.states + chunk * kHead * kHead;
            uint32_t at = 4 * g * kHead + value;
            asm volatile("" : "+v"(at));  // 32 bits behind a scalar pointer; hoisted as 64-bit addresses they took too many registers
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[q][i] = from[at + (16 * q + i) * kHead];
#pragma unroll
            for (int q = 0; q < 4; ++q) *(f32x4_t*)&lds.grads.d[wave & 3][m][16 * q + 4 * g] = acc[q];
        }
        if (!ENDS && !REV && p.states) {
            float* to = p.states + (chunk * kHead + value) * kHead + 4 * g;
#pragma unroll
            for (int q = 0; q < 4; ++q) *(f32x4_t*)(to + 16 * q) = acc[q];
        }
        const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
        f32x4_t to_sa[4], to_y[4], fs[4], fx[4], v = zero;
        if (!map) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = b.x[4 * g + i][value];
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) to_sa[q] = *(const f32x4_t*)&b.to_sa[m][16 * q + 4 * g];
        const f32x4_t sa_x = mat.sa_x[lane], inv = mat.inv[lane];
        f32x4_t z[2] = {zero, zero}, y[2] = {zero, zero}, y_sa, y_x;
        if (!map) z[0] = mma16(sa_x, v, z[0]);
#pragma unroll
        for (int q = 0; q < 4; ++q) z[q & 1] = mma16(to_sa[q], acc[q], z[q & 1]);
        z[0] += z[1];
        if constexpr (!ENDS) {
#pragma unroll
            for (int q = 0; q < 4; ++q) to_y[q] = *(const f32x4_t*)&b.to_y[m][16 * q + 4 * g];
            y_sa = mat.y_sa[lane];
            y_x = mat.y_x[lane];
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q & 1] = mma16(to_y[q], acc[q], y[q & 1]);
            y[1] = mma16(y_x, v, y[1]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                fs[q][i] = b.from_sa[4 * g + i][16 * q + m];
                fx[q][i] = b.from_x[4 * g + i][16 * q + m];
            }
        }
        const f32x4_t sa = mma16(inv, z[0], zero);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q] *= *(const f32x4_t*)&b.decay[16 * q + 4 * g];
        if (!map) {
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[q] = mma16(fx[q], v, acc[q]);
        }
        if constexpr (!ENDS) y[0] = mma16(y_sa, sa, y[0]);
#pragma unroll
        for (int i = 0; i < 4; ++i)  // one step of each sum in turn
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[q] = mfma4(fs[q][i], sa[i], acc[q]);
        if constexpr (!ENDS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) lds.y[odd(c)][4 * g + i][value] = y[0][i] + y[1][i];
            if constexpr (GRADS) {
#pragma unroll
                for (int i = 0; i < 4; ++i) lds.grads.dz[4 * g + i][value] = sa[i];
            }
            if (!REV && p.sa) {  // 0 for tokens that are not there
#pragma unroll
                for (int i = 0; i < 4; ++i) p.sa[(chunk * kChunk + 4 * g + i) * kHead + value] = sa[i];
            }
        }
        __syncthreads();
        if constexpr (GRADS) {
            chunk_grads(s, b.x, lds.grads, lane, wave & 3);
            __syncthreads();
        }
    }
    float* to = ENDS ? p.seg.ends + ((slot * H + head) * 2 * kHead + (map ? kHead : 0) + value) * kHead
                : p.state_out && seg.last ? p.state_out + ((seg.seq * H + head) * kHead + value) * kHead
                                          : nullptr;
    if (to) {
#pragma unroll
        for (int q = 0; q < 4; ++q) *(f32x4_t*)(to + 16 * q + 4 * g) = acc[q];
    }
}

// The states at the segments' beginnings, S' = S M + N from one to the next: a block is 16 values of a head of
// a sequence, its four waves 16 keys each.  A step's 64 x 64 x 64 product is 0.9 us of one CU's fp32 MFMAs, and a step
// of all values in one block took 1.75 us; the values do not need each other.
__global__ __launch_bounds__(256) void wkv7_join_kernel(WkvShape shape, WkvSegments seg, const float* state) {
    __shared__ Rows states[2];              // [value][key]
    __shared__ float maps[2][kHead][kRow];  // [from key][to key]
    const int lane = threadIdx.x & 63, q = wave_index();
    const int g = lane >> 4, m = lane & 15;
    const int64_t H = shape.heads, which = blockIdx.x / 4, seq = which / H, head = which % H;
    const Span span = span_of(shape, seq);
    const int64_t count = (span.chunks() + seg.chunks - 1) / seg.chunks;
    if (count < 2) return;
    const int64_t slot0 = shape.cu ? span.start / (seg.chunks * kChunk) + seq
                                   : seq * (((shape.time + kChunk - 1) / kChunk + seg.chunks - 1) / seg.chunks);
    const int value = 16 * (blockIdx.x & 3) + m, row = threadIdx.x >> 4, column = 4 * (threadIdx.x & 15);
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
    if (state) s = *(const f32x4_t*)(state + ((seq * H + head) * kHead + value) * kHead + 16 * q + 4 * g);
    // the first segment's too: the last one's block may write the same memory before the first one's has read it
    *(f32x4_t*)(seg.begins + ((slot0 * H + head) * kHead + value) * kHead + 16 * q + 4 * g) = s;
    // of the next steps: the thread's share of M, N[value][key 16q + 4g + i].  Registers by turns, not handed on:
    // a copy of what is on its way waits for it.
    constexpr int kTurns = 4;
    f32x4_t map[kTurns][4], add[kTurns];
    const auto load = [&](int at, int64_t j) {
        const float* from = seg.ends + ((slot0 + (j < count - 1 ? j : count - 2)) * H + head) * 2 * kHead * kHead;
#pragma unroll
        for (int x = 0; x < 4; ++x) map[at][x] = *(const f32x4_t*)(from + (kHead + 16 * x + row) * kHead + column);
        add[at] = *(const f32x4_t*)(from + value * kHead + 16 * q + 4 * g);
    };
#pragma unroll
    for (int j = 0; j + 1 < kTurns; ++j) load(j, j);
    for (int64_t j0 = 0; j0 + 1 < count; j0 += kTurns) {
#pragma unroll
        for (int o = 0; o < kTurns; ++o) {
            const int64_t j = j0 + o;
            if (j + 1 >= count) return;
            load((o + kTurns - 1) % kTurns, j + kTurns - 1);
            *(f32x4_t*)&states[o & 1][m][16 * q + 4 * g] = s;
#pragma unroll
            for (int x = 0; x < 4; ++x) *(f32x4_t*)&maps[o & 1][16 * x + row][column] = map[o][x];
            __syncthreads();
            f32x4_t sum[2] = {add[o], {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                f32x4_t a;
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = maps[o & 1][16 * x + 4 * g + i][16 * q + m];
                sum[x & 1] = mma16(a, *(const f32x4_t*)&states[o & 1][m][16 * x + 4 * g], sum[x & 1]);
            }
            s = sum[0] + sum[1];
            *(f32x4_t*)(seg.begins + (((slot0 + j + 1) * H + head) * kHead + value) * kHead + 16 * q + 4 * g) = s;
        }
    }
}

// ----------------------------------------------------------------- one token

// A block is one head of one sequence: four lanes a row of the state, 16 keys each, which stays in registers between
// the state's one reading and one writing.  Bound by these: 128 sequences of 32 heads 19-21 us (134 MB, 6.4-6.9 TB/s:
// part of it from the last-level cache); one sequence of 12 heads 3.1 us, a launch and two trips to memory.
template <int DT, int YDT>
__global__ __launch_bounds__(256) void wkv7_step_kernel(WkvStep p) {
    __shared__ float in[6][kHead];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, value = tid >> 2, part = tid & 3;
    f32x4_t s[4];
    const int64_t at = (row * kHead + value) * kHead + 4 * part;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        s[j] = p.state ? *(const f32x4_t*)(p.state + at + 16 * j) : f32x4_t{0.f, 0.f, 0.f, 0.f};
    const void* const of[6] = {p.in.r, p.in.w, p.in.k, p.in.v, p.in.a, p.in.b};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = tid + 256 * j, which = i >> 6;
        if (which < 6) {
            const void* from = which == 0 ? of[0] : which == 1 ? of[1] : which == 2 ? of[2] : which == 3 ? of[3] : which == 4 ? of[4] : of[5];
            const float x = load_dt(from, DT, row * kHead + (i & 63));
            in[which][i & 63] = which == 1 ? exp2_hw(log2_decay(x)) : x;
        }
    }
    __syncthreads();
    float sa = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f32x4_t a = *(const f32x4_t*)&in[4][16 * j + 4 * part];
#pragma unroll
        for (int i = 0; i < 4; ++i) sa = fmaf(s[j][i], a[i], sa);
    }
    sa += __shfl_xor(sa, 1);
    sa += __shfl_xor(sa, 2);
    const float v = in[3][value];
    float y = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = 16 * j + 4 * part;
        const f32x4_t r = *(const f32x4_t*)&in[0][c], d = *(const f32x4_t*)&in[1][c], k = *(const f32x4_t*)&in[2][c],
                      b = *(const f32x4_t*)&in[5][c];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[j][i] = fmaf(s[j][i], d[i], fmaf(sa, b[i], v * k[i]));
            y = fmaf(s[j][i], r[i], y);
        }
        if (p.state_out) *(f32x4_t*)(p.state_out + at + 16 * j) = s[j];
    }
    y += __shfl_xor(y, 1);
    y += __shfl_xor(y, 2);
    if (part == 0) store_dt(p.y, YDT, row * kHead + value, y);
}

template <int DT, int XDT, int YDT, bool REV>
hipError_t scan_all(const WkvScan& a, hipStream_t s) {
    const int64_t heads = a.shape.heads;
    if (a.seg.chunks) {
        const dim3 grid((unsigned)(a.seg.slots * heads));
        wkv7_scan_kernel<DT, XDT, YDT, REV, true><<<grid, kScanThreads<REV, true>, 0, s>>>(a);
        wkv7_join_kernel<<<dim3((unsigned)(4 * a.shape.seqs * heads)), 256, 0, s>>>(a.shape, a.seg, a.state);
        wkv7_scan_kernel<DT, XDT, YDT, REV, false><<<grid, kScanThreads<REV, false>, 0, s>>>(a);
    } else {
        wkv7_scan_kernel<DT, XDT, YDT, REV, false>
            <<<dim3((unsigned)(a.shape.seqs * heads)), kScanThreads<REV, false>, 0, s>>>(a);
    }
    return hipGetLastError();
}

template <int DT, int ODT>
hipError_t scan_dt(const WkvScan& a, hipStream_t s) {
    return a.reverse ? scan_all<DT, ODT, DT, true>(a, s) : scan_all<DT, DT, ODT, false>(a, s);
}

template <int DT, int ODT>
hipError_t step_dt(const WkvStep& a, hipStream_t s) {
    wkv7_step_kernel<DT, ODT><<<dim3((unsigned)a.rows), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

namespace rq {

#define RQ_BY_TYPES(F, DT_, ODT_, ...)                                        \
    if (DT_ == RQ_F32) return F<RQ_F32, RQ_F32>(__VA_ARGS__);                 \
    if (DT_ == RQ_BF16)                                                       \
        return ODT_ == RQ_F32 ? F<RQ_BF16, RQ_F32>(__VA_ARGS__) : F<RQ_BF16, RQ_BF16>(__VA_ARGS__); \
    return ODT_ == RQ_F32 ? F<RQ_F16, RQ_F32>(__VA_ARGS__) : F<RQ_F16, RQ_F16>(__VA_ARGS__);

hipError_t launch_wkv_scan(const WkvScan& a, hipStream_t s) {
    RQ_BY_TYPES(scan_dt, a.in.dt, (a.reverse ? a.x_dt : a.y_dt), a, s)
}

hipError_t launch_wkv_step(const WkvStep& a, hipStream_t s) { RQ_BY_TYPES(step_dt, a.in.dt, a.y_dt, a, s) }

}  // namespace rq
