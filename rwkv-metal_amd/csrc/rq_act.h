// rq_act.h -- the activations of rq_act and their slopes, in fp32.
#pragma once

#include "rq_common.h"
#include "../../include/rwkvq_train.h"

namespace {

// e^x for x <= 0 to about two units in the last place: 2^(x log2 e) by the
// hardware's v_exp_f32 for the rounded product, times 1 + ln 2 times its rounding
// error.  NaN stays; results below 2^-126 are 0.
RQ_DEV float exp_neg(float x) {
    x = x < -110.f ? -110.f : x;
    const float h = x * 1.44269504f;
    const float l = __builtin_fmaf(x, 1.92596303e-8f, __builtin_fmaf(x, 1.44269504f, -h));
    return __builtin_amdgcn_exp2f(h) * __builtin_fmaf(l, 0.693147181f, 1.f);
}

// act(v) and act'(v).  One exponential of a value <= 0 and one reciprocal
// (v_rcp_f32, one unit in the last place) serve both: the output stage of a large
// tile runs one wave to a SIMD, where their instructions are felt (x [4096, 2048],
// w [8192, 2048] with slopes: library expf, erff and divisions 179 us with silu and
// 228 with gelu, these 158 and 155; tanh 171, relu2 134, no activation 114).  `act` is
// the same in every lane, so the switch is a scalar branch.
//   sigmoid  e = exp(-|v|), r = 1 / (1 + e):  r or e r,  slope e r^2, which keep their
//            relative precision where the function has saturated
//   tanh     e = exp(-2 |v|):  +-(1 - e) r,  slope 4 e r^2;  below 1/4, where 1 - e
//            cancels, its series to v^9
//   gelu     v Phi(v): Phi(-x) = exp(-x^2 / 2) t P(t) with t = 1 / (1 + 0.35 x), P of degree
//            8 fitted to the least relative error over x >= 0 (3.4e-8; 3.6e-7 = 6 units of
//            2^-24 with the fp32 steps), so that the tail at v < 0 keeps its precision.  x^2's
//            rounding error, up to 5e-6 of the exponential, is put back; the exponential
//            is also the slope's density
RQ_DEV void act_both(int act, float v, float& a, float& s) {
    switch (act) {
        case RQ_ACT_RELU:
            a = v < 0.f ? 0.f : v;  // NaN stays
            s = v <= 0.f ? 0.f : 1.f;  // of NaN: 1, the gradient goes on
            return;
        case RQ_ACT_RELU2: {
            const float c = v < 0.f ? 0.f : v;
            a = c * c;
            s = v <= 0.f ? 0.f : 2.f * v;
            return;
        }
        case RQ_ACT_SILU:
        case RQ_ACT_SIGMOID: {
            const float e = exp_neg(-fabsf(v)), r = __builtin_amdgcn_rcpf(1.f + e);
            const float sg = v < 0.f ? e * r : r, d = e * r * r;
            a = act == RQ_ACT_SILU ? v * sg : sg;
            s = act == RQ_ACT_SILU ? __builtin_fmaf(v, d, sg) : d;
            return;
        }
        case RQ_ACT_GELU: {
            const float x = __builtin_amdgcn_fmed3f(fabsf(v), 0.f, 16.f);  // past 16 the tail is 0
            // exp(-x^2 / 2) = 2^-(x c x), the rounding errors of both products in l
            const float p = x * 0.721347520f, h = p * x;
            const float l = __builtin_fmaf(x, __builtin_fmaf(x, 0.721347520f, -p) + x * 9.62981495e-9f, __builtin_fmaf(p, x, -h));
            const float e = __builtin_amdgcn_exp2f(-h) * __builtin_fmaf(l, -0.693147181f, 1.f);
            const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(x, 0.35f, 1.f));
            float q = __builtin_fmaf(t, -0.029163115f, 0.14405745f);
            q = __builtin_fmaf(t, q, -0.25589612f);
            q = __builtin_fmaf(t, q, 0.15938762f);
            q = __builtin_fmaf(t, q, -0.023261009f);
            q = __builtin_fmaf(t, q, 0.10557393f);
            q = __builtin_fmaf(t, q, 0.11981564f);
            q = __builtin_fmaf(t, q, 0.13986433f);
            q = __builtin_fmaf(t, q, 0.13962126f);
            const float tail = t * q * e;  // Phi(-|v|)
            const float phi = v < 0.f ? tail : 1.f - tail;
            a = v * phi;
            s = __builtin_fmaf(v * 0.398942280f, e, phi);
            return;
        }
        case RQ_ACT_TANH: {
            const float x = fabsf(v), e = exp_neg(-2.f * x), r = __builtin_amdgcn_rcpf(1.f + e);
            const float q = v * v;
            float p = __builtin_fmaf(q, 0.0218694885f, -0.0539682540f);
            p = __builtin_fmaf(q, p, 0.133333333f);
            p = __builtin_fmaf(q, p, -0.333333333f);
            a = x < 0.25f ? __builtin_fmaf(v * q, p, v) : copysignf((1.f - e) * r, v);
            s = 4.f * e * r * r;
            return;
        }
        default:
            a = v;
            s = 1.f;
    }
}

RQ_DEV float act_value(int act, float v) {
    float a, s;
    act_both(act, v, a, s);
    return a;
}

RQ_DEV float act_slope(int act, float v) {
    float a, s;
    act_both(act, v, a, s);
    return s;
}

// The same of four values; one scalar branch for all of them.
RQ_DEV f32x4_t act_value4(int act, f32x4_t v) {
    switch (act) {
#define RQ_ACT4(A)                                               \
    case A:                                                      \
        return f32x4_t{act_value(A, v[0]), act_value(A, v[1]),   \
                       act_value(A, v[2]), act_value(A, v[3])};
        RQ_ACT4(RQ_ACT_RELU)
        RQ_ACT4(RQ_ACT_RELU2)
        RQ_ACT4(RQ_ACT_SILU)
        RQ_ACT4(RQ_ACT_GELU)
        RQ_ACT4(RQ_ACT_SIGMOID)
        RQ_ACT4(RQ_ACT_TANH)
#undef RQ_ACT4
        default: return v;
    }
}

RQ_DEV f32x4_t act_slope4(int act, f32x4_t v) {
    switch (act) {
#define RQ_ACT4(A)                                               \
    case A:                                                      \
        return f32x4_t{act_slope(A, v[0]), act_slope(A, v[1]),   \
                       act_slope(A, v[2]), act_slope(A, v[3])};
        RQ_ACT4(RQ_ACT_RELU)
        RQ_ACT4(RQ_ACT_RELU2)
        RQ_ACT4(RQ_ACT_SILU)
        RQ_ACT4(RQ_ACT_GELU)
        RQ_ACT4(RQ_ACT_SIGMOID)
        RQ_ACT4(RQ_ACT_TANH)
#undef RQ_ACT4
        default: return f32x4_t{1.f, 1.f, 1.f, 1.f};
    }
}

// RQ_SLOPE_BOUND16: a slope |s| < 2 - 2^-11 in 16 bits: its float16 bits, of which no such
// slope needs the codes 0x4000 - 0x7bff.  A saturated sigmoid's or tanh's slope goes far
// below 2^-14, where float16 loses bits (from |v| = 10 and 5 on) and then everything
// (17.5 and 9.4): those codes hold its bf16 bits.
RQ_DEV uint32_t bound16_bits(float s) {
    return fabsf(s) < 6.103515625e-05f ? (f32_to_bf16_bits(s) + 0x4000u) & 0xffffu : f32_to_f16_bits(s);
}
// Two of them, without a branch: the output stage feels every instruction.
RQ_DEV uint32_t bound16_pair(float s0, float s1) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2_t, pack_bf16x2(s0, s1)) + (uint16_t)0x4000);
    const uint32_t lo = fabsf(s0) < 6.103515625e-05f ? b : f32_to_f16_bits(s0);
    const uint32_t hi = fabsf(s1) < 6.103515625e-05f ? b : f32_to_f16_bits(s1) << 16;
    return (lo & 0xffffu) | (hi & 0xffff0000u);
}
RQ_DEV float bound16_value(uint32_t b) {
    const uint32_t c = b & 0x7fffu;
    if (c < 0x4000u || c >= 0x7c00u) return f16_bits_to_f32(b);
    return __uint_as_float((b & 0x8000u) << 16 | (c - 0x4000u) << 16);
}

// RQ_SLOPE_WIDE16: a slope s >= 0 in 16 bits, float16 in [2^-14, 2^15), where that
// keeps 11 bits, else bf16 with the unused sign bit as the mark.  Values >= 0
// compare like their bits.
RQ_DEV uint32_t wide16_bits(float s) {
    constexpr uint32_t lo = 0x38800000u, hi = 0x47000000u;  // 2^-14 and 2^15
    return __float_as_uint(s) - lo < hi - lo ? f32_to_f16_bits(s) : (f32_to_bf16_bits(s) | 0x8000u);
}
RQ_DEV float wide16_value(uint32_t b) {
    return b & 0x8000u ? bf16_bits_to_f32(b & 0x7fffu) : f16_bits_to_f32(b);
}

// The 16 bits of a slope of `act`, and of two.
RQ_DEV uint32_t slope16_bits(int act, float s) { return act == RQ_ACT_RELU2 ? wide16_bits(s) : bound16_bits(s); }
RQ_DEV uint32_t slope16_pair(int act, float s0, float s1) {
    return act == RQ_ACT_RELU2 ? wide16_bits(s0) | wide16_bits(s1) << 16 : bound16_pair(s0, s1);
}

// act'(v) from y = act(v): relu and relu2 only (relu2: v = sqrt(y)).
RQ_DEV float act_slope_of_y(int act, float y) {
    if (y <= 0.f) return 0.f;  // NaN is neither: as from v itself
    return act == RQ_ACT_RELU ? 1.f : 2.f * sqrtf(y);
}

}  // namespace
