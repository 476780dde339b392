// rq_act.h -- the activations of rq_act and their slopes, in fp32.
#pragma once

#include "rq_common.h"
#include "../../include/rwkvq_train.h"

namespace {

RQ_DEV float sigmoid_f(float v) { return 1.f / (1.f + expf(-v)); }

// act(v).  `act` is the same in every lane, so the switch is a scalar branch.
RQ_DEV float act_value(int act, float v) {
    switch (act) {
        case RQ_ACT_RELU: return v < 0.f ? 0.f : v;  // NaN stays
        case RQ_ACT_RELU2: {
            const float c = v < 0.f ? 0.f : v;
            return c * c;
        }
        case RQ_ACT_SILU: return v * sigmoid_f(v);
        case RQ_ACT_GELU: return v * (0.5f * (1.f + erff(v * 0.70710678118654752f)));
        case RQ_ACT_SIGMOID: return sigmoid_f(v);
        case RQ_ACT_TANH: return tanhf(v);
        default: return v;
    }
}

// act'(v).  The slopes of sigmoid and tanh are written in e = exp(-|v|), which
// keeps their relative precision where the function has saturated: s (1 - s) =
// e / (1 + e)^2, and 1 - tanh^2 v = 4 e' / (1 + e')^2 with e' = exp(-2 |v|).
RQ_DEV float act_slope(int act, float v) {
    switch (act) {
        case RQ_ACT_RELU: return v > 0.f ? 1.f : 0.f;
        case RQ_ACT_RELU2: return v > 0.f ? 2.f * v : 0.f;
        case RQ_ACT_SILU: {
            const float s = sigmoid_f(v), e = expf(-fabsf(v));
            return s + v * (e / ((1.f + e) * (1.f + e)));
        }
        case RQ_ACT_GELU:
            return 0.5f * (1.f + erff(v * 0.70710678118654752f)) +
                   v * (0.39894228040143268f * expf(-0.5f * v * v));
        case RQ_ACT_SIGMOID: {
            const float e = expf(-fabsf(v));
            return e / ((1.f + e) * (1.f + e));
        }
        case RQ_ACT_TANH: {
            const float e = expf(-2.f * fabsf(v));
            return 4.f * e / ((1.f + e) * (1.f + e));
        }
        default: return 1.f;
    }
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

// act'(v) from y = act(v): relu and relu2 only (relu2: v = sqrt(y)).
RQ_DEV float act_slope_of_y(int act, float y) {
    if (act == RQ_ACT_RELU) return y > 0.f ? 1.f : 0.f;
    return y > 0.f ? 2.f * sqrtf(y) : 0.f;
}

}  // namespace
