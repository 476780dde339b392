// rq_sample.hip -- one token for each row of logits from a given uniform number.
//
//   e_i = exp((l_i - max l) / temperature)
//   the top_k largest stay; of these, from the largest, those before whom less than top_p of
//   their sum lies; of these, those with e_i >= min_p
//   the token: the first by index at which the running sum of what stays exceeds u times the whole
//
// Nothing is sorted: what stays is everything above a threshold and the first few, by
// index, of those that equal it.  The threshold of top_k is found by counts of the logits'
// bits, eight at a time from the top, that of top_p by sums in the same way.
//
// The sums decide which token comes, so they are exact: every e_i is a float64 rounded to
// a multiple of 2^-36 (coarser for a vocabulary past 2^17), and a row's sum of such
// numbers needs no more than 53 bits.  The order in which they are added does not
// matter then, and tokens that the rounding takes to 0 have less than 2^-36 of the most
// likely one's probability.
#include <algorithm>

#include "rq_common.h"
#include "rq_error.h"
#include "rq_sample.h"
#include "rq_vec.h"

namespace {

using namespace rq;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kLane = 8;               // neighbouring logits a lane takes
constexpr int kStep = 64 * kLane;      // a wave's

// A float's bits in the order of its values; -0 and 0 are one.
RQ_DEV uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
RQ_DEV float of_key(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }

// 2^x for x <= 0: 2^n times the Taylor series of exp(f ln 2), |f| <= 1/2; twelve terms leave
// 0.35^12 / 12! = 6e-15.
RQ_DEV double exp2_64(double x) {
    if (!(x > -80.0)) return 0.0;
    const double n = __builtin_rint(x), t = (x - n) * 0.6931471805599453;
    double s = 1.0 / 39916800;
    s = fma(s, t, 1.0 / 3628800);
    s = fma(s, t, 1.0 / 362880);
    s = fma(s, t, 1.0 / 40320);
    s = fma(s, t, 1.0 / 5040);
    s = fma(s, t, 1.0 / 720);
    s = fma(s, t, 1.0 / 120);
    s = fma(s, t, 1.0 / 24);
    s = fma(s, t, 1.0 / 6);
    s = fma(s, t, 0.5);
    s = fma(s, t, 1.0);
    s = fma(s, t, 1.0);
    return __builtin_ldexp(s, (int)n);
}

struct Weights {
    double top, scale;  // the largest logit, log2(e) / temperature
    double grid;        // 1.5 * 2^52 quanta: a sum with it is rounded to whole quanta
    bool inf;           // the largest logit is +inf
    RQ_DEV double exact(float l) const {
        if (inf) return l == INFINITY ? 1.0 : 0.0;
        return exp2_64(((double)l - top) * scale);
    }
    RQ_DEV double quanta(double e) const { return (e + grid) - grid; }
};

struct Lds {
    double sums[256];
    uint32_t counts[256];
    double wave_sum[kWaves];
    uint32_t wave_count[kWaves];
    float wave_max[kWaves];
    int64_t wave_at[kWaves];
    double found_sum;
    uint32_t found_bin, found_count;
    int nan;
};

RQ_DEV double wave_sum64(double x) {
#pragma unroll
    for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
    return x;
}

template <int DT>
struct Row {
    const uint8_t* p;
    int64_t n, from, steps;  // the wave's first logit and its steps
    int lane;
    // f(index of the first, eight logits), in the order of the index within a wave; -inf past the end
    template <class F>
    RQ_DEV void each(F f) const {
        for (int64_t s = 0; s < steps; ++s) {
            float l[kLane];
            const int64_t at = load(s, l);
            f(at, l);
        }
    }
    RQ_DEV int64_t load(int64_t s, float* l) const {
        const int64_t at = from + s * kStep + lane * kLane;
        if (at + kLane <= n) {
#pragma unroll
            for (int i = 0; i < kLane; i += kVec<DT>) load_vec<DT>(p + (at + i) * kSize<DT>, l + i);
        } else {
#pragma unroll
            for (int i = 0; i < kLane; ++i) l[i] = at + i < n ? load_dt(p, DT, at + i) : -INFINITY;
        }
        return at;
    }
};

// The class of equal keys in which the running total from the largest key reaches `want` (counts, or
// sums where SUMS): its key, and in `before` the total of the larger ones.  `weight(l, key)` is
// what a logit adds, 0 for one that is out; `extra` is added for `extra_key`.
template <bool SUMS, int DT, class W>
RQ_DEV uint32_t select_key(const Row<DT>& row, Lds& lds, double want, double& before, W weight, uint32_t extra_key,
                           double extra) {
    uint32_t prefix = 0, mask = 0;
    before = 0.0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) {
            lds.sums[threadIdx.x] = 0.0;
            lds.counts[threadIdx.x] = 0;
        }
        __syncthreads();
        row.each([&](int64_t, const float* l) {
#pragma unroll
            for (int i = 0; i < kLane; ++i) {
                const uint32_t key = key_of(l[i]);
                if (l[i] == -INFINITY || (key & mask) != prefix) continue;
                const double x = weight(l[i], key);
                if constexpr (SUMS) {
                    if (x > 0.0) unsafeAtomicAdd(&lds.sums[(key >> shift) & 255], x);
                } else {
                    atomicAdd(&lds.counts[(key >> shift) & 255], (uint32_t)x);
                }
            }
        });
        __syncthreads();
        if (threadIdx.x < 64) {  // four bins a lane, from the largest
            const int lane = threadIdx.x;
            double bin[4], sum = 0.0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = 255 - 4 * lane - i;
                bin[i] = SUMS ? lds.sums[b] : (double)lds.counts[b];
                if (extra > 0.0 && (extra_key & mask) == prefix && (int)((extra_key >> shift) & 255) == b) bin[i] += extra;
                sum += bin[i];
            }
            double upto = sum;
            for (int d = 1; d < 64; d <<= 1) {
                const double x = __shfl_up(upto, d);
                if (lane >= d) upto += x;
            }
            double at = before + (upto - sum);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (at < want && at + bin[i] >= want) {
                    lds.found_bin = 255 - 4 * lane - i;
                    lds.found_sum = at;
                }
                at += bin[i];
            }
        }
        __syncthreads();
        before = lds.found_sum;
        prefix |= (lds.found_bin & 255u) << shift;
        mask |= 0xffu << shift;
    }
    return prefix;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs p) {
    __shared__ Lds lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = blockIdx.x, n = p.vocab;
    const int64_t steps = (n + kWaves * kStep - 1) / (kWaves * kStep);
    const Row<DT> row{(const uint8_t*)p.logits + r * n * kSize<DT>, n, wave * steps * kStep, steps, lane};
    const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
    const int64_t top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
    float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
    min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;

    // the largest logit, and the first place that has it
    float top = -INFINITY;
    int64_t top_at = n;
    uint32_t there = 0;
    bool nan = false;
    row.each([&](int64_t at, const float* l) {
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            nan |= l[i] != l[i];
            there += l[i] > -INFINITY;
            if (l[i] > top) {
                top = l[i];
                top_at = at + i;
            }
        }
    });
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const float x = __shfl_xor(top, d);
        const int64_t at = __shfl_xor((long long)top_at, d);
        there += __shfl_xor(there, d);
        if (x > top || (x == top && at < top_at)) {
            top = x;
            top_at = at;
        }
    }
    if (threadIdx.x == 0) lds.nan = 0;
    __syncthreads();
    if (__any(nan) && lane == 0) lds.nan = 1;
    if (lane == 0) {
        lds.wave_max[wave] = top;
        lds.wave_at[wave] = top_at;
        lds.wave_count[wave] = there;
    }
    __syncthreads();
    there = 0;
    for (int i = 0; i < kWaves; ++i) {
        there += lds.wave_count[i];
        if (lds.wave_max[i] > top || (lds.wave_max[i] == top && lds.wave_at[i] < top_at)) {
            top = lds.wave_max[i];
            top_at = lds.wave_at[i];
        }
    }
    if (lds.nan || there == 0) {  // nothing to choose from
        if (threadIdx.x == 0) {
            p.token[r] = -1;
            if (p.logprob) p.logprob[r] = NAN;
        }
        return;
    }
    if (!(temperature > 0.f) || top_k == 1) {
        if (threadIdx.x == 0) {
            p.token[r] = top_at;
            if (p.logprob) p.logprob[r] = 0.f;
        }
        return;
    }
    const int bits = n <= (1 << 17) ? 36 : 33;
    const Weights w{(double)top, 1.4426950408889634 / (double)temperature,
                    6755399441055744.0 / (double)(1ll << bits), top == INFINITY};
    const double quantum = 1.0 / (double)(1ll << bits);

    // what stays: keys above `least`, and the first `ties` that equal it
    uint32_t least = 0;
    int64_t ties = 0;
    if (top_k > 0 && top_k < (int64_t)there) {
        double before;
        least = select_key<false, DT>(row, lds, (double)top_k, before, [](float, uint32_t) { return 1.0; }, 0, 0.0);
        ties = top_k - (int64_t)before;
    }
    if (top_p < 1.f) {
        const double tied = ties ? (double)ties * w.quanta(w.exact(of_key(least))) : 0.0;
        const auto weight = [&](float l, uint32_t key) { return key > least ? w.quanta(w.exact(l)) : 0.0; };
        double sum = 0.0;
        row.each([&](int64_t, const float* l) {
#pragma unroll
            for (int i = 0; i < kLane; ++i)
                if (l[i] > -INFINITY) sum += weight(l[i], key_of(l[i]));
        });
        sum = wave_sum64(sum);
        __syncthreads();
        if (lane == 0) lds.wave_sum[wave] = sum;
        __syncthreads();
        sum = tied;
        for (int i = 0; i < kWaves; ++i) sum += lds.wave_sum[i];
        const double want = fmax(top_p > 0.f ? (double)top_p * sum : 0.0, quantum);
        double before;
        const uint32_t key = select_key<true, DT>(row, lds, want, before, weight, least, tied);
        // as many of that class as are needed to reach it
        const double each = w.quanta(w.exact(of_key(key)));
        double more = __builtin_ceil((want - before) / each);
        if (more > 1.0 && before + (more - 1.0) * each >= want) more -= 1.0;
        if (before + more * each < want) more += 1.0;
        ties = ties && key == least ? std::min<int64_t>(ties, (int64_t)more) : (int64_t)more;
        least = key;
    }

    // each wave's part of what stays, by index
    const double tie_e = ties ? w.exact(of_key(least)) : 0.0;
    const double tie = ties && tie_e >= (double)min_p ? w.quanta(tie_e) : 0.0;
    const auto above = [&](float l, uint32_t key) {
        if (!(l > -INFINITY) || key <= least) return 0.0;
        const double e = w.exact(l);
        return e >= (double)min_p ? w.quanta(e) : 0.0;
    };
    double sum = 0.0;
    uint32_t equal = 0;
    row.each([&](int64_t, const float* l) {
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            const uint32_t key = key_of(l[i]);
            sum += above(l[i], key);
            equal += key == least;
        }
    });
    sum = wave_sum64(sum);
#pragma unroll
    for (int d = 32; d; d >>= 1) equal += __shfl_xor(equal, d);
    __syncthreads();
    if (lane == 0) {
        lds.wave_sum[wave] = sum;
        lds.wave_count[wave] = equal;
    }
    __syncthreads();
    const auto kept = [&](int64_t so_far, uint32_t here) {  // of `here` ties behind `so_far`
        const int64_t left = ties - so_far;
        return left <= 0 ? 0.0 : (double)std::min<int64_t>(left, here);
    };
    double whole = 0.0;
    int64_t so_far = 0;
    for (int i = 0; i < kWaves; ++i) {
        whole += lds.wave_sum[i] + kept(so_far, lds.wave_count[i]) * tie;
        so_far += lds.wave_count[i];
    }
    const float u = p.u[r];
    // at most one quantum below the whole: the last that stays, where u is 1 or more
    const double target = u > 0.f ? fmin((double)u * whole, whole - quantum) : 0.0;
    double at = 0.0;
    int mine = -1;
    so_far = 0;
    for (int i = 0; i < kWaves && mine < 0; ++i) {
        const double here = lds.wave_sum[i] + kept(so_far, lds.wave_count[i]) * tie;
        if (at + here > target) {
            mine = i;
        } else {
            at += here;
            so_far += lds.wave_count[i];
        }
    }
    if (wave != mine) return;
    for (int64_t s = 0; s < steps; ++s) {
        float l[kLane];
        const int64_t first = row.load(s, l);
        double x[kLane], lane_sum = 0.0;
        uint32_t lane_ties = 0;
#pragma unroll
        for (int i = 0; i < kLane; ++i) lane_ties += key_of(l[i]) == least;
        uint32_t ties_upto = lane_ties;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t y = __shfl_up(ties_upto, d);
            if (lane >= d) ties_upto += y;
        }
        int64_t before_me = so_far + (ties_upto - lane_ties);
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            const uint32_t key = key_of(l[i]);
            if (key == least) {
                x[i] = before_me < ties ? tie : 0.0;
                ++before_me;
            } else {
                x[i] = above(l[i], key);
            }
            lane_sum += x[i];
        }
        double upto = lane_sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double y = __shfl_up(upto, d);
            if (lane >= d) upto += y;
        }
        const uint64_t over = __ballot(at + upto > target);
        if (over) {
            if (lane == __builtin_ctzll(over)) {
                double here = at + (upto - lane_sum);
                bool done = false;
#pragma unroll
                for (int i = 0; i < kLane; ++i) {
                    here += x[i];
                    if (!done && here > target) {
                        done = true;
                        p.token[r] = first + i;
                        if (p.logprob) {
                            const double z = w.inf ? 0.0 : ((double)l[i] - w.top) / (double)temperature;
                            p.logprob[r] = (float)(z - log(whole));
                        }
                    }
                }
            }
            return;
        }
        at += __shfl(upto, 63);
        so_far += __shfl(ties_upto, 63);
    }
}

}  // namespace

namespace rq {

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.rows);
    if (a.dt == RQ_F32) sample_kernel<RQ_F32><<<grid, kThreads, 0, s>>>(a);
    else if (a.dt == RQ_BF16) sample_kernel<RQ_BF16><<<grid, kThreads, 0, s>>>(a);
    else sample_kernel<RQ_F16><<<grid, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace rq
