// rq_sample.hip -- one token for each row of logits from a given uniform number.
//
//   e_i = exp((l_i - max l) / temperature)
//   the top_k largest stay; of these, from the largest, those before whom less than top_p of
//   their sum lies; of these, those with e_i >= min_p
//   the token: the first by index at which the running sum of what stays exceeds u times the whole
//
// Nothing is sorted: what stays is everything above a threshold and the first few, by
// index, of those that equal it.  A block takes a row, in few passes over it:
//   1. the largest logit;
//   2. a bound that everything that stays reaches and little else does.  top_k up to 1024: the
//      k-th largest of the 1024 lanes' maxima.  top_p alone: the sums of e_i in 2048 bins of
//      equal width below the largest logit, then the bin in which the border lies;
//   3. the logits that reach it, by index, into LDS: few enough for everything else.
// Where they are too many for that (a flat row) or nothing bounds them, the row is read
// again instead: for the border by bins and then among the logits of one bin, or, where
// too many share a bin (many equal ones, a range of 10^38), by the logits' bits, eight at a time
// from the top; and for the sums of what stays.
//
// The sums decide which token comes, so they are exact: every e_i is a float64 rounded to
// a multiple of 2^-36 (2^-33 for a vocabulary past 2^17), and a row's sum of such
// numbers needs no more than 53 bits.  The order in which they are added does not
// matter then.  Tokens whose e_i is below half of that are rounded to 0 and never come: each has less than 2^-37
// (2^-34) of the most likely one's probability, and n of them at most n times as much of the whole.
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

constexpr int kTable = 32;  // powers 2^(j / 32): each in banks of its own

// e^((l - top) / temperature) in float64: x = 32 log2 of it is split into a whole number and f, |f| <= 1/2; with
// t = f ln 2 / 32, |t| <= 0.0109, four terms of the series of e^t leave t^5 / 120 = 1.3e-12, less than a quantum's share.
struct Weights {
    double top, scale;    // the largest logit, 32 log2(e) / temperature; beside +inf a number past all others, 1
    double grid;          // 1.5 * 2^52 quanta: a sum with it is rounded to whole quanta
    const double* table;
    bool inf;             // the largest logit is +inf
    RQ_DEV double at(float l) const {
        constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52
        constexpr double k = 0.6931471805599453 / kTable;
        // past 2^-40 everything is rounded to 0
        const double x = fmin(fmax(((double)l - top) * scale, -40.0 * kTable), 0.0);
        const double r = x + kWhole;
        const int n = (int)(uint32_t)__double_as_longlong(r);
        const double f = x - (r - kWhole);
        double s = k * k * k * k / 24;
        s = fma(s, f, k * k * k / 6);
        s = fma(s, f, k * k / 2);
        s = fma(s, f, k);
        s = fma(s, f, 1.0);
        long long power = __double_as_longlong(table[n & (kTable - 1)]);
        power += (long long)(n >> 5) << 52;
        return s * __longlong_as_double(power);
    }
    RQ_DEV double quanta(double e) const { return (e + grid) - grid; }
};

// Whole units, for sums in LDS: integer atomics run at twice the rate of float64 ones.
struct Units {
    double grid, unit;  // 1.5 * 2^52 units, and one
    RQ_DEV unsigned long long of(double x) const {  // x <= 1
        return (unsigned long long)(__double_as_longlong(x + grid) - __double_as_longlong(grid));
    }
    RQ_DEV unsigned long long of_sum(double x) const { return (unsigned long long)(x / unit); }
};

constexpr int kBins = 2048;  // for sums below the largest logit
constexpr int kBin = 1024;   // logits of one bin that are told apart in LDS
constexpr int kFew = 400;    // of these, the number up to which each is compared with all
constexpr int kPart = 384;   // logits of a wave's part of the row that are kept in LDS

struct Lds {
    double table[kTable];
    unsigned long long sums[kBins];  // of the bins, in quanta; of 256 of them by bits
    double bin_sums[kBin];
    uint32_t bin_keys[kBin];
    uint32_t in_bin;
    double part_e[kWaves][kPart];  // what each adds
    uint32_t part_key[kWaves][kPart], part_at[kWaves][kPart];
    uint32_t part_n[kWaves];
    uint32_t digits[2][kWaves][16];
    double wave_sum[kWaves];
    uint32_t wave_count[kWaves];
    uint32_t wave_max[kWaves], wave_min[kWaves];  // keys, and their complements
    unsigned long long first;
    double found_sum, total;
    uint32_t found, found_key;
};

// Over a wave by data-parallel moves: rows of 16 lanes, then the rows.
template <int CTRL, int ROWS = 0xf>
RQ_DEV uint32_t moved(uint32_t x, uint32_t none) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
RQ_DEV double moved64(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    const uint64_t lo = moved<CTRL, ROWS>((uint32_t)u, 0), hi = moved<CTRL, ROWS>((uint32_t)(u >> 32), 0);
    return __longlong_as_double((long long)(lo | (hi << 32)));
}
// each lane's and all before it
template <class T, class F, class M>
RQ_DEV T scan_by(T x, F join, M) {
    x = join(x, M::template of<0x111>(x));
    x = join(x, M::template of<0x112>(x));
    x = join(x, M::template of<0x114>(x));
    x = join(x, M::template of<0x118>(x));
    x = join(x, M::template of<0x142, 0xa>(x));
    x = join(x, M::template of<0x143, 0xc>(x));
    return x;
}
struct Moved32 {
    template <int CTRL, int ROWS = 0xf>
    static RQ_DEV uint32_t of(uint32_t x) { return moved<CTRL, ROWS>(x, 0); }
};
struct Moved64 {
    template <int CTRL, int ROWS = 0xf>
    static RQ_DEV double of(double x) { return moved64<CTRL, ROWS>(x); }
};
RQ_DEV uint32_t scan32(uint32_t x) {
    return scan_by(x, [](uint32_t a, uint32_t b) { return a + b; }, Moved32());
}
RQ_DEV double scan64(double x) {
    return scan_by(x, [](double a, double b) { return a + b; }, Moved64());
}
RQ_DEV uint32_t last32(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
RQ_DEV double last64(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)((uint64_t)last32((uint32_t)u) | ((uint64_t)last32((uint32_t)(u >> 32)) << 32)));
}
RQ_DEV double wave_sum64(double x) { return last64(scan64(x)); }
RQ_DEV uint32_t wave_sum32(uint32_t x) { return last32(scan32(x)); }
RQ_DEV uint32_t wave_max32(uint32_t x) {  // of keys: 0 is below all
    return last32(scan_by(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; }, Moved32()));
}

// Eight neighbouring logits as they are stored.
template <int DT>
struct Raw8 {
    Bytes16 v[kLane / kVec<DT>];
};

// A wave's logits, a run of whole steps of 512; every pass reads them again, from the caches but
// for the first.
template <int DT>
struct Row {
    const uint8_t* p;
    int64_t n, from;  // the wave's first logit
    int whole, steps; // steps of 512 logits, and with the last one, of fewer
    int lane;

    RQ_DEV Row(const void* logits, int64_t row, int64_t vocab, int wave, int lane_)
        : p((const uint8_t*)logits + row * vocab * kSize<DT>), n(vocab), lane(lane_) {
        const int64_t per = (vocab + kWaves * kStep - 1) / (kWaves * kStep);
        from = wave * per * kStep;
        const int64_t left = vocab > from ? vocab - from : 0;
        whole = (int)std::min<int64_t>(per, left / kStep);
        steps = (int)std::min<int64_t>(per, (left + kStep - 1) / kStep);
    }
    RQ_DEV int64_t at(int s) const { return from + (int64_t)s * kStep + lane * kLane; }
    RQ_DEV void fetch(int s, Raw8<DT>& to) const {  // a whole step
        const uint8_t* q = p + at(s) * kSize<DT>;
#pragma unroll
        for (int j = 0; j < kLane / kVec<DT>; ++j) to.v[j] = *(const Bytes16*)(q + j * kVec<DT> * kSize<DT>);
    }
    RQ_DEV void fetch_last(int s, Raw8<DT>& to) const {  // -inf past the end
        const int64_t i = at(s);
        uint32_t w[kLane];
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            const int64_t x = std::min(i + j, n - 1);
            if constexpr (DT == RQ_F32) w[j] = ((const uint32_t*)p)[x];
            else w[j] = ((const uint16_t*)p)[x];
        }
        constexpr uint32_t kNone = DT == RQ_F32 ? 0xff800000u : DT == RQ_BF16 ? 0xff80u : 0xfc00u;
#pragma unroll
        for (int j = 0; j < kLane; ++j) w[j] = i + j < n ? w[j] : kNone;
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
            uint32_t& word = to.v[j / kVec<DT>].w[DT == RQ_F32 ? j % 4 : j / 2];
            if constexpr (DT == RQ_F32) word = w[j];
            else word = j % 2 ? word | (w[j] << 16) : w[j];
        }
    }
    template <class F>
    static RQ_DEV void take(int s, const Raw8<DT>& held, F f) {
        float l[kLane];
#pragma unroll
        for (int j = 0; j < kLane / kVec<DT>; ++j) unpack_vec<DT>(held.v[j], l + j * kVec<DT>);
        f(s, l);
    }
    // f(step, eight logits) in the order of the index; three steps in flight, in registers by turns (a copy of what is
    // on its way waits for it, and so does the end of a condition or a loop that a load may leave early: with
    // these 37 rows of 50021 took 59 us instead of 46)
    template <class F>
    RQ_DEV void each(F f) const {
        constexpr int kTurns = 4;
        if (whole > 0) {
            Raw8<DT> held[kTurns];
#pragma unroll
            for (int o = 0; o + 1 < kTurns; ++o) fetch(o < whole ? o : 0, held[o]);
            int s0 = 0;
            for (; s0 + kTurns <= whole; s0 += kTurns) {
#pragma unroll
                for (int o = 0; o < kTurns; ++o) {
                    const int ahead = s0 + o + kTurns - 1;
                    fetch(ahead < whole ? ahead : 0, held[(o + kTurns - 1) % kTurns]);
                    take(s0 + o, held[o], f);
                }
            }
#pragma unroll
            for (int o = 0; o + 1 < kTurns; ++o)
                if (s0 + o < whole) take(s0 + o, held[o], f);
        }
        if (whole < steps) {
            Raw8<DT> last;
            fetch_last(whole, last);
            take(whole, last, f);
        }
    }
};

// Bins of equal width that grow as the logits fall.  The scale stays finite (3.4e38) where the range is below 6e-36: a bin's
// lower edge follows from it.
struct Bins {
    float top, scale;
    RQ_DEV Bins(float top_, float range) : top(top_), scale(fminf((float)(kBins - 1) / range, 3.4e38f)) {}
    RQ_DEV int of(float l) const {
        const float x = l == top ? 0.f : (top - l) * scale;
        return x < (float)(kBins - 1) ? (int)x : kBins - 1;
    }
};

template <int BINS>
RQ_DEV void clear_bins(Lds& lds) {
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += kThreads) lds.sums[i] = 0;
    if (threadIdx.x == 0) lds.in_bin = 0;
    __syncthreads();
}

// The bin, from the first, in which the running total reaches `want` (less than 0: `share` of the
// whole, at least a unit); lds.found, the total before it lds.found_sum, what was looked for lds.total.
template <int BINS>
RQ_DEV void find_bin(Lds& lds, const Units& units, double before, double want, double share) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int PER = BINS > kThreads ? BINS / kThreads : 1;  // bins a thread
    __syncthreads();
    double own[PER], sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += own[i] = (int)threadIdx.x * PER < BINS ? (double)lds.sums[threadIdx.x * PER + i] * units.unit : 0.0;
    const double upto = scan64(sum);
    if (lane == 63) lds.wave_sum[wave] = upto;
    __syncthreads();
    double waves = lds.wave_sum[lane & 15];
    waves += Moved64::of<0x111>(waves);
    waves += Moved64::of<0x112>(waves);
    waves += Moved64::of<0x114>(waves);
    waves += Moved64::of<0x118>(waves);
    if (want < 0.0) want = fmax(share * last64(waves), units.unit);
    double at = before + (upto - sum) + (wave ? __shfl(waves, wave - 1) : 0.0);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (at < want && at + own[i] >= want) {
            lds.found = threadIdx.x * PER + i;
            lds.found_sum = at;
            lds.total = want;
        }
        at += own[i];
    }
    __syncthreads();
}

// Among the logits of one bin, whose keys and terms lie in LDS: the class of equal keys in which the running total
// from the largest key reaches `want`, and in `before` the total of the larger ones.  `extra` is added
// for extra_key, which is below all others.
RQ_DEV uint32_t key_in_bin(Lds& lds, double base, double want, double& before, uint32_t extra_key, bool with_extra) {
    const uint32_t n = lds.in_bin;
    if (threadIdx.x == 0 && with_extra) {  // reached where none of the others is
        lds.found_key = extra_key;
        lds.found_sum = -1.0;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const uint32_t key = lds.bin_keys[i];
        double above = base, same = 0.0;
        for (uint32_t j = 0; j < n; ++j) {
            const uint32_t other = lds.bin_keys[j];
            const double x = lds.bin_sums[j];
            above += other > key ? x : 0.0;
            same += other == key ? x : 0.0;
        }
        if (above < want && above + same >= want) {
            lds.found_key = key;
            lds.found_sum = above;
        }
    }
    __syncthreads();
    before = lds.found_sum;
    const uint32_t key = lds.found_key;
    if (before < 0.0) {
        before = base;
        for (uint32_t j = 0; j < n; ++j) before += lds.bin_sums[j];
    }
    __syncthreads();
    return key;
}

RQ_DEV void add_to_bin(Lds& lds, uint32_t key, double x) {
    const uint32_t at = atomicAdd(&lds.in_bin, 1u);
    if (at < kBin) {
        lds.bin_keys[at] = key;
        lds.bin_sums[at] = x;
    }
}

// The same over the whole row, once its bin is found.  weight(l, key) is what a logit adds, and
// may_weigh(l, key) whether that is more than 0 without working it out.
template <int DT, class M, class W>
RQ_DEV uint32_t key_in_row(const Row<DT>& row, Lds& lds, const Bins& bins, const Units& units, int bin, double base, double want,
                           double& before, M may_weigh, W weight, uint32_t extra_key, double extra) {
    row.each([&](int, const float* l) {
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            const uint32_t key = key_of(l[i]);
            if (!may_weigh(l[i], key) || bins.of(l[i]) != bin) continue;
            const double x = weight(l[i], key);
            if (x > 0.0) add_to_bin(lds, key, x);
        }
    });
    __syncthreads();
    const bool with_extra = extra > 0.0 && bins.of(of_key(extra_key)) == bin;
    if (lds.in_bin <= kBin) return key_in_bin(lds, base, want, before, extra_key, with_extra);
    // by bits: digit d of a key goes to bin 255 - d
    uint32_t prefix = 0, mask = 0;
    before = base;
    for (int shift = 24; shift >= 0; shift -= 8) {
        clear_bins<256>(lds);
        row.each([&](int, const float* l) {
#pragma unroll
            for (int i = 0; i < kLane; ++i) {
                const uint32_t key = key_of(l[i]);
                if ((key & mask) != prefix || !may_weigh(l[i], key) || bins.of(l[i]) != bin) continue;
                const double x = weight(l[i], key);
                if (x > 0.0) atomicAdd(&lds.sums[255 - ((key >> shift) & 255)], units.of(x));
            }
        });
        if (threadIdx.x == 0 && with_extra && (extra_key & mask) == prefix)
            atomicAdd(&lds.sums[255 - ((extra_key >> shift) & 255)], units.of_sum(extra));
        find_bin<256>(lds, units, before, want, 0.0);
        before = lds.found_sum;
        prefix |= (255u - lds.found) << shift;
        mask |= 0xffu << shift;
    }
    return prefix;
}

// The k-th largest of the keys that the waves hold, four bits at a time: `n` a lane, key(j) its j-th (0:
// none).  `above` is the number of larger ones.  1 <= k <= their number.
// BITS: of the leading bits only, the others 0: not above the k-th largest.
template <int BITS, class K>
RQ_DEV uint32_t kth_key(Lds& lds, int n, K key, uint32_t k, uint32_t& above) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t prefix = 0;
    above = 0;
#pragma unroll 1
    for (int shift = 28, turn = 0; shift >= 32 - BITS; shift -= 4, turn ^= 1) {
        uint32_t mine = 0;  // lane d: the keys of this wave that are at least prefix with digit d
        for (int j = 0; j < n; ++j) {
            const uint32_t x = key(j);
#pragma unroll
            for (uint32_t d = 1; d < 16; ++d) {
                const uint32_t c = __popcll(__ballot(x >= (prefix | (d << shift))));
                mine += lane == (int)d ? c : 0;
            }
        }
        if (lane < 16) lds.digits[turn][wave][lane] = mine;
        __syncthreads();
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) c += lds.digits[turn][i][lane & 15];
        // the largest digit that k keys reach
        const uint64_t reach = __ballot(lane > 0 && lane < 16 && c >= k);
        const int d = reach ? 63 - __builtin_clzll(reach) : 0;
        const uint32_t over = __shfl(c, d + 1);  // keys with a larger digit
        if (d < 15) above = over;
        prefix |= (uint32_t)d << shift;
    }
    return prefix;
}

// A value that at least k of the lanes' maxima reach, a little below the k-th largest: the largest maxima are
// told apart by 256 bins between the smallest and the largest of them.  k <= the lanes that hold a logit.
RQ_DEV float bound_of_maxima(Lds& lds, float mine, float top, uint32_t k) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t* const counts = (uint32_t*)lds.sums;
    const uint32_t low = wave_max32(mine > -INFINITY ? ~key_of(mine) : 0u);
    __syncthreads();
    if (lane == 0) lds.wave_min[wave] = low;
    if (threadIdx.x < 256) counts[threadIdx.x] = 0;
    __syncthreads();
    const float least = of_key(~wave_max32(lds.wave_min[lane & 15])), width = (top - least) * (1.f / 255.f);
    if (!(width > 0.f) || !(width < INFINITY)) return least;  // all equal, or a range past the type's
    const auto edge = [&](int b) { return top - (float)b * width; };
    int bin = (int)fminf((top - mine) / width, 255.f);
    while (bin < 255 && mine < edge(bin + 1)) ++bin;  // in its bin whatever the rounding: mine >= edge(bin + 1)
    if (mine > -INFINITY) atomicAdd(&counts[bin], 1u);
    __syncthreads();
    uint32_t four[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += four[i] = counts[4 * lane + i];
    uint32_t before = scan32(sum) - sum;
    int found = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (before < k && before + four[i] >= k) found = 4 * lane + i;
        before += four[i];
    }
    const uint64_t who = __ballot(found >= 0);
    if (!who) return least;
    const int b = __shfl(found, __builtin_ctzll(who));
    return b >= 255 ? least : fmaxf(least, edge(b + 1));
}

// The row's logits of `bound` (above -inf) and more into LDS, each wave's by index.  Whether they fit.
template <int DT>
RQ_DEV bool gather(const Row<DT>& row, Lds& lds, float bound) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t have = 0;
    row.each([&](int s, const float* l) {
        const float most = fmaxf(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), fmaxf(fmaxf(l[4], l[5]), fmaxf(l[6], l[7])));
        if (have > kPart || !__any(most >= bound)) return;
        uint32_t in = 0;
#pragma unroll
        for (int i = 0; i < kLane; ++i) in |= (uint32_t)(l[i] >= bound) << i;
        const uint32_t upto = scan32(__popc(in));
        uint32_t at = have + upto - __popc(in);
        have += last32(upto);
        if (have > kPart) return;
        const uint32_t first = (uint32_t)row.at(s);
        for (; in; in &= in - 1) lds.part_at[wave][at++] = first + __builtin_ctz(in);
    });
    if (lane == 0) lds.part_n[wave] = have;
    if (!__syncthreads_and(have <= kPart)) return false;
    for (uint32_t i = lane; i < have; i += 64) lds.part_key[wave][i] = key_of(load_dt(row.p, DT, lds.part_at[wave][i]));
    __syncthreads();
    return true;
}

// How many of `here` equal logits behind `so_far` others stay.
RQ_DEV uint32_t staying(int64_t ties, uint32_t so_far, uint32_t here) {
    const int64_t left = ties - (int64_t)so_far;
    return left <= 0 ? 0u : (uint32_t)std::min<int64_t>(left, here);
}

// Of the waves' sums and equal logits (lds.wave_sum, wave_count): the whole, the number that the
// running sum has to exceed, and the wave in which it does, with what lies before it.
struct Place {
    double whole, target, at;
    uint32_t so_far;
    int wave;
};
RQ_DEV Place find_wave(const Lds& lds, int64_t ties, double tie, float u, double quantum) {
    const int i = threadIdx.x & 15;  // four rows of lanes do the same
    const uint32_t equal = lds.wave_count[i];
    uint32_t equals = equal;
    equals += Moved32::of<0x111>(equals);
    equals += Moved32::of<0x112>(equals);
    equals += Moved32::of<0x114>(equals);
    equals += Moved32::of<0x118>(equals);
    const double here = lds.wave_sum[i] + staying(ties, equals - equal, equal) * tie;
    double upto = here;
    upto += Moved64::of<0x111>(upto);
    upto += Moved64::of<0x112>(upto);
    upto += Moved64::of<0x114>(upto);
    upto += Moved64::of<0x118>(upto);
    Place f;
    f.whole = last64(upto);
    // at most one quantum below the whole: the last that stays, where u is 1 or more
    f.target = u > 0.f ? fmin((double)u * f.whole, f.whole - quantum) : 0.0;
    f.wave = (int)__builtin_ctzll(__ballot(upto > f.target) | (1ull << 15));
    f.at = __shfl(upto - here, f.wave);
    f.so_far = __shfl(equals - equal, f.wave);
    return f;
}

RQ_DEV void choose(const SampleArgs& p, int64_t r, int64_t at, float l, const Weights& w, float temperature, double whole) {
    p.token[r] = at;
    if (p.logprob) {
        const double z = w.inf ? 0.0 : ((double)l - w.top) / (double)temperature;
        p.logprob[r] = (float)(z - log(whole));
    }
}

// A block of 16 waves for each row, whatever their number: bound by a CU's VALU where all of a row needs its e_i (some 30
// operations, most in float64) and by the latency of its passes elsewhere.  Rows of 65536: one with top_p 30 us, 128 with
// top_k 50 and top_p 19 us, 512 of which everything stays 45 us (67 MB at 1.5 TB/s; VALU instructions for 60 % of the cycles at
// four each, and float64 ones take more).  A row's work over several CUs is not built: it needs launches more, for the
// largest logit and for the bins, and a workspace.
template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs p) {
    __shared__ Lds lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // known to be the same in all lanes
    const int64_t r = blockIdx.x, n = p.vocab;
    const Row<DT> row(p.logits, r, n, wave, lane);
    const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
    int64_t top_k = p.top_k ? p.top_k[r] : p.top_k_all;
    const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
    float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
    const float u = p.u[r];
    min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;

    // a NaN is above +inf as an integer without its sign; below, `low` is -inf where some logits are masked
    float top = -INFINITY, low = INFINITY;
    uint32_t size = 0;
    row.each([&](int, const float* l) {
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            top = fmaxf(top, l[i]);
            low = fminf(low, l[i]);
            size = std::max(size, __float_as_uint(l[i]) & 0x7fffffffu);
        }
    });
    const uint32_t lane_top = top > -INFINITY ? key_of(top) : 0;
    if (threadIdx.x == 0) lds.first = ~0ull;
    if (threadIdx.x < kTable) lds.table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
    {
        const uint32_t a = wave_max32(key_of(top)), b = wave_max32(~key_of(low)), c = wave_max32(size);
        if (lane == 0) {
            lds.wave_max[wave] = a;
            lds.wave_min[wave] = b;
            lds.wave_count[wave] = c;
        }
    }
    __syncthreads();
    {
        const uint32_t a = wave_max32(lds.wave_max[lane & 15]), b = wave_max32(lds.wave_min[lane & 15]);
        size = wave_max32(lds.wave_count[lane & 15]);
        top = of_key(a);
        low = of_key(~b);
    }
    if (size > 0x7f800000u || top == -INFINITY) {  // nothing to choose from
        if (threadIdx.x == 0) {
            p.token[r] = -1;
            if (p.logprob) p.logprob[r] = NAN;
        }
        return;
    }
    if (!(temperature > 0.f) || top_k == 1) {  // the first that has the largest
        unsigned long long first = ~0ull;
        row.each([&](int s, const float* l) {
#pragma unroll
            for (int i = kLane - 1; i >= 0; --i)
                if (l[i] == top) first = std::min<unsigned long long>(first, row.at(s) + i);
        });
        if (first != ~0ull) atomicMin(&lds.first, first);
        __syncthreads();
        if (threadIdx.x == 0) {
            p.token[r] = (int64_t)lds.first;
            if (p.logprob) p.logprob[r] = 0.f;
        }
        return;
    }
    const int bits = n <= (1 << 17) ? 36 : 33;
    const bool inf = top == INFINITY;
    const Weights w{inf ? 6.8e38 : (double)top, inf ? 1.0 : kTable * 1.4426950408889634 / (double)temperature,
                    6755399441055744.0 / (double)(1ll << bits), lds.table, inf};
    const double quantum = 1.0 / (double)(1ll << bits);
    const Units units{w.grid, quantum};
    if (top_k < 0 || top_k >= n) top_k = 0;
    const bool by_sum = top_p < 1.f;
    // past 26 temperatures below the largest, e_i is rounded to 0
    const Bins sum_bins(top, fminf(top - low, 26.f * temperature));

    // what stays: keys above `least`, and the first `ties` that equal it
    uint32_t least = 0;
    int64_t ties = 0;
    bool listed = false;
    if (top_k > 0) {
        uint32_t above;
        if (top_k <= kThreads && __syncthreads_count(lane_top != 0) >= (int)top_k) {
            listed = gather(row, lds, bound_of_maxima(lds, lane_top ? of_key(lane_top) : -INFINITY, top, (uint32_t)top_k));
        }
        if (listed) {
            uint32_t longest = 0, all = 0;
#pragma unroll
            for (int i = 0; i < kWaves; ++i) {
                longest = std::max(longest, lds.part_n[i]);
                all += lds.part_n[i];
            }
            if (all <= kFew) {  // each against all
                uint32_t base = 0;
#pragma unroll
                for (int i = 0; i < kWaves; ++i) base += i < wave ? lds.part_n[i] : 0;
                for (uint32_t i = lane; i < lds.part_n[wave]; i += 64) lds.bin_keys[base + i] = lds.part_key[wave][i];
                if (threadIdx.x < 8) lds.bin_keys[all + threadIdx.x] = 0;
                __syncthreads();
                const uint32_t key = threadIdx.x < all ? lds.bin_keys[threadIdx.x] : 0;
                uint32_t larger = 0, same = 0;
                if (wave * 64 < all) {
                    for (uint32_t j = 0; j < all; j += 8) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const uint32_t other = lds.bin_keys[j + x];
                            larger += other > key;
                            same += other == key;
                        }
                    }
                }
                if (key && larger < top_k && larger + same >= top_k) {
                    lds.found_key = key;
                    lds.found = larger;
                }
                __syncthreads();
                least = lds.found_key;
                above = lds.found;
                __syncthreads();
            } else {
                // the bits that the type's values have
                least = kth_key<DT == RQ_BF16 ? 16 : DT == RQ_F16 ? 20 : 32>(
                    lds, (longest + 63) / 64,
                    [&](int j) {
                        const uint32_t i = lane + 64 * j;
                        return i < lds.part_n[wave] ? lds.part_key[wave][i] : 0u;
                    },
                    (uint32_t)top_k, above);
                if (DT != RQ_F32 && !(least >> 31)) least |= DT == RQ_BF16 ? 0xffffu : 0xfffu;  // a negative value's complement
            }
            ties = top_k - above;
        } else {
            // logits further below count as one bin: their range may be that of the type
            const Bins bins(top, fminf(top - low, 64.f));
            const auto any = [](float l, uint32_t) { return l > -INFINITY; };
            double before;
            clear_bins<kBins>(lds);
            row.each([&](int, const float* l) {
#pragma unroll
                for (int i = 0; i < kLane; ++i)
                    if (l[i] > -INFINITY) atomicAdd(&lds.sums[bins.of(l[i])], 1ull);
            });
            if (threadIdx.x == 0) lds.total = 0.0;
            const Units ones{6755399441055744.0, 1.0};
            find_bin<kBins>(lds, ones, 0.0, (double)top_k, 0.0);
            if (lds.total > 0.0) {  // as many logits are there
                least = key_in_row(row, lds, bins, ones, (int)lds.found, lds.found_sum, lds.total, before, any, [](float, uint32_t) { return 1.0; }, 0, 0.0);
                ties = top_k - (int64_t)before;
                listed = gather(row, lds, of_key(least));
            } else {
                top_k = 0;
            }
        }
    }
    if (by_sum) {
        double before, want;
        uint32_t key;
        if (top_k == 0) {
            // sums by bins over the row, and then what lies in the border's bin and above
            clear_bins<kBins>(lds);
            row.each([&](int, const float* l) {
                unsigned long long x[kLane];
#pragma unroll
                for (int i = 0; i < kLane; ++i) x[i] = units.of(w.at(l[i]));
#pragma unroll
                for (int i = 0; i < kLane; ++i)
                    if (x[i]) atomicAdd(&lds.sums[sum_bins.of(l[i])], x[i]);
            });
            find_bin<kBins>(lds, units, 0.0, -1.0, fmax((double)top_p, 0.0));
            want = lds.total;
            const int bin = lds.found;
            const double base = lds.found_sum;
            // a little below the bin, whatever the rounding
            const float bound = top - (float)(bin + 1) / sum_bins.scale * 1.00001f - 1e-6f * fabsf(top);
            if (bound > -INFINITY) listed = gather(row, lds, bound);
            if (listed) {
                for (uint32_t i = lane; i < lds.part_n[wave]; i += 64) {
                    const uint32_t k = lds.part_key[wave][i];
                    if (sum_bins.of(of_key(k)) != bin) continue;
                    const double x = w.quanta(w.at(of_key(k)));
                    if (x > 0.0) add_to_bin(lds, k, x);
                }
                __syncthreads();
            }
            if (listed && lds.in_bin <= kBin) {
                key = key_in_bin(lds, base, want, before, 0, false);
            } else {
                __syncthreads();
                if (threadIdx.x == 0) lds.in_bin = 0;
                __syncthreads();
                key = key_in_row(row, lds, sum_bins, units, bin, base, want, before, [](float l, uint32_t) { return l > -INFINITY; },
                                 [&](float l, uint32_t) { return w.quanta(w.at(l)); }, 0, 0.0);
            }
        } else {
            const double tied = (double)ties * w.quanta(w.at(of_key(least)));
            const bool with_tied = ties > 0;
            clear_bins<kBins>(lds);
            if (threadIdx.x == 0 && with_tied) atomicAdd(&lds.sums[sum_bins.of(of_key(least))], units.of_sum(tied));
            if (listed) {
                for (uint32_t i = lane; i < lds.part_n[wave]; i += 64) {
                    const uint32_t k = lds.part_key[wave][i];
                    if (k <= least) continue;
                    const double x = w.quanta(w.at(of_key(k)));
                    lds.part_e[wave][i] = x;
                    atomicAdd(&lds.sums[sum_bins.of(of_key(k))], units.of(x));
                }
            } else {
                row.each([&](int, const float* l) {
#pragma unroll
                    for (int i = 0; i < kLane; ++i) {
                        if (!(l[i] > -INFINITY) || key_of(l[i]) <= least) continue;
                        const double x = w.quanta(w.at(l[i]));
                        if (x > 0.0) atomicAdd(&lds.sums[sum_bins.of(l[i])], units.of(x));
                    }
                });
            }
            find_bin<kBins>(lds, units, 0.0, -1.0, fmax((double)top_p, 0.0));
            want = lds.total;
            const int bin = lds.found;
            const double base = lds.found_sum;
            const bool tied_in_bin = with_tied && sum_bins.of(of_key(least)) == bin;
            if (listed) {
                for (uint32_t i = lane; i < lds.part_n[wave]; i += 64) {
                    const uint32_t k = lds.part_key[wave][i];
                    if (k > least && sum_bins.of(of_key(k)) == bin && lds.part_e[wave][i] > 0.0) add_to_bin(lds, k, lds.part_e[wave][i]);
                }
                __syncthreads();
            }
            if (listed && lds.in_bin <= kBin) {
                key = key_in_bin(lds, base, want, before, least, tied_in_bin);
            } else {
                __syncthreads();
                if (threadIdx.x == 0) lds.in_bin = 0;
                __syncthreads();
                key = key_in_row(row, lds, sum_bins, units, bin, base, want, before,
                                 [&](float l, uint32_t k) { return k > least && l > -INFINITY; },
                                 [&](float l, uint32_t) { return w.quanta(w.at(l)); }, least, with_tied ? tied : 0.0);
            }
        }
        // as many of that class as are needed to reach it
        const double each = w.quanta(w.at(of_key(key)));
        double more = __builtin_ceil((want - before) / each);
        if (more > 1.0 && before + (more - 1.0) * each >= want) more -= 1.0;
        if (before + more * each < want) more += 1.0;
        ties = ties && key == least ? std::min<int64_t>(ties, (int64_t)more) : (int64_t)more;
        least = key;
    }
    if (!listed && top_k == 0 && !by_sum && min_p > 0.f) {
        // a little below the border (NaN where any logit may stay): the terms themselves decide
        const float border = (float)(log((double)min_p) * (double)temperature) * 1.0001f - 1e-6f * fabsf(top);
        // (of l, not of l - top: rounded by half a step of top's)
        if (!w.inf && border > -INFINITY) listed = gather(row, lds, top + border - 1e-6f * fabsf(top));
    }

    const double tie_e = ties ? w.at(of_key(least)) : 0.0;
    const double tie = ties && tie_e >= (double)min_p ? w.quanta(tie_e) : 0.0;
    const auto above = [&](float l, uint32_t key) {
        const double e = w.at(l);
        return l > -INFINITY && key > least && e >= (double)min_p ? w.quanta(e) : 0.0;
    };

    if (listed) {
        double sum = 0.0;
        uint32_t equal = 0;
        const uint32_t mine = lds.part_n[wave];
        for (uint32_t i = lane; i < mine; i += 64) {
            const uint32_t key = lds.part_key[wave][i];
            const double x = above(of_key(key), key);
            lds.part_e[wave][i] = x;
            sum += x;
            equal += ties && key == least;
        }
        sum = wave_sum64(sum);
        equal = wave_sum32(equal);
        __syncthreads();
        if (lane == 0) {
            lds.wave_sum[wave] = sum;
            lds.wave_count[wave] = equal;
        }
        __syncthreads();
        Place f = find_wave(lds, ties, tie, u, quantum);
        if (wave != f.wave) return;
        for (uint32_t i0 = 0; i0 < mine; i0 += 64) {
            const uint32_t i = i0 + lane;
            const uint32_t key = i < mine ? lds.part_key[wave][i] : 0u;
            double x = i < mine ? lds.part_e[wave][i] : 0.0;
            const uint32_t is = i < mine && ties && key == least;
            const uint32_t equals = scan32(is);
            if (is) x = staying(ties, f.so_far + equals - 1, 1) ? tie : 0.0;
            const double upto = scan64(x);
            const uint64_t over = __ballot(f.at + upto > f.target);
            if (over) {
                if (lane == __builtin_ctzll(over)) choose(p, r, lds.part_at[wave][i], of_key(key), w, temperature, f.whole);
                return;
            }
            f.at += last64(upto);
            f.so_far += last32(equals);
        }
        return;
    }

    // from the row: each wave's part, then the one in which the token lies, by all waves
    const float border = least ? of_key(least) : -INFINITY;
    const bool everything = top_k == 0 && !by_sum && !(min_p > 0.f);
    double sum = 0.0;
    uint32_t equal = 0;
    row.each([&](int, const float* l) {
        if (everything) {  // -inf adds 0
            double x[kLane];
#pragma unroll
            for (int i = 0; i < kLane; ++i) x[i] = w.quanta(w.at(l[i]));
            sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
            return;
        }
        const float most = fmaxf(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])), fmaxf(fmaxf(l[4], l[5]), fmaxf(l[6], l[7])));
        if (!__any(most >= border)) return;
        double x[kLane];
#pragma unroll
        for (int i = 0; i < kLane; ++i) {
            const double e = w.at(l[i]);
            x[i] = l[i] > border ? w.quanta(e) : 0.0;
            if (min_p > 0.f) x[i] = e >= (double)min_p ? x[i] : 0.0;
        }
        if (ties) {
#pragma unroll
            for (int i = 0; i < kLane; ++i) equal += l[i] == border;
        }
        sum += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    });
    sum = wave_sum64(sum);
    equal = wave_sum32(equal);
    __syncthreads();
    if (lane == 0) {
        lds.wave_sum[wave] = sum;
        lds.wave_count[wave] = equal;
    }
    __syncthreads();
    Place f = find_wave(lds, ties, tie, u, quantum);
    const Row<DT> part(p.logits, r, n, f.wave, lane);
    const int64_t end = std::min<int64_t>(n, part.from + (int64_t)part.steps * kStep);
    constexpr int kOwn = 4;  // neighbouring logits of a thread
    for (int64_t i0 = part.from; i0 < end; i0 += kOwn * kThreads) {
        const int64_t first = i0 + (int64_t)threadIdx.x * kOwn;
        float l[kOwn];
        double x[kOwn], lane_sum = 0.0;
        uint32_t lane_equal = 0;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) l[i] = load_dt(part.p, DT, std::min(first + i, n - 1));
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            if (first + i >= end) l[i] = -INFINITY;
            const uint32_t key = key_of(l[i]);
            lane_equal += ties && key == least;
            x[i] = above(l[i], key);
        }
        uint32_t equals = scan32(lane_equal);
        __syncthreads();
        if (lane == 63) lds.wave_count[wave] = equals;
        __syncthreads();
        uint32_t so_far = f.so_far + equals - lane_equal, here_equal = 0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            so_far += i < wave ? lds.wave_count[i] : 0;
            here_equal += lds.wave_count[i];
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            if (ties && key_of(l[i]) == least) x[i] = staying(ties, so_far++, 1) ? tie : 0.0;
            lane_sum += x[i];
        }
        const double upto = scan64(lane_sum);
        if (lane == 63) lds.wave_sum[wave] = upto;
        __syncthreads();
        double at = f.at, here = 0.0;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            at += i < wave ? lds.wave_sum[i] : 0.0;
            here += lds.wave_sum[i];
        }
        if (f.at + here > f.target) {
            const uint64_t over = __ballot(at + upto > f.target);
            if (at <= f.target && over && lane == __builtin_ctzll(over)) {
                at += upto - lane_sum;
                int i = 0;
#pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    at += x[j];
                    i += at <= f.target;
                }
                float chosen = l[0];
#pragma unroll
                for (int j = 1; j < kOwn; ++j) chosen = i == j ? l[j] : chosen;
                choose(p, r, first + i, chosen, w, temperature, f.whole);
            }
            return;
        }
        f.at += here;
        f.so_far += here_equal;
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
