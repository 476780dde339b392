// rq_vec.h -- 16-byte accesses of rows of any width and element alignment.
#pragma once

#include "rq_common.h"

namespace {

// 16 bytes at any address that is a multiple of the element size: global
// memory takes unaligned dwordx4 accesses, so that odd row widths run the same
// wide path.
struct __attribute__((packed, aligned(2))) Bytes16 {
    uint32_t w[4];
};

template <int DT>
constexpr int kVec = DT == RQ_F32 ? 4 : 8;  // elements of 16 bytes
template <int DT>
constexpr int kSize = DT == RQ_F32 ? 4 : 2;

// Its values as fp32.
template <int DT>
RQ_DEV void unpack_vec(const Bytes16& v, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == RQ_F32) {
            f[i] = __uint_as_float(v.w[i]);
        } else {
            f[2 * i] = dt_traits<DT>::to_f32((uint16_t)(v.w[i] & 0xffffu));
            f[2 * i + 1] = dt_traits<DT>::to_f32((uint16_t)(v.w[i] >> 16));
        }
    }
}

template <int DT>
RQ_DEV void load_vec(const uint8_t* p, float* f) {
    unpack_vec<DT>(*(const Bytes16*)p, f);
}

template <int DT>
RQ_DEV void store_vec(uint8_t* p, const float* f) {
    Bytes16 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == RQ_F32) v.w[i] = __float_as_uint(f[i]);
        else if constexpr (DT == RQ_BF16) v.w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
        else v.w[i] = f32_to_f16_bits(f[2 * i]) | (f32_to_f16_bits(f[2 * i + 1]) << 16);
    }
    *(Bytes16*)p = v;
}

// Columns [c, c + kVec) of a row of `dim`: whole vectors, or the row's last few elements.
template <int DT>
RQ_DEV void load_cols(const uint8_t* row, int64_t c, int64_t dim, float* f) {
    if (c + kVec<DT> <= dim) {
        load_vec<DT>(row + c * kSize<DT>, f);
    } else {
#pragma unroll
        for (int i = 0; i < kVec<DT>; ++i) f[i] = c + i < dim ? load_dt(row, DT, c + i) : 0.f;
    }
}

template <int DT>
RQ_DEV void store_cols(uint8_t* row, int64_t c, int64_t dim, const float* f) {
    if (c + kVec<DT> <= dim) {
        store_vec<DT>(row + c * kSize<DT>, f);
    } else {
#pragma unroll
        for (int i = 0; i < kVec<DT>; ++i)
            if (c + i < dim) store_dt(row, DT, c + i, f[i]);
    }
}

}  // namespace
