// Device helpers of the microscaled cache: blocks of 32 channels that share a power of two,
// codes of 8 bits (e4m3) or 4 (e2m1).
#pragma once

#include <hip/hip_runtime.h>

#include "dcn_attention_device.hpp"

namespace dcn {
namespace fa {

typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_u32x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kMxNan = 255;  // the scale byte of a block that reads as NaN

// The scale byte of a block whose largest magnitude has these bits (finite): the smallest power of
// two that takes it to 448 = 1.75 * 2^8 (6 = 1.5 * 2^2) at most. A fraction past 0.75 (0.5) carries
// into the exponent.
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale(uint32_t magnitude) {
    const int e = (int)((magnitude + (BITS == 8 ? 0x1fffffu : 0x3fffffu)) >> 23) - (BITS == 8 ? 8 : 2);
    return e < 0 ? 0 : e;
}
// 2^(byte - 127) as the scaled conversions take it: they read the exponent's bits alone (0: 2^-127,
// 255: NaN).
__device__ __forceinline__ float mx_factor(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// The largest magnitude whose code reads back as a finite value of T.
template <typename T, int BITS>
__device__ __forceinline__ float mx_most() {
    if constexpr (__is_same(T, _Float16)) return BITS == 8 ? 61440.f : 49152.f;
    return BITS == 8 ? 0x1.ep127f : 0x1.8p127f;
}

// Eight values over a power of two as codes, to the nearest, ties to even.
template <int BITS>
__device__ __forceinline__ mx_u32x2 mx_encode(const float* x, float factor) {
    mx_u32x2 r = {0, 0};
    if constexpr (BITS == 8) {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s16x2 w = {0, 0};
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i], x[4 * i + 1], factor, false);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[4 * i + 2], x[4 * i + 3], factor, true);
            r[i] = __builtin_bit_cast(uint32_t, w);
        }
    } else {
        r[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r[0], x[0], x[1], factor, 0);
        r[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r[0], x[2], x[3], factor, 1);
        r[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r[0], x[4], x[5], factor, 2);
        r[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r[0], x[6], x[7], factor, 3);
    }
    return r;
}

// Four codes of 8 bits (eight of 4) as 16-bit values, one rounding to nearest even (exact but for
// FP16's range): T's two in each word.
template <typename T, int BITS>
__device__ __forceinline__ void mx_decode(uint32_t codes, float factor, uint32_t* out) {
    if constexpr (__is_same(T, _Float16)) {
        if constexpr (BITS == 8) {
            out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, factor, false));
            out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, factor, true));
        } else {
            out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, factor, 0));
            out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, factor, 1));
            out[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, factor, 2));
            out[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, factor, 3));
        }
    } else {
        if constexpr (BITS == 8) {
            out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, factor, false));
            out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, factor, true));
        } else {
            out[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, factor, 0));
            out[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, factor, 1));
            out[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, factor, 2));
            out[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, factor, 3));
        }
    }
}
// The same in FP32 (exact).
template <int BITS>
__device__ __forceinline__ void mx_decode32(uint32_t codes, float factor, float* out) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    f2 t[4];
    if constexpr (BITS == 8) {
        t[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, factor, false);
        t[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, factor, true);
    } else {
        t[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, factor, 0);
        t[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, factor, 1);
        t[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, factor, 2);
        t[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, factor, 3);
    }
#pragma unroll
    for (int i = 0; i < 32 / BITS; ++i) out[i] = t[i >> 1][i & 1];
}

// Row of token j's head in the pool (rows of dim channels), or -1.
__device__ __forceinline__ int64_t mx_row(const PagesArgs& pg, int heads, int s, int head, int j) {
    const int page = pg.table[(int64_t)s * pg.width + (j >> pg.shift)];
    if ((unsigned)page >= (unsigned)pg.pages) return -1;
    return (((int64_t)page * heads + head) << pg.shift) + (j & ((1 << pg.shift) - 1));
}

// The sequence of `token`: the last one that starts at or before it (0 if none does). A wave looks
// for its first token's with 64 starts at a time, which is one load for up to 64 sequences, and
// every lane goes on from there: the lanes' tokens ascend. All lanes of the wave take part.
__device__ __forceinline__ int find_sequence(const int32_t* cu, int sequences, int64_t token) {
    const int lane = __lane_id();
    const int64_t first = ((int64_t)__builtin_amdgcn_readfirstlane((int)(token >> 32)) << 32) |
                          (uint32_t)__builtin_amdgcn_readfirstlane((int)token);
    int low = 0, count = sequences;  // the sequence is in [low, low + count)
    while (count > 1) {
        const int step = (int)(((unsigned)count + 63) >> 6), at = lane * step;
        const unsigned long long votes = __ballot(at < count && cu[low + at] <= first);
        const int last = votes ? 63 - __builtin_clzll(votes) : 0;
        low += last * step;
        count = step < count - last * step ? step : count - last * step;
    }
    while (low + 1 < sequences && cu[low + 1] <= token) ++low;
    return low;
}

}  // namespace fa
}  // namespace dcn
