// What the attention kernels of any type and head size share: loads as FP32, FP32 products, lines of parts.
#pragma once

#include "dcn_attention_mfma.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr float kSlack = 8.f;

// Channels at .. at + 3 of a row, as FP32; zeros past its end. Loads without a branch around
// them, which would wait for each before the next.
template <typename T, bool VEC>
__device__ __forceinline__ f32x4 load4(const T* row, int at, int dim) {
    f32x4 v;
    if constexpr (VEC) {
        typedef T four __attribute__((ext_vector_type(4)));
        const four t = *(const four*)(row + (at < dim ? at : dim - 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = at < dim ? widen((T)t[i]) : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float t = widen(row[at + i < dim ? at + i : dim - 1]);
            v[i] = at + i < dim ? t : 0.f;
        }
    }
    return v;
}
__device__ __forceinline__ f32x16 mma32(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ bool finite32(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7f800000u) != 0x7f800000u; }

// FP32 values of a part: the channels, then maximum and sum.
__device__ __host__ inline int part_line(int dim) { return (dim + 3) / 4 * 4 + 4; }

// Whether rows of a tensor lie on multiples of four elements.
template <typename T>
bool fours(const HeadsIn& h) {
    return (uintptr_t)h.p % (4 * sizeof(T)) == 0 && h.ts % 4 == 0 && h.hs % 4 == 0;
}

}  // namespace
}  // namespace fa
}  // namespace dcn
