// Building blocks of the matrix-core attention kernels: tiles of key (or query) rows in LDS,
// their copy from HBM, and the operand layouts of v_mfma_f32_32x32x16.
//
// The products are arranged so that the softmax never leaves a lane. S^T = K Q^T has M = keys
// and N = rows: lane l holds row l % 32 and, of each block of 32 keys, the 16 keys
// 8a + 4h + b (h = l / 32, a and b = 0..3, in register 4a + b). Registers 8s .. 8s + 7 are then
// the B operand of the next product's step s as they are (O^T += V^T P^T, K index = keys), as
// long as the A operand takes its keys in that order too: two reads of four adjacent keys at
// one channel, which is what the transposing LDS read gives from row-major rows. A row's
// maximum and sum are over the lane's own registers and those of lane l ^ 32.
#pragma once

#include <hip/hip_runtime.h>

#include "dcn_attention_device.hpp"

namespace dcn {
namespace fa {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// Eight FP32 values to 16 bits, nearest even.
template <typename T>
__device__ __forceinline__ u32x4 pack8(const f32x16& v, int first) {
    typedef T vec __attribute__((ext_vector_type(8)));
    vec r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)v[first + i];
    return __builtin_bit_cast(u32x4, r);
}

// The other half of the wave's value (lane ^ 32) combined with the own one.
__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// The packed rows of one (sequence, key head): row r is token r / group, head kh * group + r % group.
struct Rows {
    int group, shift;  // shift >= 0: group is 1 << shift
    __device__ __forceinline__ int token(int r) const { return shift >= 0 ? r >> shift : r / group; }
};
__device__ __forceinline__ Rows rows_of(int group) {
    return Rows{group, (group & (group - 1)) == 0 ? 31 - __builtin_clz((unsigned)group) : -1};
}

// A tile: ROWS rows of D 16-bit channels, row-major, the 16-byte chunks of row r at chunk ^
// swizzle(r). Eight adjacent rows put one chunk in eight places, and four adjacent rows
// (4n .. 4n + 3) one 32-byte pair in four, so that both kinds of read are free of bank conflicts.
__device__ __forceinline__ int swizzle(int row) { return ((row & 3) << 1) | ((row >> 2) & 1); }

template <int D>
struct Tile {
    static constexpr int kChunks = D / 8;           // 16-byte chunks a row
    static constexpr int kRowsPerCopy = 64 / kChunks;  // rows that one wave's copy instruction fills

    // A operand with M = rows: row 32 mb + l % 32, channels 16 s + 8 h .. + 7.
    static __device__ __forceinline__ u32x4 rows(const char* tile, int mb, int s, int lane) {
        const int r = 32 * mb + (lane & 31);
        return *(const u32x4*)(tile + (r * kChunks + ((2 * s + (lane >> 5)) ^ swizzle(r))) * 16);
    }
    // A operand with M = channels 32 blk + l % 32: rows 32 mb + 16 s + {4h + b, 8 + 4h + b}.
    static __device__ __forceinline__ u32x4 columns(const char* tile, int mb, int s, int blk, int lane) {
        u32x4 r;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int row = 32 * mb + 16 * s + 8 * a + 4 * (lane >> 5) + ((lane & 15) >> 2);
            const int chunk = 4 * blk + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            const char* p = tile + (row * kChunks + (chunk ^ swizzle(row))) * 16 + (lane & 1) * 8;
            const u32x2 v = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
            r[2 * a] = v[0];
            r[2 * a + 1] = v[1];
        }
        return r;
    }
    // Where lane `lane` of copy instruction n reads: its row and channel.
    static __device__ __forceinline__ int copy_row(int n, int lane) { return n * kRowsPerCopy + lane / kChunks; }
    static __device__ __forceinline__ int copy_channel(int row, int lane) {
        return ((lane % kChunks) ^ swizzle(row)) * 8;
    }
};

// 64 lanes x 16 bytes from HBM (base + at, at per lane) into LDS at dst + 16 lane; base and dst
// are uniform. In asm because the compiler, seeing the builtin, holds every later LDS read back
// until all copies have arrived (it does not tell the two halves of a double buffer apart).
// There is no output register; wait_copies() and a barrier or its own memory clobber order the
// reads.
__device__ __forceinline__ void copy16(const char* base, uint32_t at, char* dst) {
    const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(at), "s"(base) : "memory");
}
// The same from an address per lane.
__device__ __forceinline__ void copy16(const char* from, char* dst) {
    const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
// All but the last LEFT of this wave's copies have arrived.
template <int LEFT>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
// The LDS reads before this have been made: their place may be written.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <typename T>
__device__ __forceinline__ bool finite16(uint16_t bits) {
    constexpr uint16_t e = __is_same(T, _Float16) ? 0x7c00 : 0x7f80;
    return (bits & e) != e;
}
// Zeros in the place of infinities and NaN; whether there were any.
template <typename T>
__device__ __forceinline__ bool clean16(u32x4& v) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!finite16<T>((uint16_t)v[i])) v[i] &= 0xffff0000u, bad = true;
        if (!finite16<T>((uint16_t)(v[i] >> 16))) v[i] &= 0xffffu, bad = true;
    }
    return bad;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

}  // namespace fa
}  // namespace dcn
