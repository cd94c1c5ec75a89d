// Helpers of the kernels that move tokens: rotary positions, the appends to a cache and its read back.
#pragma once

#include "dcn_attention_device.hpp"

namespace dcn {
namespace fa {

constexpr int kTokenThreads = 256;

// N adjacent elements (16 bytes, or one element).
template <typename T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N)));
    static __device__ __forceinline__ void load(const T* p, T* v) {
        const type t = *(const type*)p;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = t[i];
    }
    static __device__ __forceinline__ void store(T* p, const T* v) {
        type t;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = v[i];
        *(type*)p = t;
    }
};
template <typename T>
struct Vec<T, 1> {
    static __device__ __forceinline__ void load(const T* p, T* v) { *v = *p; }
    static __device__ __forceinline__ void store(T* p, const T* v) { *p = *v; }
};

// cos and sin of position * freq. The angle is taken and reduced to a fraction of a turn in
// FP64 (its error is below 2^-51 of itself: 1e-12 rad at an angle of 5,000), so at any
// position the result's error is that of FP32 cos and sin alone.
__device__ __forceinline__ void turn(const RotaryArgs& r, const int32_t* pos, int pair, float* c, float* s) {
    const int p = pos[pair < r.st ? 0 : (pair < r.sh ? 1 : 2)];
    const double half_turns = (double)p * (double)r.freq[pair] * 0.318309886183790671537767526745;
    const double f = half_turns - 2.0 * rint(half_turns * 0.5);
    sincospif((float)f, s, c);
    *s *= r.sign;
}

// The rotation as a list of chunks of N channels: first the rotated ones (halves: the
// chunk and its partner `pairs` channels on; interleaved: the pairs inside the chunk, or
// for N = 1 the next channel as the partner), then those that pass. A thread keeps a
// chunk's cosines and sines over its heads.
template <typename T, int N>
struct Chunk {
    int at, partner;  // channel offsets; partner 0: none
    bool inside;      // the chunk holds whole pairs
    float c[N], s[N];

    static __device__ __host__ int rotated(const RotaryArgs& r) {
        return r.interleaved && N > 1 ? 2 * r.pairs / N : r.pairs / N;
    }
    static __device__ __host__ int count(const RotaryArgs& r) { return rotated(r) + (r.dim - 2 * r.pairs) / N; }
    __device__ __forceinline__ void set(const RotaryArgs& r, int index, const int32_t* pos) {
        const int turned = rotated(r);
        partner = 0;
        inside = false;
        if (index >= turned) {
            at = 2 * r.pairs + (index - turned) * N;
            return;
        }
        int first = index * N;  // the chunk's first pair
        int n = N;
        at = first;
        if (!r.interleaved) {
            partner = r.pairs;
        } else if (N == 1) {
            at = 2 * first;
            partner = 1;
        } else {
            inside = true;
            first /= 2;
            n = N / 2;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) turn(r, pos, first + i, &c[i], &s[i]);
    }
    // The chunk of up to U heads, turned or copied: their loads are all in flight before the first
    // is used. from(u), to(u): the head's row, null where there is none.
    template <int U, typename From, typename To>
    __device__ __forceinline__ void apply_all(From from, To to, bool turn_them) const {
        T a[U][N], b[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (const T* f = from(u)) {
                Vec<T, N>::load(f + at, a[u]);
                if (partner) Vec<T, N>::load(f + at + partner, b[u]);
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (T* t = to(u)) {
                if (turn_them && partner) {
#pragma unroll
                    for (int i = 0; i < N; ++i) rotate(a[u][i], b[u][i], c[i], s[i]);
                } else if (turn_them && inside) {
#pragma unroll
                    for (int i = 0; i + 1 < N; i += 2) rotate(a[u][i], a[u][i + 1], c[i / 2], s[i / 2]);
                }
                Vec<T, N>::store(t + at, a[u]);
                if (partner) Vec<T, N>::store(t + at + partner, b[u]);
            }
    }
    static __device__ __forceinline__ void rotate(T& a, T& b, float c, float s) {
        const float x = widen(a), y = widen(b);
        a = narrow<T>(fmaf(x, c, -(y * s)));
        b = narrow<T>(fmaf(x, s, y * c));
    }
};

inline bool aligned(const void* p, int64_t ts, int64_t hs, int size) {
    return (uintptr_t)p % 16 == 0 && ts * size % 16 == 0 && hs * size % 16 == 0;
}

// Whole vectors of n channels everywhere in a head.
inline bool divides(const RotaryArgs& r, int n) {
    return r.dim % n == 0 && (r.interleaved ? 2 * r.pairs : r.pairs) % n == 0;
}

// Heads a launch spreads over grid.y (65,535 at most): as many as give the card about 2,048 waves a slice.
inline unsigned head_slices(int64_t items, int heads) {
    const int64_t want = (131072 + items - 1) / items, most = heads < 65535 ? heads : 65535;
    return (unsigned)(want < 1 ? 1 : (want > most ? most : want));
}

// launch(first, grid) over all items.
template <typename F>
hipError_t in_launches(int64_t items, int heads, F launch) {
    for (int64_t first = 0; first < items; first += kMostThreads) {
        const int64_t n = items - first < kMostThreads ? items - first : kMostThreads;
        launch(first, dim3((unsigned)((n + kTokenThreads - 1) / kTokenThreads), head_slices(items, heads)));
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace fa
}  // namespace dcn
