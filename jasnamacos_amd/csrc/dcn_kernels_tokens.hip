// Rotary positions with three axes, and the append of rotated keys and values to a paged
// cache. Both are copies with a rotation on the way: bound by HBM (each element read once,
// written once), small calls by the call itself. A thread keeps one chunk of a token's channels, whose
// angles it takes once for all heads (sine and cosine cost more than a head's copy), and has four
// heads' loads in flight. Queries and keys of 108,000 tokens, 24 BF16 heads of 64: 92 us (4.8 of the 5.1 TB/s
// that a large copy reaches); a frame of 3,600 tokens for 8 streams, 24 heads of 64, appended: 47 us
// (3.8 TB/s); 64 tokens of one frame: 3.5 us of kernel.
#include "dcn_attention_device.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // heads whose loads are in flight at once

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

// One thread: one chunk of one token, over the heads blockIdx.y, blockIdx.y + gridDim.y, ...
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs r, int64_t first, int64_t tokens, int heads,
                                                          HeadsIn x, HeadsOut out) {
    const int chunks = Chunk<T, N>::count(r);
    const int64_t item = first + (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t token = item / chunks;
    if (token >= tokens) return;
    Chunk<T, N> c;
    c.set(r, (int)(item - token * chunks), r.positions + token * 3);
    const T* from = (const T*)x.p + token * x.ts;
    T* to = (T*)out.p + token * out.ts;
    const int step = gridDim.y;
    for (int h = blockIdx.y; h < heads; h += kBatch * step)
        c.template apply_all<kBatch>([&](int u) { return h + u * step < heads ? from + (h + u * step) * x.hs : nullptr; },
                                     [&](int u) { return h + u * step < heads ? to + (h + u * step) * out.hs : nullptr; }, true);
}

// One thread: one chunk of one new token; heads as above, q's, then k's, then v's.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void append_kernel(RotaryArgs r, AppendArgs a, int64_t first) {
    const int chunks = Chunk<T, N>::count(r);
    const int64_t item = first + (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t token = item / chunks;
    if (token >= a.tokens) return;
    // The sequence: the last one that starts at or before the token.
    int low = 0, high = a.sequences;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (a.cu_q[mid] <= token) low = mid;
        else high = mid;
    }
    const int64_t from = a.cu_q[low], to = a.cu_q[low + 1];
    if (token < from || token >= to) return;
    const int64_t place = (int64_t)a.kv_lens[low] - (to - token);
    int64_t row = -1;
    if (place >= 0 && place < (int64_t)a.pages.width << a.pages.shift) row = paged_row(a.pages, low, (int)place);
    const int nq = a.q.p ? a.q_heads : 0;
    const int heads = row < 0 ? nq : nq + 2 * a.kv_heads;
    if ((int)blockIdx.y >= heads) return;
    Chunk<T, N> c;
    c.set(r, (int)(item - token * chunks), r.positions + token * 3);
    // q's and k's heads turn, v's do not: two runs.
    const int step = gridDim.y, turned = row < 0 ? nq : nq + a.kv_heads;
    auto from_of = [&](int h) -> const T* {
        if (h < nq) return (const T*)a.q.p + token * a.q.ts + h * a.q.hs;
        if (h < turned) return (const T*)a.k.p + token * a.k.ts + (h - nq) * a.k.hs;
        return (const T*)a.v.p + token * a.v.ts + (h - turned) * a.v.hs;
    };
    auto to_of = [&](int h) -> T* {
        if (h < nq) return (T*)a.q_out.p + token * a.q_out.ts + h * a.q_out.hs;
        if (h < turned) return (T*)a.k_pages.p + row * a.k_pages.ts + (h - nq) * a.k_pages.hs;
        return (T*)a.v_pages.p + row * a.v_pages.ts + (h - turned) * a.v_pages.hs;
    };
    int h = blockIdx.y;
    for (; h < turned; h += kBatch * step)
        c.template apply_all<kBatch>([&](int u) { return h + u * step < turned ? from_of(h + u * step) : nullptr; },
                                     [&](int u) { return h + u * step < turned ? to_of(h + u * step) : nullptr; }, true);
    // v's first head of this slice: the next of blockIdx.y, blockIdx.y + step, ... past the turned ones.
    h = blockIdx.y + (turned > (int)blockIdx.y ? (turned - (int)blockIdx.y + step - 1) / step * step : 0);
    for (; h < heads; h += kBatch * step)
        c.template apply_all<kBatch>([&](int u) { return h + u * step < heads ? from_of(h + u * step) : nullptr; },
                                     [&](int u) { return h + u * step < heads ? to_of(h + u * step) : nullptr; }, false);
}

bool aligned(const void* p, int64_t ts, int64_t hs, int size) {
    return (uintptr_t)p % 16 == 0 && ts * size % 16 == 0 && hs * size % 16 == 0;
}

// Whole vectors of n channels everywhere in a head.
bool divides(const RotaryArgs& r, int n) {
    return r.dim % n == 0 && (r.interleaved ? 2 * r.pairs : r.pairs) % n == 0;
}

// Heads a launch spreads over grid.y (65,535 at most): as many as give the card about 2,048 waves a slice.
unsigned head_slices(int64_t items, int heads) {
    const int64_t want = (131072 + items - 1) / items, most = heads < 65535 ? heads : 65535;
    return (unsigned)(want < 1 ? 1 : (want > most ? most : want));
}

// launch(first, grid) over all items.
template <typename F>
hipError_t in_launches(int64_t items, int heads, F launch) {
    for (int64_t first = 0; first < items; first += kMostThreads) {
        const int64_t n = items - first < kMostThreads ? items - first : kMostThreads;
        launch(first, dim3((unsigned)((n + kThreads - 1) / kThreads), head_slices(items, heads)));
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

template <typename T, int N>
hipError_t rotary(int64_t tokens, int heads, const HeadsIn& x, const HeadsOut& out, const RotaryArgs& r,
                  hipStream_t stream) {
    const int64_t items = tokens * Chunk<T, N>::count(r);
    return in_launches(items, heads, [&](int64_t first, dim3 grid) {
        rotary_kernel<T, N><<<grid, kThreads, 0, stream>>>(r, first, tokens, heads, x, out);
    });
}

template <typename T>
hipError_t rotary_of(int64_t tokens, int heads, const HeadsIn& x, const HeadsOut& out, const RotaryArgs& r,
                     hipStream_t stream) {
    constexpr int n = 16 / sizeof(T);
    if (divides(r, n) && aligned(x.p, x.ts, x.hs, sizeof(T)) && aligned(out.p, out.ts, out.hs, sizeof(T)))
        return rotary<T, n>(tokens, heads, x, out, r, stream);
    return rotary<T, 1>(tokens, heads, x, out, r, stream);
}

template <typename T, int N>
hipError_t append(const AppendArgs& a, const RotaryArgs& r, hipStream_t stream) {
    const int64_t items = a.tokens * Chunk<T, N>::count(r);
    const int heads = (a.q.p ? a.q_heads : 0) + 2 * a.kv_heads;
    return in_launches(items, heads, [&](int64_t first, dim3 grid) {
        append_kernel<T, N><<<grid, kThreads, 0, stream>>>(r, a, first);
    });
}

template <typename T>
hipError_t append_of(const AppendArgs& a, const RotaryArgs& r, hipStream_t stream) {
    constexpr int n = 16 / sizeof(T);
    bool wide = divides(r, n);
    for (const HeadsIn* h : {&a.q, &a.k, &a.v}) wide = wide && (!h->p || aligned(h->p, h->ts, h->hs, sizeof(T)));
    for (const HeadsOut* h : {&a.q_out, &a.k_pages, &a.v_pages})
        wide = wide && (!h->p || aligned(h->p, h->ts, h->hs, sizeof(T)));
    return wide ? append<T, n>(a, r, stream) : append<T, 1>(a, r, stream);
}

}  // namespace
}  // namespace fa

hipError_t launch_rotary(int dtype, int64_t tokens, int heads, const HeadsIn& x, const HeadsOut& out,
                         const RotaryArgs& r, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16) return fa::rotary_of<_Float16>(tokens, heads, x, out, r, stream);
    if (dtype == DCN_DTYPE_BF16) return fa::rotary_of<fa::bf16>(tokens, heads, x, out, r, stream);
    return fa::rotary_of<float>(tokens, heads, x, out, r, stream);
}

hipError_t launch_append(int dtype, const AppendArgs& a, const RotaryArgs& r, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16) return fa::append_of<_Float16>(a, r, stream);
    if (dtype == DCN_DTYPE_BF16) return fa::append_of<fa::bf16>(a, r, stream);
    return fa::append_of<float>(a, r, stream);
}

}  // namespace dcn
