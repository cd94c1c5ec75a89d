// Device helpers of the frame-attention kernels (gfx950 only).
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

#include "dcn_attention.hpp"
#include "dcn_internal.hpp"

namespace dcn {
namespace fa {

typedef __bf16 bf16;

template <typename T>
__device__ __forceinline__ float widen(T v) {
    return (float)v;
}
// One rounding, to nearest even. FP16 through round_f16: a conversion folded into the
// operation before it (v_fma_mixlo_f16) is off by a whole step on subnormal results.
template <typename T>
__device__ __forceinline__ T narrow(float v) {
    if constexpr (__is_same(T, _Float16)) return round_f16(v);
    return (T)v;
}

// The rows of one sequence, whatever the index arrays hold: inside [0, tokens).
struct Run {
    int64_t first;
    int count;
};
__device__ __forceinline__ Run run_of(const int32_t* cu, int s, int each, int64_t tokens) {
    if (!cu) return Run{(int64_t)s * each, each};
    int64_t a = cu[s], b = cu[s + 1];
    a = a < 0 ? 0 : (a > tokens ? tokens : a);
    b = b < a ? a : (b > tokens ? tokens : b);
    return Run{a, (int)(b - a)};
}
__device__ __forceinline__ Run kv_run_of(const AttentionArgs& a, int s) {
    if (!a.pages.table) return run_of(a.cu_kv, s, a.max_kv, a.kv_tokens);
    const int64_t most = (int64_t)a.pages.width << a.pages.shift;
    int64_t n = a.cu_kv[s];
    n = n < 0 ? 0 : (n > most ? most : n);
    return Run{0, (int)n};
}

// Keys that the query at position p sees: [0, sink) and [lo, hi), sink <= lo, of n keys.
struct Span {
    int sink, lo, hi;
};
__device__ __forceinline__ Span span_of(const AttentionArgs& a, int p, int n) {
    if (p < 0) return Span{0, 0, 0};
    const int64_t f = p / a.frame, fr = a.frame;
    int64_t hi = a.ahead < 0 ? n : (f + a.ahead + 1) * fr;
    hi = hi > n ? n : hi;
    int64_t lo = a.back < 0 ? 0 : (f - a.back) * fr;
    lo = lo < 0 ? 0 : (lo > hi ? hi : lo);
    int64_t sink = (int64_t)a.sinks * fr;
    sink = sink > lo ? lo : sink;
    return Span{(int)sink, (int)lo, (int)hi};
}
__device__ __forceinline__ bool sees(const Span& s, int j) { return j < s.hi && (j >= s.lo || j < s.sink); }

// Positions that see key j: [from, to), and from `from` on without an end for a sink.
struct Seen {
    int from, to;
};
__device__ __forceinline__ Seen seen_of(const AttentionArgs& a, int j, int n) {
    const int64_t f = j / a.frame, fr = a.frame;
    int64_t from = a.ahead < 0 ? 0 : (f - a.ahead) * fr, to = a.back < 0 || f < a.sinks ? n : (f + a.back + 1) * fr;
    from = from < 0 ? 0 : (from > n ? n : from);
    to = to > n ? n : to;
    return Seen{(int)from, (int)to};
}

// Row of token j of sequence s in the paged cache, in tokens of the pool, or -1.
__device__ __forceinline__ int64_t paged_row(const PagesArgs& pg, int s, int j) {
    const int page = pg.table[(int64_t)s * pg.width + (j >> pg.shift)];
    if ((unsigned)page >= (unsigned)pg.pages) return -1;
    return ((int64_t)page << pg.shift) + (j & ((1 << pg.shift) - 1));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

}  // namespace fa
}  // namespace dcn
