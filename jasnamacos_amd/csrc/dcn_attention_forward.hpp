// Attention forward on the matrix cores: one wave's rows over a tile of keys in LDS, and the parts
// of a row whose keys several workgroups share.
#pragma once

#include "dcn_attention_mfma.hpp"

namespace dcn {
namespace fa {
namespace {

// A weight is 2^(score - maximum + kLift): FP16 keeps weights of 2^-20 of the largest normal.
template <typename T>
constexpr float kLift = __is_same(T, _Float16) ? 6.f : 0.f;
constexpr float kSlack = 8.f;
// Weights are rounded to T for the product with the values, half a step each (BF16 2^-8 of a weight, FP16 2^-11):
// FP32 products have a sixteenth of the 16-bit ones' rate. Their sum is of the unrounded ones. The outputs are
// 1.2 to 1.45 times as far from 64 bits as with FP32 weights, most of it being their own rounding.

// One wave's 32 rows: queries, sums and the running maximum.
template <typename T, int D>
struct RowState {
    u32x4 q[D / 16];
    f32x16 o[D / 32];
    float m, l;  // m: in units of log2, over the scaled scores
    Span sp;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
        m = -INFINITY;
        l = 0.f;
    }
    // The queries are there: no wait for them later, which would wait for the copies too.
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(q[i]));
    }
    // ROWS keys from t0. masked: some row may not see some key (holes: bit per key that is not there).
    // BY_HALF: 32 keys' reads at a time, for kernels whose registers the reads of 64 do not fit.
    template <int ROWS, bool BY_HALF = false>
    __device__ __forceinline__ void add(const char* kt, const char* vt, int t0, float c, bool masked, unsigned long long holes,
                                        int lane) {
        constexpr int MB = ROWS / 32;
        using Ti = Tile<D>;
        f32x16 s[MB];
        // All reads of a product are in flight before its first step, those of the values before
        // the softmax: left to itself the compiler keeps two, and each step waits for LDS.
        {
            u32x4 kf[MB][D / 16];
            if constexpr (!BY_HALF)
#pragma unroll
                for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) kf[mb][i] = Ti::rows(kt, mb, i, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                if constexpr (BY_HALF) {
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) kf[mb][i] = Ti::rows(kt, mb, i, lane);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) s[mb][r] = 0.f;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) s[mb] = mma<T>(kf[mb][i], q[i], s[mb]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        constexpr int early = D == 64 ? MB * 2 : MB;  // steps whose values are read before the softmax
        u32x4 vf[MB * 2][D / 32];
#pragma unroll
        for (int st = 0; st < early; ++st)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) vf[st][i] = Ti::columns(vt, st >> 1, st & 1, i, lane);
        __builtin_amdgcn_sched_barrier(0);
        if (masked) {
            const unsigned long long seen = (seen_bits(sp, t0) & ~holes) >> (4 * (lane >> 5));
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[mb][r] = keep_or(s[mb][r], spread_bit(seen, 32 * mb + 8 * (r >> 2) + (r & 3)), -INFINITY);
        }
        float top = s[0][0];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[mb][r]);
        top = both_max(top) * c;
        const bool raise = top > m + kSlack;
        if (__builtin_expect(__any(raise), 0)) {
            const float next = raise ? top : m;  // the other rows stay: no row's bits go by its neighbours'
            const float old = exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= old;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= old;
        }
        const float ref = kLift<T> - (m == -INFINITY ? 0.f : m);
        float sum[4] = {};
        u32x4 p[MB * 2];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[mb][r] = __builtin_amdgcn_exp2f(fmaf(s[mb][r], c, ref));
                sum[r & 3] += s[mb][r];
            }
            p[2 * mb] = pack8<T>(s[mb], 0);
            p[2 * mb + 1] = pack8<T>(s[mb], 8);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int st = early; st < MB * 2; ++st)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) vf[st][i] = Ti::columns(vt, st >> 1, st & 1, i, lane);
#pragma unroll
        for (int st = 0; st < MB * 2; ++st)
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] = mma<T>(vf[st][i], p[st], o[i]);
    }
};

// A row's result, or its part (splits > 1): FP32 sums with the weights' reference.
template <typename T, int D>
__device__ __forceinline__ void store_row4(const AttentionArgs& a, const Place& pl, int64_t index, int64_t row, int head, int at,
                                           const float* o, float inv) {
    if (pl.splits == 1) {
        typedef T four __attribute__((ext_vector_type(4)));
        four v;
#pragma unroll
        for (int b = 0; b < 4; ++b) v[b] = narrow<T>(o[b] * inv);
        *(four*)((T*)a.out.p + row * a.out.ts + head * a.out.hs + at) = v;
    } else {
        float* w = (float*)a.workspace + (index * pl.splits + pl.split) * (D + 4) + at;
        *(f32x4*)w = f32x4{o[0], o[1], o[2], o[3]};
    }
}
template <int D>
__device__ __forceinline__ void store_sums(const AttentionArgs& a, const Place& pl, int64_t index, float m, float l, float lift) {
    if (pl.splits == 1) {
        if (a.lse) a.lse[index] = l == 0.f ? -INFINITY : (m - lift + __builtin_amdgcn_logf(l)) * kLn2;
    } else {
        float* w = (float*)a.workspace + (index * pl.splits + pl.split) * (D + 4) + D;
        w[0] = m;
        w[1] = l;
    }
}

// The parts of all splits (32 at most) of a row and head, by PER waves: lane s of each has split
// s's maximum and sum; the waves take the splits' sums in turn and are added in order.
template <typename T, int D, int PER>
__global__ __launch_bounds__(kThreads) void attention_join_kernel(AttentionArgs a, int splits) {
    typedef float vec __attribute__((ext_vector_type(2)));
    constexpr int N = D / 64;
    __shared__ vec sums[kWaves][64];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const Run q = run_of(a.cu_q, blockIdx.z, a.max_q, a.q_tokens);
    const int64_t item = (int64_t)blockIdx.x * (kWaves / PER) + wave / PER;
    const int tok = (int)(item / a.q_heads), head = (int)(item % a.q_heads);
    const bool there = tok < q.count && tok < a.max_q;
    const int64_t row = q.first + (there ? tok : 0), index = row * a.q_heads + head;
    const float* parts = (const float*)a.workspace + index * splits * (D + 4);
    float m = -INFINITY, l = 0.f;
    if (there && lane < splits) {
        m = parts[lane * (D + 4) + D];
        l = parts[lane * (D + 4) + D + 1];
    }
    const float top = wave_max(m);
    const float w = exp2f(m - (top == -INFINITY ? 0.f : top)), sum = wave_sum(w * l);
    float o[2] = {};
    if (there) {
        const float* at = parts + lane * N;
        for (int s = wave % PER; s < splits; s += 4 * PER) {
            // Four splits' loads at once.
            float v[4][N];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i) v[u][i] = s + u * PER < splits ? at[(s + u * PER) * (D + 4) + i] : 0.f;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float ws = __shfl(w, (s + u * PER) & 63);
#pragma unroll
                for (int i = 0; i < N; ++i) o[i] = s + u * PER < splits ? fmaf(ws, v[u][i], o[i]) : o[i];
            }
        }
    }
    if constexpr (PER > 1) {
        sums[wave][lane] = vec{o[0], o[1]};
        __syncthreads();
        if (wave % PER) return;
#pragma unroll
        for (int g = 1; g < PER; ++g) {
            o[0] += sums[wave + g][lane][0];
            o[1] += sums[wave + g][lane][1];
        }
    }
    if (!there) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = (T*)a.out.p + row * a.out.ts + head * a.out.hs + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = narrow<T>(o[i] * inv);
    if (a.lse && lane == 0) a.lse[index] = sum == 0.f ? -INFINITY : (top - kLift<T> + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace
}  // namespace fa
}  // namespace dcn
