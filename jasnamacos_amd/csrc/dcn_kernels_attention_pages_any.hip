// Attention over microscaled pages, or with a prefix that the sequences share, of any type, head
// size (microscaled: multiples of 32), stride and alignment. The 16-bit heads of 64 and 128 channels have
// kernels of their own; this takes the rest, one query row a workgroup and its keys straight from memory.
//
// Keys are counted through: the prefix's P first, then the sequence's own, whose places in memory
// two tables give. The four waves take 64 visible keys in turn: a lane has one key's score, then
// the lanes have the channels and the weights go round. The running maximum, the sum and the output
// are FP32; the waves are joined through LDS. What a row does not see is not read.
#include "dcn_attention_mfma.hpp"
#include "dcn_mx.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr int kMaxDim = DCN_ATTENTION_MAX_HEAD_DIM;

// Where key j of the prefix and a sequence lies: the row of the pool, or -1.
template <int BITS>
__device__ __forceinline__ int64_t key_row(const PagesAttention& p, int s, int kh, int prefix, int j) {
    const PagesArgs& pg = j < prefix ? p.prefix : p.a.pages;
    const int seq = j < prefix ? 0 : s, at = j < prefix ? j : j - prefix;
    if constexpr (BITS == 0)
        return paged_row(pg, seq, at);
    else
        return mx_row(pg, p.mx.heads, seq, kh, at);
}
__device__ __forceinline__ int prefix_of(const PagesAttention& p) {
    if (!p.prefix.table) return 0;
    const int n = *p.prefix_len;
    return n < 0 ? 0 : (n > p.max_prefix ? p.max_prefix : n);
}

// Channels at .. at + 7 of a row, as FP32.
template <typename T, int BITS>
__device__ __forceinline__ void load8(const PagesAttention& p, bool value, int kh, int64_t row, int at, int dim, float* x) {
    if constexpr (BITS == 0) {
        const HeadsIn& h = value ? p.a.v : p.a.k;
        const T* from = (const T*)h.p + row * h.ts + kh * h.hs;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = at + i < dim ? widen(from[at + i]) : 0.f;
    } else {
        const uint8_t *codes = (value ? p.mx.v : p.mx.k) + (row * dim + at) * BITS / 8, *scales = value ? p.mx.vs : p.mx.ks;
        const float factor = mx_factor(scales[row * (dim / 32) + at / 32]);
        if constexpr (BITS == 8) {
            const mx_u32x2 w = *(const mx_u32x2*)codes;
            mx_decode32<8>(w[0], factor, x);
            mx_decode32<8>(w[1], factor, x + 4);
        } else {
            mx_decode32<4>(*(const uint32_t*)codes, factor, x);
        }
    }
}
template <typename T, int BITS>
__device__ __forceinline__ float load1(const PagesAttention& p, bool value, int kh, int64_t row, int ch, int dim) {
    if constexpr (BITS == 0) {
        const HeadsIn& h = value ? p.a.v : p.a.k;
        return widen(((const T*)h.p)[row * h.ts + kh * h.hs + ch]);
    } else {
        const uint8_t *codes = value ? p.mx.v : p.mx.k, *scales = value ? p.mx.vs : p.mx.ks;
        const float factor = mx_factor(scales[row * (dim / 32) + ch / 32]);
        float x[8];
        mx_decode32<BITS>(codes[(row * dim + ch) * BITS / 8], factor, x);
        return x[BITS == 8 ? 0 : ch & 1];
    }
}

template <typename T, int BITS>
__global__ __launch_bounds__(kThreads) void attention_pages_any_kernel(PagesAttention p, int64_t first) {
    __shared__ float q[kMaxDim], out[kWaves][kMaxDim], top_of[kWaves], sum_of[kWaves];
    const AttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int64_t item = first + blockIdx.x, token = item / a.q_heads;
    const int head = (int)(item - token * a.q_heads), kh = head / a.group;
    int s;
    if (a.cu_q) {
        s = find_sequence(a.cu_q, a.sequences, token);
    } else {
        const int64_t n = token / a.max_q;
        if (n >= a.sequences) return;
        s = (int)n;
    }
    const Run run = run_of(a.cu_q, s, a.max_q, a.q_tokens), kv = kv_run_of(a, s);
    const int64_t in = token - run.first;
    if (in < 0 || in >= run.count || in >= a.max_q) return;
    const int prefix = prefix_of(p), keys = prefix + kv.count;
    const Span sp = span_of(a, keys - run.count + (int)in, keys);
    for (int i = threadIdx.x; i < a.dim; i += kThreads)
        q[i] = widen(((const T*)a.q.p)[token * a.q.ts + head * a.q.hs + i]) * a.scale * kLog2e;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[kMaxDim / 64] = {};
    const int near = (sp.sink + 63) / 64, lo = sp.lo / 64 < near ? near : sp.lo / 64, end = (sp.hi + 63) / 64;
    for (int i = wave; i < near + (end > lo ? end - lo : 0); i += kWaves) {
        const int t0 = (i < near ? i : lo + (i - near)) * 64, j = t0 + lane;
        const int64_t row = sees(sp, j) ? key_row<BITS>(p, s, kh, prefix, j) : -1;
        float score = -INFINITY;
        if (row >= 0) {
            score = 0.f;
            for (int at = 0; at < a.dim; at += 8) {
                float x[8];
                load8<T, BITS>(p, false, kh, row, at, a.dim, x);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (BITS || at + e < a.dim) score = fmaf(q[at + e], x[e], score);
            }
        }
        const float top = fmaxf(m, wave_max(score)), ref = top == -INFINITY ? 0.f : top;
        const float old = exp2f(m - ref), w = row >= 0 ? exp2f(score - ref) : 0.f;
        m = top;
        l = l * old + wave_sum(w);
#pragma unroll
        for (int c = 0; c < kMaxDim / 64; ++c) o[c] *= old;
        for (unsigned long long left = __ballot(row >= 0); left; left &= left - 1) {
            const int k = __builtin_ctzll(left);
            const float weight = __shfl(w, k);
            const int64_t at = __shfl(row, k);
#pragma unroll
            for (int c = 0; c < kMaxDim / 64; ++c)
                if (lane + 64 * c < a.dim) o[c] = fmaf(weight, load1<T, BITS>(p, true, kh, at, lane + 64 * c, a.dim), o[c]);
        }
    }
    if (lane == 0) {
        top_of[wave] = m;
        sum_of[wave] = l;
    }
#pragma unroll
    for (int c = 0; c < kMaxDim / 64; ++c)
        if (lane + 64 * c < a.dim) out[wave][lane + 64 * c] = o[c];
    __syncthreads();
    float most = top_of[0], sum = 0.f, f[kWaves];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) most = fmaxf(most, top_of[w]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        f[w] = exp2f(top_of[w] - (most == -INFINITY ? 0.f : most));
        sum = fmaf(f[w], sum_of[w], sum);
    }
    const bool empty = most == -INFINITY && sum == 0.f;
    const float inv = empty ? 0.f : 1.f / sum;
    for (int i = threadIdx.x; i < a.dim; i += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v = fmaf(f[w], out[w][i], v);
        ((T*)a.out.p)[token * a.out.ts + head * a.out.hs + i] = narrow<T>(v * inv);
    }
    if (a.lse && threadIdx.x == 0) a.lse[token * a.q_heads + head] = empty ? -INFINITY : (most + log2f(sum)) * kLn2;
}

template <typename T, int BITS>
hipError_t any(const PagesAttention& p, hipStream_t stream) {
    const int64_t items = p.a.q_tokens * p.a.q_heads, most = kMostThreads / kThreads;
    for (int64_t first = 0; first < items; first += most) {
        const int64_t n = items - first < most ? items - first : most;
        attention_pages_any_kernel<T, BITS><<<dim3((unsigned)n), kThreads, 0, stream>>>(p, first);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}
template <typename T>
hipError_t any_of(const PagesAttention& p, hipStream_t stream) {
    return p.mx.bits == 8 ? any<T, 8>(p, stream) : (p.mx.bits == 4 ? any<T, 4>(p, stream) : any<T, 0>(p, stream));
}

}  // namespace
}  // namespace fa

hipError_t launch_attention_pages_any(int dtype, const PagesAttention& p, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16) return fa::any_of<_Float16>(p, stream);
    if (dtype == DCN_DTYPE_BF16) return fa::any_of<fa::bf16>(p, stream);
    return fa::any_of<float>(p, stream);
}

}  // namespace dcn
