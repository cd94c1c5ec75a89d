// Gradients of frame attention one row at a time, for heads of 129 to 256 channels: FP16, BF16 and
// FP32, any stride and alignment. Smaller heads have tiled kernels, of whose sums these are the
// plain statement.
//
// One wave per query row, or per key row for the gradients of keys and values. A pass handles
// 64 rows of the other side: lane = row for the dot products (the wave's own vector is in LDS as
// FP32), then lane = channel for the weighted sum, the 64 weights in LDS. Rows that do not see each
// other are never read, so nothing in them can reach the result. Bound: the dot products' strided
// loads (1,024 causal tokens, 8 heads of 256: FP32 11.4 ms, BF16 10.9).
#include "dcn_attention_device.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr int kWave = 64;
constexpr int kMaxDim = DCN_ATTENTION_MAX_HEAD_DIM;
constexpr int kPer = kMaxDim / kWave;  // channels a lane owns at most

template <typename T>
__device__ __forceinline__ float dot(const float* a, const T* b, int dim) {
    float s = 0.f;
    for (int d = 0; d < dim; ++d) s = fmaf(a[d], widen(b[d]), s);
    return s;
}

template <typename T>
__device__ __forceinline__ const T* kv_row(const HeadsIn& h, const Run& kv, int head, int j) {
    return (const T*)h.p + (kv.first + j) * h.ts + head * h.hs;
}

// The two intervals that a row sees as one index range: i < sink is key i, else lo + i - sink.
__device__ __forceinline__ int span_key(const Span& sp, int i) { return i < sp.sink ? i : sp.lo + (i - sp.sink); }
__device__ __forceinline__ int span_size(const Span& sp) { return sp.sink + (sp.hi - sp.lo); }

// delta[row][head] = sum of dout * out, and dq = scale * sum over keys of dS k.
template <typename T>
__global__ __launch_bounds__(kWave) void attention_row_dq_kernel(AttentionArgs a) {
    __shared__ float qs[kMaxDim], dos[kMaxDim], ps[kWave];
    __shared__ const T* ks[kWave];
    const int lane = threadIdx.x, s = blockIdx.z, head = blockIdx.y, i = blockIdx.x;
    const Run q = run_of(a.cu_q, s, a.max_q, a.q_tokens);
    if (i >= q.count) return;
    const Run kv = kv_run_of(a, s);
    const int64_t row = q.first + i;
    const Span sp = span_of(a, kv.count - q.count + i, kv.count);
    const T* qp = (const T*)a.q.p + row * a.q.ts + head * a.q.hs;
    const T* op = (const T*)a.o.p + row * a.o.ts + head * a.o.hs;
    const T* dp = (const T*)a.dout.p + row * a.dout.ts + head * a.dout.hs;
    float delta = 0.f;
    for (int d = lane; d < a.dim; d += kWave) {
        qs[d] = widen(qp[d]) * a.scale;
        dos[d] = widen(dp[d]);
        delta = fmaf(dos[d], widen(op[d]), delta);
    }
    delta = wave_sum(delta);
    if (lane == 0) ((float*)a.workspace)[row * a.q_heads + head] = delta;
    __syncthreads();
    const float lse = a.lse_in[row * a.q_heads + head];
    const int total = span_size(sp), kh = head / a.group;
    float acc[kPer] = {};
    for (int base = 0; base < total; base += kWave) {
        const bool in = base + lane < total;
        const int j = in ? span_key(sp, base + lane) : 0;
        float ds = 0.f;
        const T* kp = nullptr;
        if (in) {
            kp = kv_row<T>(a.k, kv, kh, j);
            const T* vp = kv_row<T>(a.v, kv, kh, j);
            ds = expf(dot(qs, kp, a.dim) - lse) * (dot(dos, vp, a.dim) - delta);
        }
        ps[lane] = ds;
        ks[lane] = kp;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
            const int d = lane + c * kWave;
            if (d >= a.dim) break;
            for (int n = 0; n < kWave; ++n)
                if (ks[n]) acc[c] = fmaf(ps[n], widen(ks[n][d]), acc[c]);
        }
        __syncthreads();
    }
    T* gp = (T*)a.dq.p + row * a.dq.ts + head * a.dq.hs;
#pragma unroll
    for (int c = 0; c < kPer; ++c)
        if (lane + c * kWave < a.dim) gp[lane + c * kWave] = narrow<T>(acc[c] * a.scale);
}

// dk and dv of one key: the queries that see it lie in [from, to) of the sequence, lane = query.
template <typename T>
__global__ __launch_bounds__(kWave) void attention_row_dkv_kernel(AttentionArgs a) {
    __shared__ float ks[kMaxDim], vs[kMaxDim], ps[kWave], ds[kWave];
    const int lane = threadIdx.x, s = blockIdx.z, kh = blockIdx.y, j = blockIdx.x;
    const Run kv = run_of(a.cu_kv, s, a.max_kv, a.kv_tokens);
    if (j >= kv.count) return;
    const Run q = run_of(a.cu_q, s, a.max_q, a.q_tokens);
    const int64_t row = kv.first + j;
    const T* kp = (const T*)a.k.p + row * a.k.ts + kh * a.k.hs;
    const T* vp = (const T*)a.v.p + row * a.v.ts + kh * a.v.hs;
    for (int d = lane; d < a.dim; d += kWave) {
        ks[d] = widen(kp[d]) * a.scale;
        vs[d] = widen(vp[d]);
    }
    __syncthreads();
    const int off = kv.count - q.count;
    const int64_t fj = j / a.frame, fr = a.frame;
    int64_t from = a.ahead < 0 ? 0 : (fj - a.ahead) * fr, to = kv.count;
    if (a.back >= 0 && fj >= a.sinks) to = (fj + a.back + 1) * fr;
    from = from - off < 0 ? 0 : from - off;
    to = to - off > q.count ? q.count : to - off;
    float dk[kPer] = {}, dv[kPer] = {};
    for (int g = 0; g < a.group; ++g) {
        const int head = kh * a.group + g;
        for (int64_t base = from; base < to; base += kWave) {
            const int64_t i = base + lane;
            float p = 0.f, t = 0.f;
            bool on = false;
            if (i < to) on = sees(span_of(a, (int)(off + i), kv.count), j);
            if (on) {
                const int64_t qr = q.first + i;
                p = expf(dot(ks, (const T*)a.q.p + qr * a.q.ts + head * a.q.hs, a.dim) -
                         a.lse_in[qr * a.q_heads + head]);
                t = p * (dot(vs, (const T*)a.dout.p + qr * a.dout.ts + head * a.dout.hs, a.dim) -
                         ((const float*)a.workspace)[qr * a.q_heads + head]);
            }
            ps[lane] = p;
            ds[lane] = t;
            const unsigned long long seen = __ballot(on);
            __syncthreads();
#pragma unroll
            for (int c = 0; c < kPer; ++c) {
                const int d = lane + c * kWave;
                if (d >= a.dim) break;
                for (int n = 0; n < kWave; ++n) {
                    if (!(seen >> n & 1)) continue;
                    const int64_t qr = q.first + base + n;
                    dv[c] = fmaf(ps[n], widen(((const T*)a.dout.p + qr * a.dout.ts + head * a.dout.hs)[d]), dv[c]);
                    dk[c] = fmaf(ds[n], widen(((const T*)a.q.p + qr * a.q.ts + head * a.q.hs)[d]), dk[c]);
                }
            }
            __syncthreads();
        }
    }
    T* gk = (T*)a.dk.p + row * a.dk.ts + kh * a.dk.hs;
    T* gv = (T*)a.dv.p + row * a.dv.ts + kh * a.dv.hs;
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
        const int d = lane + c * kWave;
        if (d >= a.dim) break;
        gk[d] = narrow<T>(dk[c] * a.scale);
        gv[d] = narrow<T>(dv[c]);
    }
}

template <typename T>
hipError_t rows_backward(const AttentionArgs& a, hipStream_t stream) {
    constexpr int most = (int)((INT64_C(1) << 32) / kWave) - 1;  // fewer than 2^32 threads
    if (a.max_q > most || a.max_kv > most) return hipErrorInvalidConfiguration;
    if (a.max_q > 0) {
        attention_row_dq_kernel<T><<<dim3(a.max_q, a.q_heads, a.sequences), kWave, 0, stream>>>(a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    if (a.max_kv > 0)
        attention_row_dkv_kernel<T><<<dim3(a.max_kv, a.kv_heads, a.sequences), kWave, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace
}  // namespace fa

hipError_t launch_attention_rows_backward(int dtype, const AttentionArgs& a, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16) return fa::rows_backward<_Float16>(a, stream);
    if (dtype == DCN_DTYPE_BF16) return fa::rows_backward<fa::bf16>(a, stream);
    return fa::rows_backward<float>(a, stream);
}

}  // namespace dcn
