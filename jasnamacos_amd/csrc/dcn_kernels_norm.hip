// The norms around a block's residual addition, forward and backward:
//   n = h r1, u = n w_post, x' = x + alpha g u;  m = x' r2, y = m w_pre.
// Backward, with t = dx' + r2 (dy w_pre - m mean(dy w_pre m)) the whole gradient of x':
//   dx = t, dg = alpha sum t u, dw_post = alpha sum t g n, dw_pre = sum dy m,
//   dn = alpha t g w_post, dh = r1 (dn - n mean(dn n)).
// A group of lanes owns a row: its channels stay in registers between the two norms, so
// every tensor is read once and written once. Bound: HBM. 36,000 tokens of 512 BF16 channels: forward
// 37 us, backward 56 us and its joining 7 us (3.8 TB/s over the step; 88 us at the rate of a large
// copy); 64 FP32 tokens: 3.7 us of kernel.
//
// Sums over tokens (dg, dw): a slot (one row's lanes) walks units of rows of one gate
// row, keeping its channels' sums in registers; a unit's dg goes straight out when the
// unit is the whole gate run, else to the workspace; a workgroup's dw goes to the
// workspace, and a second kernel adds the parts in a fixed order.
#include "dcn_attention_device.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;             // adjacent channels a lane owns
constexpr int kMaxGroups = 1024;    // workgroups of the backward: each leaves one row of dw

template <typename T>
struct alignas(16) Pack {
    T v[kVec];
};

// Channels [at, at + 8) of a row, as FP32; zeros past the row's end.
template <typename T, bool WIDE>
__device__ __forceinline__ void load_row(const T* row, int at, int channels, float fill, float* v) {
    if constexpr (WIDE) {
        if (at < channels) {
            const Pack<T> p = *(const Pack<T>*)(row + at);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] = widen(p.v[i]);
            return;
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = fill;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = at + i < channels ? widen(row[at + i]) : fill;
    }
}
template <typename T, bool WIDE>
__device__ __forceinline__ void store_row(T* row, int at, int channels, const float* v) {
    if constexpr (WIDE) {
        if (at < channels) {
            Pack<T> p;
#pragma unroll
            for (int i = 0; i < kVec; ++i) p.v[i] = narrow<T>(v[i]);
            *(Pack<T>*)(row + at) = p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (at + i < channels) row[at + i] = narrow<T>(v[i]);
    }
}

// What rounding x to T takes from it, in 16 bits, and x again. BF16: the distance of the
// FP32 patterns (x is back to the bit, but for ties, one FP32 step off); FP16: 2048 (x - T(x))
// in FP16, 22 bits of x in all.
template <typename T>
__device__ __forceinline__ uint16_t low_half(float x) {
    const T r = narrow<T>(x);
    if constexpr (sizeof(T) == 4) return 0;
    if constexpr (__is_same(T, bf16)) {
        const int d = __builtin_bit_cast(int, x) - (int)((uint32_t)__builtin_bit_cast(uint16_t, r) << 16);
        return (uint16_t)(d > 32767 ? 32767 : d);
    } else {
        const float d = (x - widen(r)) * 2048.f;
        return __builtin_bit_cast(uint16_t, fabsf(d) <= 65504.f ? (_Float16)d : (_Float16)0.f);
    }
}
template <typename T>
__device__ __forceinline__ float with_low(float rounded, uint16_t low) {
    if constexpr (__is_same(T, bf16))
        return __builtin_bit_cast(float, __builtin_bit_cast(int, rounded) + (int)(int16_t)low);
    else
        return fmaf((float)__builtin_bit_cast(_Float16, low), 1.f / 2048.f, rounded);
}

// A row's r1 and r2 in `low`, and its halves.
__device__ __forceinline__ float* low_stats(const NormArgs& a, int64_t row) {
    return (float*)((char*)a.low + row / kLowRows * norm_low_block(a.channels)) + row % kLowRows * 2;
}
__device__ __forceinline__ uint16_t* low_row(const NormArgs& a, int64_t row) {
    return (uint16_t*)((char*)a.low + row / kLowRows * norm_low_block(a.channels) + kLowRows * 8) + row % kLowRows * a.channels;
}

// A lane's channels of one row's tensors, as they are stored: loaded a row ahead.
template <typename T, int NV>
struct RawRow {
    Pack<T> dy[NV], x_out[NV], dx_out[NV], h[NV];
    Pack<uint16_t> low[NV];
    float r1, r2, low1, low2;

    template <bool WIDE, typename U>
    static __device__ __forceinline__ void get(const U* from, int at, int channels, Pack<U>* to) {
        if constexpr (WIDE) {
            if (at < channels) *to = *(const Pack<U>*)(from + at);
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                if (at + i < channels) to->v[i] = from[at + i];
        }
    }
    template <int LANES, bool WIDE>
    __device__ __forceinline__ void load(const NormArgs& a, int64_t row, int lane) {
        const int64_t base = row * a.channels;
        const int c = a.channels;
        r1 = a.rstd[row * 2];
        r2 = a.rstd[row * 2 + 1];
        if (sizeof(T) == 2 && a.low) {
            low1 = low_stats(a, row)[0];
            low2 = low_stats(a, row)[1];
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int at = (n * LANES + lane) * kVec;
            if (a.dy) {
                get<WIDE>((const T*)a.dy + base, at, c, &dy[n]);
                get<WIDE>((const T*)a.x_out + base, at, c, &x_out[n]);
                if (sizeof(T) == 2 && a.low)
                    get<WIDE>((const uint16_t*)low_row(a, row), at, c, &low[n]);
            }
            get<WIDE>((const T*)a.dx_out + base, at, c, &dx_out[n]);
            get<WIDE>((const T*)a.h + base, at, c, &h[n]);
        }
    }
};
// Channel i of a lane's chunk at `at`, zero past the row's end.
template <typename T>
__device__ __forceinline__ float raw(const Pack<T>& p, int i, int at, int channels) {
    return at + i < channels ? widen(p.v[i]) : 0.f;
}

// The sum over a row's LANES lanes, in every one of them.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
#pragma unroll
    for (int m = 1; m < (LANES < 64 ? LANES : 64); m <<= 1) v += __shfl_xor(v, m);
    if constexpr (LANES > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < LANES / 64; ++w) v += scratch[w];
    }
    return v;
}

template <typename T, int LANES, int NV, bool WIDE>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(NormArgs a, int64_t first) {
    __shared__ float scratch[kThreads / 64];
    constexpr int slots = kThreads / LANES;
    const int lane = threadIdx.x % LANES, c = a.channels;
    const int64_t row = first + (int64_t)blockIdx.x * slots + threadIdx.x / LANES;
    if (row >= a.tokens) return;  // whole slots; a row of 256 lanes is the whole workgroup
    const int64_t base = row * c;
    float h[NV][kVec], sum = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        load_row<T, WIDE>((const T*)a.h + base, (n * LANES + lane) * kVec, c, 0.f, h[n]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum = fmaf(h[n][i], h[n][i], sum);
    }
    const float r1 = 1.f / sqrtf(row_sum<LANES>(sum, scratch) / (float)c + a.eps);
    sum = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
        const int at = (n * LANES + lane) * kVec;
        float x[kVec], w[kVec], g[kVec];
        load_row<T, WIDE>((const T*)a.x + base, at, c, 0.f, x);
        if (a.w_post) load_row<T, WIDE>((const T*)a.w_post, at, c, 0.f, w);
        if (a.gate) load_row<T, WIDE>((const T*)a.gate + row / a.gate_tokens * c, at, c, 0.f, g);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            float u = h[n][i] * r1;
            if (a.w_post) u *= w[i];
            if (a.gate) u *= g[i];
            h[n][i] = fmaf(a.alpha, u, x[i]);
            sum = fmaf(h[n][i], h[n][i], sum);
        }
        store_row<T, WIDE>((T*)a.x_out + base, at, c, h[n]);
        if (a.low) {
            uint16_t* to = low_row(a, row);
            if constexpr (WIDE) {
                if (at < c) {
                    Pack<uint16_t> p;
#pragma unroll
                    for (int i = 0; i < kVec; ++i) p.v[i] = low_half<T>(h[n][i]);
                    *(Pack<uint16_t>*)(to + at) = p;
                }
            } else {
                for (int i = 0; i < kVec; ++i)
                    if (at + i < c) to[at + i] = low_half<T>(h[n][i]);
            }
        }
    }
    const float r2 = 1.f / sqrtf(row_sum<LANES>(sum, scratch) / (float)c + a.eps);
    if (a.y) {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int at = (n * LANES + lane) * kVec;
            float w[kVec];
            if (a.w_pre) load_row<T, WIDE>((const T*)a.w_pre, at, c, 0.f, w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                h[n][i] *= r2;
                if (a.w_pre) h[n][i] *= w[i];
            }
            store_row<T, WIDE>((T*)a.y + base, at, c, h[n]);
        }
    }
    if (a.rstd && lane == 0) {
        a.rstd[row * 2] = r1;
        a.rstd[row * 2 + 1] = r2;
    }
    if (a.low && lane == 0) {
        low_stats(a, row)[0] = r1;
        low_stats(a, row)[1] = r2;
    }
}

// How the backward cuts its rows: units of `rows` rows of one gate run, `per_gate` of them
// a run, walked by `groups` workgroups of `slots` slots.
struct Cut {
    int64_t units;
    int rows, per_gate, slots, groups;
};

__host__ __device__ inline int lanes_of(int channels) { return channels <= 128 ? 16 : (channels <= 1024 ? 64 : 256); }

Cut cut_of(int channels, int64_t tokens, int64_t gate_tokens) {
    Cut c{};
    if (tokens <= 0) return c;  // no rows: the join writes zeros
    c.slots = kThreads / lanes_of(channels);
    // About one unit a slot, but no fewer than 4 rows (a unit's dg row costs the workspace
    // two row-sized FP32 passes) and no more than 64.
    int64_t rows = tokens / ((int64_t)kMaxGroups * c.slots) + 1;
    rows = rows < 4 ? 4 : (rows > 64 ? 64 : rows);
    if (rows > gate_tokens) rows = gate_tokens;
    c.rows = (int)rows;
    c.per_gate = (int)((gate_tokens + rows - 1) / rows);
    const int64_t gates = (tokens + gate_tokens - 1) / gate_tokens;
    c.units = gates * c.per_gate;
    const int64_t groups = (c.units + c.slots - 1) / c.slots;
    c.groups = (int)(groups < kMaxGroups ? groups : kMaxGroups);
    return c;
}

template <typename T, int LANES, int NV, bool WIDE>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(NormArgs a, Cut cut, float* gate_parts,
                                                                 float* w_parts) {
    __shared__ float scratch[kThreads / 64];
    __shared__ float sums[kThreads * kVec];
    constexpr int slots = kThreads / LANES;
    const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES, c = a.channels;
    // One vector a lane: weights and gates stay in registers; more: they come from the cache each row.
    constexpr bool keep = NV == 1;
    float dw1[NV][kVec] = {}, dw2[NV][kVec] = {}, w1[keep ? NV : 1][kVec], w2[keep ? NV : 1][kVec], g[keep ? NV : 1][kVec];
    auto factor = [&](const T* row, int n, float* to) {
        if (row) {
            load_row<T, WIDE>(row, (n * LANES + lane) * kVec, c, 0.f, to);
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i) to[i] = 1.f;
        }
    };
    if constexpr (keep) {
        factor((const T*)a.w_post, 0, w1[0]);
        factor((const T*)a.w_pre, 0, w2[0]);
    }
    for (int64_t unit = (int64_t)blockIdx.x * slots + slot; unit < cut.units; unit += (int64_t)gridDim.x * slots) {
        const int64_t gate = unit / cut.per_gate, first = gate * a.gate_tokens;
        const int64_t from = first + (unit - gate * cut.per_gate) * cut.rows;
        int64_t to = from + cut.rows;
        to = to > first + a.gate_tokens ? first + a.gate_tokens : to;
        to = to > a.tokens ? a.tokens : to;
        float dg[NV][kVec] = {};
        const T* gates = a.gate ? (const T*)a.gate + gate * c : nullptr;
        if constexpr (keep) factor(gates, 0, g[0]);
        // Short rows are loaded a row ahead; a long one alone has enough bytes in flight.
        constexpr bool ahead = NV == 1;
        RawRow<T, NV> now, next;
        if (ahead && from < to) next.template load<LANES, WIDE>(a, from, lane);
        for (int64_t row = from; row < to; ++row) {
            const int64_t base = row * c;
            if constexpr (ahead) {
                now = next;
                if (row + 1 < to) next.template load<LANES, WIDE>(a, row + 1, lane);
            } else {
                now.template load<LANES, WIDE>(a, row, lane);
            }
            float t[NV][kVec], m[NV][kVec], sum = 0.f;
            if (a.dy) {
                const bool whole = sizeof(T) == 2 && a.low && now.low1 == now.r1 && now.low2 == now.r2;
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    const int at = (n * LANES + lane) * kVec;
                    if constexpr (!keep) factor((const T*)a.w_pre, n, w2[0]);
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        t[n][i] = raw(now.dy[n], i, at, c);
                        float x = raw(now.x_out[n], i, at, c);
                        if (sizeof(T) == 2 && whole && at + i < c) x = with_low<T>(x, now.low[n].v[i]);
                        m[n][i] = x * now.r2;
                        dw2[n][i] = fmaf(t[n][i], m[n][i], dw2[n][i]);
                        t[n][i] *= w2[keep ? n : 0][i];
                        sum = fmaf(t[n][i], m[n][i], sum);
                    }
                }
                const float mean = row_sum<LANES>(sum, scratch) / (float)c;
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int i = 0; i < kVec; ++i) t[n][i] = now.r2 * fmaf(-mean, m[n][i], t[n][i]);
            }
            sum = 0.f;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int at = (n * LANES + lane) * kVec;
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float d = raw(now.dx_out[n], i, at, c);
                    t[n][i] = a.dy ? t[n][i] + d : d;
                }
                store_row<T, WIDE>((T*)a.dx + base, at, c, t[n]);
                if constexpr (!keep) {
                    factor((const T*)a.w_post, n, w1[0]);
                    factor(gates, n, g[0]);
                }
                const float *w = w1[keep ? n : 0], *gt = g[keep ? n : 0];
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    m[n][i] = raw(now.h[n], i, at, c) * now.r1;
                    const float s = a.alpha * t[n][i];
                    dg[n][i] = fmaf(s * w[i], m[n][i], dg[n][i]);
                    dw1[n][i] = fmaf(s * gt[i], m[n][i], dw1[n][i]);
                    t[n][i] = s * gt[i] * w[i];
                    sum = fmaf(t[n][i], m[n][i], sum);
                }
            }
            const float mean = row_sum<LANES>(sum, scratch) / (float)c;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
#pragma unroll
                for (int i = 0; i < kVec; ++i) t[n][i] = now.r1 * fmaf(-mean, m[n][i], t[n][i]);
                store_row<T, WIDE>((T*)a.dh + base, (n * LANES + lane) * kVec, c, t[n]);
            }
        }
        if (a.dgate) {
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int at = (n * LANES + lane) * kVec;
                if (cut.per_gate == 1) store_row<T, WIDE>((T*)a.dgate + gate * c, at, c, dg[n]);
                else store_row<float, false>(gate_parts + unit * c, at, c, dg[n]);
            }
        }
    }
    // The workgroup's dw: its slots' sums, added in order of the slots.
    for (int which = 0; which < 2; ++which) {
        if (!(which ? a.dw_pre : a.dw_post)) continue;
        float* parts = w_parts + ((int64_t)which * gridDim.x + blockIdx.x) * c;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int at = (n * LANES + lane) * kVec;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kVec; ++i) sums[threadIdx.x * kVec + i] = which ? dw2[n][i] : dw1[n][i];
            __syncthreads();
            if (slot == 0) {
                float v[kVec];
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    v[i] = 0.f;
                    for (int s = 0; s < slots; ++s) v[i] += sums[(s * LANES + lane) * kVec + i];
                }
                store_row<float, false>(parts, at, c, v);
            }
        }
    }
}

// out[channel] = the sum over `count` parts of a row, for 64 channels a workgroup: 16 threads
// have four channels each, 64 groups of them take parts in turn and are added in their order.
constexpr int kJoinThreads = 1024;
template <typename T>
__device__ __forceinline__ void add_parts(const float* parts, int64_t count, int c, T* out, float* sums) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const int at = blockIdx.x * 64 + (threadIdx.x & 15) * 4, group = threadIdx.x >> 4;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (at + 3 < c && c % 4 == 0) {
#pragma unroll 8
        for (int64_t p = group; p < count; p += kJoinThreads / 16) {
            const f32x4 x = *(const f32x4*)(parts + p * c + at);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += x[i];
        }
    } else {
        for (int64_t p = group; p < count; p += kJoinThreads / 16)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] += at + i < c ? parts[p * c + at + i] : 0.f;
    }
    *(f32x4*)(sums + threadIdx.x * 4) = s;
    __syncthreads();
    if (threadIdx.x < 64 && blockIdx.x * 64 + (int)threadIdx.x < c) {
        float t = 0.f;
#pragma unroll 8
        for (int g = 0; g < kJoinThreads / 16; ++g) t += sums[g * 64 + threadIdx.x];
        out[blockIdx.x * 64 + threadIdx.x] = narrow<T>(t);
    }
    __syncthreads();
}

// Rows 0 .. gates - 1: dgate from its units; then dw_post and dw_pre from the workgroups.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void norm_join_kernel(NormArgs a, Cut cut, int gates, const float* gate_parts,
                                                                 const float* w_parts) {
    __shared__ __attribute__((aligned(16))) float sums[kJoinThreads * 4];
    const int64_t c = a.channels;
    for (int row = blockIdx.y; row < gates + 2; row += gridDim.y) {
        if (row < gates) {
            add_parts(gate_parts + (int64_t)row * cut.per_gate * c, cut.per_gate, a.channels, (T*)a.dgate + row * c, sums);
        } else {
            const int which = row - gates;
            float* out = which ? a.dw_pre : a.dw_post;
            if (out) add_parts(w_parts + which * cut.groups * c, cut.groups, a.channels, out, sums);
        }
    }
}

template <typename T, int LANES, int NV, bool WIDE>
hipError_t run(const NormArgs& a, bool backward, hipStream_t stream) {
    if (!backward) {
        constexpr int64_t slots = kThreads / LANES, most = kMostThreads / LANES;  // rows of a workgroup, a launch
        for (int64_t first = 0; first < a.tokens; first += most) {
            const int64_t rows = a.tokens - first < most ? a.tokens - first : most;
            norm_forward_kernel<T, LANES, NV, WIDE><<<(unsigned)((rows + slots - 1) / slots), kThreads, 0, stream>>>(a, first);
            if (hipError_t e = hipGetLastError()) return e;
        }
        return hipSuccess;
    }
    const Cut cut = cut_of(a.channels, a.tokens, a.gate_tokens);
    float* w_parts = a.workspace;
    float* gate_parts = a.workspace + 2 * (int64_t)cut.groups * a.channels;
    if (cut.groups) {
        norm_backward_kernel<T, LANES, NV, WIDE><<<cut.groups, kThreads, 0, stream>>>(a, cut, gate_parts, w_parts);
        if (hipError_t e = hipGetLastError()) return e;
    }
    const int64_t gates = a.dgate && cut.per_gate > 1 ? (a.tokens + a.gate_tokens - 1) / a.gate_tokens : 0;
    if (!gates && !a.dw_post && !a.dw_pre) return hipSuccess;
    const int64_t rows = gates + 2;
    norm_join_kernel<T><<<dim3((a.channels + 63) / 64, (unsigned)(rows < 32768 ? rows : 32768)), kJoinThreads, 0, stream>>>(
        a, cut, (int)gates, gate_parts, w_parts);
    return hipGetLastError();
}

template <typename T, bool WIDE>
hipError_t by_channels(const NormArgs& a, bool backward, hipStream_t stream) {
    const int c = a.channels;
    if (c <= 128) return run<T, 16, 1, WIDE>(a, backward, stream);
    if (c <= 512) return run<T, 64, 1, WIDE>(a, backward, stream);
    if (c <= 1024) return run<T, 64, 2, WIDE>(a, backward, stream);
    if (c <= 2048) return run<T, 256, 1, WIDE>(a, backward, stream);
    if (c <= 4096) return run<T, 256, 2, WIDE>(a, backward, stream);
    return run<T, 256, 4, WIDE>(a, backward, stream);
}

template <typename T>
hipError_t by_alignment(const NormArgs& a, bool backward, hipStream_t stream) {
    bool wide = a.channels % kVec == 0;
    for (const void* p : {a.h, a.x, a.gate, a.w_post, a.w_pre, (const void*)a.x_out, (const void*)a.y, a.dx_out, a.dy,
                          (const void*)a.dh, (const void*)a.dx, (const void*)a.dgate})
        wide = wide && (uintptr_t)p % 16 == 0;
    return wide ? by_channels<T, true>(a, backward, stream) : by_channels<T, false>(a, backward, stream);
}

hipError_t by_type(int dtype, const NormArgs& a, bool backward, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16) return by_alignment<_Float16>(a, backward, stream);
    if (dtype == DCN_DTYPE_BF16) return by_alignment<bf16>(a, backward, stream);
    return by_alignment<float>(a, backward, stream);
}

}  // namespace
}  // namespace fa

hipError_t launch_norm_forward(int dtype, const NormArgs& a, hipStream_t stream) {
    return fa::by_type(dtype, a, false, stream);
}
hipError_t launch_norm_backward(int dtype, const NormArgs& a, hipStream_t stream) {
    return fa::by_type(dtype, a, true, stream);
}
size_t norm_workspace_bytes(int channels, int64_t tokens, int64_t gate_tokens) {
    const fa::Cut c = fa::cut_of(channels, tokens, gate_tokens);
    const int64_t gates = c.per_gate > 1 ? c.units : 0;
    return (size_t)(2 * (int64_t)c.groups + gates) * channels * sizeof(float);
}

}  // namespace dcn
