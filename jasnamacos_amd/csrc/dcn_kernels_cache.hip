// The microscaled cache: the append of rotated keys and values as codes, and the read back.
//
// A block of 32 channels has x^ = code 2^e, e the smallest with max|x| <= 448 2^e (6 2^e in 4 bits). A
// thread has eight channels of a token, four adjacent lanes a block: its largest magnitude (as bits,
// which order as numbers do and put infinities and NaN on top) takes two moves between lanes, the
// scaled conversions round. Both kernels are bound by HBM, small calls by the call itself. A frame of 3,600
// tokens for 8 streams, 8 heads of 64 with queries, appended in 8 bits: 40 us (3.7 of the 5.1 TB/s that a large
// copy reaches; four heads' loads in flight: six 41, eight 61 us; a thread a head, which takes its sines again,
// 97). 4 x 14,400 tokens, 8 heads of 128, read from 8 bits to BF16: 77 us (4.7 TB/s); 256 tokens of 4 heads of 64
// in 4 bits: 3.2 us of kernel.
#include "dcn_mx.hpp"
#include "dcn_tokens.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr int kThreads = kTokenThreads;
constexpr int kBatch = 4;  // heads whose loads are in flight at once

// Where a new token goes: its sequence's page row, -1 if it has none; false: of no sequence.
struct Target {
    int sequence, place;  // place -1: nowhere in the cache
};
template <typename A>
__device__ __forceinline__ bool target_of(const A& a, const int32_t* cu, int64_t token, Target* t) {
    t->sequence = find_sequence(cu, a.sequences, token);
    const int64_t from = cu[t->sequence], to = cu[t->sequence + 1];
    if (token < from || token >= to) return false;
    const int64_t place = (int64_t)a.kv_lens[t->sequence] - (to - token);
    t->place = place >= 0 && place < (int64_t)a.pages.width << a.pages.shift ? (int)place : -1;
    return true;
}

// The larger of a value's bits over four adjacent lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    const uint32_t a = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true);  // lanes 1 0 3 2
    v = v > a ? v : a;
    const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true);  // lanes 2 3 0 1
    return v > b ? v : b;
}

// The rotation of channels at .. at + 7. A channel is fma(a, u, b v) of its pair's two, a first: u, v are
// cosine and minus sine for the first of a pair, sine and cosine for the second.
template <bool WIDE>
struct Turn8 {
    float u[8], v[8];
    int a[WIDE ? 1 : 8], b[WIDE ? 1 : 8];  // where the two are (WIDE: those of the first channel); b < 0: the channel passes
    bool inside;                           // WIDE: pairs inside the eight channels: u cosines, v sines

    __device__ __forceinline__ void pass(int at) {
        inside = false;
#pragma unroll
        for (int i = 0; i < (WIDE ? 1 : 8); ++i) {
            a[i] = at + i;
            b[i] = -1;
        }
    }
    __device__ __forceinline__ void set(const RotaryArgs& r, int at, const int32_t* pos) {
        pass(at);
        if constexpr (WIDE) {
            if (at >= 2 * r.pairs) return;
            inside = r.interleaved;
            const bool second = !inside && at >= r.pairs;
            const int first = inside ? at >> 1 : (second ? at - r.pairs : at);
            if (!inside) {
                a[0] = first;
                b[0] = first + r.pairs;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < (inside ? 4 : 8)) take(r, pos, first + i, second, inside, i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int ch = at + i;
                if (ch >= 2 * r.pairs) continue;
                const bool second = r.interleaved ? ch & 1 : ch >= r.pairs;
                const int pair = r.interleaved ? ch >> 1 : (second ? ch - r.pairs : ch);
                a[i] = r.interleaved ? ch & ~1 : pair;
                b[i] = r.interleaved ? ch | 1 : pair + r.pairs;
                take(r, pos, pair, second, false, i);
            }
        }
    }
    __device__ __forceinline__ void take(const RotaryArgs& r, const int32_t* pos, int pair, bool second, bool plain, int i) {
        float c, s;
        turn(r, pos, pair, &c, &s);
        u[i] = second ? s : c;
        v[i] = plain ? s : (second ? c : -s);
    }
};

// Eight values as codes, and their block's scale where the lane is the first of its four.
template <typename T, int BITS>
__device__ __forceinline__ void store_codes(const MxArgs& mx, bool value, int64_t row, int dim, int at, float* z) {
    constexpr uint32_t infinity = 0x7f800000u;
    const float most = mx_most<T, BITS>();
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __builtin_bit_cast(uint32_t, z[i]) & 0x7fffffffu;
        top = bits > top ? bits : top;
    }
    top = quad_max(top);
    // Rare: a block that reads as NaN, or magnitudes past the largest (whose clamped bits are its own then).
    const bool bad = top >= infinity;
    const uint32_t limit = __builtin_bit_cast(uint32_t, most);
    if (__builtin_expect(__any(top > limit), 0)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = bad ? 0.f : fminf(fmaxf(z[i], -most), most);
        top = top > limit ? limit : top;
    }
    const uint32_t scale = bad ? kMxNan : mx_scale<BITS>(top);
    const mx_u32x2 codes = mx_encode<BITS>(z, mx_factor(bad ? 127 : scale));
    uint8_t* to = (value ? mx.v : mx.k) + (row * dim + at) * BITS / 8;
    if constexpr (BITS == 8)
        *(mx_u32x2*)to = codes;
    else
        *(uint32_t*)to = codes[0];
    if ((at & 31) == 0) (value ? mx.vs : mx.ks)[row * (dim / 32) + at / 32] = (uint8_t)scale;
}

// One thread: eight channels of one new token, over the heads blockIdx.y, blockIdx.y + gridDim.y, ...: q's, then
// k's, then v's. Sines and cosines cost more than a head's copy, so they are taken once for all heads.
template <typename T, int BITS, bool WIDE>
__global__ __launch_bounds__(kThreads) void append_mx_kernel(RotaryArgs r, AppendArgs a, MxArgs mx, int64_t first) {
    const int chunks = r.dim / 8;
    const int64_t item = first + (int64_t)blockIdx.x * kThreads + threadIdx.x, given = item / chunks;
    const int64_t token = given < a.tokens ? given : a.tokens - 1;
    Target t;
    if (!target_of(a, a.cu_q, token, &t) || given >= a.tokens) return;
    const int64_t row0 = t.place < 0 ? -1 : mx_row(a.pages, mx.heads, t.sequence, 0, t.place);
    const int at = (int)(item - given * chunks) * 8, nq = a.q.p ? a.q_heads : 0, nk = a.kv_heads, step = gridDim.y;
    const int heads = row0 < 0 ? nq : nq + 2 * nk, turned = row0 < 0 ? nq : nq + nk;
    if ((int)blockIdx.y >= heads) return;
    Turn8<WIDE> turns;
    turns.pass(at);
    if ((int)blockIdx.y < turned) turns.set(r, at, r.positions + token * 3);
    for (int h0 = blockIdx.y; h0 < heads; h0 += kBatch * step) {
        T x[kBatch][8], y[kBatch][8];
        // The loads of all heads before the first is used.
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int h = h0 + u * step;
            if (h >= heads) continue;
            const HeadsIn& in = h < nq ? a.q : (h < nq + nk ? a.k : a.v);
            const T* p = (const T*)in.p + token * in.ts + (h < nq ? h : (h < nq + nk ? h - nq : h - nq - nk)) * in.hs;
            const bool turn = h < turned;
            if constexpr (WIDE) {
                Vec<T, 8>::load(p + (turn ? turns.a[0] : at), x[u]);
                if (turn && turns.b[0] >= 0) Vec<T, 8>::load(p + turns.b[0], y[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[u][i] = p[turn ? turns.a[i] : at + i];
                    if (turn && turns.b[i] >= 0) y[u][i] = p[turns.b[i]];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int h = h0 + u * step;
            if (h >= heads) break;
            float z[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = widen(x[u][i]);
            if (h < turned) {
                if (turns.inside) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = z[2 * i], q = z[2 * i + 1];
                        z[2 * i] = fmaf(p, turns.u[i], -(q * turns.v[i]));
                        z[2 * i + 1] = fmaf(p, turns.v[i], q * turns.u[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (turns.b[WIDE ? 0 : i] >= 0) z[i] = fmaf(z[i], turns.u[i], widen(y[u][i]) * turns.v[i]);
                }
            }
            if (h < nq) {
                T out[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) out[i] = narrow<T>(z[i]);
                T* to = (T*)a.q_out.p + token * a.q_out.ts + h * a.q_out.hs + at;
                if constexpr (WIDE) {
                    Vec<T, 8>::store(to, out);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) to[i] = out[i];
                }
            } else {
                const bool value = h >= nq + nk;
                store_codes<T, BITS>(mx, value, row0 + ((int64_t)(value ? h - nq - nk : h - nq) << a.pages.shift), r.dim, at, z);
            }
        }
    }
}

// One thread: 16 channels of one head of one token, of keys and of values.
template <typename T, int BITS, bool WIDE>
__global__ __launch_bounds__(kThreads) void cache_read_kernel(ReadArgs a, MxArgs mx, int64_t first) {
    const int chunks = mx.dim / 16, each = chunks * mx.heads;
    const int64_t item = first + (int64_t)blockIdx.x * kThreads + threadIdx.x, given = item / each;
    const int64_t token = given < a.tokens ? given : a.tokens - 1;
    Target t;
    if (!target_of(a, a.cu, token, &t) || given >= a.tokens || t.place < 0) return;
    const int in = (int)(item - given * each), head = in / chunks, at = (in - head * chunks) * 16;
    const int64_t row = mx_row(a.pages, mx.heads, t.sequence, head, t.place);
    if (row < 0) return;
    constexpr int WORDS = BITS / 2;  // of 16 codes
    typedef uint32_t words __attribute__((ext_vector_type(WORDS)));
    const words kc = *(const words*)(mx.k + (row * mx.dim + at) * BITS / 8), vc = *(const words*)(mx.v + (row * mx.dim + at) * BITS / 8);
    const float kf = mx_factor(mx.ks[row * (mx.dim / 32) + at / 32]), vf = mx_factor(mx.vs[row * (mx.dim / 32) + at / 32]);
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const words codes = part ? vc : kc;
        const float factor = part ? vf : kf;
        const HeadsOut& out = part ? a.v : a.k;
        T* to = (T*)out.p + token * out.ts + head * out.hs + at;
        T x[16];
        if constexpr (__is_same(T, float)) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) mx_decode32<BITS>(codes[w], factor, x + w * (32 / BITS));
        } else {
            typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                uint32_t two[16 / BITS];
                mx_decode<T, BITS>(codes[w], factor, two);
#pragma unroll
                for (int i = 0; i < 16 / BITS; ++i) {
                    const pair p = __builtin_bit_cast(pair, two[i]);
                    x[w * (32 / BITS) + 2 * i] = p[0];
                    x[w * (32 / BITS) + 2 * i + 1] = p[1];
                }
            }
        }
        constexpr int N = WIDE ? 16 / sizeof(T) : 1;
#pragma unroll
        for (int i = 0; i < 16; i += N) Vec<T, N>::store(to + i, x + i);
    }
}

template <typename T, int BITS, bool WIDE>
hipError_t append_mx(const AppendArgs& a, const MxArgs& mx, const RotaryArgs& r, hipStream_t stream) {
    return in_launches(a.tokens * (r.dim / 8), (a.q.p ? a.q_heads : 0) + 2 * a.kv_heads, [&](int64_t first, dim3 grid) {
        append_mx_kernel<T, BITS, WIDE><<<grid, kThreads, 0, stream>>>(r, a, mx, first);
    });
}

template <typename T, int BITS>
hipError_t append_mx_of(const AppendArgs& a, const MxArgs& mx, const RotaryArgs& r, hipStream_t stream) {
    bool wide = divides(r, 8);
    for (const HeadsIn* h : {&a.q, &a.k, &a.v}) wide = wide && (!h->p || aligned(h->p, h->ts, h->hs, sizeof(T)));
    if (a.q.p) wide = wide && aligned(a.q_out.p, a.q_out.ts, a.q_out.hs, sizeof(T));
    return wide ? append_mx<T, BITS, true>(a, mx, r, stream) : append_mx<T, BITS, false>(a, mx, r, stream);
}

template <typename T, int BITS>
hipError_t read_of(const ReadArgs& a, const MxArgs& mx, hipStream_t stream) {
    const int64_t items = a.tokens * mx.heads * (mx.dim / 16);
    const bool wide = aligned(a.k.p, a.k.ts, a.k.hs, sizeof(T)) && aligned(a.v.p, a.v.ts, a.v.hs, sizeof(T));
    return in_launches(items, 1, [&](int64_t first, dim3 grid) {
        if (wide) cache_read_kernel<T, BITS, true><<<grid, kThreads, 0, stream>>>(a, mx, first);
        else cache_read_kernel<T, BITS, false><<<grid, kThreads, 0, stream>>>(a, mx, first);
    });
}

}  // namespace
}  // namespace fa

hipError_t launch_append_mx(int dtype, const AppendArgs& a, const MxArgs& mx, const RotaryArgs& r, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16)
        return mx.bits == 8 ? fa::append_mx_of<_Float16, 8>(a, mx, r, stream) : fa::append_mx_of<_Float16, 4>(a, mx, r, stream);
    if (dtype == DCN_DTYPE_BF16)
        return mx.bits == 8 ? fa::append_mx_of<fa::bf16, 8>(a, mx, r, stream) : fa::append_mx_of<fa::bf16, 4>(a, mx, r, stream);
    return mx.bits == 8 ? fa::append_mx_of<float, 8>(a, mx, r, stream) : fa::append_mx_of<float, 4>(a, mx, r, stream);
}

hipError_t launch_cache_read(int dtype, const ReadArgs& a, const MxArgs& mx, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16)
        return mx.bits == 8 ? fa::read_of<_Float16, 8>(a, mx, stream) : fa::read_of<_Float16, 4>(a, mx, stream);
    if (dtype == DCN_DTYPE_BF16)
        return mx.bits == 8 ? fa::read_of<fa::bf16, 8>(a, mx, stream) : fa::read_of<fa::bf16, 4>(a, mx, stream);
    return mx.bits == 8 ? fa::read_of<float, 8>(a, mx, stream) : fa::read_of<float, 4>(a, mx, stream);
}

}  // namespace dcn
