// The microscaled cache: the append of rotated keys and values as codes, and the read back.
//
// A block of 32 channels has x^ = code 2^e, e the smallest with max|x| <= 448 2^e (6 2^e in 4 bits). A
// thread has eight channels of a token, four adjacent lanes a block: its largest magnitude (as bits,
// which order as numbers do and put infinities and NaN on top) takes two moves between lanes, the
// scaled conversions round. Both kernels are bound by HBM, small calls by the call itself.
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

// The rotation of channels at .. at + 7: channel c turns into x[c] cos + x[partner] sin (with the
// sine's sign), where it turns at all.
template <bool WIDE>
struct Turn8 {
    float c[8], s[8];
    int partner[WIDE ? 1 : 8];  // WIDE: of the first channel; -1: passes
    bool inside;                // WIDE: pairs inside the eight channels

    __device__ __forceinline__ void set(const RotaryArgs& r, int at, const int32_t* pos) {
        inside = WIDE && r.interleaved;
        if constexpr (WIDE) {
            partner[0] = at >= 2 * r.pairs ? -1 : (r.interleaved ? at : (at < r.pairs ? at + r.pairs : at - r.pairs));
            if (partner[0] < 0) return;
            const int first = r.interleaved ? at >> 1 : (at < r.pairs ? at : at - r.pairs), n = r.interleaved ? 4 : 8;
            const float sign = at < r.pairs ? -1.f : 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) {
                    turn(r, pos, first + i, &c[i], &s[i]);
                    if (!r.interleaved) s[i] *= sign;
                }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int ch = at + i;
                partner[i] = -1;
                if (ch >= 2 * r.pairs) continue;
                const bool second = r.interleaved ? ch & 1 : ch >= r.pairs;
                turn(r, pos, r.interleaved ? ch >> 1 : (second ? ch - r.pairs : ch), &c[i], &s[i]);
                if (!second) s[i] = -s[i];
                partner[i] = r.interleaved ? ch ^ 1 : (second ? ch - r.pairs : ch + r.pairs);
            }
        }
    }
};

// One thread: eight channels of one new token, over the heads of its slice. Slices below q_slices
// turn queries (a pair of channels by one thread: q_out may be q), the others take keys, then values.
template <typename T, int BITS, bool WIDE>
__global__ __launch_bounds__(kThreads) void append_mx_kernel(RotaryArgs r, AppendArgs a, MxArgs mx, int64_t first, int q_slices) {
    const int chunks = r.dim / 8;
    const int64_t item = first + (int64_t)blockIdx.x * kThreads + threadIdx.x, given = item / chunks;
    const int64_t token = given < a.tokens ? given : a.tokens - 1;
    Target t;
    if (!target_of(a, a.cu_q, token, &t) || given >= a.tokens) return;
    const int index = (int)(item - given * chunks);
    const int32_t* pos = r.positions + token * 3;
    if ((int)blockIdx.y < q_slices) {
        constexpr int N = WIDE ? 16 / sizeof(T) : 1;
        const T* from = (const T*)a.q.p + token * a.q.ts;
        T* to = (T*)a.q_out.p + token * a.q_out.ts;
        for (int i = index; i < Chunk<T, N>::count(r); i += chunks) {
            Chunk<T, N> c;
            c.set(r, i, pos);
            for (int h = blockIdx.y; h < a.q_heads; h += kBatch * q_slices)
                c.template apply_all<kBatch>(
                    [&](int u) { return h + u * q_slices < a.q_heads ? from + (h + u * q_slices) * a.q.hs : nullptr; },
                    [&](int u) { return h + u * q_slices < a.q_heads ? to + (h + u * q_slices) * a.q_out.hs : nullptr; }, true);
        }
        return;
    }
    const int64_t row0 = t.place < 0 ? -1 : mx_row(a.pages, mx.heads, t.sequence, 0, t.place);
    if (row0 < 0) return;
    const int at = index * 8, slice = blockIdx.y - q_slices, step = gridDim.y - q_slices, nk = a.kv_heads;
    Turn8<WIDE> turn8;
    if (slice < nk) turn8.set(r, at, pos);
    for (int h0 = slice; h0 < 2 * nk; h0 += kBatch * step) {
        T x[kBatch][8], y[kBatch][8];
        bool turns[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int h = h0 + u * step;
            turns[u] = h < nk;
            if (h >= 2 * nk) continue;
            const T* p = h < nk ? (const T*)a.k.p + token * a.k.ts + h * a.k.hs : (const T*)a.v.p + token * a.v.ts + (h - nk) * a.v.hs;
            if constexpr (WIDE) {
                Vec<T, 8>::load(p + at, x[u]);
                turns[u] = turns[u] && turn8.partner[0] >= 0;
                if (turns[u] && !turn8.inside) Vec<T, 8>::load(p + turn8.partner[0], y[u]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[u][i] = p[at + i];
                    if (turns[u] && turn8.partner[i] >= 0) y[u][i] = p[turn8.partner[i]];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int h = h0 + u * step;
            if (h >= 2 * nk) break;
            float z[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = widen(x[u][i]);
            if (turns[u]) {
                if constexpr (WIDE) {
                    if (turn8.inside) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float p = z[2 * i], q = z[2 * i + 1];
                            z[2 * i] = fmaf(p, turn8.c[i], -(q * turn8.s[i]));
                            z[2 * i + 1] = fmaf(p, turn8.s[i], q * turn8.c[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) z[i] = fmaf(z[i], turn8.c[i], widen(y[u][i]) * turn8.s[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (turn8.partner[i] >= 0) z[i] = fmaf(z[i], turn8.c[i], widen(y[u][i]) * turn8.s[i]);
                }
            }
            constexpr uint32_t infinity = 0x7f800000u;
            uint32_t top = 0;
            const float most = mx_most<T, BITS>();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t bits = __builtin_bit_cast(uint32_t, z[i]) & 0x7fffffffu;
                if (bits < infinity) {
                    z[i] = fminf(fmaxf(z[i], -most), most);
                    bits = __builtin_bit_cast(uint32_t, z[i]) & 0x7fffffffu;
                }
                top = bits > top ? bits : top;
            }
            top = quad_max(top);
            const bool bad = top >= infinity;
            const uint32_t scale = bad ? kMxNan : mx_scale<BITS>(top);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = bad ? 0.f : z[i];
            const mx_u32x2 codes = mx_encode<BITS>(z, mx_factor(bad ? 127 : scale));
            const int64_t row = row0 + ((int64_t)(h < nk ? h : h - nk) << a.pages.shift);
            uint8_t *to = h < nk ? mx.k : mx.v, *scales = h < nk ? mx.ks : mx.vs;
            uint8_t* place = to + (row * r.dim + at) * BITS / 8;
            if constexpr (BITS == 8)
                *(mx_u32x2*)place = codes;
            else
                *(uint32_t*)place = codes[0];
            if ((index & 3) == 0) scales[row * (r.dim / 32) + (index >> 2)] = (uint8_t)scale;
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
    const int64_t items = a.tokens * (r.dim / 8);
    const int nq = a.q.p ? a.q_heads : 0, heads = nq + 2 * a.kv_heads;
    for (int64_t first = 0; first < items; first += kMostThreads) {
        const int64_t n = items - first < kMostThreads ? items - first : kMostThreads;
        // Slices for queries and for keys and values by their heads, one each at least.
        const int slices = (int)head_slices(items, heads);
        int q = nq ? (int)((int64_t)slices * nq / heads) : 0;
        if (nq && q < 1) q = 1;
        const int kv = slices - q < 1 ? 1 : slices - q;
        append_mx_kernel<T, BITS, WIDE><<<dim3((unsigned)((n + kThreads - 1) / kThreads), q + kv), kThreads, 0, stream>>>(r, a, mx, first, q);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
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
