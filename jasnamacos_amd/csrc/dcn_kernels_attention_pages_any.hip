// Attention over microscaled pages, or with a prefix that the sequences share, of any type, head
// size up to 256 (microscaled: multiples of 32), stride and alignment: FP32 products on
// v_mfma_f32_32x32x2_f32. The 16-bit heads of 64 and 128 channels have kernels of their own.
//
// Keys are counted through: the prefix's P first, then the sequence's own, whose places in memory two tables
// give; each block of rows reads the prefix itself. As in the kernel of any type without a prefix,
// S^T = K Q^T has 32 keys as rows and 32 packed query rows as columns: a lane has one query row and the keys
// 8a + 4h + b (h = lane / 32), and its weights are the second product's B operand as they are. Keys and
// queries share their order of channels, which is free: a lane takes 16 adjacent ones of each 32, 16 bytes
// of codes and one scale. So is the outputs' order: block b of the second product has the channels
// n NB + b (n = lane % 32), so a lane's share of a value row lies together.
//
// Four waves take the tiles in turn and are joined through LDS; where rows are few, workgroups share the
// keys of a block of rows, and a second kernel joins their parts. Codes are taken to FP32 exactly. Bound: the
// FP32 products, of which up to half the rate is reached; for few rows the loads' latency. Queries of more than
// 64 channels lie in LDS, which leaves registers to the loads (256 channels: 437 us with them in registers,
// 199 so); 61 to 102 registers are spilled above 128 channels, 33 to 507 where pages are off four elements.
// 1,024 causal tokens on 2,000 keys of 8 bits, 8 FP32 heads of 64: 61 us, of 128: 87 us (72 of the 157
// TFLOP/s), of 256: 199 us, 8 BF16 heads of 96 on 4 bits: 87 us. One FP32 token for 8 sequences of 32 heads of
// 128 on 8: 83 us on 8,000 keys of 8 bits, 107 us on a shared prefix of as many FP32 keys. A row a workgroup with
// its products on the vector units took 859, 1,049 (tokens) and 1,706 us.
#include "dcn_attention_any.hpp"
#include "dcn_mx.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr int kRowsWg = 32, kTile = 32;

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
    return uniform(n < 0 ? 0 : (n > p.max_prefix ? p.max_prefix : n));
}

// 16 adjacent channels of a key.
template <typename T, int BITS, bool VEC>
struct KeyPart {
    static constexpr int kWords = BITS / 2;
    typedef uint32_t words __attribute__((ext_vector_type(kWords)));
    words codes;
    uint32_t scale;

    __device__ __forceinline__ void load(const PagesAttention& p, int, int64_t row, int at) {
        const int dim = p.a.dim, in = at < dim ? at : 0;
        codes = *(const words*)(p.mx.k + (row * dim + in) * BITS / 8);
        scale = p.mx.ks[row * (dim / 32) + in / 32];
    }
    __device__ __forceinline__ void get(const PagesAttention& p, int at, float* x) const {
#pragma unroll
        for (int w = 0; w < kWords; ++w) mx_decode32<BITS>(codes[w], mx_factor(scale), x + w * (32 / BITS));
        if (at >= p.a.dim)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.f;
    }
};
template <typename T, bool VEC>
struct KeyPart<T, 0, VEC> {
    f32x4 v[4];

    __device__ __forceinline__ void load(const PagesAttention& p, int kh, int64_t row, int at) {
        const T* from = (const T*)p.a.k.p + row * p.a.k.ts + kh * p.a.k.hs;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = load4<T, VEC>(from, at + 4 * i, p.a.dim);
    }
    __device__ __forceinline__ void get(const PagesAttention&, int, float* x) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = v[i >> 2][i & 3];
    }
};

// N adjacent channels of a value row (zeros past its end).
template <typename T, int N, int BITS, bool VEC>
struct ValuePart {
    static constexpr int kBytes = N * BITS / 8;
    uint32_t codes[kBytes > 4 ? 2 : 1], scale;

    __device__ __forceinline__ void load(const PagesAttention& p, int, int64_t row, int at) {
        const int dim = p.a.dim, in = at < dim ? at : 0;
        const uint8_t* from = p.mx.v + (row * dim + in) * BITS / 8;
        if constexpr (kBytes == 1) {
            codes[0] = *from;
        } else if constexpr (kBytes == 2) {
            codes[0] = *(const uint16_t*)from;
        } else {
#pragma unroll
            for (int i = 0; i < kBytes / 4; ++i) codes[i] = ((const uint32_t*)from)[i];
        }
        scale = p.mx.vs[row * (dim / 32) + in / 32];
    }
    __device__ __forceinline__ void get(const PagesAttention& p, int at, float* x) const {
#pragma unroll
        for (int i = 0; i < (kBytes > 4 ? 2 : 1); ++i) {
            float t[32 / BITS];
            mx_decode32<BITS>(codes[i], mx_factor(scale), t);
#pragma unroll
            for (int e = 0; e < 32 / BITS; ++e)
                if (i * (32 / BITS) + e < N) x[i * (32 / BITS) + e] = at < p.a.dim ? t[e] : 0.f;
        }
    }
};
template <typename T, int N, bool VEC>
struct ValuePart<T, N, 0, VEC> {
    float v[N];

    __device__ __forceinline__ void load(const PagesAttention& p, int kh, int64_t row, int at) {
        const T* from = (const T*)p.a.v.p + row * p.a.v.ts + kh * p.a.v.hs;
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const f32x4 t = load4<T, VEC>(from, at + 4 * i, p.a.dim);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = t[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float t = widen(from[at + i < p.a.dim ? at + i : p.a.dim - 1]);
                v[i] = at + i < p.a.dim ? t : 0.f;
            }
        }
    }
    __device__ __forceinline__ void get(const PagesAttention&, int, float* x) const {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = v[i];
    }
};

// NB: blocks of 32 channels. VEC: pages of the type whose rows have four-element alignment and heads whole fours.
template <typename T, int NB, int BITS, bool VEC>
__global__ __launch_bounds__(kThreads, NB <= 4 ? 2 : 1) void attention_pages_any_kernel(PagesAttention p, BlockMap map, int splits) {
    constexpr int LINE = NB * 32 + 4, KEYS = BITS ? (NB == 8 ? 4 : NB) : (NB == 8 ? 1 : 2), VALUES = NB == 8 ? 4 : (BITS && NB == 2 ? 16 : 8);  // parts whose loads are in flight
    constexpr bool HELD = NB == 2;  // queries in registers: those of more channels would not fit them
    constexpr int AT_ONCE = NB == 2 ? 2 : 4;
    typedef float channels __attribute__((ext_vector_type(AT_ONCE)));
    __shared__ __attribute__((aligned(16))) float sums[kRowsWg][LINE];  // the queries (more than 64 channels), then the sums
    __shared__ float top_of[kWaves][kRowsWg], sum_of[kWaves][kRowsWg], inverse[kRowsWg];
    const AttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
    Place pl;
    if (!place_of<kRowsWg>(a, map, splits, &pl)) return;
    // Positions and keys count from the prefix's first.
    const int prefix = prefix_of(p), keys = prefix + pl.kv.count;
    pl.offset += prefix;
    pl.kv.count = keys;
    const Rows rw = rows_of(a.group);
    const int last_row = pl.rows - 1 < pl.row0 + kRowsWg - 1 ? pl.rows - 1 : pl.row0 + kRowsWg - 1;
    const Spread all = spread_of(a, pl, rw, pl.row0, last_row);
    const int r = pl.row0 + n, rc = r < last_row ? r : last_row;
    const int tok = rw.token(rc), head = pl.kh * a.group + (rc - tok * a.group);
    const Span sp = r <= last_row ? span_of(a, pl.offset + tok, keys) : Span{0, 0, 0};
    f32x4 q[HELD ? NB : 1][4];
    if constexpr (HELD) {
        const T* qp = (const T*)a.q.p + (pl.q.first + tok) * a.q.ts + head * a.q.hs;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) q[b][e] = load4<T, false>(qp, 32 * b + 16 * h + 4 * e, a.dim);
    } else {
        const int in = threadIdx.x >> 3, row = pl.row0 + in < last_row ? pl.row0 + in : last_row, t = rw.token(row);
        const T* qp = (const T*)a.q.p + (pl.q.first + t) * a.q.ts + (pl.kh * a.group + (row - t * a.group)) * a.q.hs;
#pragma unroll
        for (int e = 0; e < NB; ++e) {
            const int ch = 32 * e + 4 * (threadIdx.x & 7);
            *(f32x4*)&sums[in][ch] = load4<T, false>(qp, ch, a.dim);
        }
        __syncthreads();
    }
    const float c = a.scale * kLog2e;
    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] = 0.f;
    float m = -INFINITY, l = 0.f;
    const TileList<kTile> list(all);
    const int per = (list.count + splits - 1) / splits, from = pl.split * per;
    const int stop = from + per < list.count ? from + per : list.count;
    for (int i = from + wave; i < stop; i += kWaves) {
        const int t0 = list.tile(i), j = t0 + n;
        // Row of this lane's key in the pool; keys that are not there are a hole, and row 0 stands in for them.
        int64_t at = key_row<BITS>(p, pl.seq, pl.kh, prefix, j < keys ? j : keys - 1);
        const uint32_t holes = (uint32_t)__ballot(at < 0);
        at = at < 0 ? 0 : at;
        const bool partial = !all_see<kTile>(all, t0) || holes;
        ValuePart<T, NB, BITS, VEC> v[VALUES];
        // Value row x of 16: keys 8a + b (h = 0) and 8a + 4 + b (h = 1), x = 4a + b.
        auto load_values = [&](int first) {
#pragma unroll
            for (int u = 0; u < VALUES; ++u) {
                const int x = first + u;
                v[u].load(p, pl.kh, __shfl(at, 8 * (x >> 2) + 4 * h + (x & 3)), n * NB);
            }
        };
        f32x16 s;
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = 0.f;
#pragma unroll
        for (int b = 0; b < NB; b += KEYS) {
            KeyPart<T, BITS, VEC> k[KEYS];
#pragma unroll
            for (int u = 0; u < KEYS; ++u) k[u].load(p, pl.kh, at, 32 * (b + u) + 16 * h);
            if (b + KEYS >= NB) load_values(0);
#pragma unroll
            for (int u = 0; u < KEYS; ++u) {
                float x[16];
                k[u].get(p, 32 * (b + u) + 16 * h, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x4 row = HELD ? q[HELD ? b + u : 0][e] : *(const f32x4*)&sums[n][32 * (b + u) + 16 * h + 4 * e];
#pragma unroll
                    for (int y = 0; y < 4; ++y) s = mma32(x[4 * e + y], row[y], s);
                }
            }
        }
        if (partial) {
            const unsigned long long seen = (seen_bits(sp, t0) & ~(unsigned long long)holes) >> (4 * h);
#pragma unroll
            for (int x = 0; x < 16; ++x) s[x] = keep_or(s[x] * c, spread_bit(seen, 8 * (x >> 2) + (x & 3)), -INFINITY);
        } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) s[x] *= c;
        }
        float top = s[0];
#pragma unroll
        for (int x = 1; x < 16; ++x) top = fmaxf(top, s[x]);
        top = both_max(top);
        const bool raise = top > m + kSlack;
        if (__any(raise)) {
            const float next = raise ? top : m, old = exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= old;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int x = 0; x < 16; ++x) o[b][x] *= old;
        }
        // fmaxf drops NaN: a NaN score keeps m and makes its own weight, and the row, NaN.
        const float ref = m == -INFINITY ? 0.f : m;
        float part = 0.f;
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            s[x] = __builtin_amdgcn_exp2f(s[x] - ref);
            part += s[x];
        }
        l += part;
        bool bad = false;
#pragma unroll
        for (int first = 0; first < 16; first += VALUES) {
            if (first) load_values(first);
#pragma unroll
            for (int u = 0; u < VALUES; ++u) {
                float x[NB];
                v[u].get(p, n * NB, x);
                // A value that is not finite would reach rows that do not see it (0 x NaN): zero here, and
                // added below where it is seen.
                if (partial) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const bool fine = finite32(x[b]);
                        bad |= !fine;
                        x[b] = fine ? x[b] : 0.f;
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] = mma32(x[b], s[first + u], o[b]);
            }
        }
        if (__builtin_expect(__any(bad), 0)) {
            for (int in = 0; in < kTile; ++in) {
                const bool on = sees(sp, t0 + in) && !(holes >> in & 1);
                const int64_t row = __shfl(at, in);
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const int ch = (8 * (x >> 2) + 4 * h + (x & 3)) * NB;
                    ValuePart<T, NB, BITS, VEC> again;
                    float one[NB];
                    again.load(p, pl.kh, row, ch);
                    again.get(p, ch, one);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        if (on && !finite32(one[b])) o[b][x] += one[b];
                    asm volatile("" ::: "memory");  // few registers: this is rare
                }
            }
        }
    }
    // The waves' sums, in order.
    l = both_sum(l);
    if (lane < 32) {
        top_of[wave][n] = m;
        sum_of[wave][n] = l;
    }
    __syncthreads();
    float mt = top_of[0][n], lt = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mt = fmaxf(mt, top_of[w][n]);
    const float ref = mt == -INFINITY ? 0.f : mt, f = exp2f(m - ref);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) lt += sum_of[w][n] * exp2f(top_of[w][n] - ref);
    for (int w = 0; w < kWaves; ++w) {
        if (wave == w)
#pragma unroll
            for (int x = 0; x < 16; ++x)
#pragma unroll
                for (int b = 0; b < NB; b += AT_ONCE) {
                    channels mine, *to = (channels*)&sums[n][(8 * (x >> 2) + 4 * h + (x & 3)) * NB + b];
#pragma unroll
                    for (int e = 0; e < AT_ONCE; ++e) mine[e] = o[b + e][x] * f;
                    *to = w ? *to + mine : mine;
                }
        __syncthreads();
    }
    const bool empty = mt == -INFINITY && lt == 0.f;
    if (splits > 1) {  // this part's sums, their reference and weight
        const int line = part_line(a.dim);
        if (wave == 0 && lane < 32 && r <= last_row) {
            float* w = (float*)a.workspace + (((pl.q.first + tok) * a.q_heads + head) * splits + pl.split) * line + line - 4;
            w[0] = mt;
            w[1] = lt;
        }
        for (int in = wave; in <= last_row - pl.row0; in += kWaves) {
            const int row = pl.row0 + in, t = rw.token(row), g = pl.kh * a.group + (row - t * a.group);
            float* to = (float*)a.workspace + (((pl.q.first + t) * a.q_heads + g) * splits + pl.split) * line;
            for (int ch = lane; ch < a.dim; ch += 64) to[ch] = sums[in][ch];
        }
        return;
    }
    if (wave == 0 && lane < 32) {
        inverse[n] = empty ? 0.f : 1.f / lt;
        if (a.lse && r <= last_row) a.lse[(pl.q.first + tok) * a.q_heads + head] = empty ? -INFINITY : (mt + log2f(lt)) * kLn2;
    }
    __syncthreads();
    for (int in = wave; in <= last_row - pl.row0; in += kWaves) {
        const int row = pl.row0 + in, t = rw.token(row), g = pl.kh * a.group + (row - t * a.group);
        T* to = (T*)a.out.p + (pl.q.first + t) * a.out.ts + g * a.out.hs;
        for (int ch = lane; ch < a.dim; ch += 64) to[ch] = narrow<T>(sums[in][ch] * inverse[in]);
    }
}

template <typename T, int NB, int BITS, bool VEC>
hipError_t run(const PagesAttention& p, hipStream_t stream) {
    const AttentionArgs& a = p.a;
    BlockMap map;
    const int64_t blocks = ((int64_t)a.max_q * a.group + kRowsWg - 1) / kRowsWg;
    if (!block_map(blocks * a.any_splits, a.kv_heads, a.sequences, &map)) return hipErrorInvalidConfiguration;
    attention_pages_any_kernel<T, NB, BITS, VEC><<<map.grid, kThreads, 0, stream>>>(p, map, a.any_splits);
    return hipGetLastError();
}
template <typename T, int NB>
hipError_t by_bits(const PagesAttention& p, hipStream_t stream) {
    if (p.mx.bits == 8) return run<T, NB, 8, true>(p, stream);
    if (p.mx.bits == 4) return run<T, NB, 4, true>(p, stream);
    return p.a.dim % 4 == 0 && fours<T>(p.a.k) && fours<T>(p.a.v) ? run<T, NB, 0, true>(p, stream) : run<T, NB, 0, false>(p, stream);
}
template <typename T>
hipError_t by_dim(const PagesAttention& p, hipStream_t stream) {
    return p.a.dim <= 64 ? by_bits<T, 2>(p, stream) : (p.a.dim <= 128 ? by_bits<T, 4>(p, stream) : by_bits<T, 8>(p, stream));
}

}  // namespace
}  // namespace fa

int attention_pages_any_splits(const dcn_attention_shape& s, int max_prefix) {
    const int group = s.q_heads / s.kv_heads;
    const int64_t blocks = ((int64_t)s.max_q * group + fa::kRowsWg - 1) / fa::kRowsWg, groups = blocks * s.kv_heads * s.sequences;
    const auto keys = [&](int most) { return attention_keys(most, s.frame_tokens, s.back, s.sinks, fa::kRowsWg / group, fa::kTile); };
    const int64_t tiles = (keys(s.max_kv) + keys(max_prefix) + fa::kTile - 1) / fa::kTile;
    if (groups < 1 || groups > 256 || tiles <= 2 * fa::kWaves) return 1;
    int64_t splits = 512 / groups;
    splits = splits < tiles / fa::kWaves ? splits : tiles / fa::kWaves;
    return (int)(splits < 32 ? splits : 32);
}

size_t attention_pages_any_workspace(const dcn_attention_shape& s, int max_prefix) {
    const int splits = attention_pages_any_splits(s, max_prefix);
    return splits == 1 ? 0 : (size_t)s.q_tokens * s.q_heads * splits * fa::part_line(s.head_dim) * sizeof(float);
}

hipError_t launch_attention_pages_any(int dtype, const PagesAttention& p, hipStream_t stream) {
    hipError_t e;
    if (dtype == DCN_DTYPE_F16) e = fa::by_dim<_Float16>(p, stream);
    else if (dtype == DCN_DTYPE_BF16) e = fa::by_dim<fa::bf16>(p, stream);
    else e = fa::by_dim<float>(p, stream);
    return e != hipSuccess || p.a.any_splits == 1 ? e : launch_attention_any_join(dtype, p.a, p.a.any_splits, stream);
}

}  // namespace dcn
