// Gradients of windowed attention on the matrix cores: FP16 and BF16 heads of 64 and 128 channels.
//
// With P = exp(S - lse) again from q, k and lse, delta = rowsum(dO * O) and dP = dO V^T:
//   dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO.
// Two passes, so that no sum is made with atomics and the same inputs give the same bits: one
// over query rows (dQ, and delta on the way), one over keys (dK and dV); seven products for
// the five of a pass that adds dQ up in memory. Both keep a wave's rows (keys) in registers as
// the B operand and as columns of the sums, as the forward does, and walk tiles of the other
// side in LDS.
//
// What bounds them: instruction issue and LDS round trips. 128 channels leave the second pass one
// wave a SIMD (its keys, values and both sums take 450 registers), where MFMA and vector instructions
// each take a third of the cycles and waits the rest. Times of a step's kernels, forward / first /
// second pass / join: 4 x 2,560 tokens, 8 heads of 64, windows of five frames of 256, BF16: 44 / 57 / 73 /
// 4 us; four sequences of up to 1,021 tokens, 8 heads of 128 on 2, windows of 256 tokens, FP16: 18 / 31 /
// 42 / 8 us; 2 x 4,096 causal tokens, 8 heads of 128, BF16: 126 / 174 / 197 us (690 TFLOP/s in the second).
//
// FP16 would lose gradients below 2^-24 and overflow above 2^16: dS enters its products
// times a power of two that follows the largest one seen of its row (first pass) or its key
// (second), P times 2^10. BF16 has FP32's range and needs neither.
#include "dcn_attention_mfma.hpp"

namespace dcn {
namespace fa {
namespace {

template <typename T>
constexpr bool kScaled = __is_same(T, _Float16);
constexpr float kWeightLift = 1024.f;  // FP16: P's factor
constexpr float kMostScaled = 32768.f;
constexpr int kFewKeys = 256;

// The power of two that brings `top` into [2^12, 2^13).
__device__ __forceinline__ float scale_for(float top) {
    int e = 12 - ((int)(__builtin_bit_cast(uint32_t, top) >> 23 & 255) - 127);
    e = e > 100 ? 100 : (e < -100 ? -100 : e);
    return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}
__device__ __forceinline__ float top_of(const f32x16& v) {
    float t = fabsf(v[0]);
#pragma unroll
    for (int r = 1; r < 16; ++r) t = fmaxf(t, fabsf(v[r]));
    return t;
}

// Lowers (or first sets) the factor of a lane's row or key where dS times it would leave FP16,
// and its sums with it.
template <int D>
__device__ __forceinline__ void follow_scale(float top, float* up, f32x16* sum) {
    top = both_max(top);
    const bool change = top * *up > kMostScaled || (*up == 0.f && top > 0.f);
    if (__builtin_expect(!__any(change), 1)) return;
    const float next = change ? scale_for(top) : *up, by = *up == 0.f ? 1.f : next / *up;
#pragma unroll
    for (int n = 0; n < D / 32; ++n)
#pragma unroll
        for (int x = 0; x < 16; ++x) sum[n][x] *= by;
    *up = next;
}

// Keys of a tile of the first pass: with 128 channels a wave's operands and sums leave registers
// for 32 keys' dS.
template <int D>
constexpr int kDqKeys = D == 64 ? 64 : 32;

// First pass: 128 packed rows a workgroup, 32 a wave, over the tiles of keys that they see.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void attention_dq_kernel(AttentionArgs a, BlockMap map) {
    constexpr int ROWS = kDqKeys<D>, BYTES = ROWS * D * 2, MB = ROWS / 32;
    using Ti = Tile<D>;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][BYTES];
    __shared__ FoundRows found;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Place pl;
    if (!place_of<32 * kWaves>(a, map, 1, &pl)) return;
    const Rows rw = rows_of(a.group);
    const int last_row = pl.rows - 1;
    const int w0 = pl.row0 + 32 * wave, w1 = w0 + 31 < last_row ? w0 + 31 : last_row;
    const Spread all = spread_of(a, pl, rw, pl.row0, pl.row0 + 32 * kWaves - 1 < last_row ? pl.row0 + 32 * kWaves - 1 : last_row);
    const bool idle = w0 > last_row;
    const Spread mine = idle ? all : spread_of(a, pl, rw, w0, w1);
    const int r = w0 + (lane & 31), rc = r < last_row ? r : last_row;
    const Span sp = r <= last_row ? span_of(a, pl.offset + rw.token(r), pl.kv.count) : Span{0, 0, 0};
    const int tok = rw.token(rc), head = pl.kh * a.group + (rc - tok * a.group);
    const int64_t row = pl.q.first + tok, index = row * a.q_heads + head;
    const TileList<ROWS> list(all);
    const Keys<false> keys(a, pl.seq, pl.kh, pl.kv);
    TilePages<D, ROWS, kWaves, false> none;
    TileCopy<D, ROWS, kWaves, false> copies;
    copies.set(keys, ROWS, wave, lane);
    if (list.count) copies.copy(keys, list.tile(0), none, lds[0][0], lds[0][1], wave, lane);
    u32x4 q[D / 16], go[D / 16];
    load_row<D>(q, a.q, a, pl, rw, r, lane);
    load_row<D>(go, a.dout, a, pl, rw, r, lane);
    float delta = 0.f;
    {
        u32x4 o[D / 16];
        load_row<D>(o, a.o, a, pl, rw, r, lane);
        typedef T vec __attribute__((ext_vector_type(8)));
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const vec x = __builtin_bit_cast(vec, o[i]), y = __builtin_bit_cast(vec, go[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf((float)x[e], (float)y[e], delta);
        }
        delta = both_sum(delta);
    }
    float lse = a.lse_in[index] * kLog2e;
    // delta from the rounded out is off by a rounding's share of it, 1 / sqrt(keys) of what dS's
    // own rounding costs. Rows of few keys take it from P and dP instead, in a pass of its own.
    const bool sum_delta = list.count * ROWS <= kFewKeys;
    if (!sum_delta && lane < 32 && r <= last_row) ((float*)a.workspace)[index] = delta;
    // Loaded: later waits for these registers would wait for the copies too.
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(q[i]), "+v"(go[i]));
    asm volatile("" : "+v"(lse), "+v"(delta));
    const float c = a.scale * kLog2e;
    f32x16 sum[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) sum[i][x] = 0.f;
    float up = kScaled<T> ? 0.f : 1.f;  // FP16: dS's factor of this row; 0: no dS seen yet
    float exact_delta = 0.f;
    if (sum_delta) delta = 0.f;
    const int steps = sum_delta ? 2 * list.count : list.count;
    for (int step = 0, i = 0; step < steps; ++step, i = i + 1 < list.count ? i + 1 : 0) {
        const int buf = step & 1, t0 = list.tile(i);
        char(*now)[BYTES] = lds[buf], (*other)[BYTES] = lds[buf ^ 1];
        wait_copies<0>();
        // Keys that are not finite, where some row does not see all of the tile: zeros in LDS, and
        // the scores of the rows that see them are NaN. Each wave looks at what it copied.
        const bool partial = !all_see<ROWS>(all, t0);
        if (partial) found.wave[buf][wave] = clean_own<T, D, ROWS, kWaves>(now[0], wave, lane);
        __syncthreads();
        if (step + 1 < steps) {
            const int next = i + 1 < list.count ? i + 1 : 0;
            if (!next) copies.set(keys, ROWS, wave, lane);
            copies.copy(keys, list.tile(next), none, other[0], other[1], wave, lane);
        }
        const bool delta_step = sum_delta && step < list.count;
        const unsigned long long poison = partial ? found.all(buf) : 0;
        if (!idle && !none_sees<ROWS>(mine, t0)) {
            const bool masked = !all_see<ROWS>(mine, t0) || poison;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                f32x16 s, dp;
                {
                    u32x4 kr[D / 16], vr[D / 16];
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) kr[n] = Ti::rows(now[0], mb, n, lane);
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) vr[n] = Ti::rows(now[1], mb, n, lane);
                    if constexpr (D == 64) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int x = 0; x < 16; ++x) s[x] = dp[x] = 0.f;
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) s = mma<T>(kr[n], q[n], s);
#pragma unroll
                    for (int n = 0; n < D / 16; ++n) dp = mma<T>(vr[n], go[n], dp);
                }
                // 64 channels leave registers to read the next product's keys before the weights are made.
                u32x4 kc[2][D / 32];
                auto read_columns = [&] {
#pragma unroll
                    for (int st = 0; st < 2; ++st)
#pragma unroll
                        for (int n = 0; n < D / 32; ++n) kc[st][n] = Ti::columns(now[0], mb, st, n, lane);
                };
                if constexpr (D == 64) {
                    __builtin_amdgcn_sched_barrier(0);
                    read_columns();
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], c, -lse)) * (dp[x] - delta);
                if (masked) {
                    if (__builtin_expect(poison != 0, 0)) {
                        const unsigned long long not_finite = poison >> (4 * (lane >> 5));
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (spread_bit(not_finite, 32 * mb + 8 * (x >> 2) + (x & 3))) s[x] = NAN;
                    }
                    const unsigned long long seen = seen_bits(sp, t0) >> (4 * (lane >> 5));
#pragma unroll
                    for (int x = 0; x < 16; ++x) s[x] = keep_or(s[x], spread_bit(seen, 32 * mb + 8 * (x >> 2) + (x & 3)), 0.f);
                }
                if (delta_step) {  // the sums are left as they are by a product with zeros
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        exact_delta += s[x];
                        s[x] = 0.f;
                    }
                }
                if constexpr (kScaled<T>) {
                    follow_scale<D>(top_of(s), &up, sum);
#pragma unroll
                    for (int x = 0; x < 16; ++x) s[x] *= up;
                }
                const u32x4 ds[2] = {pack8<T>(s, 0), pack8<T>(s, 8)};
                if constexpr (D != 64) read_columns();
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int n = 0; n < D / 32; ++n) sum[n] = mma<T>(kc[st][n], ds[st], sum[n]);
            }
        }
        if (delta_step && i + 1 == list.count) delta = both_sum(exact_delta);
    }
    if (r > last_row) return;
    if (sum_delta && lane < 32) ((float*)a.workspace)[index] = delta;
    const float f = up == 0.f ? 0.f : a.scale / up;
    T* to = (T*)a.dq.p + row * a.dq.ts + head * a.dq.hs + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            typedef T four __attribute__((ext_vector_type(4)));
            four v;
#pragma unroll
            for (int b = 0; b < 4; ++b) v[b] = narrow<T>(sum[i][4 * x + b] * f);
            *(four*)(to + 32 * i + 8 * x) = v;
        }
}

// How the key blocks (128 keys) share out their query tiles: the first `sink_blocks` hold keys
// that every later query sees, and are cut into more parts than the others.
struct KeyPlan {
    int blocks, sink_blocks, parts, sink_parts;
    __host__ __device__ int items() const { return sink_blocks * sink_parts + (blocks - sink_blocks) * parts; }
    // Items whose sums the workspace holds, the first ones: those of blocks that are cut.
    __host__ __device__ int kept() const { return parts > 1 ? items() : (sink_parts > 1 ? sink_blocks * sink_parts : 0); }
    __host__ __device__ void item(int i, int* block, int* part, int* of) const {
        if (i < sink_blocks * sink_parts) {
            *block = i / sink_parts;
            *part = i % sink_parts;
            *of = sink_parts;
        } else {
            i -= sink_blocks * sink_parts;
            *block = sink_blocks + i / parts;
            *part = i % parts;
            *of = parts;
        }
    }
};
constexpr int kKeys = 32 * kWaves;

// Positions that see all keys j .. to: `from` grows with the key, and so does `to` past the
// sinks, whose `to` is n.
__device__ __forceinline__ Seen all_seen_of(const AttentionArgs& a, int j, int to, int n) {
    const int64_t sinks = (int64_t)a.sinks * a.frame;
    return Seen{seen_of(a, to, n).from, seen_of(a, j < sinks && sinks <= to ? (int)sinks : j, n).to};
}

constexpr int kDkvRows = 64;  // query rows of a tile of the second pass

// Second pass: 128 keys a workgroup, 32 a wave, over the tiles of packed rows that see them; the rows
// of a block are split over workgroups (KeyPlan) where blocks alone do not fill the card.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, D == 64 ? 2 : 1) void attention_dkv_kernel(AttentionArgs a, BlockMap map, KeyPlan plan, float* parts) {
    constexpr int ROWS = kDkvRows, BYTES = ROWS * D * 2, MB = ROWS / 32;
    using Ti = Tile<D>;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][BYTES];
    __shared__ __attribute__((aligned(16))) float row_lse[2][ROWS], row_delta[2][ROWS];
    __shared__ FoundRows found;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    int at, block, part, of;
    Place pl;
    if (!block_of(map, &at, &pl.kh, &pl.seq)) return;
    plan.item(at, &block, &part, &of);
    pl.q = run_of(a.cu_q, pl.seq, a.max_q, a.q_tokens);
    pl.kv = run_of(a.cu_kv, pl.seq, a.max_kv, a.kv_tokens);
    pl.q.count = uniform(pl.q.count);
    pl.kv.count = uniform(pl.kv.count);
    pl.offset = pl.kv.count - pl.q.count;
    pl.rows = (pl.q.count < a.max_q ? pl.q.count : a.max_q) * a.group;
    const int k0 = block * kKeys, nk = pl.kv.count;
    if (k0 >= nk) return;
    const Rows rw = rows_of(a.group);
    // The wave's keys, as B operands (past the end: the last key's; their sums are not stored).
    const int j = k0 + 32 * wave + (lane & 31), jc = j < nk ? j : nk - 1;
    u32x4 k[D / 16], v[D / 16];
    {
        const char* kp = (const char*)a.k.p + ((pl.kv.first + jc) * a.k.ts + pl.kh * a.k.hs + 8 * (lane >> 5)) * 2;
        const char* vp = (const char*)a.v.p + ((pl.kv.first + jc) * a.v.ts + pl.kh * a.v.hs + 8 * (lane >> 5)) * 2;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            k[i] = *(const u32x4*)(kp + i * 32);
            v[i] = *(const u32x4*)(vp + i * 32);
        }
    }
    const Seen me = seen_of(a, jc, nk);
    // Positions that see some key of the block; all of them; all keys of the wave.
    const int kl = k0 + kKeys - 1 < nk ? k0 + kKeys - 1 : nk - 1;
    const int wf = k0 + 32 * wave < nk ? k0 + 32 * wave : nk - 1, wl = wf + 31 < nk ? wf + 31 : nk - 1;
    const Seen first = seen_of(a, k0, nk), last = seen_of(a, kl, nk);
    const Seen every = all_seen_of(a, k0, kl, nk), wave_every = all_seen_of(a, wf, wl, nk);
    // A sink's `to` is n: the largest `to` of a run of keys is that of its first or its last.
    int t_from = first.from - pl.offset, t_to = (first.to > last.to ? first.to : last.to) - pl.offset;
    t_from = t_from < 0 ? 0 : t_from;
    const int q_rows = pl.rows;
    const int64_t r_to = (int64_t)t_to * a.group;
    const int tile_from = (int)((int64_t)t_from * a.group / ROWS), end = r_to < q_rows ? (int)(r_to < 0 ? 0 : r_to) : q_rows;
    const int tile_to = (end + ROWS - 1) / ROWS;
    const int tiles = tile_to > tile_from ? tile_to - tile_from : 0;
    const int per = (tiles + of - 1) / of;
    const int begin = tile_from + part * per, stop = begin + per < tile_to ? begin + per : tile_to;

    // Copies of the query tile at packed row r0: byte offsets from the token of its first row, the
    // same for every tile where the group divides 64, but for the last.
    constexpr int kCopies = ROWS / Ti::kRowsPerCopy / kWaves;
    uint32_t q_at[kCopies], o_at[kCopies];
    const bool steady = ROWS % a.group == 0;
    auto offsets = [&](int r0) {
        const int rem = r0 - rw.token(r0) * a.group, last = q_rows - 1 - r0;
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            const int in = Ti::copy_row(n * kWaves + wave, lane), c = Ti::copy_channel(in, lane), r = rem + (in < last ? in : last);
            const int tok = rw.token(r), g = r - tok * a.group;
            q_at[n] = (tok * (uint32_t)a.q.ts + g * (uint32_t)a.q.hs + c) * 2;
            o_at[n] = (tok * (uint32_t)a.dout.ts + g * (uint32_t)a.dout.hs + c) * 2;
        }
    };
    auto copy = [&](int r0, char* to_q, char* to_do) {
        if (!steady || r0 + ROWS > q_rows) offsets(r0);
        const int64_t row = pl.q.first + uniform(rw.token(r0)), head = pl.kh * a.group;
        const char* qb = (const char*)a.q.p + (row * a.q.ts + head * a.q.hs) * 2;
        const char* ob = (const char*)a.dout.p + (row * a.dout.ts + head * a.dout.hs) * 2;
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            copy16(qb, q_at[n], to_q + (n * kWaves + wave) * 1024);
            copy16(ob, o_at[n], to_do + (n * kWaves + wave) * 1024);
        }
    };
    float next_lse = 0.f, next_delta = 0.f;
    auto fetch = [&](int r0) {
        const int r = r0 + (int)threadIdx.x;
        if (threadIdx.x >= ROWS || r >= q_rows) return;
        const int tok = rw.token(r), head = pl.kh * a.group + (r - tok * a.group);
        const int64_t index = (pl.q.first + tok) * a.q_heads + head;
        next_lse = a.lse_in[index] * kLog2e;
        next_delta = ((const float*)a.workspace)[index];
    };
    f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) dk[i][x] = dv[i][x] = 0.f;
    const float c = a.scale * kLog2e;
    float up = kScaled<T> ? 0.f : 1.f;  // FP16: dS's factor of this key; 0: no dS seen yet
    if (begin < stop) {
        fetch(begin * ROWS);
        offsets(begin * ROWS);
        copy(begin * ROWS, lds[0][0], lds[0][1]);
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(k[i]), "+v"(v[i]));
    for (int i = begin; i < stop; ++i) {
        const int buf = (i - begin) & 1, r0 = i * ROWS;
        char *qt = lds[buf][0], *ot = lds[buf][1];
        if (threadIdx.x < ROWS) {
            row_lse[buf][threadIdx.x] = next_lse;
            row_delta[buf][threadIdx.x] = next_delta;
        }
        // Positions of the tile's first and last row; whether this wave's keys (all of the block's)
        // are seen by all of them.
        const int rl = r0 + ROWS - 1 < q_rows ? r0 + ROWS - 1 : q_rows - 1;
        const int t0 = rw.token(r0), p0 = pl.offset + t0, p1 = pl.offset + rw.token(rl);
        const bool rows_there = r0 + ROWS <= q_rows && p0 >= 0;
        const bool whole = rows_there && p0 >= wave_every.from && p1 < wave_every.to;
        const bool partial = !(rows_there && p0 >= every.from && p1 < every.to);
        wait_copies<0>();
        // Queries and gradients that are not finite, where some pair of the tile is not visible:
        // zeros in LDS, and the weights of the pairs that are visible are NaN.
        if (partial)
            found.wave[buf][wave] = clean_own<T, D, ROWS, kWaves>(qt, wave, lane) | clean_own<T, D, ROWS, kWaves>(ot, wave, lane);
        __syncthreads();
        if (i + 1 < stop) {
            fetch(r0 + ROWS);
            copy(r0 + ROWS, lds[buf ^ 1][0], lds[buf ^ 1][1]);
        }
        if (partial)
            if (const unsigned long long poison = found.all(buf); __builtin_expect(poison != 0, 0)) {
                if (threadIdx.x < ROWS && poison >> threadIdx.x & 1) row_lse[buf][threadIdx.x] = NAN;
                __syncthreads();
            }
        // A bit for each of the tile's rows that sees this lane's key: positions grow with the rows.
        unsigned long long seen = ~0ull;
        if (!whole) {
            const int64_t rem = r0 - (int64_t)t0 * a.group;
            const int64_t lo = ((int64_t)me.from - p0) * a.group - rem, hi = ((int64_t)me.to - p0) * a.group - rem;
            const int64_t there = q_rows - r0, top = hi < there ? hi : there;
            seen = bits_below((int)(top < 64 ? (top < 0 ? 0 : top) : 64)) & ~bits_below((int)(lo < 64 ? (lo < 0 ? 0 : lo) : 64));
            seen >>= 4 * (lane >> 5);
        }
        struct Half {  // 32 rows of the tile against the wave's keys
            int mb;
            u32x4 qr[D / 16], gr[D / 16], oc[2][D / 32], qc[2][D / 32];
            f32x4 l4[4], d4[4];
            f32x16 s, dp;
        };
        auto read_rows = [&](Half& h, int mb) {
            h.mb = mb;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) h.qr[n] = Ti::rows(qt, mb, n, lane);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) h.gr[n] = Ti::rows(ot, mb, n, lane);
        };
        auto scores = [&](Half& h) {
#pragma unroll
            for (int x = 0; x < 16; ++x) h.s[x] = h.dp[x] = 0.f;
#pragma unroll
            for (int n = 0; n < D / 16; ++n) h.s = mma<T>(h.qr[n], k[n], h.s);
#pragma unroll
            for (int n = 0; n < D / 16; ++n) h.dp = mma<T>(h.gr[n], v[n], h.dp);
        };
        auto read_stats = [&](Half& h) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                h.l4[g] = *(const f32x4*)&row_lse[buf][32 * h.mb + 8 * g + 4 * (lane >> 5)];
                h.d4[g] = *(const f32x4*)&row_delta[buf][32 * h.mb + 8 * g + 4 * (lane >> 5)];
            }
        };
        auto read_columns = [&](Half& h) {
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int n = 0; n < D / 32; ++n) {
                    h.oc[st][n] = Ti::columns(ot, h.mb, st, n, lane);
                    h.qc[st][n] = Ti::columns(qt, h.mb, st, n, lane);
                }
        };
        auto weights = [&](Half& h) {
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                h.s[x] = __builtin_amdgcn_exp2f(fmaf(h.s[x], c, -h.l4[x >> 2][x & 3]));
                h.dp[x] = h.s[x] * (h.dp[x] - h.d4[x >> 2][x & 3]);
            }
            if (!whole) {
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const uint32_t on = spread_bit(seen, 32 * h.mb + 8 * (x >> 2) + (x & 3));
                    h.s[x] = keep_or(h.s[x], on, 0.f);
                    h.dp[x] = keep_or(h.dp[x], on, 0.f);
                }
            }
        };
        auto add = [&](Half& h) {
            if constexpr (kScaled<T>) {
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    h.s[x] *= kWeightLift;
                    h.dp[x] *= up;
                }
            }
            const u32x4 p16[2] = {pack8<T>(h.s, 0), pack8<T>(h.s, 8)}, ds[2] = {pack8<T>(h.dp, 0), pack8<T>(h.dp, 8)};
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int n = 0; n < D / 32; ++n) {
                    dv[n] = mma<T>(h.oc[st][n], p16[st], dv[n]);
                    dk[n] = mma<T>(h.qc[st][n], ds[st], dk[n]);
                }
        };
        if constexpr (D == 64 || !kScaled<T>) {
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                Half h;
                read_rows(h, mb);
                __builtin_amdgcn_sched_barrier(0);
                scores(h);
                __builtin_amdgcn_sched_barrier(0);
                read_stats(h);
                read_columns(h);
                __builtin_amdgcn_sched_barrier(0);
                weights(h);
                if constexpr (kScaled<T>) follow_scale<D>(top_of(h.dp), &up, dk);
                add(h);
            }
        } else {
            // FP16 of 128 channels looks at its factors once a tile: joining the sums after that
            // branch costs a copy of each (a training step of four sequences of up to 1021 tokens, two
            // key heads of four: 100 us with a look for each half, 97 so).
            Half h0, h1;
            read_rows(h0, 0);
            read_stats(h0);
            __builtin_amdgcn_sched_barrier(0);
            scores(h0);
            read_rows(h1, 1);
            __builtin_amdgcn_sched_barrier(0);
            scores(h1);
            weights(h0);
            __builtin_amdgcn_sched_barrier(0);
            read_stats(h1);
            weights(h1);
            follow_scale<D>(fmaxf(top_of(h0.dp), top_of(h1.dp)), &up, dk);
            read_columns(h0);
            add(h0);
            read_columns(h1);
            add(h1);
        }
    }
    const float fk = up == 0.f ? 0.f : a.scale / up, fv = kScaled<T> ? 1.f / kWeightLift : 1.f;
    if (of > 1) {
        // [item][dk, dv][key][D] FP32, in order of the parts
        const int64_t item = ((int64_t)pl.seq * a.kv_heads + pl.kh) * plan.kept() + at;
        float* to = parts + ((item * 2) * kKeys + 32 * wave + (lane & 31)) * D + 4 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                *(f32x4*)(to + 32 * i + 8 * x) = f32x4{dk[i][4 * x] * fk, dk[i][4 * x + 1] * fk, dk[i][4 * x + 2] * fk, dk[i][4 * x + 3] * fk};
                *(f32x4*)(to + kKeys * D + 32 * i + 8 * x) =
                    f32x4{dv[i][4 * x] * fv, dv[i][4 * x + 1] * fv, dv[i][4 * x + 2] * fv, dv[i][4 * x + 3] * fv};
            }
        return;
    }
    if (j >= nk) return;
    T* to_k = (T*)a.dk.p + (pl.kv.first + j) * a.dk.ts + pl.kh * a.dk.hs + 4 * (lane >> 5);
    T* to_v = (T*)a.dv.p + (pl.kv.first + j) * a.dv.ts + pl.kh * a.dv.hs + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            typedef T four __attribute__((ext_vector_type(4)));
            four vk, vv;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                vk[b] = narrow<T>(dk[i][4 * x + b] * fk);
                vv[b] = narrow<T>(dv[i][4 * x + b] * fv);
            }
            *(four*)(to_k + 32 * i + 8 * x) = vk;
            *(four*)(to_v + 32 * i + 8 * x) = vv;
        }
}

// The parts of one key block's gradients, in order; four channels a thread.
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void attention_dkv_join_kernel(AttentionArgs a, KeyPlan plan, const float* parts, int from_block) {
    const Run kv = run_of(a.cu_kv, blockIdx.z, a.max_kv, a.kv_tokens);
    constexpr int per = kThreads * 4 / D, groups = kKeys / per;  // keys of one workgroup
    const int block = from_block + blockIdx.x / groups, key = (blockIdx.x % groups) * per + threadIdx.x / (D / 4);
    const int j = block * kKeys + key, at = threadIdx.x % (D / 4) * 4;
    if (j >= kv.count) return;
    const int of = block < plan.sink_blocks ? plan.sink_parts : plan.parts;
    const int first = block < plan.sink_blocks ? block * plan.sink_parts
                                               : plan.sink_blocks * plan.sink_parts + (block - plan.sink_blocks) * plan.parts;
    const int64_t item = ((int64_t)blockIdx.z * a.kv_heads + blockIdx.y) * plan.kept() + first;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
        for (int p = 0; p < of; ++p) {
            const f32x4 x = *(const f32x4*)(parts + (((item + p) * 2 + which) * kKeys + key) * D + at);
#pragma unroll
            for (int b = 0; b < 4; ++b) sum[b] += x[b];
        }
        typedef T four __attribute__((ext_vector_type(4)));
        four v;
#pragma unroll
        for (int b = 0; b < 4; ++b) v[b] = narrow<T>(sum[b]);
        const HeadsOut& h = which ? a.dv : a.dk;
        *(four*)((T*)h.p + (kv.first + j) * h.ts + blockIdx.y * h.hs + at) = v;
    }
}

KeyPlan key_plan(int sequences, int kv_heads, int group, int max_q, int max_kv, int frame, int back, int ahead, int sinks) {
    KeyPlan p;
    p.blocks = (int)(((int64_t)max_kv + kKeys - 1) / kKeys);
    const int64_t all = ((int64_t)max_q * group + 63) / 64;
    // Query tiles of a block: those of its window, or all.
    int64_t tiles = all;
    p.sink_blocks = 0;
    if (back >= 0) {
        const int64_t frames = (int64_t)back + 1 + (ahead < 0 ? 0 : ahead) + ((int64_t)kKeys + frame - 1) / frame;
        const int64_t window = ahead < 0 || frames > max_q / frame ? all : (frames * frame * group + 63) / 64 + 1;
        tiles = window < all ? window : all;
        const int64_t keys = (int64_t)sinks * frame < max_kv ? (int64_t)sinks * frame : max_kv;
        if (tiles < all) p.sink_blocks = (int)((keys + kKeys - 1) / kKeys);
    }
    // A workgroup a CU where the blocks alone do not give it, of eight tiles at least.
    const int64_t groups = (int64_t)p.blocks * kv_heads * sequences;
    int64_t parts = groups > 0 ? 256 / groups : 1;
    if (parts > tiles / 8) parts = tiles / 8;
    p.parts = (int)(parts < 1 ? 1 : parts);
    // A sink block's parts are about as long as another block's, where four workgroups a CU do not share
    // its work anyhow: each part is 2 x 128 rows of the workspace, written and read again (BF16, a window of
    // 16 tokens, 4,096 sinks: 4 x 8,192 tokens, 8 heads of 64, 1,762 us and 2.2 GB without that limit, 983 us and
    // 1 MB with it; 1 x 65,536: 4,159 and 2,163 us).
    p.sink_parts = p.parts;
    if (p.sink_blocks) {
        const int64_t each = (tiles + p.parts - 1) / p.parts, most = 1024 / ((int64_t)p.sink_blocks * kv_heads * sequences);
        const int64_t wanted = each > 0 ? (all + each - 1) / each : 1;
        const int64_t sink_parts = wanted < most ? wanted : most;
        p.sink_parts = (int)(sink_parts < p.parts ? p.parts : (sink_parts > 256 ? 256 : sink_parts));
    }
    return p;
}

template <typename T, int D>
hipError_t run(const AttentionArgs& a, const KeyPlan& p, hipStream_t stream) {
    BlockMap rows, keys;  // both before a launch: a call that is too large leaves everything as it was
    if (!block_map(((int64_t)a.max_q * a.group + 127) / 128, a.kv_heads, a.sequences, &rows) ||
        !block_map(p.items(), a.kv_heads, a.sequences, &keys))
        return hipErrorInvalidConfiguration;
    if (a.max_q > 0) {
        attention_dq_kernel<T, D><<<rows.grid, kThreads, 0, stream>>>(a, rows);
        if (hipError_t e = hipGetLastError()) return e;
    }
    if (a.max_kv <= 0) return hipSuccess;
    float* parts = (float*)a.workspace + ((a.q_tokens * a.q_heads + 3) & ~INT64_C(3));
    attention_dkv_kernel<T, D><<<keys.grid, kThreads, 0, stream>>>(a, keys, p, parts);
    if (hipError_t e = hipGetLastError()) return e;
    const int joined = p.parts > 1 ? p.blocks : (p.sink_parts > 1 ? p.sink_blocks : 0);
    if (!joined) return hipSuccess;
    attention_dkv_join_kernel<T, D><<<dim3((unsigned)joined * (kKeys * D / (kThreads * 4)), a.kv_heads, a.sequences), kThreads, 0, stream>>>(a, p, parts, 0);
    return hipGetLastError();
}

template <typename T>
hipError_t by_dim(const AttentionArgs& a, const KeyPlan& p, hipStream_t stream) {
    return a.dim == 64 ? run<T, 64>(a, p, stream) : run<T, 128>(a, p, stream);
}

}  // namespace
}  // namespace fa

size_t attention_backward_workspace(const dcn_attention_shape& s) {
    const fa::KeyPlan p = fa::key_plan(s.sequences, s.kv_heads, s.q_heads / s.kv_heads, s.max_q, s.max_kv, s.frame_tokens, s.back,
                                       s.ahead, s.sinks);
    size_t n = ((size_t)s.q_tokens * s.q_heads + 3) & ~(size_t)3;
    n += (size_t)s.sequences * s.kv_heads * p.kept() * 2 * fa::kKeys * s.head_dim;
    return n * sizeof(float);
}

hipError_t launch_attention_matrix_backward(int dtype, const AttentionArgs& a, hipStream_t stream) {
    const fa::KeyPlan p = fa::key_plan(a.sequences, a.kv_heads, a.group, a.max_q, a.max_kv, a.frame, a.back, a.ahead, a.sinks);
    return dtype == DCN_DTYPE_F16 ? fa::by_dim<_Float16>(a, p, stream) : fa::by_dim<fa::bf16>(a, p, stream);
}

}  // namespace dcn
