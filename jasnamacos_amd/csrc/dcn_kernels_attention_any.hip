// Frame attention of any type, head size up to 256 (gradients: 128), stride and alignment,
// contiguous or paged: FP32 products on v_mfma_f32_32x32x2_f32. The 16-bit heads of 64 and 128 channels have
// kernels of their own where they are aligned; this takes the rest.
//
// As there, S^T = K Q^T has keys as rows and packed query rows as columns: a lane holds one
// query row and, of 32 keys, the keys 8a + 4h + b (h = lane / 32) in register 4a + b. Register r
// is then the second product's B operand of the pair of keys 8a + b and 8a + 4 + b as it is, and
// softmax stays in a lane and lane ^ 32. Channels 8s + 4h + e are step 4s + e of the first product,
// so that a lane loads four adjacent ones. Operands come straight from memory, widened on the way:
// a lane its key's channels, 32 lanes one value row's, which whole lines serve in both cases.
//
// A workgroup has 32 rows; its four (or eight) waves take the key tiles in turn, without a barrier
// until their sums are joined through LDS. Where rows are few, workgroups share the key tiles of a
// block of rows, and a second kernel joins their parts. Bound: the FP32 products, a sixteenth of the
// 16-bit rate, of which it reaches under a third: every wave loads its keys and values from memory
// itself; for few rows the loads' latency. More than 64 channels do not fit 256 registers at two
// waves a SIMD: 67 to 78 of them are spilled up to 128 channels, 168 to 174 where rows are off four
// elements, 185 and 377 above 128 (one wave a SIMD, 512 registers). 2,048 causal tokens, 8 FP32 heads
// of 64: 95 us (45 of the 157 TFLOP/s), of 128: 162 us, of 256: 772 us; FP16 heads of 96: 163 us. One
// FP32 token on 8,000 paged keys, 8 sequences of 32 heads of 128 on 8: 170 us (3.1 TB/s).
#include "dcn_attention_any.hpp"

namespace dcn {
namespace fa {
namespace {

constexpr int kRowsWg = 32, kTile = 32;

// VEC: rows of four-element alignment and heads of whole fours. NB: blocks of 32 channels.
template <typename T, int NB, bool PAGED, bool VEC, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || NB <= 4 ? 2 : 1) void attention_any_kernel(AttentionArgs a, BlockMap map, int splits) {
    constexpr int LINE = NB * 32 + 4;
    __shared__ __attribute__((aligned(16))) float sums[kRowsWg][LINE];
    __shared__ float top_of[WAVES][kRowsWg], sum_of[WAVES][kRowsWg], inverse[kRowsWg];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
    Place pl;
    if (!place_of<kRowsWg>(a, map, splits, &pl)) return;
    const Rows rw = rows_of(a.group);
    const int last_row = pl.rows - 1 < pl.row0 + kRowsWg - 1 ? pl.rows - 1 : pl.row0 + kRowsWg - 1;
    const Spread all = spread_of(a, pl, rw, pl.row0, last_row);
    const int r = pl.row0 + n, rc = r < last_row ? r : last_row;
    const int tok = rw.token(rc), head = pl.kh * a.group + (rc - tok * a.group);
    const Span sp = r <= last_row ? span_of(a, pl.offset + tok, pl.kv.count) : Span{0, 0, 0};
    f32x4 q[NB * 4];
    {
        const T* qp = (const T*)a.q.p + (pl.q.first + tok) * a.q.ts + head * a.q.hs;
#pragma unroll
        for (int i = 0; i < NB * 4; ++i) q[i] = load4<T, VEC>(qp, 8 * i + 4 * h, a.dim);
    }
    const T* kp = (const T*)a.k.p + pl.kh * a.k.hs;
    const T* vp = (const T*)a.v.p + pl.kh * a.v.hs;
    const float c = a.scale * 1.44269504088896340736f;
    f32x16 o[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[i][x] = 0.f;
    float m = -INFINITY, l = 0.f;
    const TileList<kTile> list(all);
    const int per = (list.count + splits - 1) / splits, from = pl.split * per;
    const int stop = from + per < list.count ? from + per : list.count;
    for (int i = from + wave; i < stop; i += WAVES) {
        const int t0 = list.tile(i), j = t0 + n;
        // Row of this lane's key in memory; keys that are not there stand in for the last one, unseen.
        int64_t at = pl.kv.first + (j < pl.kv.count ? j : pl.kv.count - 1);
        uint32_t holes = 0;
        if constexpr (PAGED) {
            at = paged_row(a.pages, pl.seq, j < pl.kv.count ? j : pl.kv.count - 1);
            holes = (uint32_t)__ballot(at < 0);
            at = at < 0 ? 0 : at;
        }
        const bool partial = !all_see<kTile>(all, t0) || holes;
        f32x16 s;
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = 0.f;
        const T* key = kp + at * a.k.ts;
        // Values of 32 channels: register x is the pair of keys 8a + b (h = 0) and 8a + 4 + b (h = 1).
        const int64_t value = at * a.v.ts;
        auto load_values = [&](float* v, int b) {
            const int ch = 32 * b + n, in = ch < a.dim ? ch : a.dim - 1;
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const float t = widen(vp[__shfl(value, 8 * (x >> 2) + 4 * h + (x & 3)) + in]);
                v[x] = ch < a.dim ? t : 0.f;
            }
        };
        float v[2][16];
        load_values(v[0], 0);
#pragma unroll
        for (int b = 0; b < NB * 4; b += 8) {
            f32x4 k[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) k[e] = load4<T, VEC>(key, 8 * (b + e) + 4 * h, a.dim);
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int x = 0; x < 4; ++x) s = mma32(k[e][x], q[b + e][x], s);
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
        for (int b = 0; b < NB; ++b) {
            float* now = v[b & 1];
            if (b + 1 < NB) load_values(v[b + 1 & 1], b + 1);
            // A value that is not finite would reach rows that do not see it (0 x NaN): zero here, and
            // added below where it is seen.
            if (partial) {
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const bool fine = finite32(now[x]);
                    bad |= !fine;
                    now[x] = fine ? now[x] : 0.f;
                }
            }
#pragma unroll
            for (int x = 0; x < 16; ++x) o[b] = mma32(now[x], s[x], o[b]);
        }
        if (__builtin_expect(__any(bad), 0)) {
            for (int in = 0; in < kTile; ++in) {
                const bool on = sees(sp, t0 + in) && !(holes >> in & 1);
                const int64_t row = __shfl(at, in);
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const int ch = 32 * b + 8 * (x >> 2) + 4 * h + (x & 3);
                        const float one = on && ch < a.dim ? widen(vp[row * a.v.ts + ch]) : 0.f;
                        if (!finite32(one)) o[b][x] += one;
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
    for (int w = 1; w < WAVES; ++w) mt = fmaxf(mt, top_of[w][n]);
    const float ref = mt == -INFINITY ? 0.f : mt, f = exp2f(m - ref);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) lt += sum_of[w][n] * exp2f(top_of[w][n] - ref);
    for (int w = 0; w < WAVES; ++w) {
        if (wave == w)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    f32x4* to = (f32x4*)&sums[n][32 * b + 8 * x + 4 * h];
                    const f32x4 mine = {o[b][4 * x] * f, o[b][4 * x + 1] * f, o[b][4 * x + 2] * f, o[b][4 * x + 3] * f};
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
        for (int in = wave; in <= last_row - pl.row0; in += WAVES) {
            const int row = pl.row0 + in, t = rw.token(row), g = pl.kh * a.group + (row - t * a.group);
            float* to = (float*)a.workspace + (((pl.q.first + t) * a.q_heads + g) * splits + pl.split) * line;
            for (int ch = lane; ch < a.dim; ch += 64) to[ch] = sums[in][ch];
        }
        return;
    }
    if (wave == 0 && lane < 32) {
        inverse[n] = empty ? 0.f : 1.f / lt;
        if (a.lse && r <= last_row)
            a.lse[(pl.q.first + tok) * a.q_heads + head] = empty ? -INFINITY : (mt + log2f(lt)) * 0.69314718055994530942f;
    }
    __syncthreads();
    for (int in = wave; in <= last_row - pl.row0; in += WAVES) {
        const int row = pl.row0 + in, t = rw.token(row), g = pl.kh * a.group + (row - t * a.group);
        T* to = (T*)a.out.p + (pl.q.first + t) * a.out.ts + g * a.out.hs;
        for (int ch = lane; ch < a.dim; ch += 64) to[ch] = narrow<T>(sums[in][ch] * inverse[in]);
    }
}

// The parts of all splits (32 at most) of a row and head, by a wave: lane s has split s's maximum
// and sum; the sums are added in order of the splits.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_any_join_kernel(AttentionArgs a, int splits) {
    const int lane = threadIdx.x & 63, line = part_line(a.dim);
    const Run q = run_of(a.cu_q, blockIdx.z, a.max_q, a.q_tokens);
    const int64_t item = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
    const int64_t tok = item / a.q_heads;
    const int head = (int)(item - tok * a.q_heads);
    if (tok >= q.count || tok >= a.max_q) return;
    const int64_t row = q.first + tok, index = row * a.q_heads + head;
    const float* parts = (const float*)a.workspace + index * splits * line;
    const float m = lane < splits ? parts[lane * line + line - 4] : -INFINITY;
    const float l = lane < splits ? parts[lane * line + line - 3] : 0.f;
    const float top = wave_max(m), w = exp2f(m - (top == -INFINITY ? 0.f : top)), sum = wave_sum(w * l);
    const bool empty = top == -INFINITY && sum == 0.f;
    const float inv = empty ? 0.f : 1.f / sum;
    T* out = (T*)a.out.p + row * a.out.ts + head * a.out.hs;
    for (int first = 0; first < a.dim; first += 64) {
        const int ch = first + lane, at = ch < a.dim ? ch : a.dim - 1;
        float o = 0.f;
        for (int s = 0; s < splits; s += 8) {  // eight loads at once; w is 0 past the last split
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = s + u < splits ? parts[(s + u) * line + at] : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) o = fmaf(__shfl(w, s + u), v[u], o);
        }
        if (ch < a.dim) out[ch] = narrow<T>(o * inv);
    }
    if (a.lse && lane == 0) a.lse[index] = empty ? -INFINITY : (top + log2f(sum)) * 0.69314718055994530942f;
}

// Gradients, of heads of up to 128 channels: one pass over query rows (dQ and delta) and one over
// keys (dK, dV), both as above. A lane owns a row (KEYS: a key) x1 = q, x2 = dO (k, v) as B operands
// and the workgroup's waves take tiles of 32 of the other side, y1 = k, y2 = v (q, dO):
//   S = y1 x1, dP = y2 x2, dS = P (dP - delta), sum1 = sum dS y1 (dQ, dK), sum2 = sum P y2 (dV).
// delta is the sum of dO and out as it was rounded: in 16 bits that is off by a rounding's share of
// |dO| |out|, which rows of few keys show most (the 16-bit kernels take theirs from P and dP).
// Bound as above; 2 to 113 registers are spilled, but for query gradients of 65 to 128 aligned channels. A
// step of 1,024 causal tokens, forward included: 8 FP32 heads of 64: 272 us, BF16 heads of 96: 430 us (a row
// at a time 2.7 and 4.0 ms). 128 channels leave one wave a SIMD.
template <typename T, int NB, bool KEYS, bool VEC>
__global__ __launch_bounds__(kThreads, NB == 2 ? 2 : 1) void attention_any_grad_kernel(AttentionArgs a, BlockMap map) {
    constexpr int LINE = NB * 32 + 4;
    constexpr float kLog2e = 1.44269504088896340736f;
    __shared__ __attribute__((aligned(16))) float sums[kRowsWg][LINE];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
    Place pl;
    if constexpr (KEYS) {
        int block;
        if (!block_of(map, &block, &pl.kh, &pl.seq)) return;
        pl.q = run_of(a.cu_q, pl.seq, a.max_q, a.q_tokens);
        pl.kv = kv_run_of(a, pl.seq);
        pl.q.count = uniform(pl.q.count);
        pl.kv.count = uniform(pl.kv.count);
        pl.offset = pl.kv.count - pl.q.count;
        pl.rows = (pl.q.count < a.max_q ? pl.q.count : a.max_q) * a.group;
        pl.row0 = block * kRowsWg;
        if (pl.row0 >= pl.kv.count) return;
    } else if (!place_of<kRowsWg>(a, map, 1, &pl)) {
        return;
    }
    const Rows rw = rows_of(a.group);
    // What the lane owns (past the end: the last one, and nothing sees it or is written).
    const int owned = KEYS ? pl.kv.count : pl.rows, own = pl.row0 + n, oc = own < owned ? own : owned - 1;
    const int tok = KEYS ? 0 : rw.token(oc), head = KEYS ? 0 : pl.kh * a.group + (oc - tok * a.group);
    const int64_t index = (pl.q.first + tok) * a.q_heads + head;
    auto of_row = [&](const HeadsIn& t, int row) {  // element of packed row `row`'s first channel
        const int k = rw.token(row);
        return (pl.q.first + k) * t.ts + (pl.kh * a.group + (row - k * a.group)) * t.hs;
    };
    auto of_key = [&](const HeadsIn& t, int key) { return (pl.kv.first + key) * t.ts + pl.kh * t.hs; };
    const HeadsIn &own1 = KEYS ? a.k : a.q, &own2 = KEYS ? a.v : a.dout, &other1 = KEYS ? a.q : a.k, &other2 = KEYS ? a.dout : a.v;
    const T *y1 = (const T*)other1.p, *y2 = (const T*)other2.p;
    f32x4 x1[NB * 4], x2[NB * 4];
    {
        const T* p1 = (const T*)own1.p + (KEYS ? of_key(own1, oc) : of_row(own1, oc));
        const T* p2 = (const T*)own2.p + (KEYS ? of_key(own2, oc) : of_row(own2, oc));
#pragma unroll
        for (int i = 0; i < NB * 4; ++i) {
            x1[i] = load4<T, VEC>(p1, 8 * i + 4 * h, a.dim);
            x2[i] = load4<T, VEC>(p2, 8 * i + 4 * h, a.dim);
        }
    }
    float delta = 0.f, lse = 0.f;
    Span sp{0, 0, 0};
    Seen me{0, 0};
    int count, first;  // tiles of the other side
    if constexpr (KEYS) {
        if (own < owned) me = seen_of(a, own, pl.kv.count);
        const int last = pl.row0 + kRowsWg - 1 < owned ? pl.row0 + kRowsWg - 1 : owned - 1;
        const Seen f = seen_of(a, pl.row0, pl.kv.count), l = seen_of(a, last, pl.kv.count);
        // A sink's `to` is the end: the largest of a run of keys is that of its first or its last.
        int64_t from = (int64_t)(f.from - pl.offset) * a.group, to = (int64_t)((f.to > l.to ? f.to : l.to) - pl.offset) * a.group;
        from = from < 0 ? 0 : from;
        to = to < pl.rows ? to : pl.rows;
        first = (int)(from / kTile);
        count = to > from ? (int)((to + kTile - 1) / kTile) - first : 0;
    } else {
        const T* p = (const T*)a.o.p + of_row(a.o, oc);
#pragma unroll
        for (int i = 0; i < NB * 4; ++i) {
            const f32x4 o = load4<T, VEC>(p, 8 * i + 4 * h, a.dim);
#pragma unroll
            for (int e = 0; e < 4; ++e) delta = fmaf(o[e], x2[i][e], delta);
        }
        delta = both_sum(delta);
        lse = a.lse_in[index] * kLog2e;
        if (wave == 0 && lane < 32 && own < owned) ((float*)a.workspace)[index] = delta;
        if (own < owned) sp = span_of(a, pl.offset + tok, pl.kv.count);
        first = 0;
        count = 0;
    }
    const Spread all = KEYS ? Spread{} : spread_of(a, pl, rw, pl.row0, pl.row0 + kRowsWg - 1 < owned ? pl.row0 + kRowsWg - 1 : owned - 1);
    const TileList<kTile> list(all);
    if constexpr (!KEYS) count = list.count;
    const int others = KEYS ? pl.rows : pl.kv.count;
    const float c = a.scale * kLog2e;
    f32x16 sum1[NB], sum2[KEYS ? NB : 1];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            sum1[i][x] = 0.f;
            if constexpr (KEYS) sum2[i][x] = 0.f;
        }
    for (int i = wave; i < count; i += kWaves) {
        const int t0 = KEYS ? (first + i) * kTile : list.tile(i);
        const int j = t0 + n < others ? t0 + n : others - 1;
        const int64_t at1 = KEYS ? of_row(other1, j) : of_key(other1, j), at2 = KEYS ? of_row(other2, j) : of_key(other2, j);
        // A bit for each of the tile's 32 that see (or are seen by) what the lane owns.
        unsigned long long seen;
        float their_lse = 0.f, their_delta = 0.f;
        if constexpr (KEYS) {
            int64_t lo = (int64_t)(me.from - pl.offset) * a.group - t0, hi = (int64_t)(me.to - pl.offset) * a.group - t0;
            hi = hi < pl.rows - t0 ? hi : pl.rows - t0;
            seen = bits_below((int)(hi < 64 ? (hi < 0 ? 0 : hi) : 64)) & ~bits_below((int)(lo < 64 ? (lo < 0 ? 0 : lo) : 64));
            if (me.to <= me.from) seen = 0;
            const int k = rw.token(j);
            const int64_t theirs = (pl.q.first + k) * a.q_heads + pl.kh * a.group + (j - k * a.group);
            their_lse = a.lse_in[theirs] * kLog2e;
            their_delta = ((const float*)a.workspace)[theirs];
        } else {
            seen = seen_bits(sp, t0);
        }
        const bool partial = !__all((uint32_t)seen == ~0u);
        f32x16 s, dp;
#pragma unroll
        for (int x = 0; x < 16; ++x) s[x] = dp[x] = 0.f;
        bool bad = false;
#pragma unroll
        for (int b = 0; b < NB * 4; b += 4) {
            f32x4 f1[4], f2[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f1[e] = load4<T, VEC>(y1 + at1, 8 * (b + e) + 4 * h, a.dim);
                f2[e] = load4<T, VEC>(y2 + at2, 8 * (b + e) + 4 * h, a.dim);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    s = mma32(f1[e][x], x1[b + e][x], s);
                    dp = mma32(f2[e][x], x2[b + e][x], dp);
                    bad |= !finite32(f1[e][x]) || !finite32(f2[e][x]);
                }
        }
        // Vectors that are not finite, where some pair of the tile is not visible: zeros in the second
        // product, and the weights of the pairs that are visible are NaN.
        uint32_t poison = 0;
        if (partial) {
            const unsigned long long lanes = __ballot(bad);
            poison = (uint32_t)(lanes | lanes >> 32);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const int in = 8 * (x >> 2) + 4 * h + (x & 3);
            const float ref = KEYS ? __shfl(their_lse, in) : lse, d = KEYS ? __shfl(their_delta, in) : delta;
            s[x] = __builtin_amdgcn_exp2f(fmaf(s[x], c, -ref));
            dp[x] = s[x] * (dp[x] - d);
            if (poison >> in & 1) s[x] = dp[x] = NAN;
            const uint32_t on = spread_bit(seen >> (4 * h), 8 * (x >> 2) + (x & 3));
            s[x] = keep_or(s[x], on, 0.f);
            dp[x] = keep_or(dp[x], on, 0.f);
        }
        auto product = [&](const T* y, int64_t at, const f32x16& w, f32x16& sum, int b) {
            const int ch = 32 * b + n, cc = ch < a.dim ? ch : a.dim - 1;
            float v[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
                const float t = widen(y[__shfl(at, 8 * (x >> 2) + 4 * h + (x & 3)) + cc]);
                v[x] = ch < a.dim && !(poison && !finite32(t)) ? t : 0.f;
            }
#pragma unroll
            for (int x = 0; x < 16; ++x) sum = mma32(v[x], w[x], sum);
        };
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            product(y1, at1, dp, sum1[b], b);
            if constexpr (KEYS) product(y2, at2, s, sum2[b], b);
        }
    }
    // The waves' sums, in order, and the rows (keys) of this workgroup.
    auto join = [&](const f32x16* sum, const HeadsOut& out, float by) {
        for (int w = 0; w < kWaves; ++w) {
            if (wave == w)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        f32x4* to = (f32x4*)&sums[n][32 * b + 8 * x + 4 * h];
                        const f32x4 mine = {sum[b][4 * x], sum[b][4 * x + 1], sum[b][4 * x + 2], sum[b][4 * x + 3]};
                        *to = w ? *to + mine : mine;
                    }
            __syncthreads();
        }
        for (int in = wave; in < kRowsWg && pl.row0 + in < owned; in += kWaves) {
            const int row = pl.row0 + in, k = KEYS ? 0 : rw.token(row);
            T* to = (T*)out.p + (KEYS ? (pl.kv.first + row) * out.ts + pl.kh * out.hs
                                      : (pl.q.first + k) * out.ts + (pl.kh * a.group + (row - k * a.group)) * out.hs);
            for (int ch = lane; ch < a.dim; ch += 64) to[ch] = narrow<T>(sums[in][ch] * by);
        }
        __syncthreads();
    };
    join(sum1, KEYS ? a.dk : a.dq, a.scale);
    if constexpr (KEYS) join(sum2, a.dv, 1.f);
}

template <typename T>
hipError_t join(const AttentionArgs& a, int splits, hipStream_t stream) {
    const int64_t rows = (int64_t)a.max_q * a.q_heads;
    attention_any_join_kernel<T><<<dim3((unsigned)((rows + kWaves - 1) / kWaves), 1, a.sequences), kThreads, 0, stream>>>(a, splits);
    return hipGetLastError();
}

template <typename T, int NB, bool PAGED, bool VEC>
hipError_t run(const AttentionArgs& a, hipStream_t stream) {
    BlockMap map;
    const int splits = a.any_splits;
    const int64_t blocks = ((int64_t)a.max_q * a.group + kRowsWg - 1) / kRowsWg;
    if (!block_map(blocks * splits, a.kv_heads, a.sequences, &map)) return hipErrorInvalidConfiguration;
    // Where there is no workgroup for every CU eight waves share the keys (8 sequences of 8,000 keys,
    // 32 FP32 heads of 128 on 8 key heads: 721 us with four, 487 so).
    if (NB <= 4 && blocks * a.kv_heads * a.sequences <= 256)
        attention_any_kernel<T, NB, PAGED, VEC, NB <= 4 ? 8 : 4><<<map.grid, 512, 0, stream>>>(a, map, splits);
    else
        attention_any_kernel<T, NB, PAGED, VEC, 4><<<map.grid, 256, 0, stream>>>(a, map, splits);
    if (hipError_t e = hipGetLastError()) return e;
    return splits == 1 ? hipSuccess : join<T>(a, splits, stream);
}
template <typename T, int NB, bool PAGED>
hipError_t by_rows(const AttentionArgs& a, hipStream_t stream) {
    return a.dim % 4 == 0 && fours<T>(a.q) && fours<T>(a.k) ? run<T, NB, PAGED, true>(a, stream) : run<T, NB, PAGED, false>(a, stream);
}
template <typename T, bool PAGED>
hipError_t by_dim(const AttentionArgs& a, hipStream_t stream) {
    return a.dim <= 64 ? by_rows<T, 2, PAGED>(a, stream) : (a.dim <= 128 ? by_rows<T, 4, PAGED>(a, stream) : by_rows<T, 8, PAGED>(a, stream));
}
template <typename T>
hipError_t by_keys(const AttentionArgs& a, hipStream_t stream) {
    return a.pages.table ? by_dim<T, true>(a, stream) : by_dim<T, false>(a, stream);
}

template <typename T, int NB, bool VEC>
hipError_t run_grad(const AttentionArgs& a, hipStream_t stream) {
    BlockMap rows, keys;
    if (!block_map(((int64_t)a.max_q * a.group + kRowsWg - 1) / kRowsWg, a.kv_heads, a.sequences, &rows) ||
        !block_map(((int64_t)a.max_kv + kRowsWg - 1) / kRowsWg, a.kv_heads, a.sequences, &keys))
        return hipErrorInvalidConfiguration;
    if (a.max_q > 0) {
        attention_any_grad_kernel<T, NB, false, VEC><<<rows.grid, kThreads, 0, stream>>>(a, rows);
        if (hipError_t e = hipGetLastError()) return e;
    }
    if (a.max_kv <= 0) return hipSuccess;
    attention_any_grad_kernel<T, NB, true, VEC><<<keys.grid, kThreads, 0, stream>>>(a, keys);
    return hipGetLastError();
}
template <typename T>
hipError_t grad(const AttentionArgs& a, hipStream_t stream) {
    bool vec = a.dim % 4 == 0;
    for (const HeadsIn* h : {&a.q, &a.k, &a.v, &a.o, &a.dout}) vec = vec && fours<T>(*h);
    if (a.dim <= 64) return vec ? run_grad<T, 2, true>(a, stream) : run_grad<T, 2, false>(a, stream);
    return vec ? run_grad<T, 4, true>(a, stream) : run_grad<T, 4, false>(a, stream);
}

}  // namespace
}  // namespace fa

hipError_t launch_attention_any_backward(int dtype, const AttentionArgs& a, hipStream_t stream) {
    // Two vectors and two sums of more than 128 channels do not fit a lane's registers.
    if (a.dim > 128) return launch_attention_rows_backward(dtype, a, stream);
    if (dtype == DCN_DTYPE_F16) return fa::grad<_Float16>(a, stream);
    if (dtype == DCN_DTYPE_BF16) return fa::grad<fa::bf16>(a, stream);
    return fa::grad<float>(a, stream);
}

int attention_any_splits(const dcn_attention_shape& s) {
    const int group = s.q_heads / s.kv_heads;
    const int64_t blocks = ((int64_t)s.max_q * group + fa::kRowsWg - 1) / fa::kRowsWg, groups = blocks * s.kv_heads * s.sequences;
    const int64_t keys = attention_keys(s.max_kv, s.frame_tokens, s.back, s.sinks, fa::kRowsWg / group, fa::kTile);
    const int64_t tiles = (keys + fa::kTile - 1) / fa::kTile, waves = s.head_dim <= 128 ? 8 : 4;
    // Row blocks that leave half of the CUs idle or more: a workgroup a CU, of a tile a wave at least,
    // and 32 parts the most that the join adds quickly. Up to two tiles a wave the join costs what it
    // saves. One FP32 token, whole and in parts: 540 keys of 8 heads of 64: 23.9 and 20.4 us; 8,000:
    // 224 and 24; for 8 sequences of 32 heads of 128 on 8, 488 and 170; 16 of 8 heads of 64, 309 and 174.
    if (groups < 1 || groups > 128 || tiles <= 2 * waves) return 1;
    int64_t splits = 256 / groups;
    splits = splits < tiles / waves ? splits : tiles / waves;
    return (int)(splits < 32 ? splits : 32);
}

size_t attention_any_workspace(const dcn_attention_shape& s) {
    const int splits = attention_any_splits(s);
    return splits == 1 ? 0 : (size_t)s.q_tokens * s.q_heads * splits * fa::part_line(s.head_dim) * sizeof(float);
}

hipError_t launch_attention_any_join(int dtype, const AttentionArgs& a, int splits, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16) return fa::join<_Float16>(a, splits, stream);
    if (dtype == DCN_DTYPE_BF16) return fa::join<fa::bf16>(a, splits, stream);
    return fa::join<float>(a, splits, stream);
}

hipError_t launch_attention_any(int dtype, const AttentionArgs& a, hipStream_t stream) {
    if (dtype == DCN_DTYPE_F16) return fa::by_keys<_Float16>(a, stream);
    if (dtype == DCN_DTYPE_BF16) return fa::by_keys<fa::bf16>(a, stream);
    return fa::by_keys<float>(a, stream);
}

}  // namespace dcn
