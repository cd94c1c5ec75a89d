// Attention over microscaled pages, and of sequences that share a prefix over pages of either kind, on
// the matrix cores: FP16 and BF16 heads of 64 and 128 channels.
//
// The keys of a row are two runs: the prefix's, then its sequence's own, each with a table of pages;
// tiles of keys lie in one of them. What a workgroup takes is
//   a block of packed rows of one sequence, over its own keys or over both runs, or
//   a block of packed rows of all sequences, over the prefix's keys: read once for all of them,
// and of those keys all tiles or a part. Parts of a row are joined in FP32 by a second kernel.
//
// Microscaled tiles go through registers: loaded a tile ahead, taken to 16 bits by the scaled
// conversions (exact: a code has 4 bits of significand at most; FP16 rounds below 2^-14 and beyond
// 65504), stored to LDS as rows of the 16-bit kernels, whose products then run as they are. The
// scales are in the values, so a block of 32 channels costs its scale's load and nothing else.
#include "dcn_attention_pages.hpp"
#include "dcn_attention_plan.hpp"

namespace dcn {
namespace fa {
namespace {

template <int D>
constexpr int tile_bytes() {
    return 2 * 2 * 64 * D * 2;
}
// 128 rows, 32 a wave, over tiles of 64 keys in LDS that the four waves fill together: the 16-bit kernels'
// loop, with codes loaded two tiles ahead in registers and stored one ahead. A frame of 3,600 tokens for two
// streams on 14,400 keys of 8 bits, 8 heads of 64: 340 us, 546 TFLOP/s; the vector units are busy 45 % of the
// time, the matrix units 20 %: at 64 channels the softmax is longer than its products, and two waves a SIMD do not
// hide all of its latencies (three spill: 486 us). 128 channels in microscaled pages leave no registers
// for the reads of 64 keys at once: they are taken by half (64 streams on a shared prefix: 55 -> 52 us).
template <typename T, int D, int BITS>
__device__ __forceinline__ void tile_block(const PagesCall& c, unsigned number, char* memory, FoundRows& found) {
    constexpr int ROWS = 64, BYTES = ROWS * D * 2;
    char(*lds)[2][BYTES] = (char(*)[2][BYTES])memory;
    const PagesAttention& p = c.p;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Block b;
    if (!block_place<32 * kWaves>(c, number, &b)) return;
    Place& pl = b.pl;
    const int r = pl.row0 + 32 * wave + (lane & 31);
    RowState<T, D> st;
    st.clear();
    load_queries<D / 16>(st.q, c, pl, r, 8 * (lane >> 5), 16);
    const int rows[2] = {pl.row0 + lane, pl.row0 + 64 + lane};
    int place[2], low, high, low1, high1;
    positions_of<2>(c, b, rows, lane, place);
    const int at = __shfl(wave & 2 ? place[1] : place[0], 32 * (wave & 1) + (lane & 31));
    if (b.all) {
        extremes<64>(c, b, 0, 0, place[0], &low, &high);
        extremes<64>(c, b, 0, 0, place[1], &low1, &high1);
        low = low1 < low ? low1 : low;
        high = high1 > high ? high1 : high;
    } else {
        extremes<64>(c, b, pl.row0, 32 * kWaves, 0, &low, &high);
    }
    if (high == kNowhere) return;  // no row of a sequence
    extremes<32>(c, b, pl.row0 + 32 * wave, 32, at, &low1, &high1);
    const bool idle = high1 == kNowhere;  // no rows: the wave copies only
    int count;
    Cursor<ROWS> now(c, b, low, high, &count);
    Spread all = spread_in(c, b, low, high, now.second), mine = spread_in(c, b, low1, high1, now.second);  // all: of the run ahead
    const int from = pl.split * b.per, to = last_tile(count, from, b);
    const float scale = p.a.scale * kLog2e;
    Stage<T, D, BITS, ROWS, kWaves> stage(p, pl.kh, wave, lane);
    Cursor<ROWS> ahead = now;
    bool next_part = false;  // whether some row does not see all of the tile that was found last
    auto find = [&](int i) {
        if (ahead.go(c, b, low, high, i)) all = spread_in(c, b, low, high, 1);
        const int t0 = ahead.tile(i);
        stage.find(p, ahead.run, pl.kh, t0, wave);
        next_part = stage.holes || !all_see<ROWS>(all, t0);
    };
    // Of the present tile, the one behind it, and the one behind that: holes, and whether it is seen in part.
    unsigned long long holes = 0, holes1 = 0;
    bool part = false, part1 = false;
    if (from < to) {
        find(from);
        holes = stage.holes;
        part = next_part;
        if constexpr (BITS == 16) {
            stage.copy(lds[0][0], lds[0][1], wave, lane);
            if (from + 1 < to) find(from + 1);
        } else {
            stage.load(lane);
            found.wave[0][wave] = stage.store(lds[0][0], lds[0][1], part, wave, lane);
            if (from + 1 < to) {
                find(from + 1);
                holes1 = stage.holes;
                part1 = next_part;
                stage.load(lane);
                if (from + 2 < to) find(from + 2);
            }
        }
    }
    if constexpr (BITS != 16) __syncthreads();
    st.settle();
    for (int i = from; i < to; ++i) {
        const int buf = (i - from) & 1;
        if (now.go(c, b, low, high, i)) mine = spread_in(c, b, low1, high1, 1);
        const int t0 = now.tile(i);
        char(*here)[BYTES] = lds[buf], (*other)[BYTES] = lds[buf ^ 1];
        unsigned long long holes2 = 0;
        bool part2 = false;
        if constexpr (BITS == 16) {
            wait_copies<0>();
            // Values that are not finite matter where some row does not see all of the tile: zero times
            // them is not zero. Each wave looks at what it copied.
            if (part) found.wave[buf][wave] = clean_own<T, D, ROWS, kWaves>(here[1], wave, lane);
            __syncthreads();
            if (i + 1 < to) {
                stage.copy(other[0], other[1], wave, lane);
                holes1 = stage.holes;
                part1 = next_part;
                if (i + 2 < to) find(i + 2);
            }
        } else if (i + 1 < to) {
            found.wave[buf ^ 1][wave] = stage.store(other[0], other[1], part1, wave, lane);
            if (i + 2 < to) {
                stage.load(lane);
                holes2 = stage.holes;
                part2 = next_part;
                if (i + 3 < to) find(i + 3);
            }
        }
        const bool bad = part && uniform(found.all(buf) != 0);
        if (!idle && !none_sees<ROWS>(mine, t0)) {
            const bool masked = holes || !all_see<ROWS>(mine, t0);
            if (masked || bad) st.sp = b.span(c, at, now.second);
            st.template add<ROWS, D == 128 && BITS != 16>(here[0], here[1], t0, scale, masked, holes, lane);
            if (bad) add_bad<T, D, BITS>(p, now.run, pl.kh, st.o, st.sp, t0, ROWS, holes, lane);
        }
        holes = holes1;
        part = part1;
        if constexpr (BITS != 16) {
            holes1 = holes2;
            part1 = part2;
            __syncthreads();
        }
    }
    if (at == kNowhere) return;
    number_part(c, b, &pl);
    const Target to_row = target_of(c, pl, r);
    const float l = both_sum(st.l), inv = l == 0.f ? 0.f : 1.f / l;
    if (pl.splits == 1 || st.m != -INFINITY) {  // a part that saw nothing has no output
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float o[4] = {st.o[i][4 * x], st.o[i][4 * x + 1], st.o[i][4 * x + 2], st.o[i][4 * x + 3]};
                store_row4<T, D>(p.a, pl, to_row.index, to_row.row, to_row.head, 32 * i + 8 * x + 4 * (lane >> 5), o, inv);
            }
    }
    if (lane < 32) store_sums<D>(p.a, pl, to_row.index, st.m, l, kLift<T>);
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads, 2) void pages_tile_kernel(PagesCall c) {
    __shared__ __attribute__((aligned(1024))) char lds[tile_bytes<D>()];
    __shared__ FoundRows found;
    tile_block<T, D, BITS>(c, blockIdx.x, lds, found);
}

// 32 rows, all of them for each wave, whose waves take tiles of 32 keys in turn without a barrier, each through
// LDS of its own, until they are joined. It fills the card where there are few rows, and reads the keys
// for every 32 of them: bound by the caches, about 12 TB/s. 8 continuations of a clip, a frame of 256
// tokens each, 8 FP16 heads of 64 on 4, 4,352 keys: 47 us (128 rows in parts: 57).
//
// LDS of a wave: pages of the type have two tiles, one in flight.
template <int D, int BITS>
constexpr int few_wave_bytes() {
    return (BITS == 16 ? 4 : 2) * 32 * D * 2;
}

template <typename T, int D, int BITS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || BITS != 16 ? 2 : 1) void pages_few_kernel(PagesCall c) {
    constexpr int ROWS = 32, BYTES = ROWS * D * 2, COPIES = 2 * ROWS / Tile<D>::kRowsPerCopy;
    extern __shared__ __attribute__((aligned(1024))) char lds[];  // each wave's tiles, then the join
    const PagesAttention& p = c.p;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Block b;
    if (!block_place<32>(c, blockIdx.x, &b)) return;
    Place& pl = b.pl;
    const int r = pl.row0 + (lane & (32 - 1));
    RowState<T, D> st;
    st.clear();
    load_queries<D / 16>(st.q, c, pl, r, 8 * (lane >> 5), 16);
    int place, low, high;
    positions_of<1>(c, b, &r, lane, &place);
    extremes<32>(c, b, pl.row0, 32, place, &low, &high);
    if (high == kNowhere) return;  // no row of a sequence
    int count;
    Cursor<ROWS> now(c, b, low, high, &count);
    const int from = pl.split * b.per, to = last_tile(count, from, b);
    if (from >= to && c.parts > 1) {  // nothing but that there is nothing
        if (threadIdx.x < 32 && place != kNowhere) {
            number_part(c, b, &pl);
            store_sums<D>(p.a, pl, target_of(c, pl, r).index, -INFINITY, 0.f, kLift<T>);
        }
        return;
    }
    Spread all = spread_in(c, b, low, high, now.second);
    const float scale = p.a.scale * kLog2e;
    char* own = lds + wave * few_wave_bytes<D, BITS>();
    Stage<T, D, BITS, ROWS, 1> stage(p, pl.kh, 0, lane);
    Cursor<ROWS> ahead = now;
    auto find = [&](int i) {
        ahead.go(c, b, low, high, i);
        stage.find(p, ahead.run, pl.kh, ahead.tile(i), 0);
    };
    unsigned long long holes = 0;
    int n = 0;
    if (from + wave < to) {
        find(from + wave);
        if constexpr (BITS == 16) stage.copy(own, own + BYTES, 0, lane);
        else stage.load(lane);
        holes = stage.holes;
    }
    if (from + wave + WAVES < to) find(from + wave + WAVES);
    st.settle();
    for (int i = from + wave; i < to; i += WAVES, ++n) {
        char *kt = own, *vt = kt + BYTES;
        if (now.go(c, b, low, high, i)) all = spread_in(c, b, low, high, 1);
        const int t0 = now.tile(i);
        const bool whole = !holes && all_see<ROWS>(all, t0);
        bool bad;
        unsigned long long next_holes = 0;
        if constexpr (BITS == 16) {
            kt = own + (n & 1) * 2 * BYTES;
            vt = kt + BYTES;
            char* other = own + ((n + 1) & 1) * 2 * BYTES;
            if (i + WAVES < to) {
                stage.copy(other, other + BYTES, 0, lane);
                next_holes = stage.holes;
                if (i + 2 * WAVES < to) find(i + 2 * WAVES);
                wait_copies<COPIES>();
            } else {
                wait_copies<0>();
            }
            bad = !whole && clean_own<T, D, ROWS, 1>(vt, 0, lane);
        } else {
            bad = stage.store(kt, vt, !whole, 0, lane);
            if (i + WAVES < to) {
                stage.load(lane);
                next_holes = stage.holes;
                if (i + 2 * WAVES < to) find(i + 2 * WAVES);
            }
        }
        if (!whole) st.sp = b.span(c, place, now.second);
        st.template add<ROWS>(kt, vt, t0, scale, !whole, holes, lane);
        if (bad) add_bad<T, D, BITS>(p, now.run, pl.kh, st.o, st.sp, t0, ROWS, holes, lane);
        holes = next_holes;
        if constexpr (BITS == 16) wait_reads();  // the next copies go where this tile was
    }
    // Join the waves: [wave][32 rows][D + 4] FP32 (rows of D + 4 keep the stores off each other's banks).
    __syncthreads();
    float* mem = (float*)lds;
    constexpr int LINE = D + 4;
    float* line = mem + (wave * 32 + (lane & 31)) * LINE;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x)
            *(f32x4*)(line + 32 * i + 8 * x + 4 * (lane >> 5)) =
                f32x4{st.o[i][4 * x], st.o[i][4 * x + 1], st.o[i][4 * x + 2], st.o[i][4 * x + 3]};
    const float l = both_sum(st.l);
    if (lane < 32) {
        line[D] = st.m;
        line[D + 1] = l;
        line[D + 2] = place == kNowhere ? 0.f : 1.f;
    }
    __syncthreads();
    // Two threads a row and wave.
    constexpr int share = 2 * WAVES;
    const int jr = threadIdx.x / share, part = threadIdx.x % share;
    if (mem[jr * LINE + D + 2] == 0.f) return;  // a row of no sequence
    float m = -INFINITY, sum = 0.f, w[WAVES];
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, mem[(i * 32 + jr) * LINE + D]);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        w[i] = exp2f(mem[(i * 32 + jr) * LINE + D] - (m == -INFINITY ? 0.f : m));
        sum = fmaf(w[i], mem[(i * 32 + jr) * LINE + D + 1], sum);
    }
    number_part(c, b, &pl);
    const Target to_row = target_of(c, pl, pl.row0 + jr);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int at = part * 4; at < D; at += 4 * share) {
        if (pl.splits > 1 && m == -INFINITY) break;  // a part that saw nothing has no output
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const f32x4 v = *(const f32x4*)(mem + (i * 32 + jr) * LINE + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(w[i], v[e], o[e]);
        }
        const float four[4] = {o[0], o[1], o[2], o[3]};
        store_row4<T, D>(p.a, pl, to_row.index, to_row.row, to_row.head, at, four, inv);
    }
    if (part == 0) store_sums<D>(p.a, pl, to_row.index, m, sum, kLift<T>);
}

// 16 rows, for single tokens: as above, with v_mfma_f32_16x16x32 and keys straight from memory. Loads of the
// next tile are in flight behind the products of this one. 32 streams' tokens on up to 18,001 keys, 32 heads of 128
// on 8: 156 us in 8 bits (5.3 TB/s; 32 rows a block 217), 100 in 4 (4.3 TB/s). One token on 997 keys, 8 heads of 64:
// 10.6 us, a chain of latencies (16 waves; four and a join 12.7).
//
// LDS: each wave's values, then the join.
template <int D, int WAVES>
constexpr int token_bytes() {
    constexpr int values = WAVES * 32 * D * 2, join = WAVES * 16 * (D + 4) * 4;
    return values > join ? values : join;
}
template <typename T, int D, int BITS, int WAVES>
__device__ __forceinline__ void token_block(const PagesCall& c, unsigned number, char* lds) {
    constexpr int ROWS = 32, NR = 16, BYTES = ROWS * D * 2, LINE = D + 4;
    const PagesAttention& p = c.p;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Block b;
    if (!block_place<NR>(c, number, &b)) return;
    Place& pl = b.pl;
    const int r = pl.row0 + (lane & (NR - 1));
    FewRows<T, D> st;
    st.clear();
    load_queries<D / 32>(st.q, c, pl, r, D / 4 * (lane >> 4), 8);
    int place, low, high;
    positions_of<1>(c, b, &r, lane, &place);
    extremes<NR>(c, b, pl.row0, NR, place, &low, &high);
    if (high == kNowhere) return;  // no row of a sequence
    int count;
    Cursor<ROWS> now(c, b, low, high, &count);
    const int from = pl.split * b.per, to = last_tile(count, from, b);
    if (from >= to && c.parts > 1) {  // nothing but that there is nothing
        if (threadIdx.x < NR && place != kNowhere) {
            number_part(c, b, &pl);
            store_sums<D>(p.a, pl, target_of(c, pl, r).index, -INFINITY, 0.f, kLift<T>);
        }
        return;
    }
    Spread all = spread_in(c, b, low, high, now.second);
    const float scale = p.a.scale * kLog2e;
    char* vt = lds + wave * BYTES;
    FewStage<T, D, BITS> stage;
    Cursor<ROWS> ahead = now;
    auto find = [&](int i) {
        ahead.go(c, b, low, high, i);
        stage.find(p, ahead.run, pl.kh, ahead.tile(i));
    };
    unsigned long long holes = 0;
    if (from + wave < to) {
        find(from + wave);
        stage.load(p, pl.kh, lane);
        holes = stage.holes;
    }
    if (from + wave + WAVES < to) find(from + wave + WAVES);
    for (int i = from + wave; i < to; i += WAVES) {
        if (now.go(c, b, low, high, i)) all = spread_in(c, b, low, high, 1);
        const int t0 = now.tile(i);
        const bool whole = !holes && all_see<ROWS>(all, t0);
        const bool bad = stage.store(vt, !whole, lane);
        f32x4 s[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            s[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < D / 32; ++e) s[x] = st.mma16(stage.keys(x, e), st.q[e], s[x]);
        }
        unsigned long long next_holes = 0;
        if (i + WAVES < to) {
            stage.load(p, pl.kh, lane);
            next_holes = stage.holes;
            if (i + 2 * WAVES < to) find(i + 2 * WAVES);
        }
        if (!whole) st.sp = b.span(c, place, now.second);
        const u32x4 w = st.weigh(s, t0, scale, !whole, holes, lane);
#pragma unroll
        for (int x = 0; x < D / 16; ++x) st.o[x] = st.mma16(st.values(vt, x, lane), w, st.o[x]);
        if (bad) {
            const int end = t0 + ROWS < now.run.count ? t0 + ROWS : now.run.count;
            for (int j = t0; j < end; ++j) {
                const int64_t row = now.run.template pool_row<BITS>(p, j, pl.kh);
                if (row < 0) continue;
                const bool on = sees(st.sp, j) && !(holes >> (j - t0) & 1);
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    const u32x2 four = value4<T, D, BITS>(p, row, pl.kh, 16 * x + 4 * (lane >> 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t bits = (uint16_t)(four[e >> 1] >> (16 * (e & 1)));
                        if (on && !finite16<T>(bits)) st.o[x][e] += widen(__builtin_bit_cast(T, bits));
                    }
                    asm volatile("" ::: "memory");  // few registers: this is rare
                }
            }
        }
        holes = next_holes;
    }
    // Join the waves: [wave][16 rows][D + 4] FP32 (rows of D + 4 keep the stores off each other's banks).
    __syncthreads();
    float* mem = (float*)lds;
    float* line = mem + (wave * NR + (lane & 15)) * LINE;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) *(f32x4*)(line + 16 * i + 4 * (lane >> 4)) = st.o[i];
    const float l = st.quarters_sum(st.l);
    if (lane < NR) {
        line[D] = st.m;
        line[D + 1] = l;
        line[D + 2] = place == kNowhere ? 0.f : 1.f;
    }
    __syncthreads();
    constexpr int share = 64 * WAVES / NR;  // threads a row
    const int jr = threadIdx.x / share, part = threadIdx.x % share;
    if (mem[jr * LINE + D + 2] == 0.f) return;  // a row of no sequence
    float m = -INFINITY, sum = 0.f, w[WAVES];
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, mem[(i * NR + jr) * LINE + D]);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        w[i] = exp2f(mem[(i * NR + jr) * LINE + D] - (m == -INFINITY ? 0.f : m));
        sum = fmaf(w[i], mem[(i * NR + jr) * LINE + D + 1], sum);
    }
    number_part(c, b, &pl);
    const Target to_row = target_of(c, pl, pl.row0 + jr);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int at = part * 4; at < D; at += 4 * share) {
        if (pl.splits > 1 && m == -INFINITY) break;  // a part that saw nothing has no output
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const f32x4 v = *(const f32x4*)(mem + (i * NR + jr) * LINE + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(w[i], v[e], o[e]);
        }
        const float four[4] = {o[0], o[1], o[2], o[3]};
        store_row4<T, D>(p.a, pl, to_row.index, to_row.row, to_row.head, at, four, inv);
    }
    if (part == 0) store_sums<D>(p.a, pl, to_row.index, m, sum, kLift<T>);
}

template <typename T, int D, int BITS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 16 ? 4 : 2) void pages_token_kernel(PagesCall c) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    token_block<T, D, BITS, WAVES>(c, blockIdx.x, lds);
}

// The prefix for many rows and the sequences' own keys for single tokens in one launch: the first
// is bound by the products, the second by memory, and a CU takes a workgroup of each. 64 streams' tokens
// on a prefix of 14,400 and up to 901 of their own, 32 heads of 128 on 8: 68 us with the join (in two launches 80;
// 3.3 TB/s, the prefix read once), in 8 bits 52. Workgroups for the prefix: 128 78 us, 192 68, 256 68, 320 73, 512 80; in
// 8 bits 77, 58, 52, 61, 59.
template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads, 2) void pages_mixed_kernel(PagesCall c) {
    __shared__ __attribute__((aligned(1024))) char lds[tile_bytes<D>()];
    __shared__ FoundRows found;
    static_assert(tile_bytes<D>() >= token_bytes<D, kWaves>(), "");
    const unsigned first = c.prefix.grid < 256 ? c.prefix.grid : 256, own = c.own.grid < 256 ? c.own.grid : 256;
    // A workgroup of each for every CU, then the rest; runs of 8 workgroups stay together, one on each XCD.
    unsigned i = blockIdx.x;
    if (i >= first) {
        if (i < first + own) i += c.prefix.grid - first;
        else if (i < c.prefix.grid + own) i -= own;
    }
    if (i < c.prefix.grid) tile_block<T, D, BITS>(c, i, lds, found);
    else token_block<T, D, BITS, kWaves>(c, i, lds);
}

// The parts (64 at most) of a row and head, by PER waves: lane s of each has part s's maximum and sum;
// the waves take the parts' outputs in turn and are added in order. A part that saw nothing has
// written no output. Bound by latency: 2,048 rows of 128 channels in 16 parts 6 us, in two 4.8.
template <typename T, int D, int PER>
__global__ __launch_bounds__(kThreads) void pages_join_kernel(AttentionArgs a, int parts) {
    typedef float vec __attribute__((ext_vector_type(D / 64)));
    constexpr int N = D / 64, AT_ONCE = 4;
    __shared__ vec sums[kWaves][64];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const Run q = run_of(a.cu_q, blockIdx.z, a.max_q, a.q_tokens);
    const int64_t item = (int64_t)blockIdx.x * (kWaves / PER) + wave / PER;
    const int tok = (int)(item / a.q_heads), head = (int)(item % a.q_heads);
    const bool there = tok < q.count && tok < a.max_q;
    const int64_t row = q.first + (there ? tok : 0), index = row * a.q_heads + head;
    const float* of = (const float*)a.workspace + index * parts * (D + 4);
    float m = -INFINITY, l = 0.f;
    if (there && lane < parts) {
        m = of[lane * (D + 4) + D];
        l = of[lane * (D + 4) + D + 1];
    }
    const float top = wave_max(m);
    const float w = exp2f(m - (top == -INFINITY ? 0.f : top)), sum = wave_sum(w * l);
    float o[N] = {};
    unsigned long long left = __ballot(m != -INFINITY);
    // This wave's parts: every PER-th of those with an output.
    for (int skip = wave % PER; skip && left; --skip) left &= left - 1;
    while (left) {
        vec v[AT_ONCE];
        int part[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            part[u] = left ? __builtin_ctzll(left) : -1;
            v[u] = vec(0.f);
            if (left) v[u] = *(const vec*)(of + part[u] * (D + 4) + lane * N);
#pragma unroll
            for (int i = 0; i < PER; ++i) left &= left - 1;
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const float weight = __shfl(w, part[u] & 63);
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] = part[u] < 0 ? o[i] : fmaf(weight, v[u][i], o[i]);
        }
    }
    if constexpr (PER > 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) sums[wave][lane][i] = o[i];
        __syncthreads();
        if (wave % PER) return;
#pragma unroll
        for (int g = 1; g < PER; ++g)
#pragma unroll
            for (int i = 0; i < N; ++i) o[i] += sums[wave + g][lane][i];
    }
    if (!there) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = (T*)a.out.p + row * a.out.ts + head * a.out.hs + lane * N;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = narrow<T>(o[i] * inv);
    if (a.lse && lane == 0) a.lse[index] = sum == 0.f ? -INFINITY : (top - kLift<T> + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <typename T, int D, int BITS, int WAVES>
hipError_t run_few(const PagesCall& c, hipStream_t stream) {
    constexpr int tiles = WAVES * few_wave_bytes<D, BITS>(), join = WAVES * 32 * (D + 4) * 4;
    constexpr int bytes = tiles > join ? tiles : join;
    if (hipError_t e = allow_dynamic_lds((const void*)pages_few_kernel<T, D, BITS, WAVES>, bytes)) return e;
    pages_few_kernel<T, D, BITS, WAVES><<<c.prefix.grid + c.own.grid, 64 * WAVES, bytes, stream>>>(c);
    return hipGetLastError();
}

template <typename T, int D, int BITS, int WAVES>
hipError_t run_token(const PagesCall& c, hipStream_t stream) {
    constexpr int bytes = token_bytes<D, WAVES>();
    if (hipError_t e = allow_dynamic_lds((const void*)pages_token_kernel<T, D, BITS, WAVES>, bytes)) return e;
    pages_token_kernel<T, D, BITS, WAVES><<<c.prefix.grid + c.own.grid, 64 * WAVES, bytes, stream>>>(c);
    return hipGetLastError();
}

template <typename T, int D, int BITS>
hipError_t run_blocks(const PagesCall& c, const Blocks& b, hipStream_t stream) {
    if (b.rows == 16) return b.waves == 4 ? run_token<T, D, BITS, 4>(c, stream) : run_token<T, D, BITS, D == 64 ? 16 : 8>(c, stream);
    if (b.rows == 128) {
        pages_tile_kernel<T, D, BITS><<<c.prefix.grid + c.own.grid, kThreads, 0, stream>>>(c);
        return hipGetLastError();
    }
    return b.waves == 8 ? run_few<T, D, BITS, D == 64 ? 8 : 4>(c, stream) : run_few<T, D, BITS, 4>(c, stream);
}

template <typename T, int D>
hipError_t join(const AttentionArgs& a, int parts, hipStream_t stream) {
    const int64_t rows = (int64_t)a.max_q * a.q_heads;
    if (parts <= kJoinByRow)
        pages_join_kernel<T, D, 1><<<dim3((unsigned)((rows + kWaves - 1) / kWaves), 1, a.sequences), kThreads, 0, stream>>>(a, parts);
    else
        pages_join_kernel<T, D, kWaves><<<dim3((unsigned)rows, 1, a.sequences), kThreads, 0, stream>>>(a, parts);
    return hipGetLastError();
}

template <typename T, int D, int BITS>
hipError_t run(const PagesAttention& p, const PlanOf& plan, hipStream_t stream) {
    const AttentionArgs& a = p.a;
    PagesCall c{};
    c.p = p;
    c.window = window_of(a);
    c.by_group = divide_by(a.group);
    c.prefix_splits = plan.shared ? plan.prefix.splits : 0;
    c.parts = plan.parts;
    c.both = plan.both;
    if (!pages_grid(plan.own.blocks, plan.own.splits, plan.own.per, a.kv_heads, a.sequences, &c.own)) return hipErrorInvalidConfiguration;
    if (plan.shared && !pages_grid(plan.prefix.blocks, plan.prefix.splits, plan.prefix.per, a.kv_heads, 1, &c.prefix))
        return hipErrorInvalidConfiguration;
    if (!launches_fit(plan, c.prefix.grid, c.own.grid, (int64_t)a.max_q * a.q_heads)) return hipErrorInvalidConfiguration;
    if (plan.shared && plan.prefix.rows == 128 && plan.own.rows == 16) {
        pages_mixed_kernel<T, D, BITS><<<c.prefix.grid + c.own.grid, kThreads, 0, stream>>>(c);
        if (hipError_t e = hipGetLastError()) return e;
        return join<T, D>(a, plan.parts, stream);
    }
    if (plan.shared && (plan.own.rows != plan.prefix.rows || plan.own.waves != plan.prefix.waves)) {
        PagesCall first = c;
        first.own.grid = 0;
        c.prefix.grid = 0;
        if (hipError_t e = run_blocks<T, D, BITS>(first, plan.prefix, stream)) return e;
    }
    if (hipError_t e = run_blocks<T, D, BITS>(c, plan.own, stream)) return e;
    return plan.parts == 1 ? hipSuccess : join<T, D>(a, plan.parts, stream);
}

template <typename T, int D>
hipError_t by_bits(const PagesAttention& p, const PlanOf& plan, hipStream_t stream) {
    return p.mx.bits == 8 ? run<T, D, 8>(p, plan, stream) : (p.mx.bits == 4 ? run<T, D, 4>(p, plan, stream) : run<T, D, 16>(p, plan, stream));
}
template <typename T>
hipError_t by_dim(const PagesAttention& p, const PlanOf& plan, hipStream_t stream) {
    return p.a.dim == 64 ? by_bits<T, 64>(p, plan, stream) : by_bits<T, 128>(p, plan, stream);
}

}  // namespace
}  // namespace fa

size_t attention_pages_workspace(const dcn_attention_shape& s, int bits, int max_prefix) {
    const fa::PlanOf p = fa::plan_of(s.head_dim, bits, s.sequences, s.kv_heads, s.q_heads / s.kv_heads, s.q_tokens, s.max_q, s.max_kv, max_prefix,
                                     s.frame_tokens, s.back, s.sinks);
    return p.parts == 1 ? 0 : (size_t)s.q_tokens * s.q_heads * p.parts * (s.head_dim + 4) * sizeof(float);
}

hipError_t launch_attention_pages(int dtype, const PagesAttention& p, hipStream_t stream) {
    const AttentionArgs& a = p.a;
    const fa::PlanOf plan = fa::plan_of(a.dim, p.mx.bits, a.sequences, a.kv_heads, a.group, a.q_tokens, a.max_q, a.max_kv, p.max_prefix, a.frame, a.back,
                                        a.sinks);
    return dtype == DCN_DTYPE_F16 ? fa::by_dim<_Float16>(p, plan, stream) : fa::by_dim<fa::bf16>(p, plan, stream);
}

}  // namespace dcn
