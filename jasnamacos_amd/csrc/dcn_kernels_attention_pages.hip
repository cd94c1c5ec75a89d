// Attention over microscaled pages, and of sequences that share a prefix over pages of either kind, on
// the matrix cores: FP16 and BF16 heads of 64 and 128 channels.
//
// The keys of a row are two runs: the prefix's, then its sequence's own, each with a table of pages;
// tiles of keys lie in one of them. What a workgroup takes is
//   a block of packed rows of one sequence, over its own keys or over both runs, or
//   a block of packed rows of all sequences, over the prefix's keys: read once for all of them,
// and of those keys all tiles or a split. Parts of a row are joined in FP32 by a second kernel.
//
// Microscaled tiles go through registers: loaded a tile ahead, taken to 16 bits by the scaled
// conversions (exact: a code has 4 bits of significand at most; FP16 rounds below 2^-14 and beyond
// 65504), stored to LDS as rows of the 16-bit kernels, whose products then run as they are. The
// scales are in the values, so a block of 32 channels costs its scale's load and nothing else.
#include "dcn_attention_forward.hpp"
#include "dcn_mx.hpp"

namespace dcn {
namespace fa {
namespace {

// The two launches' worth of blocks that one launch may hold: those of the prefix first.
struct PagesPlan {
    BlockMap prefix, own;
    int prefix_splits, own_splits;
    int parts;  // of a row: the prefix's, then its own
    int both;   // own blocks take the prefix too
};

// One run of keys: `count` of them on the pages of row `seq` of a table.
struct KeyRun {
    PagesArgs pages;
    int seq, count;

    // Row of the pool of key j (uniform), in tokens of one head's pages (microscaled) or of all; -1 where its
    // page is not there. A scalar load: it is not counted with the copies.
    template <int BITS>
    __device__ __forceinline__ int pool_row(int j, int heads, int head) const {
        typedef const __attribute__((address_space(4))) int* scalar;
        const int page = ((scalar)(uintptr_t)(pages.table + (int64_t)seq * pages.width))[j >> pages.shift];
        if ((unsigned)page >= (unsigned)pages.pages) return -1;
        return ((BITS == 16 ? page : page * heads + head) << pages.shift) + (j & ((1 << pages.shift) - 1));
    }
};

// The keys of a run that a span counted over both runs holds: `from` keys lie before it.
__device__ __forceinline__ int inside(int at, int from, int count) {
    at -= from;
    return at < 0 ? 0 : (at < count ? at : count);
}
__device__ __forceinline__ Span part_of(const Span& s, int from, int count) {
    return Span{inside(s.sink, from, count), inside(s.lo, from, count), inside(s.hi, from, count)};
}

// One of two by a uniform choice, field by field: an index would put both in memory.
__device__ __forceinline__ int pick(int second, int a, int b) { return second ? b : a; }
__device__ __forceinline__ Span pick(int second, const Span& a, const Span& b) {
    return Span{pick(second, a.sink, b.sink), pick(second, a.lo, b.lo), pick(second, a.hi, b.hi)};
}
__device__ __forceinline__ Spread pick(int second, const Spread* s) {
    return Spread{pick(second, s[0].first, s[1].first), pick(second, s[0].last, s[1].last)};
}
__device__ __forceinline__ KeyRun pick(int second, const KeyRun* r) {
    return KeyRun{PagesArgs{r[0].pages.pages, r[0].pages.shift, pick(second, r[0].pages.width, r[1].pages.width),
                            second ? r[1].pages.table : r[0].pages.table},
                  pick(second, r[0].seq, r[1].seq), pick(second, r[0].count, r[1].count)};
}

// The tiles of ROWS keys of both runs that a block's rows see.
template <int ROWS>
struct Tiles {
    TileList<ROWS> first, second;
    __device__ __forceinline__ Tiles(const Spread& a, const Spread& b) : first(a), second(b) {}
    __device__ __forceinline__ int count() const { return first.count + second.count; }
    __device__ __forceinline__ int run(int i) const { return i >= first.count; }
    __device__ __forceinline__ int tile(int i) const { return i < first.count ? first.tile(i) : second.tile(i - first.count); }
};

// A block's place, and what its rows see of each run.
struct Block {
    Place pl;
    KeyRun run[2];
    bool all;  // rows of all sequences
    int prefix;
};
constexpr int kNowhere = INT32_MIN;

// Position of packed row r, or kNowhere where it is none of a sequence.
__device__ __forceinline__ int position_of(const PagesAttention& p, const Block& b, const Rows& rw, int r) {
    if (r >= b.pl.rows) return kNowhere;
    const int tok = rw.token(r);
    if (!b.all) return b.pl.offset + tok;
    const AttentionArgs& a = p.a;
    int low = 0, high = a.sequences;
    if (a.cu_q) {
        while (high - low > 1) {
            const int mid = (low + high) >> 1;
            if (a.cu_q[mid] <= tok) low = mid;
            else high = mid;
        }
    } else {
        low = tok / a.max_q;
        if (low >= a.sequences) return kNowhere;
    }
    const Run q = run_of(a.cu_q, low, a.max_q, a.q_tokens), kv = kv_run_of(a, low);
    const int64_t in = tok - q.first;
    if (in < 0 || in >= q.count || in >= a.max_q) return kNowhere;
    return b.prefix + kv.count - q.count + (int)in;
}

template <int ROWS_WG>
__device__ __forceinline__ bool block_place(const PagesAttention& p, const PagesPlan& plan, Block* b) {
    const AttentionArgs& a = p.a;
    b->all = blockIdx.x < plan.prefix.grid;
    const BlockMap& map = b->all ? plan.prefix : plan.own;
    Place& pl = b->pl;
    int at;
    if (!block_of(map, b->all ? blockIdx.x : blockIdx.x - plan.prefix.grid, &at, &pl.kh, &pl.seq)) return false;
    int prefix = 0;
    if (p.prefix.table) {
        prefix = *p.prefix_len;
        prefix = uniform(prefix < 0 ? 0 : (prefix > p.max_prefix ? p.max_prefix : prefix));
    }
    b->prefix = prefix;
    b->run[0] = KeyRun{p.prefix, 0, b->all || plan.both ? prefix : 0};
    b->run[1] = KeyRun{a.pages, pl.seq, 0};
    const int splits = b->all ? plan.prefix_splits : plan.own_splits;
    pl.splits = splits;
    pl.split = at % splits;
    int64_t rows;
    if (b->all) {
        pl.q = Run{0, (int)a.q_tokens};
        pl.offset = 0;
        rows = a.q_tokens * a.group;
    } else {
        pl.q = run_of(a.cu_q, pl.seq, a.max_q, a.q_tokens);
        pl.kv = kv_run_of(a, pl.seq);
        pl.q.count = uniform(pl.q.count);
        pl.kv.count = uniform(pl.kv.count);
        b->run[1].count = pl.kv.count;
        pl.offset = prefix + pl.kv.count - pl.q.count;
        rows = (int64_t)(pl.q.count < a.max_q ? pl.q.count : a.max_q) * a.group;
    }
    pl.rows = (int)rows;
    pl.row0 = (map.x / splits - 1 - at / splits) * ROWS_WG;  // the last rows first: they see the most keys
    return pl.row0 < pl.rows;
}

// What rows from .. from + n - 1 (n a multiple of 64, or 32) see at least and at most of each run;
// false: none is of a sequence.
__device__ __forceinline__ bool spreads_of(const PagesAttention& p, const Block& b, const Rows& rw, int from, int n, int lane,
                                           Spread* first, Spread* second) {
    int low = INT32_MAX, high = kNowhere;
    if (b.all) {
        for (int r = from + (lane < n ? lane : n - 1); r < from + n; r += 64) {
            const int at = position_of(p, b, rw, r);
            if (at == kNowhere) continue;
            low = at < low ? at : low;
            high = at > high ? at : high;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            const int l = __shfl_xor(low, d), h = __shfl_xor(high, d);
            low = l < low ? l : low;
            high = h > high ? h : high;
        }
        low = uniform(low);
        high = uniform(high);
    } else if (from < b.pl.rows) {
        const int last = from + n < b.pl.rows ? from + n - 1 : b.pl.rows - 1;
        low = b.pl.offset + rw.token(from);
        high = b.pl.offset + rw.token(last);
    }
    if (high == kNowhere) {
        *first = *second = Spread{};
        return false;
    }
    // Keys that are there, for the ends of the spans: a block of all sequences looks at the prefix only.
    const int keys = b.all ? INT32_MAX : b.prefix + b.run[1].count;
    const Span lo = span_of(p.a, low, keys), hi = span_of(p.a, high, keys);
    *first = Spread{part_of(lo, 0, b.run[0].count), part_of(hi, 0, b.run[0].count)};
    *second = Spread{part_of(lo, b.prefix, b.run[1].count), part_of(hi, b.prefix, b.run[1].count)};
    return true;
}

// How a wave's share of a tile of ROWS keys gets into LDS: WAVES waves, or one, each its part of it.
// Pages of the type: by asynchronous copies (copy), as in the 16-bit kernels.
template <typename T, int D, int BITS, int ROWS, int WAVES>
struct Stage;

template <typename T, int D, int ROWS, int WAVES>
struct Stage<T, D, 16, ROWS, WAVES> {
    using Ti = Tile<D>;
    static constexpr int kCopies = ROWS / Ti::kRowsPerCopy / WAVES;
    const char *kp, *vp;
    uint32_t ks, vs;  // bytes between tokens
    uint32_t kat, vat;
    int row[kCopies];
    unsigned long long holes = 0;

    __device__ __forceinline__ Stage(const PagesAttention& p, int kh, int wave, int lane) {
        kp = (const char*)p.a.k.p + kh * p.a.k.hs * 2;
        vp = (const char*)p.a.v.p + kh * p.a.v.hs * 2;
        ks = (uint32_t)p.a.k.ts * 2;
        vs = (uint32_t)p.a.v.ts * 2;
        kat = lane / Ti::kChunks * ks;
        vat = lane / Ti::kChunks * vs;
    }
    // Looks up the pages of the tile from t0: past the run's end those of its last keys.
    __device__ __forceinline__ void find(const PagesAttention&, const KeyRun& run, int, int t0, int wave) {
        const int last = (run.count - 1) & ~7;
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            const int in = (n * WAVES + wave) * Ti::kRowsPerCopy, j = t0 + (in & ~7);
            const int r = run.pool_row<16>(j < last ? j : last, 1, 0);
            row[n] = r < 0 ? 0 : r + (in & 7);
        }
        holes = 0;
#pragma unroll
        for (int g = 0; g < ROWS / 8; ++g) {
            const int j = t0 + 8 * g;
            if (run.pool_row<16>(j < last ? j : last, 1, 0) < 0) holes |= 0xffull << (8 * g);
        }
    }
    __device__ __forceinline__ void copy(char* kt, char* vt, int wave, int lane) const {
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            const int i = n * WAVES + wave;
            const uint32_t c = Ti::copy_channel(Ti::copy_row(i, lane), lane) * 2;
            copy16(kp + (int64_t)row[n] * ks, kat + c, kt + i * 1024);
            copy16(vp + (int64_t)row[n] * vs, vat + c, vt + i * 1024);
        }
    }
};

// Microscaled pages: through registers. A wave has ROWS / WAVES adjacent keys of the tile; a lane's load
// is a chunk of one key's codes, and its block's scale.
template <typename T, int D, int BITS, int ROWS, int WAVES>
struct Stage {
    using Ti = Tile<D>;
    static constexpr int kKeys = ROWS / WAVES, kBytes = D * BITS / 8;                       // a wave's keys, a key's bytes
    static constexpr int kChunk = kKeys * kBytes >= 1024 ? 16 : kKeys * kBytes / 64;         // bytes a lane loads at once
    static constexpr int kLoads = kKeys * kBytes / (64 * kChunk), kPerLoad = kKeys / kLoads;  // keys a load takes
    static constexpr int kWords = kChunk / 4, kCodes = kChunk * 8 / BITS, kRuns = kKeys / 8;
    static_assert(kChunk >= 8 && kCodes <= 32 && kPerLoad % 8 == 0, "");
    typedef uint32_t words __attribute__((ext_vector_type(kWords)));
    const uint8_t *kp, *vp, *ksp, *vsp;
    int row[kRuns];
    unsigned long long holes = 0;
    words k[kLoads], v[kLoads];
    uint32_t kf[kLoads], vf[kLoads];

    __device__ __forceinline__ Stage(const PagesAttention& p, int kh, int wave, int lane) {
        kp = p.mx.k;
        vp = p.mx.v;
        ksp = p.mx.ks;
        vsp = p.mx.vs;
    }
    __device__ __forceinline__ void find(const PagesAttention& p, const KeyRun& run, int kh, int t0, int wave) {
        const int last = (run.count - 1) & ~7;
        holes = 0;
#pragma unroll
        for (int g = 0; g < ROWS / 8; ++g) {
            const int j = t0 + 8 * g, r = run.pool_row<BITS>(j < last ? j : last, p.mx.heads, kh);
            if (r < 0) holes |= 0xffull << (8 * g);
            if constexpr (WAVES == 1) {
                row[g] = r < 0 ? 0 : r;
            } else if (g / kRuns == wave) {
                row[g % kRuns] = r < 0 ? 0 : r;
            }
        }
    }
    static __device__ __forceinline__ int key(int n, int lane) { return n * kPerLoad + lane / (kBytes / kChunk); }
    static __device__ __forceinline__ int channel(int lane) { return lane % (kBytes / kChunk) * kCodes; }
    __device__ __forceinline__ void load(int lane) {
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int in = key(n, lane);
            int r = row[n * kPerLoad / 8];
#pragma unroll
            for (int g = 1; g < kPerLoad / 8; ++g)
                if (lane / (kBytes / kChunk) >> 3 == g) r = row[n * kPerLoad / 8 + g];
            const int64_t at = r + (in & 7);
            k[n] = *(const words*)(kp + at * kBytes + lane % (kBytes / kChunk) * kChunk);
            v[n] = *(const words*)(vp + at * kBytes + lane % (kBytes / kChunk) * kChunk);
            kf[n] = ksp[at * (D / 32) + channel(lane) / 32];
            vf[n] = vsp[at * (D / 32) + channel(lane) / 32];
        }
    }
    // The loaded tile to LDS; look: zeros for values that are not finite, and a bit, in every lane, for
    // each key of the tile that had one.
    __device__ __forceinline__ unsigned long long store(char* kt, char* vt, bool look, int wave, int lane) const {
        constexpr int kGroups = kCodes / 8;  // 16-byte chunks of LDS
        unsigned long long rows = 0;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int in = wave * kKeys + key(n, lane), c0 = channel(lane) / 8;
            const float fk = mx_factor(kf[n]), fv = mx_factor(vf[n]);
            u32x4 x[kGroups], y[kGroups];
            uint32_t two[kCodes];
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                mx_decode<T, BITS>(k[n][w], fk, two + w * (16 / BITS));
                mx_decode<T, BITS>(v[n][w], fv, two + kCodes / 2 + w * (16 / BITS));
            }
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[g][i] = two[4 * g + i];
                    y[g][i] = two[kCodes / 2 + 4 * g + i];
                }
            if (__builtin_expect(look, 0)) {
                bool bad = false;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) bad |= clean16<T>(y[g]);
                if (bad) rows |= 1ull << in;
            }
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int at = (in * Ti::kChunks + ((c0 + g) ^ Ti::swizzle(in))) * 16;
                *(u32x4*)(kt + at) = x[g];
                *(u32x4*)(vt + at) = y[g];
            }
        }
        if (look && __any(rows != 0))
            for (int d = 32; d; d >>= 1) rows |= __shfl_xor(rows, d);
        return rows;
    }
};

// Infinities and NaN of the values of a tile of keys, which stand as zeros in LDS, to the rows that see them.
template <typename T, int D, int BITS>
__device__ __forceinline__ void add_bad(const PagesAttention& p, const KeyRun& run, int kh, f32x16* o, const Span& sp, int t0, int rows,
                                        unsigned long long holes, int lane) {
    const int to = t0 + rows < run.count ? t0 + rows : run.count;
    if constexpr (BITS == 16) {
        add_nonfinite<T, D>(o, sp, t0, to, holes, lane, [&](int j) -> const uint16_t* {
            const int64_t row = run.pool_row<16>(j, 1, 0);
            return row < 0 ? nullptr : (const uint16_t*)p.a.v.p + row * p.a.v.ts + kh * p.a.v.hs;
        });
    } else {
        for (int j = t0; j < to; ++j) {
            const int64_t row = run.pool_row<BITS>(j, p.mx.heads, kh);
            if (row < 0) continue;
            const bool on = sees(sp, j) && !(holes >> (j - t0) & 1);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const float factor = mx_factor(p.mx.vs[row * (D / 32) + i]);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int ch = 32 * i + 8 * x + 4 * (lane >> 5);
                    const uint8_t* at = p.mx.v + (row * D + ch) * BITS / 8;
                    uint32_t two[16 / BITS];
                    if constexpr (BITS == 8)
                        mx_decode<T, 8>(*(const uint32_t*)at, factor, two);
                    else
                        mx_decode<T, 4>(*(const uint16_t*)at, factor, two);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t bits = (uint16_t)(two[e >> 1] >> (16 * (e & 1)));
                        if (on && !finite16<T>(bits)) o[i][4 * x + e] += widen(__builtin_bit_cast(T, bits));
                    }
                }
                asm volatile("" ::: "memory");  // few registers: this is rare
            }
        }
    }
}

// Stores a part: its number among those of the row.
__device__ __forceinline__ void number_part(const PagesPlan& plan, const Block& b, Place* pl) {
    pl->split = b.all ? pl->split : (plan.parts - plan.own_splits) + pl->split;
    pl->splits = plan.parts;
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kThreads, 2) void pages_tile_kernel(PagesAttention p, PagesPlan plan) {
    constexpr int ROWS = 64, BYTES = ROWS * D * 2;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][BYTES];
    __shared__ FoundRows found;
    const AttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Block b;
    if (!block_place<32 * kWaves>(p, plan, &b)) return;
    Place& pl = b.pl;
    const Rows rw = rows_of(a.group);
    const int w0 = pl.row0 + 32 * wave, r = w0 + (lane & 31);
    Spread all[2], mine[2];
    if (!spreads_of(p, b, rw, pl.row0, 32 * kWaves, lane, &all[0], &all[1])) return;
    const bool idle = !spreads_of(p, b, rw, w0, 32, lane, &mine[0], &mine[1]);  // no rows: the wave copies only
    const int at = position_of(p, b, rw, r);
    Span sp[2] = {};
    if (at != kNowhere) {
        const Span s = span_of(a, at, b.all ? INT32_MAX : b.prefix + b.run[1].count);
        sp[0] = part_of(s, 0, b.run[0].count);
        sp[1] = part_of(s, b.prefix, b.run[1].count);
    }
    RowState<T, D> st;
    st.clear();
    load_row<D>(st.q, a.q, a, pl, rw, r, lane);
    const Tiles<ROWS> list(all[0], all[1]);
    const int per = (list.count() + pl.splits - 1) / pl.splits;
    const int from = pl.split * per, to = from + per < list.count() ? from + per : list.count();
    const float c = a.scale * kLog2e;
    Stage<T, D, BITS, ROWS, kWaves> stage(p, pl.kh, wave, lane);
    auto find = [&](int i) { stage.find(p, pick(list.run(i), b.run), pl.kh, list.tile(i), wave); };
    auto partial = [&](int i, unsigned long long holes) { return holes || !all_see<ROWS>(pick(list.run(i), all), list.tile(i)); };
    unsigned long long holes = 0, next_holes = 0;
    if constexpr (BITS == 16) {
        if (from < to) {
            find(from);
            stage.copy(lds[0][0], lds[0][1], wave, lane);
            holes = stage.holes;
            if (from + 1 < to) find(from + 1);
        }
    } else {
        if (from < to) {
            find(from);
            stage.load(lane);
            holes = stage.holes;
            found.wave[0][wave] = stage.store(lds[0][0], lds[0][1], partial(from, holes), wave, lane);
            if (from + 1 < to) {
                find(from + 1);
                stage.load(lane);
                next_holes = stage.holes;
                if (from + 2 < to) find(from + 2);
            }
        }
        __syncthreads();
    }
    st.settle();
    for (int i = from; i < to; ++i) {
        const int buf = (i - from) & 1, t0 = list.tile(i), run = list.run(i);
        char(*now)[BYTES] = lds[buf], (*other)[BYTES] = lds[buf ^ 1];
        const bool some = partial(i, holes);
        if constexpr (BITS == 16) {
            wait_copies<0>();
            if (some) found.wave[buf][wave] = clean_own<T, D, ROWS, kWaves>(now[1], wave, lane);
            __syncthreads();
            if (i + 1 < to) {
                stage.copy(other[0], other[1], wave, lane);
                next_holes = stage.holes;
                if (i + 2 < to) find(i + 2);
            }
        } else if (i + 1 < to) {
            found.wave[buf ^ 1][wave] = stage.store(other[0], other[1], partial(i + 1, next_holes), wave, lane);
        }
        unsigned long long after = 0;
        if constexpr (BITS != 16) {
            if (i + 2 < to) {
                stage.load(lane);
                after = stage.holes;
                if (i + 3 < to) find(i + 3);
            }
        }
        const bool bad = some && uniform(found.all(buf) != 0);
        const Spread own = pick(run, mine);
        if (!idle && !none_sees<ROWS>(own, t0)) {
            st.sp = pick(run, sp[0], sp[1]);
            st.template add<ROWS>(now[0], now[1], t0, c, holes || !all_see<ROWS>(own, t0), holes, lane);
            if (bad) add_bad<T, D, BITS>(p, pick(run, b.run), pl.kh, st.o, st.sp, t0, ROWS, holes, lane);
        }
        holes = next_holes;
        if constexpr (BITS != 16) {
            next_holes = after;
            __syncthreads();
        }
    }
    if (at == kNowhere) return;
    number_part(plan, b, &pl);
    const int tok = rw.token(r), head = pl.kh * a.group + (r - tok * a.group);
    const int64_t row = pl.q.first + tok, index = row * a.q_heads + head;
    const float l = both_sum(st.l), inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float o[4] = {st.o[i][4 * x], st.o[i][4 * x + 1], st.o[i][4 * x + 2], st.o[i][4 * x + 3]};
            store_row4<T, D>(a, pl, index, row, head, 32 * i + 8 * x + 4 * (lane >> 5), o, inv);
        }
    if (lane < 32) store_sums<D>(a, pl, index, st.m, l, kLift<T>);
}

// LDS of a wave of the few kernel: pages of the type have two tiles, one in flight.
template <int D, int BITS>
constexpr int few_wave_bytes() {
    return (BITS == 16 ? 4 : 2) * 32 * D * 2;
}

template <typename T, int D, int BITS, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || BITS != 16 ? 2 : 1) void pages_few_kernel(PagesAttention p, PagesPlan plan) {
    constexpr int ROWS = 32, BYTES = ROWS * D * 2, COPIES = 2 * ROWS / Tile<D>::kRowsPerCopy;
    extern __shared__ __attribute__((aligned(1024))) char lds[];  // each wave's tiles, then the join
    const AttentionArgs& a = p.a;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Block b;
    if (!block_place<32>(p, plan, &b)) return;
    Place& pl = b.pl;
    const Rows rw = rows_of(a.group);
    const int r = pl.row0 + (lane & 31);
    Spread all[2];
    if (!spreads_of(p, b, rw, pl.row0, 32, lane, &all[0], &all[1])) return;
    const int place = position_of(p, b, rw, r);
    Span sp[2] = {};
    if (place != kNowhere) {
        const Span s = span_of(a, place, b.all ? INT32_MAX : b.prefix + b.run[1].count);
        sp[0] = part_of(s, 0, b.run[0].count);
        sp[1] = part_of(s, b.prefix, b.run[1].count);
    }
    RowState<T, D> st;
    st.clear();
    load_row<D>(st.q, a.q, a, pl, rw, r, lane);
    const Tiles<ROWS> list(all[0], all[1]);
    const int per = (list.count() + pl.splits - 1) / pl.splits;
    const int from = pl.split * per, to = from + per < list.count() ? from + per : list.count();
    const float c = a.scale * kLog2e;
    char* own = lds + wave * few_wave_bytes<D, BITS>();
    Stage<T, D, BITS, ROWS, 1> stage(p, pl.kh, 0, lane);
    auto find = [&](int i) { stage.find(p, pick(list.run(i), b.run), pl.kh, list.tile(i), 0); };
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
        const int t0 = list.tile(i), run = list.run(i);
        const bool whole = !holes && all_see<ROWS>(pick(run, all), t0);
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
        st.sp = pick(run, sp[0], sp[1]);
        st.template add<ROWS>(kt, vt, t0, c, !whole, holes, lane);
        if (bad) add_bad<T, D, BITS>(p, pick(run, b.run), pl.kh, st.o, st.sp, t0, ROWS, holes, lane);
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
    }
    __syncthreads();
    // Two threads a row and wave.
    constexpr int share = 2 * WAVES;
    const int jr = threadIdx.x / share, part = threadIdx.x % share;
    const int mine = pl.row0 + jr;
    if (mine >= pl.rows || (b.all && position_of(p, b, rw, mine) == kNowhere)) return;
    float m = -INFINITY, sum = 0.f, w[WAVES];
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, mem[(i * 32 + jr) * LINE + D]);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        w[i] = exp2f(mem[(i * 32 + jr) * LINE + D] - (m == -INFINITY ? 0.f : m));
        sum = fmaf(w[i], mem[(i * 32 + jr) * LINE + D + 1], sum);
    }
    number_part(plan, b, &pl);
    const int tok = rw.token(mine), head = pl.kh * a.group + (mine - tok * a.group);
    const int64_t row = pl.q.first + tok, index = row * a.q_heads + head;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int at = part * 4; at < D; at += 4 * share) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const f32x4 v = *(const f32x4*)(mem + (i * 32 + jr) * LINE + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(w[i], v[e], o[e]);
        }
        const float four[4] = {o[0], o[1], o[2], o[3]};
        store_row4<T, D>(a, pl, index, row, head, at, four, inv);
    }
    if (part == 0) store_sums<D>(a, pl, index, m, sum, kLift<T>);
}

// The blocks of rows of one kind, and over how many workgroups each one's key tiles are split.
struct Blocks {
    bool few;
    int waves, blocks, splits;
};
struct PlanOf {
    Blocks prefix, own;
    bool shared, both;  // shared: the prefix once for all sequences; both: own blocks take it
    int parts;
};

Blocks blocks_of(int dim, int64_t rows, int64_t pairs, int64_t keys) {
    Blocks b;
    const int64_t wide = (rows + 127) / 128 * pairs;
    b.few = rows <= 32 || (dim == 64 ? wide <= 256 && keys <= 4096 : wide <= 128 && keys <= 2048);
    const int per_block = b.few ? 32 : 128, tile = b.few ? 32 : 64;
    b.blocks = (int)((rows + per_block - 1) / per_block);
    const int64_t tiles = (keys + tile - 1) / tile, groups = (int64_t)b.blocks * pairs;
    b.waves = b.few && dim == 64 && groups <= 256 ? 8 : 4;
    const int64_t least = b.few ? b.waves : 4, room = 512;
    int64_t splits = 1;
    if (groups > 0 && groups <= 128 && tiles > 4 * least) {
        splits = (room + groups - 1) / groups;
        splits = splits < tiles / least ? splits : tiles / least;
        splits = splits < 32 ? splits : 32;
    }
    b.splits = (int)splits;
    return b;
}

PlanOf plan_of(int dim, int sequences, int kv_heads, int group, int64_t q_tokens, int max_q, int max_kv, int max_prefix, int frame, int back,
               int sinks) {
    PlanOf p{};
    const int64_t rows = (int64_t)max_q * group;
    // Keys that a block of rows sees at most.
    const auto keys_of = [&](int64_t tokens, int most) { return attention_keys(most, frame, back, sinks, tokens, 64); };
    const int64_t first = max_prefix ? keys_of(max_q, max_prefix) : 0, own = keys_of(128 / group, max_kv);
    p.shared = first > 0 && sequences > 1;
    p.both = first > 0 && !p.shared;
    p.own = blocks_of(dim, rows, (int64_t)kv_heads * sequences, own + (p.both ? first : 0));
    if (p.shared) p.prefix = blocks_of(dim, q_tokens * group, kv_heads, first);
    p.parts = p.own.splits + (p.shared ? p.prefix.splits : 0);
    return p;
}

template <typename T, int D, int BITS, int WAVES>
hipError_t run_few(const PagesAttention& p, const PagesPlan& plan, hipStream_t stream) {
    constexpr int tiles = WAVES * few_wave_bytes<D, BITS>(), join = WAVES * 32 * (D + 4) * 4;
    constexpr int bytes = tiles > join ? tiles : join;
    if (hipError_t e = allow_dynamic_lds((const void*)pages_few_kernel<T, D, BITS, WAVES>, bytes)) return e;
    pages_few_kernel<T, D, BITS, WAVES><<<plan.prefix.grid + plan.own.grid, 64 * WAVES, bytes, stream>>>(p, plan);
    return hipGetLastError();
}

template <typename T, int D, int BITS>
hipError_t run_blocks(const PagesAttention& p, const PagesPlan& plan, const Blocks& b, hipStream_t stream) {
    if (!b.few) {
        pages_tile_kernel<T, D, BITS><<<plan.prefix.grid + plan.own.grid, kThreads, 0, stream>>>(p, plan);
        return hipGetLastError();
    }
    return b.waves == 8 ? run_few<T, D, BITS, D == 64 ? 8 : 4>(p, plan, stream) : run_few<T, D, BITS, 4>(p, plan, stream);
}

template <typename T, int D, int BITS>
hipError_t run(const PagesAttention& p, const PlanOf& plan, hipStream_t stream) {
    const AttentionArgs& a = p.a;
    PagesPlan both{}, none{};
    both.prefix_splits = plan.shared ? plan.prefix.splits : 1;
    both.own_splits = plan.own.splits;
    both.parts = plan.parts;
    both.both = plan.both;
    none = both;
    if (!block_map((int64_t)plan.own.blocks * plan.own.splits, a.kv_heads, a.sequences, &both.own)) return hipErrorInvalidConfiguration;
    if (plan.shared && !block_map((int64_t)plan.prefix.blocks * plan.prefix.splits, a.kv_heads, 1, &both.prefix))
        return hipErrorInvalidConfiguration;
    // Every launch has fewer than 2^32 threads along x.
    const int64_t rows = (int64_t)a.max_q * a.q_heads, most = (INT64_C(1) << 32) / (2 * kThreads);
    if ((int64_t)both.prefix.grid + both.own.grid >= most || (plan.parts > 1 && rows >= most)) return hipErrorInvalidConfiguration;
    const bool one = !plan.shared || (plan.own.few == plan.prefix.few && plan.own.waves == plan.prefix.waves);
    if (!one) {
        none.prefix = both.prefix;
        both.prefix = BlockMap{};
        if (hipError_t e = run_blocks<T, D, BITS>(p, none, plan.prefix, stream)) return e;
    }
    if (hipError_t e = run_blocks<T, D, BITS>(p, both, plan.own, stream)) return e;
    if (plan.parts == 1) return hipSuccess;
    if (plan.parts <= 8)
        attention_join_kernel<T, D, 1><<<dim3((unsigned)((rows + kWaves - 1) / kWaves), 1, a.sequences), kThreads, 0, stream>>>(a, plan.parts);
    else
        attention_join_kernel<T, D, kWaves><<<dim3((unsigned)rows, 1, a.sequences), kThreads, 0, stream>>>(a, plan.parts);
    return hipGetLastError();
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

size_t attention_pages_workspace(const dcn_attention_shape& s, int max_prefix) {
    const fa::PlanOf p = fa::plan_of(s.head_dim, s.sequences, s.kv_heads, s.q_heads / s.kv_heads, s.q_tokens, s.max_q, s.max_kv, max_prefix,
                                     s.frame_tokens, s.back, s.sinks);
    return p.parts == 1 ? 0 : (size_t)s.q_tokens * s.q_heads * p.parts * (s.head_dim + 4) * sizeof(float);
}

hipError_t launch_attention_pages(int dtype, const PagesAttention& p, hipStream_t stream) {
    const AttentionArgs& a = p.a;
    const fa::PlanOf plan = fa::plan_of(a.dim, a.sequences, a.kv_heads, a.group, a.q_tokens, a.max_q, a.max_kv, p.max_prefix, a.frame, a.back,
                                        a.sinks);
    return dtype == DCN_DTYPE_F16 ? fa::by_dim<_Float16>(p, plan, stream) : fa::by_dim<fa::bf16>(p, plan, stream);
}

}  // namespace dcn
