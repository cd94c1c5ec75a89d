// Attention over pages of either kind with a prefix that sequences may share: what its kernels are built
// of (dcn_kernels_attention_pages.hip).
#pragma once

#include "dcn_attention_forward.hpp"
#include "dcn_mx.hpp"

namespace dcn {
namespace fa {
namespace {

// Division of 0 .. 2^31 - 1 by a number that the host knows: one product. The scalar units of a CU make
// one instruction a cycle for all its waves, and a division is about thirty.
struct Divide {
    uint32_t factor;
    int shift;
    __host__ __device__ __forceinline__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * factor) >> shift); }
};
inline Divide divide_by(int d) {
    int bits = 0;
    while ((INT64_C(1) << bits) < d) ++bits;
    return d == 1 ? Divide{1u << 31, 31} : Divide{(uint32_t)((UINT64_C(1) << (31 + bits)) / d + 1), 31 + bits};
}

// The window in tokens: from a frame's first token, how far its queries see ahead and back. Past 2^31 - 1
// there is no key.
struct Window {
    Divide by_frame;
    int frame, sinks;
    uint32_t ahead, back;

    __host__ __device__ __forceinline__ Span at(int p, int n) const {
        if (p < 0) return Span{0, 0, 0};
        const uint32_t start = by_frame(p) * frame, end = start + ahead;
        const int hi = end < (uint32_t)n ? (int)end : n;
        int lo = start > back ? (int)(start - back) : 0;
        lo = lo < hi ? lo : hi;
        return Span{sinks < lo ? sinks : lo, lo, hi};
    }
};
inline Window window_of(const AttentionArgs& a) {
    const auto tokens = [&](int64_t frames) { return frames <= INT32_MAX / a.frame ? (uint32_t)(frames * a.frame) : (uint32_t)INT32_MAX; };
    return Window{divide_by(a.frame), a.frame, (int)tokens(a.sinks), a.ahead < 0 ? (uint32_t)INT32_MAX : tokens((int64_t)a.ahead + 1),
                  a.back < 0 ? (uint32_t)INT32_MAX : tokens(a.back)};
}

// Workgroups for `x` blocks of each of `pairs` (sequence, key head), spread over the XCDs as a BlockMap
// does; x is row blocks times parts of their keys.
struct PagesGrid {
    unsigned grid;  // a multiple of 8
    int x, pairs, heads, splits, per;  // splits: parts of a row's keys, of `per` tiles each
    int share, classes;  // as powers of two
    Divide by_x, by_heads, by_splits;
};
inline bool pages_grid(int64_t blocks, int splits, int per, int heads, int64_t sequences, PagesGrid* g) {
    BlockMap m;
    if (!block_map(blocks * splits, heads, sequences, &m) || heads * sequences > INT32_MAX) return false;
    *g = PagesGrid{m.grid, m.x, m.pairs, heads, splits, per, m.classes == 8 ? 0 : (m.classes == 4 ? 1 : (m.classes == 2 ? 2 : 3)), 0,
                   divide_by(m.x), divide_by(heads), divide_by(splits)};
    g->classes = 3 - g->share;
    return true;
}

// A launch: workgroups that take rows of all sequences over the prefix, then workgroups that take rows of
// one over its own keys (both: over the prefix too).
struct PagesCall {
    PagesAttention p;
    PagesGrid prefix, own;
    int prefix_splits, parts;  // of a row: the prefix's first
    int both;
    Window window;
    Divide by_group;
};

// One run of keys: `count` of them, whose pages a table's row gives.
struct KeyRun {
    const int32_t* table;
    int count;

    // Row of the pool of key j (uniform), in tokens of one head's pages (microscaled) or of all; -1 where its
    // page is not there. A scalar load: it is not counted with the copies.
    template <int BITS>
    __device__ __forceinline__ int pool_row(const PagesAttention& p, int j, int head) const {
        typedef const __attribute__((address_space(4))) int* scalar;
        const PagesArgs& pages = p.a.pages;
        const int page = ((scalar)(uintptr_t)table)[j >> pages.shift];
        if ((unsigned)page >= (unsigned)pages.pages) return -1;
        return ((BITS == 16 ? page : page * p.mx.heads + head) << pages.shift) + (j & ((1 << pages.shift) - 1));
    }
    // Rows of the pool that the runs of eight keys of a tile start at (0 where the page is not there, with
    // a bit for each of their keys in the result). Past the end those of the last eight: rows that are
    // there, of keys that are not seen.
    template <int BITS, int ROWS>
    __device__ __forceinline__ unsigned long long tile_rows(const PagesAttention& p, int t0, int head, int* rows) const {
        const int last = (count - 1) & ~7;
        unsigned long long holes = 0;
        if ((ROWS >> p.a.pages.shift) <= 1) {  // a tile lies on one page
            const int r = pool_row<BITS>(p, t0, head);
#pragma unroll
            for (int g = 0; g < ROWS / 8; ++g) rows[g] = r < 0 ? 0 : r + 8 * g;
            return r < 0 ? ~0ull : 0ull;
        }
#pragma unroll
        for (int g = 0; g < ROWS / 8; ++g) {
            const int j = t0 + 8 * g, r = pool_row<BITS>(p, j < last ? j : last, head);
            if (r < 0) holes |= 0xffull << (8 * g);
            rows[g] = r < 0 ? 0 : r;
        }
        return holes;
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

// A block's place.
struct Block {
    Place pl;
    bool all;    // rows of all sequences
    int prefix;  // keys of the prefix
    int per;     // tiles of a part
    KeyRun run[2];

    // What a row at this position sees of one run.
    __device__ __forceinline__ Span span(const PagesCall& c, int at, int second) const {
        if (at == INT32_MIN) return Span{0, 0, 0};
        // A block of all sequences looks at the prefix only, and a span's end past it does not matter.
        const Span s = c.window.at(at, all ? INT32_MAX : prefix + run[1].count);
        return second ? part_of(s, prefix, run[1].count) : part_of(s, 0, run[0].count);
    }
};
constexpr int kNowhere = INT32_MIN;

// What rows from position low to high see at least and at most of a run.
__device__ __forceinline__ Spread spread_in(const PagesCall& c, const Block& b, int low, int high, int second) {
    if (high == kNowhere) return Spread{};
    const Span s = b.span(c, high, second);
    return low == high ? Spread{s, s} : Spread{b.span(c, low, second), s};
}

// Where a loop over a block's tiles of ROWS keys is: the tiles of the prefix that its rows see, then those of
// their own keys. Most blocks have one of the two.
template <int ROWS>
struct Cursor {
    TileList<ROWS> list;
    int base, second;  // the first tile's number; which run
    KeyRun run;

    // At the first tile; its end is *count.
    __device__ __forceinline__ Cursor(const PagesCall& c, const Block& b, int low, int high, int* count) : list(Spread{}), base(0) {
        second = !b.all && !c.both;
        run = second ? b.run[1] : b.run[0];
        list = TileList<ROWS>(spread_in(c, b, low, high, second));
        *count = list.count + (c.both ? TileList<ROWS>(spread_in(c, b, low, high, 1)).count : 0);
    }
    // On to tile i; whether that is in another run than before.
    __device__ __forceinline__ bool go(const PagesCall& c, const Block& b, int low, int high, int i) {
        if (!c.both || second || i < list.count) return false;
        base = list.count;
        second = 1;
        run = b.run[1];
        list = TileList<ROWS>(spread_in(c, b, low, high, 1));
        return true;
    }
    __device__ __forceinline__ int tile(int i) const { return list.tile(i - base); }
};

// Positions of packed rows rows[0 .. N - 1] of each lane (lane 0's first is the lowest), kNowhere where a
// row is none of a sequence. Rows of all sequences look their sequence up among 64 at a time that
// the lanes hold: a search in memory would be a chain of loads.
template <int N>
__device__ __forceinline__ void positions_of(const PagesCall& c, const Block& b, const int* rows, int lane, int* at) {
    const AttentionArgs& a = c.p.a;
    int tok[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        tok[n] = c.by_group(rows[n] < b.pl.rows ? rows[n] : b.pl.rows - 1);
        at[n] = rows[n] < b.pl.rows && !b.all ? b.pl.offset + tok[n] : kNowhere;
    }
    if (!b.all) return;
    const int most = a.pages.width << a.pages.shift;
    if (!a.cu_q) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int s = tok[n] / a.max_q;
            if (rows[n] < b.pl.rows && s < a.sequences) at[n] = b.prefix + inside(a.cu_kv[s], 0, most) - a.max_q + (tok[n] - s * a.max_q);
        }
        return;
    }
    if (a.back < 0) {
        // Without a window a row behind the prefix sees all of it, wherever it is: where no sequence has more
        // queries than keys, that is every row.
        bool behind = true;
        for (int i = lane; i < a.sequences; i += 64) {
            const int64_t n = (int64_t)a.cu_q[i + 1] - a.cu_q[i];
            behind = behind && n >= 0 && n <= a.max_q && n <= inside(a.cu_kv[i], 0, most);
        }
        if (__all(behind)) {
            const int from = a.cu_q[0], to = a.cu_q[a.sequences];
#pragma unroll
            for (int n = 0; n < N; ++n) at[n] = rows[n] < b.pl.rows && tok[n] >= from && tok[n] < to ? INT32_MAX - 1 : kNowhere;
            return;
        }
    }
    int first = a.sequences > 64 ? uniform(find_sequence(a.cu_q, a.sequences, tok[0])) : 0;  // lane 0's, the lowest
    bool found[N] = {}, all;
    do {
        // Lane i has the end of sequence first + i, and its keys.
        const int mine = first + lane < a.sequences ? first + lane : a.sequences - 1;
        const int end = a.cu_q[mine + 1], keys = inside(a.cu_kv[mine], 0, most), start = a.cu_q[first];
        all = true;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            int i = 0;  // ends at or before the token
#pragma unroll
            for (int d = 32; d; d >>= 1) i += __shfl(end, i + d - 1) <= tok[n] ? d : 0;
            const int to = __shfl(end, i), before = __shfl(end, i ? i - 1 : 0), n_keys = __shfl(keys, i);
            const bool here = to > tok[n] && first + i < a.sequences;
            if (here && !found[n] && rows[n] < b.pl.rows) {
                int64_t from = i ? before : start, until = to;
                from = from < 0 ? 0 : from;
                until = until > a.q_tokens ? a.q_tokens : until;
                const int64_t in = tok[n] - from;
                if (in >= 0 && in < a.max_q) at[n] = b.prefix + n_keys - (int)(until - from) + (int)in;
            }
            found[n] = found[n] || here;
            all = all && __all(found[n]);
        }
        first += 64;
    } while (!all && first < a.sequences);
}

template <int ROWS_WG>
__device__ __forceinline__ bool block_place(const PagesCall& c, unsigned index, Block* b) {
    const AttentionArgs& a = c.p.a;
    b->all = index < c.prefix.grid;
    const PagesGrid& g = b->all ? c.prefix : c.own;
    if (!b->all) index -= c.prefix.grid;
    Place& pl = b->pl;
    const int xcd = index & 7, item = (int)((index >> 3) << g.share) + (xcd >> g.classes);
    const int nth = g.by_x(item), pair = (xcd & ((1 << g.classes) - 1)) + (nth << g.classes);
    if (pair >= g.pairs) return false;
    pl.seq = g.by_heads(pair);
    pl.kh = pair - pl.seq * g.heads;
    const int at = item - nth * g.x, block = g.by_splits(at);
    pl.splits = g.splits;
    pl.split = at - block * g.splits;
    b->per = g.per;
    int prefix = 0;
    if (c.p.prefix.table) {
        prefix = *c.p.prefix_len;
        prefix = uniform(prefix < 0 ? 0 : (prefix > c.p.max_prefix ? c.p.max_prefix : prefix));
    }
    b->prefix = prefix;
    b->run[0] = KeyRun{c.p.prefix.table, b->all || c.both ? prefix : 0};
    int64_t rows;
    if (b->all) {
        b->run[1] = KeyRun{nullptr, 0};
        pl.q = Run{0, (int)a.q_tokens};
        pl.offset = 0;
        rows = a.q_tokens * a.group;
    } else {
        pl.q = run_of(a.cu_q, pl.seq, a.max_q, a.q_tokens);
        pl.kv = kv_run_of(a, pl.seq);
        pl.q.count = uniform(pl.q.count);
        pl.kv.count = uniform(pl.kv.count);
        b->run[1] = KeyRun{a.pages.table + (int64_t)pl.seq * a.pages.width, pl.kv.count};
        pl.offset = prefix + pl.kv.count - pl.q.count;
        rows = (int64_t)(pl.q.count < a.max_q ? pl.q.count : a.max_q) * a.group;
    }
    pl.rows = (int)rows;
    // Blocks are counted in tokens' order; the last rows first: they see the most keys.
    const int blocks = g.by_splits(g.x);
    pl.row0 = (blocks - 1 - block) * ROWS_WG;
    return pl.row0 < pl.rows;
}
// The end of a part's tiles: the last part has what the host's bound on the keys may have missed.
__device__ __forceinline__ int last_tile(int count, int from, const Block& b) {
    return b.pl.split + 1 < b.pl.splits && from + b.per < count ? from + b.per : count;
}
// Stores a part: its number among those of the row.
__device__ __forceinline__ void number_part(const PagesCall& c, const Block& b, Place* pl) {
    pl->split = b.all ? pl->split : c.prefix_splits + pl->split;
    pl->splits = c.parts;
}
// A packed row's queries, `part` channels from the lane's first on; rows past the end stand for the last.
template <int N>
__device__ __forceinline__ void load_queries(u32x4* to, const PagesCall& c, const Place& pl, int r, int first, int step) {
    const HeadsIn& t = c.p.a.q;
    r = r < pl.rows ? r : pl.rows - 1;
    const int tok = c.by_group(r), head = pl.kh * c.p.a.group + (r - tok * c.p.a.group);
    const char* at = (const char*)t.p + ((pl.q.first + tok) * t.ts + head * t.hs + first) * 2;
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = *(const u32x4*)(at + i * step * 2);
}
// Where packed row r's results go.
struct Target {
    int64_t row, index;
    int head;
};
__device__ __forceinline__ Target target_of(const PagesCall& c, const Place& pl, int r) {
    const int tok = c.by_group(r), head = pl.kh * c.p.a.group + (r - tok * c.p.a.group);
    const int64_t row = pl.q.first + tok;
    return Target{row, row * c.p.a.q_heads + head, head};
}

// The lowest and the highest position that the lanes of a wave (aligned runs of WIDTH of them) have, by
// moves inside the registers.
template <int WIDTH>
__device__ __forceinline__ int highest(int v) {
    const auto most = [](int a, int b) { return a > b ? a : b; };
    v = most(v, __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, true));   // lane ^ 1
    v = most(v, __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, true));   // lane ^ 2
    v = most(v, __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, true));  // the other half of eight
    v = most(v, __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, true));  // of sixteen
    if constexpr (WIDTH >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
        v = most((int)r[0], (int)r[1]);
    }
    if constexpr (WIDTH >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
        v = most((int)r[0], (int)r[1]);
    }
    return uniform(v);
}
// The lowest and the highest position of packed rows from .. from + n - 1, which are the lanes' (at; in
// aligned runs of WIDTH). kNowhere: none is of a sequence.
template <int WIDTH>
__device__ __forceinline__ void extremes(const PagesCall& c, const Block& b, int from, int n, int at, int* low, int* high) {
    if (b.all) {
        *high = highest<WIDTH>(at);
        *low = -highest<WIDTH>(at == kNowhere ? -INT32_MAX : -at);
    } else {  // one sequence's rows ascend
        const int last = from + n < b.pl.rows ? from + n - 1 : b.pl.rows - 1;
        *low = from <= last ? b.pl.offset + c.by_group(from) : kNowhere;
        *high = from <= last ? b.pl.offset + c.by_group(last) : kNowhere;
    }
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
    // Looks up the pages of the tile from t0.
    __device__ __forceinline__ void find(const PagesAttention& p, const KeyRun& run, int, int t0, int wave) {
        int rows[ROWS / 8];
        holes = run.tile_rows<16, ROWS>(p, t0, 0, rows);
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            const int in = (n * WAVES + wave) * Ti::kRowsPerCopy;
            int r = rows[0];
#pragma unroll
            for (int g = 1; g < ROWS / 8; ++g) {
                const int other = rows[g];
                r = in >> 3 == g ? other : r;
            }
            row[n] = r + (in & 7);
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

// Of PER_LOAD keys that a wave's lanes take in groups, the key of group i: an order in which sixteen lanes'
// stores to LDS meet different banks.
template <int D, int PER_LOAD>
__device__ __forceinline__ int shuffled(int i) {
    if constexpr (D == 128) return PER_LOAD == 8 ? (i & 1) << 2 | i >> 1 : (PER_LOAD == 16 ? (i & 3) << 2 | i >> 2 : i);
    return (i & ~6) | (i & 2) << 1 | (i & 4) >> 1;
}

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
        int rows[ROWS / 8];
        holes = run.tile_rows<BITS, ROWS>(p, t0, kh, rows);
#pragma unroll
        for (int g = 0; g < kRuns; ++g) {
            int r = rows[g];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) {
                const int other = rows[w * kRuns + g];
                r = wave == w ? other : r;
            }
            row[g] = r;
        }
    }
    static __device__ __forceinline__ int key(int lane) { return shuffled<D, kPerLoad>(lane / (kBytes / kChunk)); }  // of a load
    static __device__ __forceinline__ int channel(int lane) { return lane % (kBytes / kChunk) * kCodes; }
    __device__ __forceinline__ void load(int lane) {
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int in = key(lane);
            int r = row[n * kPerLoad / 8];
#pragma unroll
            for (int g = 1; g < kPerLoad / 8; ++g) {
                const int other = row[n * kPerLoad / 8 + g];  // read outside the choice: a choice of places would put them in memory
                r = in >> 3 == g ? other : r;
            }
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
            const int in = wave * kKeys + n * kPerLoad + key(lane), c0 = channel(lane) / 8;
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

// Four channels of a value row of the pool, in 16 bits.
template <typename T, int D, int BITS>
__device__ __forceinline__ u32x2 value4(const PagesAttention& p, int64_t row, int kh, int ch) {
    if constexpr (BITS == 16) {
        return *(const u32x2*)((const T*)p.a.v.p + row * p.a.v.ts + kh * p.a.v.hs + ch);
    } else {
        const float factor = mx_factor(p.mx.vs[row * (D / 32) + ch / 32]);
        const uint8_t* at = p.mx.v + (row * D + ch) * BITS / 8;
        uint32_t two[16 / BITS];
        if constexpr (BITS == 8)
            mx_decode<T, 8>(*(const uint32_t*)at, factor, two);
        else
            mx_decode<T, 4>(*(const uint16_t*)at, factor, two);
        return u32x2{two[0], two[1]};
    }
}
// Infinities and NaN of the values of a tile of keys, which stand as zeros in LDS, to the rows that see them.
template <typename T, int D, int BITS>
__device__ __forceinline__ void add_bad(const PagesAttention& p, const KeyRun& run, int kh, f32x16* o, const Span& sp, int t0, int rows,
                                        unsigned long long holes, int lane) {
    const int to = t0 + rows < run.count ? t0 + rows : run.count;
    for (int j = t0; j < to; ++j) {
        const int64_t row = run.pool_row<BITS>(p, j, kh);
        if (row < 0) continue;
        const bool on = sees(sp, j) && !(holes >> (j - t0) & 1);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const u32x2 four = value4<T, D, BITS>(p, row, kh, 32 * i + 8 * x + 4 * (lane >> 5));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint16_t bits = (uint16_t)(four[e >> 1] >> (16 * (e & 1)));
                    if (on && !finite16<T>(bits)) o[i][4 * x + e] += widen(__builtin_bit_cast(T, bits));
                }
                asm volatile("" ::: "memory");  // few registers: this is rare
            }
    }
}

// Sixteen rows, for single tokens: v_mfma_f32_16x16x32, whose sums and weights are half as many as those
// of 32 rows. S^T has keys as rows: lane l holds row l % 16 and, of each sixteen keys, 4h .. 4h + 3 (h = l / 16);
// two such blocks are the B operand of the second product as they are, with keys 16 a + 4h + b in the
// place of 8h + 4a + b. Channels may come in any order that keys and queries share: a lane
// takes a quarter of a head's, which lie together, so keys go from memory to the product without
// LDS, and with them one scale.
template <typename T, int D>
struct FewRows {
    u32x4 q[D / 32];
    f32x4 o[D / 16];
    float m, l;
    Span sp;

    static __device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 c) {
        if constexpr (__is_same(T, _Float16))
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    // Over the four lanes that hold a row.
    static __device__ __forceinline__ float quarters_max(float v) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
        return both_max(fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])));
    }
    static __device__ __forceinline__ float quarters_sum(float v) {
        const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
        return both_sum(__builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        l = 0.f;
    }
    // Scores of 32 keys into weights.
    __device__ __forceinline__ u32x4 weigh(f32x4* s, int t0, float c, bool masked, unsigned long long holes, int lane) {
        if (masked) {
            const unsigned long long seen = (seen_bits(sp, t0) & ~holes) >> (4 * (lane >> 4));
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[b][i] = keep_or(s[b][i], spread_bit(seen, 16 * b + i), -INFINITY);
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i >> 2][i & 3]);
        top = quarters_max(top) * c;
        const bool raise = top > m + kSlack;
        if (__builtin_expect(__any(raise), 0)) {
            const float next = raise ? top : m;  // the other rows stay: no row's bits go by its neighbours'
            const float old = exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= old;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] *= old;
        }
        const float ref = kLift<T> - (m == -INFINITY ? 0.f : m);
        f32x16 w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], c, ref));
        l += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        return pack8<T>(w, 0);
    }
    // A operand of the second product: channels 16 blk + l % 16, keys as above, from a tile in LDS.
    static __device__ __forceinline__ u32x4 values(const char* tile, int blk, int lane) {
        u32x4 r;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int row = 16 * a + 4 * (lane >> 4) + ((lane & 15) >> 2), chunk = 2 * blk + ((lane & 3) >> 1);
            const char* at = tile + (row * Tile<D>::kChunks + (chunk ^ Tile<D>::swizzle(row))) * 16 + (lane & 1) * 8;
            const u32x2 v = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
            r[2 * a] = v[0];
            r[2 * a + 1] = v[1];
        }
        return r;
    }
};

// 32 keys on their way to one wave: a lane's quarters of two keys' channels, and its share of the
// values, which go through LDS. Loaded a tile ahead.
template <typename T, int D, int BITS>
struct FewStage {
    using Ti = Tile<D>;
    static constexpr int kBytes = D * BITS / 8, kPart = kBytes / 4;  // a key's bytes, a quarter
    static constexpr int kWords = kPart / 4, kWide = kWords < 4 ? kWords : 4;
    static constexpr int kLoads = kBytes / 32 ? kBytes / 32 : 1;     // 16 bytes each, of values
    static constexpr int kPerLoad = 32 / kLoads, kLanes = 64 / kPerLoad;  // keys a load takes, lanes a key
    static constexpr int kCodes = 128 / BITS, kGroups = kCodes / 8;
    typedef uint32_t wide __attribute__((ext_vector_type(kWide)));
    int row[4];
    unsigned long long holes = 0;
    wide k[2][kWords / kWide];
    u32x4 v[kLoads];
    uint32_t kf[2], vf[kLoads];

    __device__ __forceinline__ void find(const PagesAttention& p, const KeyRun& run, int kh, int t0) {
        holes = run.tile_rows<BITS, 32>(p, t0, kh, row);
    }
    // Row of the pool of key `in` of the tile, whose run of eight is one of those from `first` on.
    template <int N>
    __device__ __forceinline__ int64_t pool(int first, int in) const {
        int r = row[first];
#pragma unroll
        for (int g = 1; g < N; ++g) {
            const int other = row[first + g];  // read outside the choice: a choice of places would put them in memory
            r = (in >> 3) - first == g ? other : r;
        }
        return r + (in & 7);
    }
    __device__ __forceinline__ void load(const PagesAttention& p, int kh, int lane) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t at = pool<2>(2 * b, 16 * b + (lane & 15));
            const char* from;
            if constexpr (BITS == 16) {
                from = (const char*)p.a.k.p + (at * p.a.k.ts + kh * p.a.k.hs) * 2 + (lane >> 4) * kPart;
            } else {
                from = (const char*)p.mx.k + at * kBytes + (lane >> 4) * kPart;
                kf[b] = p.mx.ks[at * (D / 32) + (lane >> 4) * (D / 32) / 4];
            }
#pragma unroll
            for (int i = 0; i < kWords / kWide; ++i) k[b][i] = *(const wide*)(from + i * kWide * 4);
        }
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int in = n * kPerLoad + shuffled<D, kPerLoad>(lane / kLanes), c = lane % kLanes;
            const int64_t at = pool<kPerLoad / 8 ? kPerLoad / 8 : 1>(n * kPerLoad / 8, in);
            if constexpr (BITS == 16) {
                v[n] = *(const u32x4*)((const char*)p.a.v.p + (at * p.a.v.ts + kh * p.a.v.hs) * 2 + c * 16);
            } else {
                v[n] = *(const u32x4*)(p.mx.v + at * kBytes + c * 16);
                vf[n] = p.mx.vs[at * (D / 32) + c * kCodes / 32];
            }
        }
    }
    // The values to LDS; look: zeros for what is not finite, and whether there was any.
    __device__ __forceinline__ bool store(char* vt, bool look, int lane) const {
        bool bad = false;
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const int in = n * kPerLoad + shuffled<D, kPerLoad>(lane / kLanes), c0 = lane % kLanes * kGroups;
            u32x4 x[kGroups];
            if constexpr (BITS == 16) {
                x[0] = v[n];
            } else {
                const float f = mx_factor(vf[n]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t two[16 / BITS];
                    mx_decode<T, BITS>(v[n][w], f, two);
#pragma unroll
                    for (int i = 0; i < 16 / BITS; ++i) x[w * (16 / BITS) / 4][(w * (16 / BITS) + i) & 3] = two[i];
                }
            }
            if (__builtin_expect(look, 0)) {
#pragma unroll
                for (int g = 0; g < kGroups; ++g) bad |= clean16<T>(x[g]);
            }
#pragma unroll
            for (int g = 0; g < kGroups; ++g) *(u32x4*)(vt + (in * Ti::kChunks + ((c0 + g) ^ Ti::swizzle(in))) * 16) = x[g];
        }
        return look && __any(bad);
    }
    // Step s of the first product: eight channels of key l % 16 of block b.
    __device__ __forceinline__ u32x4 keys(int b, int s) const {
        u32x4 r;
        constexpr int each = BITS / 4;  // words of eight channels
        if constexpr (BITS == 16) {
            r = k[b][s];
        } else {
#pragma unroll
            for (int w = 0; w < each; ++w) {
                uint32_t two[16 / BITS];
                const int at = s * each + w;
                mx_decode<T, BITS>(k[b][at / kWide][at % kWide], mx_factor(kf[b]), two);
#pragma unroll
                for (int i = 0; i < 16 / BITS; ++i) r[w * (16 / BITS) + i] = two[i];
            }
        }
        return r;
    }
};

}  // namespace
}  // namespace fa
}  // namespace dcn
