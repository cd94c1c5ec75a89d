// Building blocks of the matrix-core attention kernels: tiles of key (or query) rows in LDS,
// their copy from HBM, and the operand layouts of v_mfma_f32_32x32x16.
//
// The products are arranged so that the softmax never leaves a lane. S^T = K Q^T has M = keys
// and N = rows: lane l holds row l % 32 and, of each block of 32 keys, the 16 keys
// 8a + 4h + b (h = l / 32, a and b = 0..3, in register 4a + b). Registers 8s .. 8s + 7 are then
// the B operand of the next product's step s as they are (O^T += V^T P^T, K index = keys), as
// long as the A operand takes its keys in that order too: two reads of four adjacent keys at
// one channel, which is what the transposing LDS read gives from row-major rows. A row's
// maximum and sum are over the lane's own registers and those of lane l ^ 32.
#pragma once

#include <hip/hip_runtime.h>

#include "dcn_attention_device.hpp"

namespace dcn {
namespace fa {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// Eight FP32 values to 16 bits, nearest even.
template <typename T>
__device__ __forceinline__ u32x4 pack8(const f32x16& v, int first) {
    typedef T vec __attribute__((ext_vector_type(8)));
    vec r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (T)v[first + i];
    return __builtin_bit_cast(u32x4, r);
}

// The other half of the wave's value (lane ^ 32) combined with the own one.
__device__ __forceinline__ float both_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

// The packed rows of one (sequence, key head): row r is token r / group, head kh * group + r % group.
struct Rows {
    int group, shift;  // shift >= 0: group is 1 << shift
    __device__ __forceinline__ int token(int r) const { return shift >= 0 ? r >> shift : r / group; }
};
__device__ __forceinline__ Rows rows_of(int group) {
    return Rows{group, (group & (group - 1)) == 0 ? 31 - __builtin_clz((unsigned)group) : -1};
}

// A tile: ROWS rows of D 16-bit channels, row-major, the 16-byte chunks of row r at chunk ^
// swizzle(r). LDS gives 256 bytes a cycle from 64 banks: a read of rows takes sixteen lanes (one
// chunk of sixteen adjacent rows) at a time, a transposing one thirty-two (64 bytes of four
// adjacent rows). With 128 channels, a row on all banks, both lie in different banks. With 64 they
// meet in pairs: the swizzle without that has more addresses to hold, and a training step of
// 4 x 2560 tokens took 174 us with it, 170 so (128 channels, forward of 2 x 4096 tokens: 185 us
// without conflicts, 190 in pairs).
template <int D>
struct Tile {
    static constexpr int kChunks = D / 8;           // 16-byte chunks a row
    static constexpr int kRowsPerCopy = 64 / kChunks;  // rows that one wave's copy instruction fills

    static __device__ __forceinline__ int swizzle(int row) {
        return D == 64 ? ((row & 3) << 1) | (row >> 2 & 1) : ((row & 3) << 2) | (row >> 2 & 3);
    }

    // A operand with M = rows: row 32 mb + l % 32, channels 16 s + 8 h .. + 7.
    static __device__ __forceinline__ u32x4 rows(const char* tile, int mb, int s, int lane) {
        const int r = 32 * mb + (lane & 31);
        return *(const u32x4*)(tile + (r * kChunks + ((2 * s + (lane >> 5)) ^ swizzle(r))) * 16);
    }
    // A operand with M = channels 32 blk + l % 32: rows 32 mb + 16 s + {4h + b, 8 + 4h + b}.
    static __device__ __forceinline__ u32x4 columns(const char* tile, int mb, int s, int blk, int lane) {
        u32x4 r;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int row = 32 * mb + 16 * s + 8 * a + 4 * (lane >> 5) + ((lane & 15) >> 2);
            const int chunk = 4 * blk + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            const char* p = tile + (row * kChunks + (chunk ^ swizzle(row))) * 16 + (lane & 1) * 8;
            const u32x2 v = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
            r[2 * a] = v[0];
            r[2 * a + 1] = v[1];
        }
        return r;
    }
    // Where lane `lane` of copy instruction n reads: its row and channel.
    static __device__ __forceinline__ int copy_row(int n, int lane) { return n * kRowsPerCopy + lane / kChunks; }
    static __device__ __forceinline__ int copy_channel(int row, int lane) {
        return ((lane % kChunks) ^ swizzle(row)) * 8;
    }
};

// 64 lanes x 16 bytes from HBM (base + at, at per lane) into LDS at dst + 16 lane; base and dst
// are uniform. In asm because the compiler, seeing the builtin, holds every later LDS read back
// until all copies have arrived (it does not tell the two halves of a double buffer apart).
// There is no output register; wait_copies() and a barrier or its own memory clobber order the
// reads.
__device__ __forceinline__ void copy16(const char* base, uint32_t at, char* dst) {
    const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(at), "s"(base) : "memory");
}
// All but the last LEFT of this wave's copies have arrived.
template <int LEFT>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}
// The LDS reads before this have been made: their place may be written.
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <typename T>
__device__ __forceinline__ bool finite16(uint16_t bits) {
    constexpr uint16_t e = __is_same(T, _Float16) ? 0x7c00 : 0x7f80;
    return (bits & e) != e;
}
// Zeros in the place of infinities and NaN; whether there were any.
template <typename T>
__device__ __forceinline__ bool clean16(u32x4& v) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (!finite16<T>((uint16_t)v[i])) v[i] &= 0xffff0000u, bad = true;
        if (!finite16<T>((uint16_t)(v[i] >> 16))) v[i] &= 0xffffu, bad = true;
    }
    return bad;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

// Workgroups on the card's eight XCDs, each with an L2 of its own: workgroup i runs on XCD i % 8.
// The blocks of one (sequence, key head) read the same keys, so they stay on one XCD where the
// number of pairs is a multiple of 8, or else share as few XCDs as spread the work evenly, taking
// blocks in turn. `x` blocks a pair.
struct BlockMap {
    int x, heads, pairs, classes;  // classes: the greatest common divisor of pairs and 8
    unsigned grid;
};
inline bool block_map(int64_t x, int64_t heads, int64_t sequences, BlockMap* m) {
    const int64_t pairs = heads * sequences, classes = pairs % 8 == 0 ? 8 : (pairs % 4 == 0 ? 4 : (pairs % 2 == 0 ? 2 : 1));
    const int64_t share = 8 / classes, each = (pairs / classes * x + share - 1) / share;
    *m = BlockMap{(int)x, (int)heads, (int)pairs, (int)classes, (unsigned)(8 * each)};
    return x < INT32_MAX && each < (INT64_C(1) << 32) / kThreads / 8;  // fewer than 2^32 threads
}
// Block, key head and sequence of this workgroup; false for the padding.
__device__ __forceinline__ bool block_of(const BlockMap& m, int* block, int* head, int* sequence) {
    const int xcd = blockIdx.x & 7, share = 8 / m.classes;
    const int item = (int)(blockIdx.x >> 3) * share + xcd / m.classes;
    const int nth = item / m.x, pair = xcd % m.classes + m.classes * nth;
    if (pair >= m.pairs) return false;
    *block = item - nth * m.x;
    *head = pair % m.heads;
    *sequence = pair / m.heads;
    return true;
}

// Where one workgroup works.
struct Place {
    int seq, kh, split, splits;
    Run q, kv;
    int rows;   // packed rows of this (sequence, key head)
    int row0;   // the workgroup's first
    int offset; // position of query 0
};

template <bool PAGED>
struct Keys {
    HeadsIn k, v;
    PagesArgs pages;
    const char *kp, *vp;  // the head's first row (contiguous: of the sequence)
    int seq, count;

    __device__ __forceinline__ Keys(const AttentionArgs& a, int s, int kh, const Run& kv) : k(a.k), v(a.v), pages(a.pages) {
        seq = s;
        count = kv.count;
        const int64_t first = PAGED ? 0 : kv.first;
        kp = (const char*)a.k.p + (first * k.ts + kh * k.hs) * 2;
        vp = (const char*)a.v.p + (first * v.ts + kh * v.hs) * 2;
    }
    // Row of the pool of key j (uniform); -1 where its page is not there. A scalar load: it is not
    // counted with the copies, so waiting for it does not wait for them.
    __device__ __forceinline__ int pool_row(int j) const {
        typedef const __attribute__((address_space(4))) int* scalar;
        const int page = ((scalar)(uintptr_t)(pages.table + (int64_t)seq * pages.width))[j >> pages.shift];
        return (unsigned)page >= (unsigned)pages.pages ? -1 : (page << pages.shift) + (j & ((1 << pages.shift) - 1));
    }
    __device__ __forceinline__ int end(int t1) const { return t1 < count ? t1 : count; }
    // Value row of key j, or null.
    __device__ __forceinline__ const uint16_t* value(int j) const {
        const int64_t row = PAGED ? pool_row(j) : j;
        return row < 0 ? nullptr : (const uint16_t*)(vp + row * v.ts * 2);
    }
};

// Pages have 8 tokens at least, and every run of 8 keys from a multiple of 8 lies on one. What
// the copies of a tile of ROWS keys need of the table, looked up a tile ahead: the rows of the
// pool that copy instructions wave, wave + WAVES, ... start at (past the sequence's end: those
// of its last run; rows past it are in the pool, and not visible), and a bit per key whose page
// is not there.
template <int D, int ROWS, int WAVES, bool PAGED>
struct TilePages {
    static constexpr int kCopies = ROWS / Tile<D>::kRowsPerCopy / WAVES;
    int row[kCopies];
    unsigned long long holes = 0;

    __device__ __forceinline__ void find(const Keys<PAGED>& keys, int t0, int wave) {
        if constexpr (PAGED) {
            const int last = (keys.count - 1) & ~7;
#pragma unroll
            for (int n = 0; n < kCopies; ++n) {
                const int in = (n * WAVES + wave) * Tile<D>::kRowsPerCopy, j = t0 + (in & ~7);
                const int r = keys.pool_row(j < last ? j : last);
                row[n] = r < 0 ? 0 : r + (in & 7);
            }
            holes = 0;
#pragma unroll
            for (int g = 0; g < ROWS / 8; ++g) {
                const int j = t0 + 8 * g;
                if (keys.pool_row(j < last ? j : last) < 0) holes |= 0xffull << (8 * g);
            }
        }
    }
};

// This wave's part of the copies of key tiles: byte offsets of its lanes from the tile's first
// key (paged: from each instruction's first key), the same for every tile but the last.
template <int D, int ROWS, int WAVES, bool PAGED>
struct TileCopy {
    using Ti = Tile<D>;
    static constexpr int kCopies = ROWS / Ti::kRowsPerCopy / WAVES;
    static constexpr int kOffsets = PAGED ? 1 : kCopies;
    uint32_t k[kOffsets], v[kOffsets];

    // Rows past `last` stand for it (contiguous keys only: a page is there whole).
    __device__ __forceinline__ void set(const Keys<PAGED>& keys, int last, int wave, int lane) {
#pragma unroll
        for (int n = 0; n < kOffsets; ++n) {
            const int in = PAGED ? lane / Ti::kChunks : Ti::copy_row(n * WAVES + wave, lane);
            const uint32_t at = PAGED || in < last ? in : last;
            k[n] = at * (uint32_t)keys.k.ts * 2;
            v[n] = at * (uint32_t)keys.v.ts * 2;
            if (!PAGED) {
                k[n] += Ti::copy_channel(in, lane) * 2;
                v[n] += Ti::copy_channel(in, lane) * 2;
            }
        }
    }
    // The tile from key t0 (below the sequence's end) to `kt` and `vt`.
    __device__ __forceinline__ void copy(const Keys<PAGED>& keys, int t0, const TilePages<D, ROWS, WAVES, PAGED>& pages, char* kt,
                                         char* vt, int wave, int lane) {
        if (!PAGED && t0 + ROWS > keys.count) set(keys, keys.count - 1 - t0, wave, lane);
        const char* kb = keys.kp + (int64_t)t0 * keys.k.ts * 2;
        const char* vb = keys.vp + (int64_t)t0 * keys.v.ts * 2;
#pragma unroll
        for (int n = 0; n < kCopies; ++n) {
            const int i = n * WAVES + wave;
            if constexpr (PAGED) {
                const uint32_t c = Ti::copy_channel(Ti::copy_row(i, lane), lane) * 2;
                copy16(keys.kp + (int64_t)pages.row[n] * keys.k.ts * 2, k[0] + c, kt + i * 1024);
                copy16(keys.vp + (int64_t)pages.row[n] * keys.v.ts * 2, v[0] + c, vt + i * 1024);
            } else {
                copy16(kb, k[n], kt + i * 1024);
                copy16(vb, v[n], vt + i * 1024);
            }
        }
    }
};

// Whether any of eight values is infinite or NaN: its exponent's ones carry into the sign's place.
template <typename T>
__device__ __forceinline__ bool any_nonfinite(u32x4 v) {
    constexpr uint32_t e = __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u, one = __is_same(T, _Float16) ? 0x04000400u : 0x00800080u;
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) t |= (v[i] & e) + one;
    return t & 0x80008000u;
}
// Zeros for the infinities and NaN of the rows of a tile that this wave has copied (and that
// have arrived); a bit, in every lane, for each row that had one.
template <typename T, int D, int ROWS, int WAVES>
__device__ __forceinline__ unsigned long long clean_own(char* tile, int wave, int lane) {
    using Ti = Tile<D>;
    constexpr int n = ROWS / Ti::kRowsPerCopy / WAVES;
    u32x4 v[n];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < n; ++i) {
        v[i] = *(const u32x4*)(tile + (i * WAVES + wave) * 1024 + lane * 16);
        bad |= any_nonfinite<T>(v[i]);
    }
    if (__builtin_expect(!__any(bad), 1)) return 0;
    unsigned long long rows = 0;
#pragma unroll
    for (int i = 0; i < n; ++i)
        if (clean16<T>(v[i])) {
            *(u32x4*)(tile + (i * WAVES + wave) * 1024 + lane * 16) = v[i];
            rows |= 1ull << Ti::copy_row(i * WAVES + wave, lane);
        }
    for (int d = 32; d; d >>= 1) rows |= __shfl_xor(rows, d);
    return rows;
}
// What the waves of a workgroup found in a tile, exchanged over the barrier that the tile waits
// for: one slot a wave and buffer.
struct FoundRows {
    unsigned long long wave[2][kWaves];
    __device__ __forceinline__ unsigned long long all(int buf) const {
        unsigned long long r = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) r |= wave[buf][w];
        return r;
    }
};

// Infinities and NaN of one row of 16-bit channels, which stand as zeros in LDS, to a lane's sums
// (o^T: channels 32 i + 8 a + 4 h + b) if `on`.
template <typename T, int D>
__device__ __forceinline__ void add_nonfinite(f32x16* o, const uint16_t* row, bool on, int lane) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const u32x2 four = *(const u32x2*)(row + 32 * i + 8 * a + 4 * (lane >> 5));
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint16_t bits = (uint16_t)(four[b >> 1] >> (16 * (b & 1)));
                if (on && !finite16<T>(bits)) o[i][4 * a + b] += widen(__builtin_bit_cast(T, bits));
            }
            asm volatile("" ::: "memory");  // one load at a time: few registers, and this is rare
        }
}
// The same for the rows of a tile of keys, `row(j)` that of key j or null.
template <typename T, int D, typename Row>
__device__ __forceinline__ void add_nonfinite(f32x16* o, const Span& sp, int t0, int to, unsigned long long holes, int lane, Row row) {
    for (int j = t0; j < to; ++j)
        if (const uint16_t* v = row(j)) add_nonfinite<T, D>(o, v, sees(sp, j) && !(holes >> (j - t0) & 1), lane);
}

// A pair's blocks are split + splits * row block, the last rows first: they see the most keys.
template <int ROWS_WG>
__device__ __forceinline__ bool place_of(const AttentionArgs& a, const BlockMap& map, int splits, Place* pl) {
    int at;
    if (!block_of(map, &at, &pl->kh, &pl->seq)) return false;
    pl->splits = splits;
    const int block = map.x / splits - 1 - at / splits;
    pl->split = at % splits;
    pl->q = run_of(a.cu_q, pl->seq, a.max_q, a.q_tokens);
    pl->kv = kv_run_of(a, pl->seq);
    pl->q.count = uniform(pl->q.count);
    pl->kv.count = uniform(pl->kv.count);
    pl->offset = pl->kv.count - pl->q.count;
    const int64_t rows = (int64_t)(pl->q.count < a.max_q ? pl->q.count : a.max_q) * a.group;
    pl->rows = (int)rows;
    pl->row0 = block * ROWS_WG;
    return pl->row0 < pl->rows;
}

// The B operand of packed row r (past the end: of the last one): channels 16 i + 8 h .. + 7.
template <int D>
__device__ __forceinline__ void load_row(u32x4* to, const HeadsIn& t, const AttentionArgs& a, const Place& pl, const Rows& rw, int r,
                                         int lane) {
    r = r < pl.rows ? r : pl.rows - 1;
    const int tok = rw.token(r), head = pl.kh * a.group + (r - tok * a.group);
    const char* p = (const char*)t.p + ((pl.q.first + tok) * t.ts + head * t.hs + 8 * (lane >> 5)) * 2;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) to[i] = *(const u32x4*)(p + i * 32);
}

// Bits [0, n) of 64.
__device__ __forceinline__ unsigned long long bits_below(int n) {
    return n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1);
}
// A bit for each of 64 keys from t0 that a row sees.
__device__ __forceinline__ unsigned long long seen_bits(const Span& s, int t0) {
    return (bits_below(s.hi - t0) & ~bits_below(s.lo - t0)) | bits_below(s.sink - t0);
}
// All ones if bit `in` of a lane's 64 is set: a constant `in` makes it one instruction.
__device__ __forceinline__ uint32_t spread_bit(unsigned long long bits, int in) {
    return (uint32_t)((int32_t)((uint32_t)(bits >> (in & 32)) << (31 - (in & 31))) >> 31);
}
__device__ __forceinline__ float keep_or(float v, uint32_t mask, float other) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, v) & mask) | (__builtin_bit_cast(uint32_t, other) & ~mask));
}

struct Spread {
    Span first, last;  // of the first and the last row of a run of rows: all three ends grow with the position
};
__device__ __forceinline__ Spread spread_of(const AttentionArgs& a, const Place& pl, const Rows& rw, int from, int to) {
    Spread s;
    s.first = span_of(a, pl.offset + rw.token(from), pl.kv.count);
    s.last = span_of(a, pl.offset + rw.token(to), pl.kv.count);
    return s;
}
// Tiles of ROWS keys that some row of the run sees.
template <int ROWS>
struct TileList {
    int near, first, count;
    __device__ __forceinline__ TileList(const Spread& s) {
        const int end = (s.last.hi + ROWS - 1) / ROWS;
        first = s.first.lo / ROWS;
        near = (s.last.sink + ROWS - 1) / ROWS;
        if (near > first) near = first;
        count = near + (end > first ? end - first : 0);
    }
    __device__ __forceinline__ int tile(int i) const { return (i < near ? i : first + (i - near)) * ROWS; }
};
template <int ROWS>
__device__ __forceinline__ bool all_see(const Spread& s, int t0) {
    const int t1 = t0 + ROWS;
    return t1 <= s.first.hi && (t0 >= s.last.lo || t1 <= s.first.sink);
}
template <int ROWS>
__device__ __forceinline__ bool none_sees(const Spread& s, int t0) {
    return t0 >= s.last.hi || (t0 + ROWS <= s.first.lo && t0 >= s.last.sink);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

}  // namespace fa
}  // namespace dcn
