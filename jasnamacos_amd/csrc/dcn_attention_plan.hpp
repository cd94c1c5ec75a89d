// How the matrix kernels of attention over pages share a call out: which kernels take its rows, and in how many
// parts its keys are taken (dcn_kernels_attention_pages.hip).
#pragma once

#include "dcn_attention.hpp"

namespace dcn {
namespace fa {

// The blocks of rows of one kind, and in how many parts each one's key tiles are taken.
struct Blocks {
    int rows;  // of a block: 16 (token kernel), 32 (few kernel) or 128 (tile kernel)
    int waves, blocks, splits, per;
};
struct PlanOf {
    Blocks prefix, own;
    bool shared, both;  // shared: the prefix once for all sequences; both: own blocks take it
    int parts;
};

// Whether more than 32 rows take 32-row workgroups, whose waves share the keys out, and not 128-row ones.
// The small ones fill the card where there are few (wide: 128-row workgroups) and read the keys four times
// as often. Measured (us, 128 rows -> 32; 8 query heads on 4 throughout, other groups were not tried):
//   64 channels, 8 bits: wide 32 at 3,000 keys 29 -> 24; 128 at 12,000 104 -> 94; 256 at 12,000 198 -> 159;
//     456 at 4,000 100 -> 72 and at 12,000 310 -> 305; 464 at 14,400 344 -> 365; 928 at 4,000 154 -> 135;
//     2,048 at 12,000 914 -> 924. 4 bits: 256 at 16,000 252 -> 199.
//   64 channels, 16 bits: 128 at 4,000 47 -> 40 and at 8,000 73 -> 75; 192 at 4,000 74 -> 68; 456 at 4,000
//     155 -> 187.
//   128 channels, 8 bits: 128 at 3,000 55 -> 43; 256 at 12,000 274 -> 255; 928 at 4,000 221 -> 242.
//     4 bits: 4 at 300 15 -> 11; 64 at 700 28 -> 20, at 2,000 32 -> 34, at 4,000 43 -> 52; 128 at 1,200 35 -> 22, at
//     2,000 45 -> 40; 256 at 700 31 -> 32, at 4,000 112 -> 125. 16 bits: 4 at 300 18 -> 12; 64 at 600 27 -> 27; 128 at
//     600 27 -> 24, at 2,000 44 -> 52; 256 at 600 28 -> 47.
inline bool few_of(int dim, int bits, int64_t wide, int64_t keys) {
    if (dim == 64 && bits) return wide <= 256 || (wide <= 1024 && keys <= 8192);
    if (dim == 64) return wide <= 256 && keys <= 6144;
    return bits == 8 ? wide <= 256 : wide <= 128 && keys <= (bits ? 2048 : 1024);
}

// Up to 16 rows take the token kernel. Keys are taken in parts where workgroups would leave the card idle,
// until about 512 are there (two a CU): one token of 32 streams on 18,001 keys of 8 bits, 32 heads of 128
// on 8, in one part 217 us, in two 156, in six 170. Tiles of 128 rows write long parts, so only whole
// shares are taken: a frame of 3,600 tokens for two streams, 464 workgroups, 340 us in one part and 470 in
// two. Up to four tiles of 32 keys a wave go to one workgroup of many waves for single tokens: a join costs more.
// That is 64 tiles at 64 channels (16 waves; 997 keys, 8 heads: 10.6 us, in parts 12.7) and 32 at 128 (8 waves;
// 8 heads on 8 bits, in one workgroup and in parts: 1,280 keys 13.3 and 13.6, 1,500 keys 16.2 and 13.4, 2,040 keys
// 19.0 and 13.0).
inline Blocks blocks_of(int dim, int64_t rows, int64_t pairs, int64_t keys, int64_t resident, bool few) {
    Blocks b;
    b.rows = rows <= 16 ? 16 : (few ? 32 : 128);
    const int tile = few ? 32 : 64;
    b.blocks = (int)((rows + b.rows - 1) / b.rows);
    const int64_t tiles = (keys + tile - 1) / tile, groups = (int64_t)b.blocks * pairs;
    b.waves = b.rows == 32 && dim == 64 && groups <= 256 ? 8 : 4;
    if (b.rows == 16 && groups <= 256 && tiles <= 64) b.waves = dim == 64 ? 16 : 8;
    const int64_t least = few ? b.waves : 4;
    int64_t splits = 1;
    if (groups > 0 && tiles > 4 * least) {
        splits = b.rows == 128 ? resident / groups : (resident + groups - 1) / groups;
        splits = splits < tiles / least ? splits : tiles / least;
        splits = splits < 32 ? splits : 32;
    }
    splits = splits < 1 ? 1 : splits;
    b.per = (int)((tiles + splits - 1) / splits);
    b.splits = b.per ? (int)((tiles + b.per - 1) / b.per) : 1;
    return b;
}

// Bytes of the prefix that would be read again by the sequences behind the first from which on sharing it
// pays for the join of its parts: about 12 us of reading, from the caches. 24 streams on 2,175 keys
// (51 MB): shared 21 us, each on its own 12; 61 streams on 1,500 keys (180 MB): 21 and 31. Sequences whose
// rows fill blocks of their own share nothing: a block reads the prefix once either way.
constexpr double kAgain = 120e6;

inline PlanOf plan_of(int dim, int bits, int sequences, int kv_heads, int group, int64_t q_tokens, int max_q, int max_kv, int max_prefix,
                      int frame, int back, int sinks) {
    PlanOf p{};
    const int64_t rows = (int64_t)max_q * group, pairs = (int64_t)kv_heads * sequences;
    // Keys that a block of rows sees at most.
    const auto keys_of = [&](int64_t tokens, int most) { return attention_keys(most, frame, back, sinks, tokens, 64); };
    const int64_t first = max_prefix ? keys_of(max_q, max_prefix) : 0, own = keys_of(128 / group, max_kv);
    const double again = (double)(sequences - 1) * first * kv_heads * dim * (bits ? bits : 16) / 4;
    p.shared = first > 0 && sequences > 1 && rows < 128 && again > kAgain;
    p.both = first > 0 && !p.shared;
    const int64_t keys = own + (p.both ? first : 0);
    p.own = blocks_of(dim, rows, pairs, keys, 512, rows <= 32 || few_of(dim, bits, (rows + 127) / 128 * pairs, keys));
    // The prefix's rows are many and its keys long: 128-row blocks, unless they are few rows.
    if (p.shared)
        p.prefix = blocks_of(dim, q_tokens * group, kv_heads, first, p.own.rows == 16 ? 256 : 512, q_tokens * group <= 32);
    p.parts = p.own.splits + (p.shared ? p.prefix.splits : 0);
    return p;
}

// Whether every launch of a plan has fewer than 2^32 threads along x: these workgroups over the prefix and over the
// sequences' own keys (in one launch or two), and the join of `rows` rows and heads of a sequence.
constexpr int kJoinByRow = 8;  // up to so many parts a wave joins a row, else a workgroup does
inline bool launches_fit(const PlanOf& p, unsigned prefix_grid, unsigned own_grid, int64_t rows) {
    const int64_t most = (INT64_C(1) << 32) / 64;  // waves
    return (int64_t)prefix_grid * p.prefix.waves + (int64_t)own_grid * p.own.waves < most &&
           (p.parts == 1 || rows < (p.parts <= kJoinByRow ? most - 4 : most / 4));
}

}  // namespace fa
}  // namespace dcn
