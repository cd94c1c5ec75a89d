// Windowed attention forward on the matrix cores: FP16 and BF16 heads of 64 and 128 channels,
// contiguous or paged keys.
//
// Rows are packed: the heads that share a key head stand side by side (row = token, head of
// the group), so that a key tile is read once for all of them and single tokens fill a
// wave's rows. One pass over the visible key tiles with the running maximum and sum of the
// softmax; the maximum is raised (and the sums rescaled) only when a score passes it by more
// than 2^8, which FP32 sums do not notice. Two shapes:
//   tile kernel  four waves of 32 rows each share tiles of 64 keys;
//   few kernel   32 rows a workgroup, where there are no more or where 128-row workgroups would leave
//                CUs idle: four or eight waves take tiles of 32 keys in turn, each with its own
//                buffers and no barrier, and are joined at the end.
// Both may split the key tiles over workgroups; a second kernel then joins the parts.
//
// What bounds them. Tile kernel: the issue of vector and matrix instructions and the waits between
// them at two waves a SIMD (128 channels: MFMA 44 % of the cycles, vector instructions about as many,
// which overlap in part); 7,680 tokens in windows of nine frames of 256, 16 heads of 128 on 4: 140 to 150 us, 840 to
// 890 TFLOP/s of the 1,220 that a large product reaches; 2 x 4,096 causal tokens, 16 heads of 64: 116 us,
// of 128: 184 us. Few kernel: HBM where histories are long (32 tokens on 16,384 of 20,011 keys, 32 heads of 128
// on 8: 314 us, 5.5 TB/s), else the chain of launch, first tile and join (one token on 777 keys, 8 heads of 64:
// 9.1 us).
#include "dcn_attention_forward.hpp"

namespace dcn {
namespace fa {
namespace {

template <typename T, int D, bool PAGED>
__global__ __launch_bounds__(kThreads, 2) void attention_tile_kernel(AttentionArgs a, BlockMap map, int splits) {
    constexpr int ROWS = 64, BYTES = ROWS * D * 2;
    __shared__ __attribute__((aligned(1024))) char lds[2][2][BYTES];
    __shared__ FoundRows found;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Place pl;
    if (!place_of<32 * kWaves>(a, map, splits, &pl)) return;
    const Rows rw = rows_of(a.group);
    const int last_row = pl.rows - 1;
    const int w0 = pl.row0 + 32 * wave, w1 = w0 + 31 < last_row ? w0 + 31 : last_row;
    const Spread all = spread_of(a, pl, rw, pl.row0, pl.row0 + 32 * kWaves - 1 < last_row ? pl.row0 + 32 * kWaves - 1 : last_row);
    const bool idle = w0 > last_row;  // the wave has no rows: it copies only
    const Spread mine = idle ? all : spread_of(a, pl, rw, w0, w1);
    RowState<T, D> st;
    st.clear();
    const int r = w0 + (lane & 31);
    st.sp = r <= last_row ? span_of(a, pl.offset + rw.token(r), pl.kv.count) : Span{0, 0, 0};
    load_row<D>(st.q, a.q, a, pl, rw, r, lane);
    const TileList<ROWS> list(all);
    const int per = (list.count + splits - 1) / splits;
    const int from = pl.split * per, to = from + per < list.count ? from + per : list.count;
    const Keys<PAGED> keys(a, pl.seq, pl.kh, pl.kv);
    const float c = a.scale * kLog2e;
    TilePages<D, ROWS, kWaves, PAGED> pages, next;  // of the tile whose copies are next; one further
    TileCopy<D, ROWS, kWaves, PAGED> copies;
    if (from < to) {
        copies.set(keys, ROWS, wave, lane);
        pages.find(keys, list.tile(from), wave);
        copies.copy(keys, list.tile(from), pages, lds[0][0], lds[0][1], wave, lane);
    }
    unsigned long long holes = pages.holes;
    if (from + 1 < to) next.find(keys, list.tile(from + 1), wave);
    st.settle();
    for (int i = from; i < to; ++i) {
        const int buf = (i - from) & 1, t0 = list.tile(i);
        char(*now)[BYTES] = lds[buf], (*other)[BYTES] = lds[buf ^ 1];
        wait_copies<0>();
        // Values that are not finite matter where some row does not see all of the tile: zero times
        // them is not zero. Each wave looks at what it copied.
        const bool partial = holes || !all_see<ROWS>(all, t0);
        if (partial) found.wave[buf][wave] = clean_own<T, D, ROWS, kWaves>(now[1], wave, lane);
        __syncthreads();
        if (i + 1 < to) {
            pages = next;
            copies.copy(keys, list.tile(i + 1), pages, other[0], other[1], wave, lane);
            if (i + 2 < to) next.find(keys, list.tile(i + 2), wave);
        }
        const bool bad = partial && uniform(found.all(buf) != 0);
        if (!idle && !none_sees<ROWS>(mine, t0)) {
            st.template add<ROWS>(now[0], now[1], t0, c, holes || !all_see<ROWS>(mine, t0), holes, lane);
            if (bad) add_nonfinite<T, D>(st.o, st.sp, t0, keys.end(t0 + ROWS), holes, lane, [&](int j) { return keys.value(j); });
        }
        holes = pages.holes;
    }
    if (r > last_row) return;
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

template <typename T, int D, int WAVES, bool PAGED>
__global__ __launch_bounds__(64 * WAVES, 1) void attention_few_kernel(AttentionArgs a, BlockMap map, int splits) {
    constexpr int ROWS = 32, BYTES = ROWS * D * 2, COPIES = 2 * ROWS / Tile<D>::kRowsPerCopy;
    extern __shared__ __attribute__((aligned(1024))) char lds[];  // [wave][2][2][BYTES], then the join
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    Place pl;
    if (!place_of<32>(a, map, splits, &pl)) return;
    const Rows rw = rows_of(a.group);
    const int last_row = pl.rows - 1;
    const Spread all = spread_of(a, pl, rw, pl.row0, pl.row0 + 31 < last_row ? pl.row0 + 31 : last_row);
    RowState<T, D> st;
    st.clear();
    const int r = pl.row0 + (lane & 31);
    st.sp = r <= last_row ? span_of(a, pl.offset + rw.token(r), pl.kv.count) : Span{0, 0, 0};
    load_row<D>(st.q, a.q, a, pl, rw, r, lane);
    const TileList<ROWS> list(all);
    const int per = (list.count + splits - 1) / splits;
    const int from = pl.split * per, to = from + per < list.count ? from + per : list.count;
    const Keys<PAGED> keys(a, pl.seq, pl.kh, pl.kv);
    const float c = a.scale * kLog2e;
    char* own = lds + wave * 4 * BYTES;
    int n = 0;
    TilePages<D, ROWS, 1, PAGED> pages, next;
    TileCopy<D, ROWS, 1, PAGED> copies;
    if (from + wave < to) {
        copies.set(keys, ROWS, 0, lane);
        pages.find(keys, list.tile(from + wave), 0);
        copies.copy(keys, list.tile(from + wave), pages, own, own + BYTES, 0, lane);
    }
    unsigned long long holes = pages.holes;
    if (from + wave + WAVES < to) next.find(keys, list.tile(from + wave + WAVES), 0);
    st.settle();
    for (int i = from + wave; i < to; i += WAVES, ++n) {
        char *kt = own + (n & 1) * 2 * BYTES, *vt = kt + BYTES, *other = own + ((n + 1) & 1) * 2 * BYTES;
        const int t0 = list.tile(i);
        if (i + WAVES < to) {
            pages = next;
            copies.copy(keys, list.tile(i + WAVES), pages, other, other + BYTES, 0, lane);
            if (i + 2 * WAVES < to) next.find(keys, list.tile(i + 2 * WAVES), 0);
            wait_copies<COPIES>();
        } else {
            wait_copies<0>();
        }
        const bool whole = !holes && all_see<ROWS>(all, t0);
        const bool bad = !whole && clean_own<T, D, ROWS, 1>(vt, 0, lane);
        st.template add<ROWS>(kt, vt, t0, c, !whole, holes, lane);
        if (bad) add_nonfinite<T, D>(st.o, st.sp, t0, keys.end(t0 + ROWS), holes, lane, [&](int j) { return keys.value(j); });
        holes = pages.holes;
        wait_reads();  // the next copies go where this tile was
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
    if (pl.row0 + jr > last_row) return;
    float m = -INFINITY, sum = 0.f, w[WAVES];
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, mem[(i * 32 + jr) * LINE + D]);
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        w[i] = exp2f(mem[(i * 32 + jr) * LINE + D] - (m == -INFINITY ? 0.f : m));
        sum = fmaf(w[i], mem[(i * 32 + jr) * LINE + D + 1], sum);
    }
    const int tok = rw.token(pl.row0 + jr), head = pl.kh * a.group + (pl.row0 + jr - tok * a.group);
    const int64_t row = pl.q.first + tok, index = row * a.q_heads + head;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int at = part * 4; at < D; at += 4 * share) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const f32x4 v = *(const f32x4*)(mem + (i * 32 + jr) * LINE + at);
#pragma unroll
            for (int b = 0; b < 4; ++b) o[b] = fmaf(w[i], v[b], o[b]);
        }
        const float four[4] = {o[0], o[1], o[2], o[3]};
        store_row4<T, D>(a, pl, index, row, head, at, four, inv);
    }
    if (part == 0) store_sums<D>(a, pl, index, m, sum, kLift<T>);
}

// Row blocks, and over how many workgroups each one's key tiles are split.
struct Plan {
    bool few;
    int waves, blocks, splits;
};
Plan plan_of(int dim, int sequences, int kv_heads, int group, int max_q, int max_kv, int frame, int back, int sinks) {
    Plan p;
    const int64_t rows = (int64_t)max_q * group, wide = (rows + 127) / 128 * kv_heads * sequences;
    // Keys that one block of `block` rows sees at most.
    const auto keys_of = [&](int block, int tile) { return attention_keys(max_kv, frame, back, sinks, block / group, tile); };
    const int64_t keys = keys_of(128, 64);
    // Few rows, or so few workgroups of 128 rows that 32-row ones with four (eight) waves on the keys
    // are done sooner, though each key tile is read four times as often (256 x 128 rows, 64
    // channels: 29.9 -> 21.5 us; 64 x 128 rows of 8,000 keys, 128 channels: 59 -> 103).
    p.few = rows <= 32 || (dim == 64 ? wide <= 256 && keys <= 4096 : wide <= 128 && keys <= 2048);
    const int per_block = p.few ? 32 : 128, tile = p.few ? 32 : 64;
    p.blocks = (int)((rows + per_block - 1) / per_block);
    const int64_t tiles = (keys_of(per_block, tile) + tile - 1) / tile, groups = (int64_t)p.blocks * kv_heads * sequences;
    p.waves = p.few && dim == 64 && groups <= 256 ? 8 : 4;
    // Blocks that leave half of the CUs idle or more split their tiles: until every CU has as many
    // workgroups as its LDS takes (one of the few kernel's with 128 channels, else two), a tile a
    // wave (tile kernel: four) being the least, and 32 parts the most that the join adds quickly.
    // Up to four tiles a wave the join would cost more than it saves: one token of 777 keys, 8
    // heads of 64: 8.9 us in one part, 9.7 in three; of 1,500 keys 12.8 and 10.0.
    const int64_t least = p.few ? p.waves : 4, room = p.few && dim == 128 ? 256 : 512;
    int64_t splits = 1;
    if (groups > 0 && groups <= 128 && tiles > 4 * least) {
        splits = (room + groups - 1) / groups;
        splits = splits < tiles / least ? splits : tiles / least;
        splits = splits < 32 ? splits : 32;
    }
    p.splits = (int)splits;
    return p;
}

template <typename T, int D, int WAVES, bool PAGED>
hipError_t run_few(const AttentionArgs& a, const Plan& p, const BlockMap& map, hipStream_t stream) {
    constexpr int copies = WAVES * 4 * 32 * D * 2, join = WAVES * 32 * (D + 4) * 4;
    constexpr int bytes = copies > join ? copies : join;
    if (hipError_t e = allow_dynamic_lds((const void*)attention_few_kernel<T, D, WAVES, PAGED>, bytes)) return e;
    attention_few_kernel<T, D, WAVES, PAGED><<<map.grid, 64 * WAVES, bytes, stream>>>(a, map, p.splits);
    return hipGetLastError();
}

template <typename T, int D, bool PAGED>
hipError_t run(const AttentionArgs& a, const Plan& p, hipStream_t stream) {
    BlockMap map;
    if (!block_map((int64_t)p.blocks * p.splits, a.kv_heads, a.sequences, &map)) return hipErrorInvalidConfiguration;
    if (p.few) {
        if (hipError_t e = p.waves == 8 ? run_few<T, D, D == 64 ? 8 : 4, PAGED>(a, p, map, stream)
                                                   : run_few<T, D, 4, PAGED>(a, p, map, stream))
            return e;
    } else {
        attention_tile_kernel<T, D, PAGED><<<map.grid, kThreads, 0, stream>>>(a, map, p.splits);
    }
    if (hipError_t e = hipGetLastError()) return e;
    if (p.splits == 1) return hipSuccess;
    const int64_t rows = (int64_t)a.max_q * a.q_heads;
    if (p.splits <= 8)
        attention_join_kernel<T, D, 1><<<dim3((unsigned)((rows + kWaves - 1) / kWaves), 1, a.sequences), kThreads, 0, stream>>>(a, p.splits);
    else
        attention_join_kernel<T, D, kWaves><<<dim3((unsigned)rows, 1, a.sequences), kThreads, 0, stream>>>(a, p.splits);
    return hipGetLastError();
}

template <typename T, int D>
hipError_t by_keys(const AttentionArgs& a, const Plan& p, hipStream_t stream) {
    return a.pages.table ? run<T, D, true>(a, p, stream) : run<T, D, false>(a, p, stream);
}
template <typename T>
hipError_t by_dim(const AttentionArgs& a, const Plan& p, hipStream_t stream) {
    return a.dim == 64 ? by_keys<T, 64>(a, p, stream) : by_keys<T, 128>(a, p, stream);
}

}  // namespace
}  // namespace fa

size_t attention_forward_workspace(const dcn_attention_shape& s) {
    const fa::Plan p = fa::plan_of(s.head_dim, s.sequences, s.kv_heads, s.q_heads / s.kv_heads, s.max_q, s.max_kv, s.frame_tokens, s.back, s.sinks);
    return p.splits == 1 ? 0 : (size_t)s.q_tokens * s.q_heads * p.splits * (s.head_dim + 4) * sizeof(float);
}

hipError_t launch_attention_matrix(int dtype, const AttentionArgs& a, hipStream_t stream) {
    const fa::Plan p = fa::plan_of(a.dim, a.sequences, a.kv_heads, a.group, a.max_q, a.max_kv, a.frame, a.back, a.sinks);
    return dtype == DCN_DTYPE_F16 ? fa::by_dim<_Float16>(a, p, stream) : fa::by_dim<fa::bf16>(a, p, stream);
}

}  // namespace dcn
