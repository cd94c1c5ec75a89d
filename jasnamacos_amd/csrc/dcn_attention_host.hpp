// Host-side checks shared by the C entries of the frame-attention operators.
#pragma once

#include <cmath>
#include <exception>
#include <string>

#include "dcn_attention.hpp"
#include "dcn_host.hpp"
#include "dcn_internal.hpp"

namespace dcn {
namespace host {

// Runs an entry point's body: a null context and C++ exceptions become a status.
template <typename F>
inline dcn_status entry(dcn_context* ctx, F body) noexcept {
    if (!ctx) return DCN_INVALID_ARGUMENT;
    try {
        DeviceGuard guard(ctx->device);
        return body();
    } catch (const std::exception&) {
        return DCN_COMMAND_FAILED;
    }
}

inline dcn_status shape_fail(dcn_context* ctx, const std::string& what) { return fail(ctx, DCN_INVALID_SHAPE, what); }
inline dcn_status null_fail(dcn_context* ctx, const char* what) {
    return fail(ctx, DCN_INVALID_ARGUMENT, std::string(what) + " is null");
}

#define REQUIRE_SHAPE(cond, what) \
    if (!(cond)) return shape_fail(ctx, what)
#define REQUIRE_POINTER(p) \
    if (!(p)) return null_fail(ctx, #p)

inline bool known_dtype(int dtype) { return dtype >= DCN_DTYPE_F16 && dtype <= DCN_DTYPE_F32; }
inline int size_of(int dtype) { return dtype == DCN_DTYPE_F32 ? 4 : 2; }

// A pointer the kernels take as elements of this type.
inline dcn_status check_pointer(dcn_context* ctx, const char* name, const void* p, int dtype) {
    if (!p) return null_fail(ctx, name);
    if ((uintptr_t)p % size_of(dtype))
        return fail(ctx, DCN_INVALID_ARGUMENT, std::string(name) + " is not aligned to its type");
    return DCN_OK;
}

// One that may be null.
inline dcn_status check_optional(dcn_context* ctx, const char* name, const void* p, int dtype) {
    return p ? check_pointer(ctx, name, p, dtype) : DCN_OK;
}

constexpr int kMaxHeads = 65535;        // grid.y
constexpr int kMaxSequences = 65535;    // grid.z
constexpr int64_t kMaxStride = INT64_C(1) << 40;

inline dcn_status check_strides(dcn_context* ctx, const char* name, const int64_t* s) {
    REQUIRE_SHAPE(s[0] >= 0 && s[1] >= 0 && s[0] < kMaxStride && s[1] < kMaxStride,
                  std::string(name) + " strides must be in [0, 2^40)");
    return DCN_OK;
}
// An output's rows must not lie on each other.
inline dcn_status check_out_strides(dcn_context* ctx, const char* name, const int64_t* s, int64_t tokens, int heads, int dim) {
    DCN_TRY(check_strides(ctx, name, s));
    const bool rows = tokens <= 1 || s[0] >= (heads > 1 && s[0] >= s[1] ? (heads - 1) * s[1] + dim : dim);
    const bool across = heads <= 1 || s[1] >= (tokens > 1 && s[1] > s[0] ? (tokens - 1) * s[0] + dim : dim);
    REQUIRE_SHAPE(rows && across, std::string(name) + " rows overlap");
    return DCN_OK;
}

// Whether an output's rows lie on an input's ([tokens][heads][dim] each, on their element size): exact where both have
// the same strides; among rows of other strides they are taken to.
inline bool rows_meet(const void* in, const int64_t* in_s, int in_heads, const void* out, const int64_t* out_s, int out_heads, int64_t tokens,
                      int dim, int size) {
    typedef __int128 wide;  // a stride has 40 bits, a count 31
    const auto last = [&](const int64_t* s, int heads) { return (wide)(tokens - 1) * s[0] + (wide)(heads - 1) * s[1] + dim; };
    const wide apart = ((wide)(uintptr_t)out - (wide)(uintptr_t)in) / size;
    if (apart >= last(in_s, in_heads) || -apart >= last(out_s, out_heads)) return false;
    if ((tokens > 1 && in_s[0] != out_s[0]) || ((in_heads > 1 || out_heads > 1) && in_s[1] != out_s[1])) return true;
    // Row i, head h of the output is at apart + (i - j) ts + (h - g) hs from row j, head g of the input.
    const wide ts = tokens > 1 ? in_s[0] : 0;
    for (int64_t heads = 1 - (int64_t)in_heads; heads < out_heads; ++heads) {
        const wide from = apart + heads * (wide)in_s[1];
        wide rows = ts ? -from / ts : 0;  // the nearest are this one and its neighbours
        rows = rows > tokens - 1 ? tokens - 1 : (rows < 1 - tokens ? 1 - tokens : rows);
        for (wide r = rows - 1; r <= rows + 1; ++r) {
            const wide at = from + r * ts;
            if (r > -tokens && r < tokens && at < dim && -at < dim) return true;
        }
    }
    return false;
}

inline dcn_status check_rotary(dcn_context* ctx, const dcn_rotary* r, dcn::RotaryArgs* out) {
    REQUIRE_SHAPE(known_dtype(r->dtype), "rotary dtype " + std::to_string(r->dtype) + " is unknown");
    REQUIRE_SHAPE(r->head_dim >= 1 && r->head_dim <= 65536, "rotary head_dim must be 1..65536");
    int64_t sum = 0;
    for (int p : r->pairs) {
        REQUIRE_SHAPE(p >= 0, "rotary pairs must not be negative");
        sum += p;
    }
    REQUIRE_SHAPE(2 * sum <= r->head_dim, "rotary pairs exceed head_dim / 2");
    out->dim = r->head_dim;
    out->st = r->pairs[0];
    out->sh = r->pairs[0] + r->pairs[1];
    out->pairs = (int)sum;
    out->interleaved = r->interleaved != 0;
    out->sign = 1.f;
    out->positions = nullptr;
    out->freq = nullptr;
    return DCN_OK;
}

inline dcn_status check_cache(dcn_context* ctx, const dcn_cache* c, dcn::PagesArgs* out) {
    REQUIRE_SHAPE(known_dtype(c->dtype), "cache dtype " + std::to_string(c->dtype) + " is unknown");
    REQUIRE_SHAPE(c->pages >= 1 && c->table_width >= 1 && c->kv_heads >= 1 && c->kv_heads <= kMaxHeads &&
                      c->head_dim >= 1 && c->head_dim <= 65536,
                  "cache sizes must be positive (heads up to 65535, head_dim up to 65536)");
    REQUIRE_SHAPE(c->page_tokens >= 1 && (c->page_tokens & (c->page_tokens - 1)) == 0,
                  "page_tokens must be a power of two");
    REQUIRE_SHAPE((int64_t)c->table_width * c->page_tokens <= INT32_MAX, "table_width * page_tokens must be below 2^31");
    out->pages = c->pages;
    out->width = c->table_width;
    out->shift = 0;
    while ((1 << out->shift) < c->page_tokens) ++out->shift;
    return DCN_OK;
}

// The sizes of an append.
inline dcn_status check_append(dcn_context* ctx, const dcn_cache* cache, const dcn_append_shape* shape, const dcn_rotary* rotary,
                               bool has_q, dcn::RotaryArgs* r) {
    if (rotary) {
        DCN_TRY(check_rotary(ctx, rotary, r));
        REQUIRE_SHAPE(rotary->dtype == cache->dtype && rotary->head_dim == cache->head_dim,
                      "rotary and cache have different types or head sizes");
    }
    REQUIRE_SHAPE(shape->sequences >= 0 && shape->tokens >= 0 && shape->tokens <= INT32_MAX,
                  "append sequences and tokens must be 0..2^31-1");
    REQUIRE_SHAPE(!has_q || (shape->q_heads >= 1 && shape->q_heads <= kMaxHeads), "q_heads must be 1..65535");
    DCN_TRY(check_strides(ctx, "k", shape->k_stride));
    DCN_TRY(check_strides(ctx, "v", shape->v_stride));
    if (has_q) {
        DCN_TRY(check_strides(ctx, "q", shape->q_stride));
        DCN_TRY(check_out_strides(ctx, "q_out", shape->q_out_stride, shape->tokens, shape->q_heads, r->dim));
    }
    return DCN_OK;
}
// Its pointers, but for the cache's buffers.
inline dcn_status check_append_pointers(dcn_context* ctx, const dcn_cache* cache, const dcn_append_shape* shape,
                                        const dcn::RotaryArgs& r, const void* d_q, const void* d_k, const void* d_v,
                                        const int32_t* d_positions, const float* d_freq, const int32_t* d_cu_q,
                                        const int32_t* d_kv_lens, const int32_t* d_table, const void* d_q_out) {
    if (d_q) {
        DCN_TRY(check_pointer(ctx, "q", d_q, cache->dtype));
        DCN_TRY(check_pointer(ctx, "q_out", d_q_out, cache->dtype));
        if (d_q == d_q_out && (shape->q_stride[0] != shape->q_out_stride[0] || shape->q_stride[1] != shape->q_out_stride[1]))
            return fail(ctx, DCN_INVALID_ARGUMENT, "q_out is q with other strides");
    }
    DCN_TRY(check_pointer(ctx, "k", d_k, cache->dtype));
    DCN_TRY(check_pointer(ctx, "v", d_v, cache->dtype));
    DCN_TRY(check_pointer(ctx, "cu_q", d_cu_q, DCN_DTYPE_F32));
    DCN_TRY(check_pointer(ctx, "kv_lens", d_kv_lens, DCN_DTYPE_F32));
    DCN_TRY(check_pointer(ctx, "table", d_table, DCN_DTYPE_F32));
    if (r.pairs) {
        DCN_TRY(check_pointer(ctx, "positions", d_positions, DCN_DTYPE_F32));
        DCN_TRY(check_pointer(ctx, "freq", d_freq, DCN_DTYPE_F32));
    }
    return DCN_OK;
}
inline void fill_append(dcn::AppendArgs* a, dcn::RotaryArgs* r, const dcn_cache* cache, const dcn_append_shape* shape, const void* d_q,
                        const void* d_k, const void* d_v, const int32_t* d_positions, const float* d_freq, const int32_t* d_cu_q,
                        const int32_t* d_kv_lens, const int32_t* d_table, void* d_q_out) {
    r->positions = d_positions;
    r->freq = d_freq;
    a->sequences = shape->sequences;
    a->q_heads = shape->q_heads;
    a->kv_heads = cache->kv_heads;
    a->tokens = shape->tokens;
    a->q = {d_q, shape->q_stride[0], shape->q_stride[1]};
    a->k = {d_k, shape->k_stride[0], shape->k_stride[1]};
    a->v = {d_v, shape->v_stride[0], shape->v_stride[1]};
    a->q_out = {d_q ? d_q_out : nullptr, shape->q_out_stride[0], shape->q_out_stride[1]};
    a->cu_q = d_cu_q;
    a->kv_lens = d_kv_lens;
    a->pages.table = d_table;
}

// The bounds of the sequences' lengths are not above the rows that there are: plans and launches are
// made for lengths that occur. (The paged call's keys are bounded by its table, in the kernels.)
inline dcn_attention_shape fitted(const dcn_attention_shape& shape, bool paged) {
    dcn_attention_shape s = shape;
    if (s.q_tokens >= 0 && s.max_q > s.q_tokens) s.max_q = (int32_t)s.q_tokens;
    if (!paged && s.kv_tokens >= 0 && s.max_kv > s.kv_tokens) s.max_kv = (int32_t)s.kv_tokens;
    return s;
}

// The sizes, spans and strides of one attention call; pointers come later.
inline dcn_status check_attention(dcn_context* ctx, const dcn_attention_shape* s, bool paged, dcn::AttentionArgs* a) {
    REQUIRE_SHAPE(known_dtype(s->dtype), "attention dtype " + std::to_string(s->dtype) + " is unknown");
    REQUIRE_SHAPE(s->sequences >= 0 && s->sequences <= kMaxSequences, "sequences must be 0..65535");
    REQUIRE_SHAPE(s->q_heads >= 1 && s->kv_heads >= 1 && s->q_heads <= kMaxHeads && s->q_heads % s->kv_heads == 0,
                  "q_heads must be a positive multiple of kv_heads, up to 65535");
    REQUIRE_SHAPE(s->head_dim >= 1 && s->head_dim <= DCN_ATTENTION_MAX_HEAD_DIM, "attention head_dim must be 1..256");
    REQUIRE_SHAPE(s->frame_tokens >= 1, "frame_tokens must be positive");
    REQUIRE_SHAPE(s->sinks >= 0, "sinks must not be negative");
    REQUIRE_SHAPE(s->max_q >= 0 && s->max_kv >= 0, "max_q and max_kv must not be negative");
    REQUIRE_SHAPE(s->q_tokens >= 0 && s->kv_tokens >= 0, "q_tokens and kv_tokens must not be negative");
    REQUIRE_SHAPE(std::isfinite(s->scale), "scale must be finite");
    // Packed rows are counted by an int.
    REQUIRE_SHAPE((int64_t)s->max_q * (s->q_heads / s->kv_heads) < INT32_MAX - 256,
                  "max_q times the heads that share a key head must be below 2^31 - 256");
    a->sequences = s->sequences;
    a->q_heads = s->q_heads;
    a->kv_heads = s->kv_heads;
    a->dim = s->head_dim;
    a->group = s->q_heads / s->kv_heads;
    a->frame = s->frame_tokens;
    a->back = s->back;
    a->ahead = s->ahead;
    a->sinks = s->sinks;
    a->max_q = s->max_q;
    a->max_kv = s->max_kv;
    a->scale = s->scale;
    a->q_tokens = s->q_tokens;
    a->kv_tokens = s->kv_tokens;
    DCN_TRY(check_strides(ctx, "q", s->q_stride));
    if (!paged) {
        DCN_TRY(check_strides(ctx, "k", s->k_stride));
        DCN_TRY(check_strides(ctx, "v", s->v_stride));
    }
    a->q = {nullptr, s->q_stride[0], s->q_stride[1]};
    a->k = {nullptr, s->k_stride[0], s->k_stride[1]};
    a->v = {nullptr, s->v_stride[0], s->v_stride[1]};
    a->out = {nullptr, s->out_stride[0], s->out_stride[1]};
    return DCN_OK;
}

// Without index arrays the sequences are max_q (max_kv) rows each.
inline dcn_status check_even(dcn_context* ctx, const dcn_attention_shape* s, const void* cu_q, const void* cu_kv) {
    REQUIRE_SHAPE(cu_q || (int64_t)s->sequences * s->max_q <= s->q_tokens, "sequences * max_q exceeds q_tokens");
    REQUIRE_SHAPE(cu_kv || (int64_t)s->sequences * s->max_kv <= s->kv_tokens, "sequences * max_kv exceeds kv_tokens");
    return DCN_OK;
}

// Whether the 16-bit matrix kernels take heads of this kind: 64 or 128 channels, and a scale that
// keeps the order of the scores. The kernels of any type take the rest, and tensors that are not
// aligned to 16 bytes.
inline bool matrix_heads(const dcn_attention_shape* s) {
    return s->dtype != DCN_DTYPE_F32 && (s->head_dim == 64 || s->head_dim == 128) && s->scale > 0.f;
}
// 16-byte rows, and the rows of one tile (64 tokens, the heads of a group) within 32-bit offsets.
template <typename H>
inline bool matrix_tensor(const H& h, int group = 1) {
    return (uintptr_t)h.p % 16 == 0 && h.ts % 8 == 0 && h.hs % 8 == 0 && h.ts < (INT64_C(1) << 24) &&
           (group - 1) * h.hs < (INT64_C(1) << 29);
}
// Pages of whole runs of 8 keys, and rows of the pool that an int counts.
inline bool matrix_pool(const dcn_cache* c) { return c->page_tokens >= 8 && (int64_t)c->pages * c->page_tokens <= INT32_MAX; }

inline dcn_status check_workspace(dcn_context* ctx, const void* p, size_t have, size_t need) {
    if (!need) return DCN_OK;
    REQUIRE_POINTER(p);
    if ((uintptr_t)p % 16) return fail(ctx, DCN_INVALID_ARGUMENT, "workspace is not aligned to 16 bytes");
    if (have < need)
        return fail(ctx, DCN_INVALID_ARRAY_COUNT,
                    "workspace has " + std::to_string(have) + " bytes; expected " + std::to_string(need));
    return DCN_OK;
}

}  // namespace host
}  // namespace dcn
