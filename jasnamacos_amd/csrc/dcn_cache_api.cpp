// C-ABI host layer of the microscaled cache (append, read back) and of the attention over it
// and over prefixes that sequences share. Checks every size, stride and pointer that a kernel relies on,
// then launches; nothing here allocates or synchronises.
#include "dcn_attention_host.hpp"

using namespace dcn::host;

namespace {

// The sizes of a cache and how it holds them; as_is: pages of the dtype are taken too.
dcn_status check_pages(dcn_context* ctx, const dcn_pages* p, bool as_is, dcn::PagesArgs* pages, dcn::MxArgs* mx) {
    DCN_TRY(check_cache(ctx, &p->cache, pages));
    REQUIRE_SHAPE(p->bits == 8 || p->bits == 4 || (as_is && p->bits == 0),
                  "pages of " + std::to_string(p->bits) + " bits: microscaled ones have 8 or 4");
    REQUIRE_SHAPE(p->reserved == 0, "pages reserved must be 0");
    REQUIRE_SHAPE(!p->bits || p->cache.head_dim % 32 == 0, "a microscaled cache needs a head_dim of whole blocks of 32");
    *mx = dcn::MxArgs{p->bits, p->cache.kv_heads, p->cache.head_dim, (uint8_t*)p->k, (uint8_t*)p->v, (uint8_t*)p->k_scales, (uint8_t*)p->v_scales};
    return DCN_OK;
}

dcn_status check_aligned(dcn_context* ctx, const char* name, const void* p, size_t to) {
    if (!p) return null_fail(ctx, name);
    if ((uintptr_t)p % to)
        return fail(ctx, DCN_INVALID_ARGUMENT, std::string(name) + " is not aligned to " + std::to_string(to) + " bytes");
    return DCN_OK;
}

// The buffers of a cache.
dcn_status check_buffers(dcn_context* ctx, const dcn_pages* p) {
    if (!p->bits) {
        DCN_TRY(check_pointer(ctx, "k_pages", p->k, p->cache.dtype));
        return check_pointer(ctx, "v_pages", p->v, p->cache.dtype);
    }
    DCN_TRY(check_aligned(ctx, "k codes", p->k, 16));
    DCN_TRY(check_aligned(ctx, "v codes", p->v, 16));
    DCN_TRY(check_aligned(ctx, "k_scales", p->k_scales, 4));
    return check_aligned(ctx, "v_scales", p->v_scales, 4);
}

// The sizes of an attention call, after which p has everything but the pointers.
dcn_status check_call(dcn_context* ctx, const dcn_attention_shape* shape, const dcn_pages* pages, const dcn_prefix* prefix,
                      dcn::PagesAttention* p) {
    DCN_TRY(check_pages(ctx, pages, prefix != nullptr, &p->a.pages, &p->mx));
    DCN_TRY(check_attention(ctx, shape, true, &p->a));
    const dcn_cache& c = pages->cache;
    REQUIRE_SHAPE(c.dtype == shape->dtype && c.kv_heads == shape->kv_heads && c.head_dim == shape->head_dim,
                  "attention and cache have different types, key heads or head sizes");
    p->prefix = p->a.pages;
    p->prefix.table = nullptr;
    p->prefix.width = 0;
    // The kernels' tiles end up to 64 keys past the last.
    REQUIRE_SHAPE((!prefix || prefix->width >= 0) && ((int64_t)(prefix ? prefix->width : 0) + c.table_width) * c.page_tokens <= INT32_MAX - 63,
                  "(prefix width + table_width) * page_tokens must be below 2^31 - 63");
    if (prefix) {
        REQUIRE_SHAPE(prefix->max_tokens >= 0 && prefix->max_tokens <= (int64_t)prefix->width * c.page_tokens,
                      "prefix max_tokens must be 0..width * page_tokens");
        p->prefix.width = prefix->width;
        p->max_prefix = prefix->max_tokens;
    }
    return DCN_OK;
}

// Whether the matrix kernels take a call of these sizes: as in the paged call, and rows of all sequences
// and of the pool that an int counts.
bool matrix_call(const dcn_attention_shape* s, const dcn_pages* p) {
    // By division: the products of sizes that no memory has may pass 64 bits.
    return matrix_heads(s) && matrix_pool(&p->cache) &&
           (!p->bits || (int64_t)p->cache.pages * p->cache.page_tokens <= INT32_MAX / p->cache.kv_heads) &&
           s->q_tokens <= (INT32_MAX - 257) / (s->q_heads / s->kv_heads);
}
size_t workspace_of(const dcn_attention_shape* s, const dcn_pages* pages, const dcn::PagesAttention& p) {
    return matrix_call(s, pages) ? dcn::attention_pages_workspace(*s, pages->bits, p.max_prefix)
                                 : dcn::attention_pages_any_workspace(*s, p.max_prefix);
}

}  // namespace

extern "C" {

dcn_status dcn_cache_append_mx_dev(dcn_context* ctx, const dcn_pages* pages, const dcn_append_shape* shape,
                                   const dcn_rotary* rotary, const void* d_q, const void* d_k, const void* d_v,
                                   const int32_t* d_positions, const float* d_freq, const int32_t* d_cu_q,
                                   const int32_t* d_kv_lens, const int32_t* d_table, void* d_q_out, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        REQUIRE_POINTER(pages);
        REQUIRE_POINTER(shape);
        const dcn_cache* cache = &pages->cache;
        dcn::AppendArgs a{};
        dcn::MxArgs mx;
        DCN_TRY(check_pages(ctx, pages, false, &a.pages, &mx));
        dcn::RotaryArgs r{};
        r.dim = cache->head_dim;
        DCN_TRY(check_append(ctx, cache, shape, rotary, d_q != nullptr, &r));
        if (!shape->tokens || !shape->sequences) return DCN_OK;
        DCN_TRY(check_append_pointers(ctx, cache, shape, r, d_q, d_k, d_v, d_positions, d_freq, d_cu_q, d_kv_lens, d_table, d_q_out));
        if (d_q && d_q == d_q_out) return fail(ctx, DCN_INVALID_ARGUMENT, "q_out is q: an append of this kind does not turn in place");
        // Workgroups read rows that others may have written by then.
        const auto meets = [&](const void* in, const int64_t* strides, int heads) {
            return rows_meet(in, strides, heads, d_q_out, shape->q_out_stride, shape->q_heads, shape->tokens, r.dim, size_of(cache->dtype));
        };
        if (d_q && (meets(d_q, shape->q_stride, shape->q_heads) || meets(d_k, shape->k_stride, cache->kv_heads) ||
                    meets(d_v, shape->v_stride, cache->kv_heads)))
            return fail(ctx, DCN_INVALID_ARGUMENT, "q_out lies on q, k or v, or among their rows with other strides");
        DCN_TRY(check_buffers(ctx, pages));
        fill_append(&a, &r, cache, shape, d_q, d_k, d_v, d_positions, d_freq, d_cu_q, d_kv_lens, d_table, d_q_out);
        DCN_HIP(ctx, dcn::launch_append_mx(cache->dtype, a, mx, r, (hipStream_t)stream));
        return DCN_OK;
    });
}

dcn_status dcn_cache_read_dev(dcn_context* ctx, const dcn_pages* pages, const dcn_read_shape* shape, const int32_t* d_cu,
                              const int32_t* d_kv_lens, const int32_t* d_table, void* d_k_out, void* d_v_out, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        REQUIRE_POINTER(pages);
        REQUIRE_POINTER(shape);
        const dcn_cache* cache = &pages->cache;
        dcn::ReadArgs a{};
        dcn::MxArgs mx;
        DCN_TRY(check_pages(ctx, pages, false, &a.pages, &mx));
        REQUIRE_SHAPE(shape->reserved == 0, "read reserved must be 0");
        REQUIRE_SHAPE(shape->sequences >= 0 && shape->tokens >= 0 && shape->tokens <= INT32_MAX,
                      "read sequences and tokens must be 0..2^31-1");
        DCN_TRY(check_out_strides(ctx, "k_out", shape->k_stride, shape->tokens, cache->kv_heads, cache->head_dim));
        DCN_TRY(check_out_strides(ctx, "v_out", shape->v_stride, shape->tokens, cache->kv_heads, cache->head_dim));
        if (!shape->tokens || !shape->sequences) return DCN_OK;
        DCN_TRY(check_buffers(ctx, pages));
        DCN_TRY(check_pointer(ctx, "cu", d_cu, DCN_DTYPE_F32));
        DCN_TRY(check_pointer(ctx, "kv_lens", d_kv_lens, DCN_DTYPE_F32));
        DCN_TRY(check_pointer(ctx, "table", d_table, DCN_DTYPE_F32));
        DCN_TRY(check_pointer(ctx, "k_out", d_k_out, cache->dtype));
        DCN_TRY(check_pointer(ctx, "v_out", d_v_out, cache->dtype));
        a.sequences = shape->sequences;
        a.tokens = shape->tokens;
        a.cu = d_cu;
        a.kv_lens = d_kv_lens;
        a.pages.table = d_table;
        a.k = {d_k_out, shape->k_stride[0], shape->k_stride[1]};
        a.v = {d_v_out, shape->v_stride[0], shape->v_stride[1]};
        DCN_HIP(ctx, dcn::launch_cache_read(cache->dtype, a, mx, (hipStream_t)stream));
        return DCN_OK;
    });
}

size_t dcn_attention_pages_workspace_bytes(const dcn_attention_shape* shape, const dcn_pages* pages, const dcn_prefix* prefix) {
    dcn::PagesAttention p{};
    try {
        if (!shape || !pages) return 0;
        const dcn_attention_shape s = fitted(*shape, true);
        if (check_call(nullptr, &s, pages, prefix, &p) != DCN_OK) return 0;
        return workspace_of(&s, pages, p);
    } catch (const std::exception&) {
        return 0;
    }
}

dcn_status dcn_attention_pages_dev(dcn_context* ctx, const dcn_attention_shape* given, const dcn_pages* pages,
                                   const dcn_prefix* prefix, const void* d_q, const int32_t* d_cu_q,
                                   const int32_t* d_kv_lens, const int32_t* d_table, void* d_out, float* d_lse,
                                   void* d_workspace, size_t workspace_bytes, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        if (!given) return null_fail(ctx, "shape");
        REQUIRE_POINTER(pages);
        REQUIRE_SHAPE(d_cu_q || (int64_t)given->sequences * given->max_q <= given->q_tokens,
                      "sequences * max_q exceeds q_tokens");
        const dcn_attention_shape own = fitted(*given, true), *shape = &own;
        dcn::PagesAttention p{};
        DCN_TRY(check_call(ctx, shape, pages, prefix, &p));
        DCN_TRY(check_out_strides(ctx, "out", shape->out_stride, shape->q_tokens, shape->q_heads, shape->head_dim));
        if (!shape->sequences || !shape->max_q || !shape->q_tokens) return DCN_OK;
        DCN_TRY(check_buffers(ctx, pages));
        DCN_TRY(check_pointer(ctx, "q", d_q, shape->dtype));
        DCN_TRY(check_pointer(ctx, "out", d_out, shape->dtype));
        DCN_TRY(check_pointer(ctx, "kv_lens", d_kv_lens, DCN_DTYPE_F32));
        DCN_TRY(check_pointer(ctx, "table", d_table, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "lse", d_lse, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "cu_q", d_cu_q, DCN_DTYPE_F32));
        DCN_TRY(check_workspace(ctx, d_workspace, workspace_bytes, workspace_of(shape, pages, p)));
        const bool shared = prefix && prefix->max_tokens;
        if (shared) {
            DCN_TRY(check_pointer(ctx, "prefix table", prefix->table, DCN_DTYPE_F32));
            DCN_TRY(check_pointer(ctx, "prefix tokens", prefix->tokens, DCN_DTYPE_F32));
        }
        const int64_t ts = (int64_t)pages->cache.kv_heads * pages->cache.head_dim;
        p.a.q.p = d_q;
        p.a.k = {pages->k, ts, pages->cache.head_dim};
        p.a.v = {pages->v, ts, pages->cache.head_dim};
        p.a.out.p = d_out;
        p.a.lse = d_lse;
        p.a.cu_q = d_cu_q;
        p.a.cu_kv = d_kv_lens;
        p.a.pages.table = d_table;
        p.prefix.table = shared ? prefix->table : nullptr;
        p.prefix_len = shared ? prefix->tokens : nullptr;
        p.a.workspace = d_workspace;
        // Tensors that keep a call of the matrix kernels' sizes from them have no room for the others' parts.
        p.a.any_splits = matrix_call(shape, pages) ? 1 : dcn::attention_pages_any_splits(*shape, p.max_prefix);
        const bool matrix = matrix_call(shape, pages) && matrix_tensor(p.a.q) && matrix_tensor(p.a.out) &&
                            (pages->bits || (matrix_tensor(p.a.k) && matrix_tensor(p.a.v)));
        DCN_HIP(ctx, (matrix ? dcn::launch_attention_pages : dcn::launch_attention_pages_any)(shape->dtype, p, (hipStream_t)stream));
        return DCN_OK;
    });
}

}  // extern "C"
