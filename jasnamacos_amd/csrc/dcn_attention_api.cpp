// C-ABI host layer of the frame-attention operators: rotary positions, the paged cache's
// append, windowed attention and the gated norms. Checks every size, stride and pointer that
// a kernel relies on, then launches; nothing here allocates or synchronises.
#include "dcn_attention_host.hpp"

using namespace dcn::host;

namespace {

size_t attention_workspace(const dcn_attention_shape* s, int pass) {
    if (pass == DCN_ATTENTION_BACKWARD)  // the rows' delta at least
        return matrix_heads(s) ? dcn::attention_backward_workspace(*s) : (size_t)s->q_tokens * s->q_heads * sizeof(float);
    return matrix_heads(s) ? dcn::attention_forward_workspace(*s) : dcn::attention_any_workspace(*s);
}

// The workspace of heads that the matrix kernels take is for their parts, whichever kernel runs.
int any_splits(const dcn_attention_shape* s) { return matrix_heads(s) ? 1 : dcn::attention_any_splits(*s); }

dcn_status check_low(dcn_context* ctx, const void* low) {
    if ((uintptr_t)low % 16) return fail(ctx, DCN_INVALID_ARGUMENT, "low is not aligned to 16 bytes");
    return DCN_OK;
}

dcn_status check_norm(dcn_context* ctx, const dcn_norm_shape* s, dcn::NormArgs* a) {
    REQUIRE_SHAPE(known_dtype(s->dtype), "norm dtype " + std::to_string(s->dtype) + " is unknown");
    REQUIRE_SHAPE(s->channels >= 1 && s->channels <= DCN_NORM_MAX_CHANNELS, "norm channels must be 1..8192");
    REQUIRE_SHAPE(s->tokens >= 0 && s->tokens <= INT32_MAX, "norm tokens must be 0..2^31-1");
    REQUIRE_SHAPE(s->gate_tokens >= 1, "gate_tokens must be positive");
    REQUIRE_SHAPE(s->eps >= 0.f && std::isfinite(s->eps) && std::isfinite(s->residual_scale),
                  "eps must be finite and not negative, residual_scale finite");
    *a = dcn::NormArgs{};
    a->channels = s->channels;
    a->tokens = s->tokens;
    a->gate_tokens = s->gate_tokens < s->tokens ? s->gate_tokens : s->tokens;
    a->alpha = s->residual_scale;
    a->eps = s->eps;
    return DCN_OK;
}

}  // namespace

extern "C" {

dcn_status dcn_rotary_dev(dcn_context* ctx, const dcn_rotary* rotary, int64_t tokens, int heads, const void* d_x,
                          int64_t x_token_stride, int64_t x_head_stride, const int32_t* d_positions,
                          const float* d_freq, int inverse, void* d_out, int64_t out_token_stride,
                          int64_t out_head_stride, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        REQUIRE_POINTER(rotary);
        dcn::RotaryArgs r;
        DCN_TRY(check_rotary(ctx, rotary, &r));
        REQUIRE_SHAPE(tokens >= 0 && tokens <= INT32_MAX && heads >= 0 && heads <= kMaxHeads,
                      "rotary tokens must be 0..2^31-1 and heads 0..65535");
        const int64_t xs[2] = {x_token_stride, x_head_stride}, os[2] = {out_token_stride, out_head_stride};
        DCN_TRY(check_strides(ctx, "x", xs));
        DCN_TRY(check_out_strides(ctx, "out", os, tokens, heads, r.dim));
        if (!tokens || !heads) return DCN_OK;
        DCN_TRY(check_pointer(ctx, "x", d_x, rotary->dtype));
        DCN_TRY(check_pointer(ctx, "out", d_out, rotary->dtype));
        if (r.pairs) {
            DCN_TRY(check_pointer(ctx, "positions", d_positions, DCN_DTYPE_F32));
            DCN_TRY(check_pointer(ctx, "freq", d_freq, DCN_DTYPE_F32));
        }
        if (d_x == d_out && (xs[0] != os[0] || xs[1] != os[1]))
            return fail(ctx, DCN_INVALID_ARGUMENT, "out is x with other strides");
        r.positions = d_positions;
        r.freq = d_freq;
        r.sign = inverse ? -1.f : 1.f;
        DCN_HIP(ctx, dcn::launch_rotary(rotary->dtype, tokens, heads, {d_x, xs[0], xs[1]}, {d_out, os[0], os[1]}, r,
                                        (hipStream_t)stream));
        return DCN_OK;
    });
}

dcn_status dcn_cache_append_dev(dcn_context* ctx, const dcn_cache* cache, const dcn_append_shape* shape,
                                const dcn_rotary* rotary, const void* d_q, const void* d_k, const void* d_v,
                                const int32_t* d_positions, const float* d_freq, const int32_t* d_cu_q,
                                const int32_t* d_kv_lens, const int32_t* d_table, void* d_q_out, void* d_k_pages,
                                void* d_v_pages, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        REQUIRE_POINTER(cache);
        REQUIRE_POINTER(shape);
        dcn::AppendArgs a{};
        DCN_TRY(check_cache(ctx, cache, &a.pages));
        dcn::RotaryArgs r{};
        r.dim = cache->head_dim;
        DCN_TRY(check_append(ctx, cache, shape, rotary, d_q != nullptr, &r));
        if (!shape->tokens || !shape->sequences) return DCN_OK;
        DCN_TRY(check_append_pointers(ctx, cache, shape, r, d_q, d_k, d_v, d_positions, d_freq, d_cu_q, d_kv_lens, d_table, d_q_out));
        DCN_TRY(check_pointer(ctx, "k_pages", d_k_pages, cache->dtype));
        DCN_TRY(check_pointer(ctx, "v_pages", d_v_pages, cache->dtype));
        fill_append(&a, &r, cache, shape, d_q, d_k, d_v, d_positions, d_freq, d_cu_q, d_kv_lens, d_table, d_q_out);
        const int64_t ts = (int64_t)cache->kv_heads * cache->head_dim;
        a.k_pages = {d_k_pages, ts, cache->head_dim};
        a.v_pages = {d_v_pages, ts, cache->head_dim};
        DCN_HIP(ctx, dcn::launch_append(cache->dtype, a, r, (hipStream_t)stream));
        return DCN_OK;
    });
}

size_t dcn_attention_workspace_bytes(const dcn_attention_shape* shape, dcn_attention_pass pass) {
    dcn::AttentionArgs a{};
    try {
        if (!shape) return 0;
        const dcn_attention_shape s = fitted(*shape, pass == DCN_ATTENTION_PAGED);
        if (check_attention(nullptr, &s, pass == DCN_ATTENTION_PAGED, &a) != DCN_OK) return 0;
        return attention_workspace(&s, pass);
    } catch (const std::exception&) {
        return 0;
    }
}

dcn_status dcn_attention_forward_dev(dcn_context* ctx, const dcn_attention_shape* given, const void* d_q,
                                     const void* d_k, const void* d_v, const int32_t* d_cu_q,
                                     const int32_t* d_cu_kv, void* d_out, float* d_lse, void* d_workspace,
                                     size_t workspace_bytes, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        if (!given) return null_fail(ctx, "shape");
        DCN_TRY(check_even(ctx, given, d_cu_q, d_cu_kv));
        const dcn_attention_shape own = fitted(*given, false), *shape = &own;
        dcn::AttentionArgs a{};
        DCN_TRY(check_attention(ctx, shape, false, &a));
        DCN_TRY(check_out_strides(ctx, "out", shape->out_stride, shape->q_tokens, shape->q_heads, shape->head_dim));
        if (!shape->sequences || !shape->max_q || !shape->q_tokens) return DCN_OK;
        DCN_TRY(check_pointer(ctx, "q", d_q, shape->dtype));
        DCN_TRY(check_pointer(ctx, "out", d_out, shape->dtype));
        if (shape->kv_tokens) {
            DCN_TRY(check_pointer(ctx, "k", d_k, shape->dtype));
            DCN_TRY(check_pointer(ctx, "v", d_v, shape->dtype));
        }
        DCN_TRY(check_optional(ctx, "lse", d_lse, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "cu_q", d_cu_q, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "cu_kv", d_cu_kv, DCN_DTYPE_F32));
        DCN_TRY(check_workspace(ctx, d_workspace, workspace_bytes, attention_workspace(shape, DCN_ATTENTION_FORWARD)));
        a.q.p = d_q;
        a.k.p = d_k;
        a.v.p = d_v;
        a.out.p = d_out;
        a.lse = d_lse;
        a.cu_q = d_cu_q;
        a.cu_kv = d_cu_kv;
        a.workspace = d_workspace;
        a.any_splits = any_splits(shape);
        const bool matrix = matrix_heads(shape) && matrix_tensor(a.q) && matrix_tensor(a.k) && matrix_tensor(a.v) && matrix_tensor(a.out);
        DCN_HIP(ctx, (matrix ? dcn::launch_attention_matrix : dcn::launch_attention_any)(shape->dtype, a, (hipStream_t)stream));
        return DCN_OK;
    });
}

dcn_status dcn_attention_paged_dev(dcn_context* ctx, const dcn_attention_shape* given, const dcn_cache* cache,
                                   const void* d_q, const void* d_k_pages, const void* d_v_pages,
                                   const int32_t* d_cu_q, const int32_t* d_kv_lens, const int32_t* d_table,
                                   void* d_out, float* d_lse, void* d_workspace, size_t workspace_bytes,
                                   void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        if (!given) return null_fail(ctx, "shape");
        REQUIRE_POINTER(cache);
        REQUIRE_SHAPE(d_cu_q || (int64_t)given->sequences * given->max_q <= given->q_tokens,
                      "sequences * max_q exceeds q_tokens");
        const dcn_attention_shape own = fitted(*given, true), *shape = &own;
        dcn::AttentionArgs a{};
        DCN_TRY(check_cache(ctx, cache, &a.pages));
        DCN_TRY(check_attention(ctx, shape, true, &a));
        REQUIRE_SHAPE(cache->dtype == shape->dtype && cache->kv_heads == shape->kv_heads &&
                          cache->head_dim == shape->head_dim,
                      "attention and cache have different types, key heads or head sizes");
        DCN_TRY(check_out_strides(ctx, "out", shape->out_stride, shape->q_tokens, shape->q_heads, shape->head_dim));
        if (!shape->sequences || !shape->max_q || !shape->q_tokens) return DCN_OK;
        DCN_TRY(check_pointer(ctx, "q", d_q, shape->dtype));
        DCN_TRY(check_pointer(ctx, "out", d_out, shape->dtype));
        DCN_TRY(check_pointer(ctx, "k_pages", d_k_pages, shape->dtype));
        DCN_TRY(check_pointer(ctx, "v_pages", d_v_pages, shape->dtype));
        DCN_TRY(check_pointer(ctx, "kv_lens", d_kv_lens, DCN_DTYPE_F32));
        DCN_TRY(check_pointer(ctx, "table", d_table, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "lse", d_lse, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "cu_q", d_cu_q, DCN_DTYPE_F32));
        DCN_TRY(check_workspace(ctx, d_workspace, workspace_bytes, attention_workspace(shape, DCN_ATTENTION_PAGED)));
        const int64_t ts = (int64_t)cache->kv_heads * cache->head_dim;
        a.q.p = d_q;
        a.k = {d_k_pages, ts, cache->head_dim};
        a.v = {d_v_pages, ts, cache->head_dim};
        a.out.p = d_out;
        a.lse = d_lse;
        a.cu_q = d_cu_q;
        a.cu_kv = d_kv_lens;
        a.pages.table = d_table;
        a.workspace = d_workspace;
        a.any_splits = any_splits(shape);
        const bool matrix = matrix_heads(shape) && matrix_pool(cache) && matrix_tensor(a.q) && matrix_tensor(a.k) &&
                            matrix_tensor(a.v) && matrix_tensor(a.out);
        DCN_HIP(ctx, (matrix ? dcn::launch_attention_matrix : dcn::launch_attention_any)(shape->dtype, a, (hipStream_t)stream));
        return DCN_OK;
    });
}

dcn_status dcn_attention_backward_dev(dcn_context* ctx, const dcn_attention_shape* given, const void* d_q,
                                      const void* d_k, const void* d_v, const void* d_out, const float* d_lse,
                                      const void* d_dout, const int32_t* d_cu_q, const int32_t* d_cu_kv, void* d_dq,
                                      void* d_dk, void* d_dv, void* d_workspace, size_t workspace_bytes,
                                      void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        if (!given) return null_fail(ctx, "shape");
        DCN_TRY(check_even(ctx, given, d_cu_q, d_cu_kv));
        const dcn_attention_shape own = fitted(*given, false), *shape = &own;
        dcn::AttentionArgs a{};
        DCN_TRY(check_attention(ctx, shape, false, &a));
        const int dim = shape->head_dim;
        DCN_TRY(check_strides(ctx, "out", shape->out_stride));
        DCN_TRY(check_strides(ctx, "dout", shape->dout_stride));
        DCN_TRY(check_out_strides(ctx, "dq", shape->dq_stride, shape->q_tokens, shape->q_heads, dim));
        DCN_TRY(check_out_strides(ctx, "dk", shape->dk_stride, shape->kv_tokens, shape->kv_heads, dim));
        DCN_TRY(check_out_strides(ctx, "dv", shape->dv_stride, shape->kv_tokens, shape->kv_heads, dim));
        if (!shape->sequences) return DCN_OK;
        if (shape->q_tokens && shape->max_q) {
            DCN_TRY(check_pointer(ctx, "q", d_q, shape->dtype));
            DCN_TRY(check_pointer(ctx, "out", d_out, shape->dtype));
            DCN_TRY(check_pointer(ctx, "dout", d_dout, shape->dtype));
            DCN_TRY(check_pointer(ctx, "lse", d_lse, DCN_DTYPE_F32));
            DCN_TRY(check_pointer(ctx, "dq", d_dq, shape->dtype));
        }
        if (shape->kv_tokens && shape->max_kv) {
            DCN_TRY(check_pointer(ctx, "k", d_k, shape->dtype));
            DCN_TRY(check_pointer(ctx, "v", d_v, shape->dtype));
            DCN_TRY(check_pointer(ctx, "dk", d_dk, shape->dtype));
            DCN_TRY(check_pointer(ctx, "dv", d_dv, shape->dtype));
        }
        DCN_TRY(check_optional(ctx, "cu_q", d_cu_q, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "cu_kv", d_cu_kv, DCN_DTYPE_F32));
        DCN_TRY(check_workspace(ctx, d_workspace, workspace_bytes, attention_workspace(shape, DCN_ATTENTION_BACKWARD)));
        a.q.p = d_q;
        a.k.p = d_k;
        a.v.p = d_v;
        a.o = {d_out, shape->out_stride[0], shape->out_stride[1]};
        a.dout = {d_dout, shape->dout_stride[0], shape->dout_stride[1]};
        a.dq = {d_dq, shape->dq_stride[0], shape->dq_stride[1]};
        a.dk = {d_dk, shape->dk_stride[0], shape->dk_stride[1]};
        a.dv = {d_dv, shape->dv_stride[0], shape->dv_stride[1]};
        a.lse_in = d_lse;
        a.cu_q = d_cu_q;
        a.cu_kv = d_cu_kv;
        a.workspace = d_workspace;
        if (!shape->q_tokens) a.max_q = 0;
        if (!shape->kv_tokens) a.max_kv = 0;
        bool matrix = matrix_heads(shape);
        for (const dcn::HeadsIn* h : {&a.q, &a.k, &a.v, &a.o, &a.dout}) matrix = matrix && matrix_tensor(*h, a.group);
        for (const dcn::HeadsOut* h : {&a.dq, &a.dk, &a.dv}) matrix = matrix && matrix_tensor(*h);
        DCN_HIP(ctx, (matrix ? dcn::launch_attention_matrix_backward : dcn::launch_attention_any_backward)(shape->dtype, a,
                                                                                                          (hipStream_t)stream));
        return DCN_OK;
    });
}

dcn_status dcn_gated_norm_forward_dev(dcn_context* ctx, const dcn_norm_shape* shape, const void* d_h,
                                      const void* d_x, const void* d_gate, const void* d_w_post, const void* d_w_pre,
                                      void* d_x_out, void* d_y, float* d_rstd, void* d_low, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        REQUIRE_POINTER(shape);
        dcn::NormArgs a;
        DCN_TRY(check_norm(ctx, shape, &a));
        if (!shape->tokens) return DCN_OK;
        DCN_TRY(check_pointer(ctx, "h", d_h, shape->dtype));
        DCN_TRY(check_pointer(ctx, "x", d_x, shape->dtype));
        DCN_TRY(check_pointer(ctx, "x_out", d_x_out, shape->dtype));
        DCN_TRY(check_optional(ctx, "gate", d_gate, shape->dtype));
        DCN_TRY(check_optional(ctx, "w_post", d_w_post, shape->dtype));
        DCN_TRY(check_optional(ctx, "w_pre", d_w_pre, shape->dtype));
        DCN_TRY(check_optional(ctx, "y", d_y, shape->dtype));
        DCN_TRY(check_optional(ctx, "rstd", d_rstd, DCN_DTYPE_F32));
        a.h = d_h;
        a.x = d_x;
        a.gate = d_gate;
        a.w_post = d_w_post;
        a.w_pre = d_w_pre;
        a.x_out = d_x_out;
        a.y = d_y;
        a.rstd = d_rstd;
        DCN_TRY(check_low(ctx, d_low));
        a.low = shape->dtype == DCN_DTYPE_F32 ? nullptr : d_low;
        DCN_HIP(ctx, dcn::launch_norm_forward(shape->dtype, a, (hipStream_t)stream));
        return DCN_OK;
    });
}

size_t dcn_gated_norm_low_bytes(const dcn_norm_shape* shape) {
    dcn::NormArgs a;
    try {
        if (!shape || check_norm(nullptr, shape, &a) != DCN_OK || shape->dtype == DCN_DTYPE_F32) return 0;
        return dcn::norm_low_bytes(a.tokens, a.channels);
    } catch (const std::exception&) {
        return 0;
    }
}

size_t dcn_gated_norm_workspace_bytes(const dcn_norm_shape* shape) {
    dcn::NormArgs a;
    try {
        if (!shape || check_norm(nullptr, shape, &a) != DCN_OK) return 0;
        return dcn::norm_workspace_bytes(a.channels, a.tokens, a.gate_tokens);
    } catch (const std::exception&) {
        return 0;
    }
}

dcn_status dcn_gated_norm_backward_dev(dcn_context* ctx, const dcn_norm_shape* shape, const void* d_h,
                                       const void* d_x_out, const void* d_gate, const void* d_w_post,
                                       const void* d_w_pre, const float* d_rstd, const void* d_low,
                                       const void* d_dx_out, const void* d_dy, void* d_dh, void* d_dx, void* d_dgate, float* d_dw_post,
                                       float* d_dw_pre, void* d_workspace, size_t workspace_bytes, void* stream) {
    return entry(ctx, [&]() -> dcn_status {
        REQUIRE_POINTER(shape);
        dcn::NormArgs a;
        DCN_TRY(check_norm(ctx, shape, &a));
        const hipStream_t st = (hipStream_t)stream;
        DCN_TRY(check_workspace(ctx, d_workspace, workspace_bytes,
                                dcn::norm_workspace_bytes(a.channels, a.tokens, a.gate_tokens)));
        if (shape->tokens) {
            DCN_TRY(check_pointer(ctx, "h", d_h, shape->dtype));
            DCN_TRY(check_pointer(ctx, "x_out", d_x_out, shape->dtype));
            DCN_TRY(check_pointer(ctx, "rstd", d_rstd, DCN_DTYPE_F32));
            DCN_TRY(check_pointer(ctx, "dx_out", d_dx_out, shape->dtype));
            DCN_TRY(check_pointer(ctx, "dh", d_dh, shape->dtype));
            DCN_TRY(check_pointer(ctx, "dx", d_dx, shape->dtype));
        }
        DCN_TRY(check_optional(ctx, "gate", d_gate, shape->dtype));
        DCN_TRY(check_optional(ctx, "w_post", d_w_post, shape->dtype));
        DCN_TRY(check_optional(ctx, "w_pre", d_w_pre, shape->dtype));
        DCN_TRY(check_optional(ctx, "dy", d_dy, shape->dtype));
        DCN_TRY(check_optional(ctx, "dgate", d_dgate, shape->dtype));
        DCN_TRY(check_optional(ctx, "dw_post", d_dw_post, DCN_DTYPE_F32));
        DCN_TRY(check_optional(ctx, "dw_pre", d_dw_pre, DCN_DTYPE_F32));
        a.h = d_h;
        a.x_out = const_cast<void*>(d_x_out);
        a.gate = d_gate;
        a.w_post = d_w_post;
        a.w_pre = d_w_pre;
        a.rstd = const_cast<float*>(d_rstd);
        DCN_TRY(check_low(ctx, d_low));
        a.low = shape->dtype == DCN_DTYPE_F32 ? nullptr : const_cast<void*>(d_low);
        a.dx_out = d_dx_out;
        a.dy = d_dy;
        a.dh = d_dh;
        a.dx = d_dx;
        a.dgate = d_dgate;
        a.dw_post = d_dw_post;
        a.dw_pre = d_dw_pre;
        a.workspace = (float*)d_workspace;
        DCN_HIP(ctx, dcn::launch_norm_backward(shape->dtype, a, st));
        return DCN_OK;
    });
}

}  // extern "C"
