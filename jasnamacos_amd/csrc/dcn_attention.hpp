// Frame attention: kernel arguments shared by the C-ABI layer and the kernel files, and the
// device helpers of its kernels.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstddef>
#include <cstdint>

#include "dcn/dcn.h"

namespace dcn {

// A [tokens][heads][head_dim] tensor: element strides, adjacent channels.
struct HeadsIn {
    const void* p;
    int64_t ts, hs;
};
struct HeadsOut {
    void* p;
    int64_t ts, hs;
};

struct RotaryArgs {
    int dim, st, sh, pairs, interleaved;  // pairs < st: time, < sh: height, else width
    float sign;                           // -1: the inverse
    const int32_t* positions;             // null: no rotation
    const float* freq;
};

struct PagesArgs {
    int pages, shift, width;  // tokens a page = 1 << shift; entries a table row
    const int32_t* table;
};

struct AttentionArgs {
    int sequences, q_heads, kv_heads, dim, group;
    int frame, back, ahead, sinks;
    int max_q, max_kv;
    float scale;
    int64_t q_tokens, kv_tokens;
    const int32_t* cu_q;
    const int32_t* cu_kv;   // the paged call: kv_lens
    PagesArgs pages;        // table null: contiguous keys
    HeadsIn q, k, v;        // paged: k and v are pages, ts between a page's tokens
    HeadsOut out;
    float* lse;             // may be null
    // backward
    HeadsIn o, dout;
    HeadsOut dq, dk, dv;
    const float* lse_in;
    void* workspace;
    int any_splits;  // launch_attention_any: workgroups that share a row block's keys
};

// A launch has fewer than 2^32 threads along x: rows or items past that go into launches of their own,
// of this many threads each.
constexpr int64_t kMostThreads = INT64_C(1) << 31;

// Keys that `tokens` adjacent queries see at most, in tiles of `tile`.
inline int64_t attention_keys(int max_kv, int frame, int back, int sinks, int64_t tokens, int tile) {
    const int64_t frames = (int64_t)back + 1 + sinks;
    if (back < 0 || frames > max_kv / frame) return max_kv;
    const int64_t window = frames * frame + tokens + 2 * tile;
    return window < max_kv ? window : (int64_t)max_kv;
}

hipError_t launch_rotary(int dtype, int64_t tokens, int heads, const HeadsIn& x, const HeadsOut& out,
                         const RotaryArgs& r, hipStream_t stream);

struct AppendArgs {
    int sequences, q_heads, kv_heads;
    int64_t tokens;
    HeadsIn q, k, v;  // q.p null: keys and values only
    HeadsOut q_out, k_pages, v_pages;
    const int32_t* cu_q;
    const int32_t* kv_lens;
    PagesArgs pages;
};
hipError_t launch_append(int dtype, const AppendArgs& a, const RotaryArgs& r, hipStream_t stream);

struct NormArgs {
    int channels;
    int64_t tokens, gate_tokens;
    float alpha, eps;
    const void *h, *x, *gate, *w_post, *w_pre;
    void *x_out, *y;
    float* rstd;
    void* low;  // rounded-off halves of x_out (norm_low_bytes); may be null
    // backward
    const void *dx_out, *dy;
    void *dh, *dx, *dgate;
    float *dw_post, *dw_pre;
    float* workspace;
};
hipError_t launch_norm_forward(int dtype, const NormArgs& a, hipStream_t stream);
hipError_t launch_norm_backward(int dtype, const NormArgs& a, hipStream_t stream);
// `low` in blocks of 16 rows: r1 and r2 (FP32) of each, then [16][channels] of 16 bits. A row's place
// does not depend on how many there are, so its statistics and its halves are always of one forward.
constexpr int kLowRows = 16;
constexpr int64_t norm_low_block(int channels) { return kLowRows * (8 + 2 * (int64_t)channels); }
constexpr size_t norm_low_bytes(int64_t tokens, int channels) {
    return (size_t)((tokens + kLowRows - 1) / kLowRows * norm_low_block(channels));
}
size_t norm_workspace_bytes(int channels, int64_t tokens, int64_t gate_tokens);

// Any head size, type, stride and alignment (dcn_kernels_attention_any.hip, _rows.hip).
hipError_t launch_attention_any(int dtype, const AttentionArgs& a, hipStream_t stream);
int attention_any_splits(const dcn_attention_shape& s);
size_t attention_any_workspace(const dcn_attention_shape& s);
hipError_t launch_attention_any_backward(int dtype, const AttentionArgs& a, hipStream_t stream);
hipError_t launch_attention_rows_backward(int dtype, const AttentionArgs& a, hipStream_t stream);

// Matrix-core kernels: 16-bit heads of 64 and 128 channels (dcn_kernels_attention.hip).
hipError_t launch_attention_matrix(int dtype, const AttentionArgs& a, hipStream_t stream);
size_t attention_forward_workspace(const dcn_attention_shape& s);
hipError_t launch_attention_matrix_backward(int dtype, const AttentionArgs& a, hipStream_t stream);
size_t attention_backward_workspace(const dcn_attention_shape& s);

}  // namespace dcn
