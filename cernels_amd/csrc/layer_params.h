// Launch parameters of the decoder-layer kernels, filled in and checked by the C entries (layer_capi.cpp).
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

namespace cmoe {

constexpr int kDtBf16 = 0, kDtF16 = 1, kDtF32 = 2, kDtF64 = 3;

struct NormParams {
    const void *x, *weight, *bias, *dy;  // [rows, cols]; [cols] (bias may be null); dy: backward
    void *y, *dx, *dweight, *dbias;      // backward: each may be null
    float* stats;                        // [rows, 2] mean and 1 / standard deviation; forward: may be null
    float* partial;                      // backward: norm_backward_partials() rows of [2, cols]
    long long rows;
    int cols, dtype, wdtype;
    float eps;
};
int norm_backward_partials(long long rows, int cols, int dtype);
hipError_t launch_norm(const NormParams& p, hipStream_t s);
hipError_t launch_norm_backward(const NormParams& p, hipStream_t s);

// A [tokens, heads, dim] tensor whose last dimension is contiguous, strides in elements.
struct HeadsView {
    const void* p;
    long long token, head;
    int heads;
};
// A page pool: element (page, slot, head, d) at page * page_stride + slot * slot + head * head + d.
struct PagesView {
    void* p;
    long long page, slot, head;
};
// The sequences of a step: sequence b has the new tokens offsets[b] .. offsets[b + 1] - 1 (uniform many where offsets is null),
// which are the last of its lengths[b] tokens.
struct StepView {
    const int32_t *table, *lengths, *offsets;
    long long table_stride;
    int seqs, tokens, uniform, pages, page_size, blocks;
};

struct RotaryParams {
    HeadsView q, k, v;        // v, and k's destination in the pages: append only
    void *q_out, *k_out;      // [tokens, heads, dim] contiguous
    PagesView k_pages, v_pages;
    StepView step;            // append
    const void* positions;    // rotary: [tokens] int32 or int64
    const void* inv_freq;     // [pairs] fp32 or fp64
    int tokens, dim, pairs, interleaved, position_i64, freq_f64, backward, append, dtype;
    float scale;
};
hipError_t launch_rotary(const RotaryParams& p, hipStream_t s);

struct AttentionParams {
    HeadsView q;
    void* out;                // [tokens, heads, dim] contiguous
    PagesView k, v;
    StepView step;
    const float* sinks;       // [heads] or null
    int kv_heads, dim, window, dtype, max_new;
    float scale;
    float* ws;
};
size_t attention_workspace_bytes(const AttentionParams& p);
bool attention_dim_ok(int dim);
hipError_t launch_attention(const AttentionParams& p, hipStream_t s);

}  // namespace cmoe
