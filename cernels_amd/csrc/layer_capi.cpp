// extern "C" entry points of the decoder layer around the experts (declared in include/cernels_moe.h): argument checks and launch
// parameters; no device allocation, no host sync.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/cernels_moe.h"
#include "layer_params.h"

namespace {

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
int hip_status(hipError_t e) { return e == hipSuccess ? CERNELS_MOE_OK : CERNELS_MOE_HIP_ERROR; }
unsigned size_of(int dtype) { return dtype == CERNELS_DTYPE_F32 ? 4 : 2; }
bool row_dtype(int dtype) { return dtype >= CERNELS_DTYPE_BF16 && dtype <= CERNELS_DTYPE_F32; }

int norm_checks(int64_t rows, int32_t cols, int32_t dtype, int32_t weight_dtype) {
    if (rows < 0 || cols <= 0 || !row_dtype(dtype) || !row_dtype(weight_dtype)) return CERNELS_MOE_INVALID_ARGUMENT;
    if (weight_dtype != dtype && weight_dtype != CERNELS_DTYPE_F32) return CERNELS_MOE_INVALID_ARGUMENT;
    if (rows >= (1LL << 31) || cols > (1 << 24)) return CERNELS_MOE_UNSUPPORTED_SHAPE;
    return CERNELS_MOE_OK;
}

int step_checks(const cmoe::StepView& s) {
    if (s.tokens < 0 || s.seqs < 0 || s.pages < 0 || s.blocks < 0 || s.page_size <= 0) return CERNELS_MOE_INVALID_ARGUMENT;
    if (s.tokens == 0 || s.seqs == 0) return CERNELS_MOE_OK;
    if (!s.table || !s.lengths) return CERNELS_MOE_INVALID_ARGUMENT;
    if (s.table_stride < s.blocks || (!s.offsets && s.tokens % s.seqs)) return CERNELS_MOE_INVALID_ARGUMENT;
    if (s.page_size % 16 || s.pages < 1 || s.seqs > 65535 || (long long)s.blocks * s.page_size >= (1LL << 31))
        return CERNELS_MOE_UNSUPPORTED_SHAPE;
    if (!aligned(s.table, 4) || !aligned(s.lengths, 4) || !aligned(s.offsets, 4)) return CERNELS_MOE_MISALIGNED;
    return CERNELS_MOE_OK;
}

// Pages are read and written in 16-byte vectors.
bool pages_ok(const cmoe::PagesView& v) {
    return aligned(v.p, 16) && v.page % 8 == 0 && v.slot % 8 == 0 && v.head % 8 == 0 && v.page >= 0 && v.slot >= 0 && v.head >= 0;
}
// A run of 16 slots is reached by 32-bit offsets.
bool runs_ok(const cmoe::PagesView& v) { return v.slot < (1LL << 26); }

cmoe::StepView step_of(const int32_t* table, int64_t table_stride, const int32_t* lengths, const int32_t* offsets, int32_t seqs,
                       int32_t tokens, int32_t pages, int32_t page_size, int32_t blocks) {
    return cmoe::StepView{table, lengths, offsets, table_stride, seqs, tokens, seqs > 0 ? tokens / seqs : 0, pages, page_size, blocks};
}

}  // namespace

extern "C" {

int cernels_layer_norm(const void* x, const void* weight, const void* bias, int64_t rows, int32_t cols, int32_t dtype,
                       int32_t weight_dtype, float eps, void* y, float* stats, hipStream_t stream) {
    const int st = norm_checks(rows, cols, dtype, weight_dtype);
    if (st != CERNELS_MOE_OK || rows == 0) return st;
    if (!x || !weight || !y) return CERNELS_MOE_INVALID_ARGUMENT;
    const unsigned n = size_of(dtype), w = size_of(weight_dtype);
    if (!aligned(x, n) || !aligned(y, n) || !aligned(weight, w) || !aligned(bias, w) || !aligned(stats, 4)) return CERNELS_MOE_MISALIGNED;
    cmoe::NormParams p{};
    p.x = x, p.weight = weight, p.bias = bias, p.y = y, p.stats = stats;
    p.rows = rows, p.cols = cols, p.dtype = dtype, p.wdtype = weight_dtype, p.eps = eps;
    return hip_status(cmoe::launch_norm(p, stream));
}

size_t cernels_layer_norm_backward_workspace_bytes(int64_t rows, int32_t cols, int32_t dtype) {
    if (norm_checks(rows, cols, dtype, dtype) != CERNELS_MOE_OK) return 0;
    return (size_t)cmoe::norm_backward_partials(rows, cols, dtype) * 2 * (size_t)cols * sizeof(float);
}

int cernels_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* stats, int64_t rows, int32_t cols,
                                int32_t dtype, int32_t weight_dtype, void* dx, void* dweight, void* dbias, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
    const int st = norm_checks(rows, cols, dtype, weight_dtype);
    if (st != CERNELS_MOE_OK) return st;
    const bool sums = dweight || dbias;
    if (!weight || (rows > 0 && (!dy || !x || !stats)) || (sums && !workspace)) return CERNELS_MOE_INVALID_ARGUMENT;
    if ((!sums && !dx) || (!sums && rows == 0)) return CERNELS_MOE_OK;
    const unsigned n = size_of(dtype), w = size_of(weight_dtype);
    if (!aligned(dy, n) || !aligned(x, n) || !aligned(dx, n) || !aligned(weight, w) || !aligned(dweight, w) || !aligned(dbias, w) ||
        !aligned(stats, 4) || !aligned(workspace, 4))
        return CERNELS_MOE_MISALIGNED;
    if (sums && workspace_bytes < cernels_layer_norm_backward_workspace_bytes(rows, cols, dtype)) return CERNELS_MOE_WORKSPACE_TOO_SMALL;
    cmoe::NormParams p{};
    p.dy = dy, p.x = x, p.weight = weight, p.stats = const_cast<float*>(stats);
    p.dx = dx, p.dweight = dweight, p.dbias = dbias, p.partial = static_cast<float*>(workspace);
    p.rows = rows, p.cols = cols, p.dtype = dtype, p.wdtype = weight_dtype;
    return hip_status(cmoe::launch_norm_backward(p, stream));
}

int cernels_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads, const void* k,
                   int64_t k_token_stride, int64_t k_head_stride, int32_t k_heads, const void* positions, int32_t position_type,
                   const void* inv_freq, int32_t freq_dtype, int32_t tokens, int32_t dim, int32_t pairs, int32_t interleaved,
                   float scale, int32_t backward, int32_t dtype, void* q_out, void* k_out, hipStream_t stream) {
    if (tokens < 0 || dim <= 0 || pairs < 0 || 2LL * pairs > dim || q_heads < 0 || k_heads < 0 || !row_dtype(dtype) ||
        position_type < CERNELS_MOE_INDEX_I32 || position_type > CERNELS_MOE_INDEX_I64 ||
        (freq_dtype != CERNELS_DTYPE_F32 && freq_dtype != CERNELS_DTYPE_F64))
        return CERNELS_MOE_INVALID_ARGUMENT;
    if (tokens == 0 || (!q && !k)) return CERNELS_MOE_OK;
    if (!positions || (pairs > 0 && !inv_freq) || (q && !q_out) || (k && !k_out)) return CERNELS_MOE_INVALID_ARGUMENT;
    if (pairs > 1024 || (q_heads + (long long)k_heads) * dim >= (1LL << 30)) return CERNELS_MOE_UNSUPPORTED_SHAPE;
    const unsigned n = size_of(dtype);
    if (!aligned(q, n) || !aligned(k, n) || !aligned(q_out, n) || !aligned(k_out, n) || !aligned(positions, position_type ? 8 : 4) ||
        !aligned(inv_freq, freq_dtype == CERNELS_DTYPE_F64 ? 8 : 4))
        return CERNELS_MOE_MISALIGNED;
    cmoe::RotaryParams p{};
    p.q = {q, q_token_stride, q_head_stride, q_heads}, p.k = {k, k_token_stride, k_head_stride, k_heads};
    p.q_out = q_out, p.k_out = k_out, p.positions = positions, p.inv_freq = inv_freq;
    p.tokens = tokens, p.dim = dim, p.pairs = pairs, p.interleaved = interleaved != 0, p.position_i64 = position_type;
    p.freq_f64 = freq_dtype == CERNELS_DTYPE_F64, p.backward = backward != 0, p.dtype = dtype, p.scale = scale;
    return hip_status(cmoe::launch_rotary(p, stream));
}

int cernels_paged_append(const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads, void* q_out, const void* k,
                         int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                         int32_t kv_heads, int32_t dim, int32_t dtype, const void* inv_freq, int32_t freq_dtype, int32_t pairs,
                         int32_t interleaved, float scale, void* k_pages, void* v_pages, const int64_t* page_strides, int32_t pages,
                         int32_t page_size, const int32_t* block_table, int64_t table_stride, int32_t blocks, const int32_t* lengths,
                         const int32_t* q_offsets, int32_t seqs, int32_t tokens, hipStream_t stream) {
    if (dim <= 0 || q_heads < 0 || kv_heads <= 0 || pairs < 0 || 2LL * pairs > dim || !page_strides ||
        (dtype != CERNELS_DTYPE_BF16 && dtype != CERNELS_DTYPE_F16) ||
        (pairs > 0 && freq_dtype != CERNELS_DTYPE_F32 && freq_dtype != CERNELS_DTYPE_F64))
        return CERNELS_MOE_INVALID_ARGUMENT;
    cmoe::RotaryParams p{};
    p.step = step_of(block_table, table_stride, lengths, q_offsets, seqs, tokens, pages, page_size, blocks);
    const int st = step_checks(p.step);
    if (st != CERNELS_MOE_OK || tokens == 0 || seqs == 0) return st;
    if (!k || !v || !k_pages || !v_pages || (q && !q_out) || (pairs > 0 && !inv_freq)) return CERNELS_MOE_INVALID_ARGUMENT;
    if (pairs > 1024 || (q_heads + 2LL * kv_heads) * dim >= (1LL << 30)) return CERNELS_MOE_UNSUPPORTED_SHAPE;
    p.q = {q, q_token_stride, q_head_stride, q_heads}, p.k = {k, k_token_stride, k_head_stride, kv_heads};
    p.v = {v, v_token_stride, v_head_stride, kv_heads};
    p.q_out = q_out;
    p.k_pages = {k_pages, page_strides[0], page_strides[1], page_strides[2]};
    p.v_pages = {v_pages, page_strides[3], page_strides[4], page_strides[5]};
    p.inv_freq = inv_freq, p.tokens = tokens, p.dim = dim, p.pairs = pairs, p.interleaved = interleaved != 0;
    p.freq_f64 = freq_dtype == CERNELS_DTYPE_F64, p.append = 1, p.dtype = dtype, p.scale = scale;
    if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(q_out, 2) || !aligned(inv_freq, p.freq_f64 ? 8 : 4) ||
        !aligned(k_pages, 2) || !aligned(v_pages, 2))
        return CERNELS_MOE_MISALIGNED;
    return hip_status(cmoe::launch_rotary(p, stream));
}

static int attention_of(cmoe::AttentionParams& p, int32_t heads, int32_t kv_heads, int32_t dim, int32_t dtype, int32_t window,
                        int32_t max_new) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || window < 0 || max_new < 0 ||
        (dtype != CERNELS_DTYPE_BF16 && dtype != CERNELS_DTYPE_F16))
        return CERNELS_MOE_INVALID_ARGUMENT;
    const int st = step_checks(p.step);
    if (st != CERNELS_MOE_OK) return st;
    if (!cmoe::attention_dim_ok(dim) || kv_heads > 65535 || (long long)p.step.tokens * heads >= (1LL << 31)) return CERNELS_MOE_UNSUPPORTED_SHAPE;
    p.q.heads = heads, p.kv_heads = kv_heads, p.dim = dim, p.dtype = dtype, p.window = window;
    p.max_new = p.step.offsets ? (max_new > 0 ? max_new : p.step.tokens) : p.step.uniform;
    return CERNELS_MOE_OK;
}

size_t cernels_paged_attention_workspace_bytes(int32_t tokens, int32_t seqs, int32_t heads, int32_t kv_heads, int32_t dim,
                                               int32_t page_size, int32_t blocks, int32_t max_new) {
    if (tokens <= 0 || seqs <= 0) return 16;
    static const int32_t some[2] = {0, 0};  // stands for the arrays, which only the kernels read
    cmoe::AttentionParams p{};
    p.step = step_of(some, blocks, some, some, seqs, tokens, 1, page_size, blocks);
    if (attention_of(p, heads, kv_heads, dim, CERNELS_DTYPE_BF16, 0, max_new) != CERNELS_MOE_OK) return 0;
    return cmoe::attention_workspace_bytes(p);
}

int cernels_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t heads, int32_t kv_heads,
                            int32_t dim, int32_t dtype, const void* k_pages, const void* v_pages, const int64_t* page_strides,
                            int32_t pages, int32_t page_size, const int32_t* block_table, int64_t table_stride, int32_t blocks,
                            const int32_t* lengths, const int32_t* q_offsets, int32_t seqs, int32_t tokens, int32_t max_new,
                            float scale, int32_t window, const float* sinks, void* out, void* workspace, size_t workspace_bytes,
                            hipStream_t stream) {
    cmoe::AttentionParams p{};
    p.step = step_of(block_table, table_stride, lengths, q_offsets, seqs, tokens, pages, page_size, blocks);
    const int st = attention_of(p, heads, kv_heads, dim, dtype, window, max_new);
    if (st != CERNELS_MOE_OK) return st;
    if (!page_strides || !(scale > 0.0f) || scale > 3.0e38f) return CERNELS_MOE_INVALID_ARGUMENT;
    if (tokens == 0 || seqs == 0) return CERNELS_MOE_OK;
    if (!q || !k_pages || !v_pages || !out || !workspace) return CERNELS_MOE_INVALID_ARGUMENT;
    p.q.p = q, p.q.token = q_token_stride, p.q.head = q_head_stride;
    p.k = {const_cast<void*>(k_pages), page_strides[0], page_strides[1], page_strides[2]};
    p.v = {const_cast<void*>(v_pages), page_strides[3], page_strides[4], page_strides[5]};
    p.sinks = sinks, p.out = out, p.scale = scale, p.ws = static_cast<float*>(workspace);
    if (!aligned(q, 2) || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(sinks, 4) || !pages_ok(p.k) || !pages_ok(p.v))
        return CERNELS_MOE_MISALIGNED;
    if (!runs_ok(p.k) || !runs_ok(p.v)) return CERNELS_MOE_UNSUPPORTED_SHAPE;
    if (workspace_bytes < cmoe::attention_workspace_bytes(p)) return CERNELS_MOE_WORKSPACE_TOO_SMALL;
    return hip_status(cmoe::launch_attention(p, stream));
}

}  // extern "C"
