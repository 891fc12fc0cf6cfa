// Entry points of the 4-bit operators (include/llmini_b200_fp4.h): the checks of their arguments and their launches.
#include <atomic>

#include "fp4.h"

namespace {

using b2::launch_fp4_decode;
using b2::launch_fp4_matmul;
using b2::launch_fp4_quantize_columns;
using b2::launch_fp4_quantize_rows;

constexpr uint32_t kMaxExtent = 65535u * 128u;

cudaStream_t as_stream(void *s) { return reinterpret_cast<cudaStream_t>(s); }
bool on(const void *p, uintptr_t boundary) { return reinterpret_cast<uintptr_t>(p) % boundary == 0; }

cudaError_t sm_count(int &count) {
    static std::atomic<int> cached[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (count = cached[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    e = cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess && dev < 64) cached[dev].store(count, std::memory_order_relaxed);
    return e;
}

bool good(const b2_matrix &m) {
    if (m.type > B2_TYPE_F16 || m.reserved != 0 || m.rows > kMaxExtent || m.cols > kMaxExtent || m.ld < m.cols || m.ld >> 40) return false;
    if (m.rows == 0 || m.cols == 0) return true;
    return m.data && on(m.data, m.type == B2_TYPE_F32 ? 4 : 2);
}
bool good(const b2_nvfp4_operand &o) {
    if (o.reserved != 0 || o.rows > kMaxExtent || o.cols > kMaxExtent || o.cols == 0 || o.cols % 16 != 0) return false;
    if (o.row_bytes % 16 != 0 || o.row_bytes < o.cols / 2 || o.row_bytes >> 40) return false;
    if (o.scale_count != 1 && o.scale_count != o.rows) return false;
    if (o.rows == 0) return true;
    return o.bytes && o.scales && o.scale && on(o.bytes, 16) && on(o.scales, 16) && on(o.scale, 4);
}
uint32_t blocks_up(uint32_t values) { return (values + 15) / 16 * 16; }
bool rows_of(const b2_matrix &x, const b2_nvfp4_operand &o) {
    return good(x) && good(o) && x.cols != 0 && o.rows == x.rows && o.cols == blocks_up(x.cols) && o.scale_count == x.rows;
}
bool columns_of(const b2_matrix &x, const b2_nvfp4_operand &o) {
    return good(x) && good(o) && x.rows != 0 && o.rows == x.cols && o.cols == blocks_up(x.rows) && o.scale_count == 1;
}
// Whether two matrices may have a byte in common: whether their first and last bytes enclose one.
bool may_overlap(const b2_matrix &a, const b2_matrix &b) {
    auto first = [](const b2_matrix &m) { return reinterpret_cast<uintptr_t>(m.data); };
    auto end = [&](const b2_matrix &m) { return first(m) + ((m.rows - 1) * m.ld + m.cols) * (m.type == B2_TYPE_F32 ? 4 : 2); };
    return a.rows != 0 && b.rows != 0 && first(a) < end(b) && first(b) < end(a);
}
bool product_of(const b2_nvfp4_operand &a, const b2_nvfp4_operand &b, const b2_matrix &c) {
    return good(a) && good(b) && good(c) && a.cols == b.cols && c.rows == a.rows && c.cols == b.rows;
}
bool good(const b2_nvfp4_cache &c) {
    return c.bytes && c.scales && c.exponents && on(c.bytes, 8) && c.page_size != 0 && c.page_size <= kMaxExtent && c.heads != 0 && c.heads <= 65535u &&
           c.dim != 0 && c.dim % 16 == 0 && c.dim <= 1024;
}
bool good(const b2_vectors &v) {
    return v.data && v.type <= B2_TYPE_F16 && v.reserved == 0 && on(v.data, v.type == B2_TYPE_F32 ? 4 : 2) &&
           !(v.sequence_stride >> 40) && !(v.token_stride >> 40) && !(v.head_stride >> 40);
}
bool good(const b2_nvfp4_cache *caches, const b2_vectors *vectors, uint32_t count) {
    if (!caches || !vectors || count == 0 || count > 2) return false;
    for (uint32_t i = 0; i < count; ++i)
        if (!good(caches[i]) || !good(vectors[i]) || vectors[i].type != vectors[0].type) return false;
    return true;
}

}  // namespace

extern "C" {

int b2_nvfp4_quantize_rows(const b2_matrix *x, const b2_nvfp4_operand *out, void *stream) {
    if (!x || !out || (x->rows != 0 && !rows_of(*x, *out))) return B2_ERROR_INVALID_VALUE;
    if (x->rows == 0) return out->rows == 0 ? B2_SUCCESS : B2_ERROR_INVALID_VALUE;
    return (int)launch_fp4_quantize_rows(*x, *out, as_stream(stream));
}

int b2_nvfp4_quantize_columns(const b2_matrix *x, const b2_nvfp4_operand *out, float *d_maxima, void *stream) {
    if (!x || !out || !columns_of(*x, *out) || !d_maxima || !on(d_maxima, 4)) return B2_ERROR_INVALID_VALUE;
    if (x->cols == 0) return B2_SUCCESS;
    int sms = 0;
    cudaError_t e = sm_count(sms);
    if (e != cudaSuccess) return (int)e;
    const b2::ColumnsTask task = {x, out, nullptr, 0};
    return (int)launch_fp4_quantize_columns(&task, 1, d_maxima, sms, as_stream(stream));
}

int b2_nvfp4_decode(const b2_nvfp4_operand *in, uint32_t scale_layout, const b2_matrix *out, void *stream) {
    if (!in || !out || !good(*in) || !good(*out) || scale_layout > B2_SCALES_SM100) return B2_ERROR_INVALID_VALUE;
    if (out->rows != in->rows || blocks_up(out->cols) != in->cols) return B2_ERROR_INVALID_VALUE;
    // CSF storage and its group numbers: whole 128-value pieces of a row, and 32 bits (csf_load_scale)
    if (scale_layout == B2_SCALES_CSF && (in->cols % 128 != 0 || (uint64_t)in->rows * (in->cols / 16) > 0xffffffffu)) return B2_ERROR_INVALID_VALUE;
    if (in->rows == 0) return B2_SUCCESS;
    return (int)launch_fp4_decode(*in, scale_layout, *out, as_stream(stream));
}

int b2_nvfp4_matmul(const b2_nvfp4_operand *a, const b2_nvfp4_operand *b, const b2_matrix *c, const float *d_bias, uint32_t accumulate,
                    void *stream) {
    if (!a || !b || !c || !product_of(*a, *b, *c) || accumulate > 1 || (accumulate && c->type != B2_TYPE_F32) || !on(d_bias, 4))
        return B2_ERROR_INVALID_VALUE;
    if (c->rows == 0 || c->cols == 0) return B2_SUCCESS;
    int sms = 0;
    cudaError_t e = sm_count(sms);
    if (e != cudaSuccess) return (int)e;
    return (int)launch_fp4_matmul(*a, *b, *c, d_bias, accumulate != 0, sms, as_stream(stream));
}

int b2_nvfp4_linear_forward(const b2_matrix *x, const b2_nvfp4_operand *weight, const b2_matrix *y, const float *d_bias,
                            const b2_nvfp4_operand *scratch, void *stream) {
    if (!x || !weight || !y || !scratch || !rows_of(*x, *scratch) || !product_of(*scratch, *weight, *y) || !on(d_bias, 4))
        return B2_ERROR_INVALID_VALUE;
    if (y->rows == 0 || y->cols == 0) return B2_SUCCESS;
    int sms = 0;
    cudaError_t e = sm_count(sms);
    // a few values are quantised by every CTA of the product for itself; more, or what y lies over, once
    if (e == cudaSuccess && b2::fp4_linear_fused(x->rows, x->cols) && !may_overlap(*x, *y))
        return (int)b2::launch_fp4_linear(*x, *weight, *y, d_bias, sms, as_stream(stream));
    if (e == cudaSuccess) e = launch_fp4_quantize_rows(*x, *scratch, as_stream(stream));
    if (e == cudaSuccess) e = launch_fp4_matmul(*scratch, *weight, *y, d_bias, false, sms, as_stream(stream));
    return (int)e;
}

int b2_nvfp4_linear_backward(const b2_nvfp4_linear_gradients *g, void *stream) {
    if (!g || g->reserved != 0 || g->accumulate > 1 || !good(g->grad) || g->grad.cols == 0) return B2_ERROR_INVALID_VALUE;
    const bool to_x = g->grad_x.data != nullptr, to_weight = g->grad_weight.data != nullptr;
    const uint32_t tokens = g->grad.rows;
    if (to_x && tokens != 0 && (!rows_of(g->grad, g->grad_rows) || !product_of(g->grad_rows, g->weight_t, g->grad_x))) return B2_ERROR_INVALID_VALUE;
    if (to_weight) {
        if (!good(g->x) || g->x.rows != tokens || !good(g->grad_weight) || g->grad_weight.type != B2_TYPE_F32 || g->grad_weight.rows != g->grad.cols ||
            g->grad_weight.cols != g->x.cols)
            return B2_ERROR_INVALID_VALUE;
        if (tokens != 0 && (!columns_of(g->grad, g->grad_columns) || !columns_of(g->x, g->x_columns) || !g->d_maxima || !on(g->d_maxima, 4)))
            return B2_ERROR_INVALID_VALUE;
    }
    cudaStream_t s = as_stream(stream);
    if (tokens == 0) {   // a sum of nothing
        if (!to_weight || g->accumulate || g->x.cols == 0) return B2_SUCCESS;
        return (int)cudaMemset2DAsync(g->grad_weight.data, g->grad_weight.ld * 4, 0, (size_t)g->grad_weight.cols * 4, g->grad_weight.rows, s);
    }
    int sms = 0;
    cudaError_t e = sm_count(sms);
    const bool columns = to_weight && g->x.cols != 0;
    // x's maximum comes along with the rows of grad, which saves a launch where grad's needs none: 777 x 1600 -> 1600 25.9 -> 24.1 us,
    // 64 x 1024 -> 1024 15.0 -> 13.3; with 8192 rows 85.9 -> 86.8
    const bool along = to_x && columns && g->x.type == g->grad.type && tokens <= b2::kFewTops;
    float *x_maxima = along ? g->d_maxima + B2_NVFP4_MAXIMA : nullptr;
    // grad_x comes last of all where it lies over what the columns are still to be read from.  (Always last, 777 x 1600 -> 1600 on new inputs
    // takes 26.5 us instead of 25.7, on the same ones again 23.7 instead of 24.4.)
    const bool last = columns && (may_overlap(g->grad_x, g->grad) || may_overlap(g->grad_x, g->x));
    auto product_x = [&]() { return to_x && g->grad_x.cols != 0 ? launch_fp4_matmul(g->grad_rows, g->weight_t, g->grad_x, nullptr, false, sms, s) : cudaSuccess; };
    if (e == cudaSuccess && to_x) {
        e = along ? b2::launch_fp4_quantize_rows_and_maximum(g->grad, g->grad_rows, g->x, x_maxima, sms, s)
                  : launch_fp4_quantize_rows(g->grad, g->grad_rows, s);
        if (e == cudaSuccess && !last) e = product_x();
    }
    if (e == cudaSuccess && columns) {
        // the scales of grad's rows are scales of parts of it: with them its first pass is done
        const b2::ColumnsTask tasks[2] = {{&g->grad, &g->grad_columns, to_x ? g->grad_rows.scale : nullptr, tokens},
                                          {&g->x, &g->x_columns, x_maxima, along ? b2::fp4_maximum_parts(g->x, sms) : 0}};
        e = launch_fp4_quantize_columns(tasks, 2, g->d_maxima, sms, s);
    }
    if (e == cudaSuccess && last) e = product_x();
    if (e == cudaSuccess && columns) e = launch_fp4_matmul(g->grad_columns, g->x_columns, g->grad_weight, nullptr, g->accumulate != 0, sms, s);
    return (int)e;
}

int b2_nvfp4_status(void *stream) {
    uint32_t status = 0;
    const cudaError_t e = b2::fp4_gemm_status(&status, as_stream(stream));
    return e != cudaSuccess ? (int)e : status != 0 ? B2_ERROR_LAUNCH_TIMEOUT : B2_SUCCESS;
}

int b2_nvfp4_cache_write(const b2_nvfp4_cache *caches, const b2_vectors *tokens, uint32_t count, const int64_t *d_slots, uint32_t token_count,
                         void *stream) {
    if (token_count == 0) return count == 1 || count == 2 ? B2_SUCCESS : B2_ERROR_INVALID_VALUE;
    if (!good(caches, tokens, count) || !d_slots || !on(d_slots, 8) || token_count > kMaxExtent) return B2_ERROR_INVALID_VALUE;
    return (int)b2::launch_fp4_cache_write(caches, tokens, count, d_slots, token_count, as_stream(stream));
}

int b2_nvfp4_cache_read(const b2_nvfp4_cache *caches, const b2_vectors *out, uint32_t count, const int32_t *d_table, uint32_t table_width,
                        const int32_t *d_lengths, uint32_t sequences, uint32_t max_tokens, void *stream) {
    if (sequences == 0 || max_tokens == 0 || table_width == 0) return count == 1 || count == 2 ? B2_SUCCESS : B2_ERROR_INVALID_VALUE;
    if (!good(caches, out, count) || !d_table || !d_lengths || !on(d_table, 4) || !on(d_lengths, 4) || sequences > 65535u || max_tokens > kMaxExtent)
        return B2_ERROR_INVALID_VALUE;
    return (int)b2::launch_fp4_cache_read(caches, out, count, d_table, table_width, d_lengths, sequences, max_tokens, as_stream(stream));
}

}  // extern "C"
