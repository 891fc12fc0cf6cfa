/*
 * llmini_b200 — 4-bit operators beside the requantised weights: activations and gradients quantised to NVFP4 along either
 * axis, the product of two NVFP4 operands on the block-scaled tensor cores of sm_100a, the linear layer and its gradients
 * made of them, reading 4-bit tensors back, and a paged cache that is quantised as it is written.
 *
 * The conventions are those of llmini_b200.h: an int result (0, or a CUDA error number; 1 = B2_ERROR_INVALID_VALUE where an
 * argument is refused, before anything is launched), work enqueued on `stream` (a cudaStream_t of the current device, which
 * holds every buffer), no allocation, no synchronisation unless stated, no CPU fallback.
 *
 * The format.  A vector is cut into blocks of 16 values; a value stands for code * s * g:
 *   g     the scale on top, FP32.  The quantisers below take the power of two 2^(floor(log2 amax) - 10), amax the largest
 *         magnitude of the row (or of the tensor), never below 2^-110; any other positive value may stand there, such as the
 *         max / 1536 of the optimizer's requantised weights.
 *   s     E4M3, nearest to (largest magnitude of the block) / 6 / g
 *   code  E2M1, nearest to value / (s g), the even one between two, 0 where s is 0
 * With g a power of two all of this is exact: the codes are those of real arithmetic.  A row (tensor) that holds an infinity or
 * a NaN has g = NaN and zeros below it, so that what is computed from it is NaN.
 */
#ifndef LLMINI_B200_FP4_H
#define LLMINI_B200_FP4_H

#include "llmini_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { B2_TYPE_F32 = 0, B2_TYPE_BF16 = 1, B2_TYPE_F16 = 2 };

/* A matrix of plain values in device memory: element (r, c) at data + (r * ld + c) elements, ld >= cols. */
typedef struct b2_matrix {
    void *data;
    uint64_t ld;
    uint32_t rows, cols;
    uint32_t type;      /* B2_TYPE_* */
    uint32_t reserved;  /* 0 */
} b2_matrix;

/* A matrix in NVFP4, the operand of b2_nvfp4_matmul.  Codes: row r at bytes + r * row_bytes, two a byte, the first in the low
 * half.  Scales: B2_SCALES_SM100 (b2_nvfp4_sm100_scales_bytes(rows, cols) bytes; the quantisers below write the padding behind
 * the last block of a row as zero and leave rows behind the last one alone, the optimizer's plan writes neither: zero its
 * buffer once).  bytes and scales start on 16-byte boundaries. */
typedef struct b2_nvfp4_operand {
    uint8_t *bytes;
    uint8_t *scales;
    float *scale;          /* the scale on top: f32[scale_count] */
    uint64_t row_bytes;    /* a multiple of 16, at least cols / 2 */
    uint32_t rows, cols;   /* cols: a multiple of 16 */
    uint32_t scale_count;  /* 1 (one for the tensor) or rows (one a row) */
    uint32_t reserved;     /* 0 */
} b2_nvfp4_operand;

/* Rows of x, each with a scale of its own, in one pass.  out: x.rows rows of x.cols values rounded up to a multiple of 16
 * (zeros behind the end), scale_count = rows.  Beside the flat FP32 quantiser b2_fp32_to_nvfp4_four_six. */
int b2_nvfp4_quantize_rows(const b2_matrix *x, const b2_nvfp4_operand *out, void *stream);
/* The transpose of x, blocks along x's rows: x.cols rows of x.rows values rounded up to a multiple of 16, one scale for the
 * tensor (scale_count = 1).  Two launches, a maximum and the encode; `d_maxima` is scratch of B2_NVFP4_MAXIMA floats. */
#define B2_NVFP4_MAXIMA 1024
int b2_nvfp4_quantize_columns(const b2_matrix *x, const b2_nvfp4_operand *out, float *d_maxima, void *stream);
/* The values of `in` in out's type, rounded once.  out: in.rows rows, in.cols - 15 .. in.cols columns.  scale_layout says how
 * in.scales is laid out: B2_SCALES_SM100, B2_SCALES_RAW ([rows][cols / 16]) or B2_SCALES_CSF (cols % 128 == 0); so the
 * optimizer's weights are read back too.  CSF storage whose header describes fewer scales, or none, reads as NaN. */
int b2_nvfp4_decode(const b2_nvfp4_operand *in, uint32_t scale_layout, const b2_matrix *out, void *stream);

/* c[m][n] = sum_k a[m][k] b[n][k], + bias[n] (FP32, may be NULL), + c[m][n] where `accumulate` (FP32 c only).  a: M rows, b: N
 * rows, both of K values.  Sums are held in FP32 and rounded once to c's type.  c may not overlap the operands.  An empty c
 * (no rows or no columns) is a no-op.  The result does not depend on anything but the operands: no atomics. */
int b2_nvfp4_matmul(const b2_nvfp4_operand *a, const b2_nvfp4_operand *b, const b2_matrix *c, const float *d_bias,
                    uint32_t accumulate, void *stream);

/* y = Q(x) W^T + bias: x [tokens][inputs] quantised by rows, W [outputs][inputs] as it is.  `scratch`: memory for Q(x), an operand of
 * tokens rows, scale_count = rows; a few values are quantised on the way and do not go there, so what it holds afterwards is not
 * defined.  y may lie over x; other buffers may not overlap. */
int b2_nvfp4_linear_forward(const b2_matrix *x, const b2_nvfp4_operand *weight, const b2_matrix *y, const float *d_bias,
                            const b2_nvfp4_operand *scratch, void *stream);
/* The gradients of that, straight through the rounding:
 *   grad_x = Q(grad) W          Q by rows; weight_t is W^T [inputs][outputs], quantised along the outputs
 *   grad_weight = Q(grad^T) Q(x^T)^T   both quantised along the tokens, one scale a tensor; FP32, added to what is there where
 *                               `accumulate`
 * grad_x.data or grad_weight.data may be NULL: that gradient is left out.  grad_x may lie over grad or over x; other
 * buffers may not overlap.  Scratch: grad_rows as `scratch` above for grad,
 * grad_columns [outputs][tokens] and x_columns [inputs][tokens] as of b2_nvfp4_quantize_columns, d_maxima. */
typedef struct b2_nvfp4_linear_gradients {
    b2_matrix grad;            /* [tokens][outputs] */
    b2_matrix x;               /* [tokens][inputs] */
    b2_nvfp4_operand weight_t;
    b2_matrix grad_x;          /* [tokens][inputs] */
    b2_matrix grad_weight;     /* [outputs][inputs], FP32 */
    b2_nvfp4_operand grad_rows;
    b2_nvfp4_operand grad_columns;
    b2_nvfp4_operand x_columns;
    float *d_maxima;           /* f32[2 * B2_NVFP4_MAXIMA] */
    uint32_t accumulate;
    uint32_t reserved;         /* 0 */
} b2_nvfp4_linear_gradients;
int b2_nvfp4_linear_backward(const b2_nvfp4_linear_gradients *args, void *stream);
/* Reads back and clears the current device's status word of the product kernels (synchronises `stream`): 0 when no bounded
 * device wait ran out, else B2_ERROR_LAUNCH_TIMEOUT. */
int b2_nvfp4_status(void *stream);

/* ---- a paged cache of vectors in 4 bits ------------------------------------------------------------------------------ */
/* `pages` pages of `page_size` tokens of `heads` vectors of `dim` values (a multiple of 16, at most 1024):
 *   bytes     [pages][page_size][heads][dim / 2]    codes, two a byte
 *   scales    [pages][page_size][heads][dim / 16]   E4M3
 *   exponents [pages][page_size][heads]             g = 2^(exponent - 127), E8M0; 255 stands for NaN
 * No two vectors share a byte.  bytes starts on an 8-byte boundary. */
typedef struct b2_nvfp4_cache {
    uint8_t *bytes;
    uint8_t *scales;
    uint8_t *exponents;
    uint32_t pages, page_size, heads, dim;
} b2_nvfp4_cache;
/* Vectors of plain values: element d of head h of token t (of sequence b) at data + (b * sequence_stride + t * token_stride +
 * h * head_stride + d) elements. */
typedef struct b2_vectors {
    void *data;
    uint64_t sequence_stride, token_stride, head_stride;
    uint32_t type;      /* B2_TYPE_* */
    uint32_t reserved;  /* 0 */
} b2_vectors;
/* Quantises tokens[0 .. token_count) of `count` (1 or 2: keys, values) tensors into slots d_slots[t] = page * page_size +
 * place of each one's cache.  A slot outside [0, pages * page_size) leaves its token out.  Two tokens of a call may not have
 * the same slot. */
int b2_nvfp4_cache_write(const b2_nvfp4_cache *caches, const b2_vectors *tokens, uint32_t count, const int64_t *d_slots,
                         uint32_t token_count, void *stream);
/* Reads sequence b's tokens 0 .. d_lengths[b] (clamped to [0, min(max_tokens, table_width * page_size)]) of each cache into
 * out: token t lies in page d_table[b][t / page_size].  A page outside [0, pages) reads as NaN.  What lies behind a sequence's
 * length in out is left as it is.  Vectors of out may not overlap. */
int b2_nvfp4_cache_read(const b2_nvfp4_cache *caches, const b2_vectors *out, uint32_t count, const int32_t *d_table,
                        uint32_t table_width, const int32_t *d_lengths, uint32_t sequences, uint32_t max_tokens, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* LLMINI_B200_FP4_H */
