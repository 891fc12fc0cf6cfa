// Host-side prototypes of the 4-bit operators (fp4_kernels.cu, fp4_gemm_sm100.cu; the entry points are in fp4_api.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/llmini_b200_fp4.h"

namespace b2 {

// Every kernel of these operators waits for the launch in front of it before it touches global memory (griddepcontrol.wait),
// so all of them are launched with programmatic dependent launch: their prologues run while that one ends.
template <typename... P, typename... A>
inline cudaError_t overlapped_launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// Raises a kernel's limit of shared memory on the current device, once; `done`: the devices on which it has been.
template <typename K>
inline cudaError_t allow_smem(K kernel, uint32_t bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1u)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
    return e;
}

// ---- fp4_kernels.cu --------------------------------------------------------------------------------------------------
cudaError_t launch_fp4_quantize_rows(const b2_matrix &x, const b2_nvfp4_operand &out, cudaStream_t s);
// The same, and in the same launch the maximum of `other`, of x's type: scales on top of its fp4_maximum_parts(other) parts.
cudaError_t launch_fp4_quantize_rows_and_maximum(const b2_matrix &x, const b2_nvfp4_operand &out, const b2_matrix &other, float *maxima,
                                                 int sm_count, cudaStream_t s);
uint32_t fp4_maximum_parts(const b2_matrix &x, int sm_count);
// Scales on top of parts of a tensor that every CTA of the columns' kernel goes through for itself; more have a launch of their own.
constexpr uint32_t kFewTops = 4096;
// One or two tensors by columns.  `tops`: scales on top of parts of x where they are known (those of its rows), else null.
// maxima: B2_NVFP4_MAXIMA floats a tensor; `tops` may lie there only if there are no more of them.
struct ColumnsTask {
    const b2_matrix *x;
    const b2_nvfp4_operand *out;
    const float *tops;
    uint32_t top_count;
};
cudaError_t launch_fp4_quantize_columns(const ColumnsTask *tasks, uint32_t count, float *maxima, int sm_count, cudaStream_t s);
cudaError_t launch_fp4_decode(const b2_nvfp4_operand &in, uint32_t layout, const b2_matrix &out, cudaStream_t s);
cudaError_t launch_fp4_cache_write(const b2_nvfp4_cache *caches, const b2_vectors *tokens, uint32_t count, const int64_t *slots,
                                   uint32_t token_count, cudaStream_t s);
cudaError_t launch_fp4_cache_read(const b2_nvfp4_cache *caches, const b2_vectors *out, uint32_t count, const int32_t *table,
                                  uint32_t table_width, const int32_t *lengths, uint32_t sequences, uint32_t max_tokens,
                                  cudaStream_t s);

// ---- fp4_gemm_sm100.cu -----------------------------------------------------------------------------------------------
cudaError_t launch_fp4_matmul(const b2_nvfp4_operand &a, const b2_nvfp4_operand &b, const b2_matrix &c, const float *bias,
                              bool accumulate, int sm_count, cudaStream_t s);
// x quantised by rows on the way, for few values (fp4_linear_fused).
bool fp4_linear_fused(uint32_t rows, uint32_t cols);
cudaError_t launch_fp4_linear(const b2_matrix &x, const b2_nvfp4_operand &b, const b2_matrix &c, const float *bias, int sm_count,
                              cudaStream_t s);
cudaError_t fp4_gemm_status(uint32_t *status, cudaStream_t s);

}  // namespace b2
