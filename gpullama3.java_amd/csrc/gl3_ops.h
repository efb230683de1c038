// gl3_ops.h — the operators on device memory as the library's own plans launch them: arguments checked by the caller, nothing but launches.  What fails is the
// first launch that failed; none follows it.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/gpullama3_hip.h"

static inline int64_t op_code_ld(int64_t cols) { return (cols + GL3_CODE_BLOCK - 1) / GL3_CODE_BLOCK * GL3_CODE_BLOCK; }

struct OpProduct {             // y = (float(a w^T) * a_scale) * w_scale (+ bias)
    const int8_t* a; int64_t lda; const float* a_scale;
    const int8_t* w; int64_t ldw; const float* w_scale; const float* bias;
    int64_t m, n; int32_t k;
    void* y; int32_t y_type; int64_t ldy;
};
struct OpLogprobs {
    const void* logits; int32_t type; int64_t rows; int32_t vocab; int64_t ld;
    const int32_t* targets; int32_t top;
    float* logprob; int32_t* rank; float* entropy; int32_t* top_ids; float* top_logprobs;
};
uint64_t op_product_workspace(int64_t m, int64_t n, int32_t k);
uint64_t op_linear_workspace(int64_t m, int64_t n, int32_t k);
uint64_t op_logprobs_workspace(int64_t rows, int32_t vocab, int32_t top);
hipError_t op_quantize(hipStream_t s, const void* x, int32_t type, int64_t rows, int32_t cols, int64_t ldx, int8_t* codes, int64_t ldq, float* scale);
hipError_t op_product(hipStream_t s, const OpProduct& p, void* workspace);
hipError_t op_linear(hipStream_t s, const void* x, int32_t x_type, int64_t ldx, const OpProduct& p, void* workspace);          // p.a, lda, a_scale: not read
hipError_t op_logprobs(hipStream_t s, const OpLogprobs& p, void* workspace);
