// gl3_ops_int8.h — rows in 8-bit integers with a scale each, and their products (include/gpullama3_hip.h: gl3_quantize_rows, gl3_int8_matmul).
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

typedef int op_v4i __attribute__((ext_vector_type(4)));
typedef int op_v16i __attribute__((ext_vector_type(16)));

// element types of float rows and results
struct op_bf16 { uint16_t u; };
template <typename T> __device__ __forceinline__ float op_f32(T v);
template <> __device__ __forceinline__ float op_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float op_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float op_f32<op_bf16>(op_bf16 v) { return __uint_as_float((uint32_t)v.u << 16); }
template <typename T> __device__ __forceinline__ T op_cast(float v);
template <> __device__ __forceinline__ float op_cast<float>(float v) { return v; }
template <> __device__ __forceinline__ __half op_cast<__half>(float v) { return __float2half(v); }
template <> __device__ __forceinline__ op_bf16 op_cast<op_bf16>(float v) { return op_bf16{__builtin_bit_cast(uint16_t, (__bf16)v)}; }

// ---- rows -> codes and scales ---------------------------------------------------------------------------------------------------------
// |x| as bits: whole numbers that order like the magnitudes, an infinity and every NaN above all finite ones
constexpr uint32_t OP_INF_BITS = 0x7f800000u;
__device__ __forceinline__ uint32_t op_mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// scale of a row from the bits of its largest magnitude, and what its values are multiplied with (0: all codes are 0)
__device__ __forceinline__ void op_row_scale(uint32_t mag, float& scale, float& to_code) {
    const float a = __uint_as_float(mag);
    if (mag >= OP_INF_BITS) { scale = __uint_as_float(0x7fc00000u); to_code = 0.f; }
    else if (a < 0x1p-100f) { scale = 0.f; to_code = 0.f; }
    else { scale = a / 127.0f; to_code = 127.0f / a; }
}
__device__ __forceinline__ int op_code(float v, float to_code) {
    return to_code == 0.f ? 0 : (int)__builtin_rintf(fminf(fmaxf(v * to_code, -127.f), 127.f));
}

template <typename T>
static __global__ __launch_bounds__(256) void op_quantize_kernel(const T* __restrict__ x, int cols, int64_t ldx, int8_t* __restrict__ codes, int64_t ldq, float* __restrict__ scale) {
    __shared__ uint32_t red[4];
    const T* row = x + (int64_t)blockIdx.x * ldx;
    int8_t* out = codes + (int64_t)blockIdx.x * ldq;
    uint32_t mag = 0;
    for (int c = threadIdx.x; c < cols; c += 256) mag = max(mag, op_mag(op_f32<T>(row[c])));
    for (int d = 32; d; d >>= 1) mag = max(mag, (uint32_t)__shfl_xor((int)mag, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mag;
    __syncthreads();
    mag = max(max(red[0], red[1]), max(red[2], red[3]));
    float s, r;
    op_row_scale(mag, s, r);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    const int end = (cols + GL3_CODE_BLOCK - 1) / GL3_CODE_BLOCK * GL3_CODE_BLOCK;
    for (int c = threadIdx.x; c < end; c += 256) out[c] = c < cols ? (int8_t)op_code(op_f32<T>(row[c]), r) : (int8_t)0;
}

// ---- products -------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float op_result(int acc, float as, float ws) { return ((float)acc * as) * ws; }

// One wavefront per 16 tokens x 16 channels, both operands straight from memory: a lane holds 16 consecutive k of one row of either.
template <typename TY>
static __global__ __launch_bounds__(64) void op_product_kernel(const int8_t* __restrict__ a, int64_t lda, const float* __restrict__ as, const int8_t* __restrict__ w, int64_t ldw,
                                                               const float* __restrict__ ws, const float* __restrict__ bias, int64_t m, int64_t n, int k, TY* __restrict__ y, int64_t ldy) {
    const int lane = threadIdx.x, r16 = lane & 15, kg = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16, m0 = (int64_t)blockIdx.y * 16;
    const int8_t* ap = a + min(m0 + r16, m - 1) * lda + 16 * kg;
    const int8_t* wp = w + min(n0 + r16, n - 1) * ldw + 16 * kg;
    op_v4i acc = {0, 0, 0, 0};
    for (int c = 0; c < k; c += 64)          // (rows end on a multiple of 128)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(*reinterpret_cast<const op_v4i*>(ap + c), *reinterpret_cast<const op_v4i*>(wp + c), acc, 0, 0, 0);
    const int64_t col = n0 + r16;
    if (col >= n) return;
    const float sw = ws[col], b = bias ? bias[col] : 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = m0 + 4 * kg + r;
        if (row >= m) break;
        const float v = op_result(acc[r], as[row], sw);
        y[row * ldy + col] = op_cast<TY>(bias ? v + b : v);
    }
}
