// gl3_ops_logprobs.h — log probabilities of given tokens, entropy and the most probable tokens of rows of logits (include/gpullama3_hip.h).
#pragma once
#include "gl3_ops_int8.h"          // element types

// A token of a row as one whole number that orders like (logit, lower id first); 0: nothing.  A NaN orders as nothing.
__device__ __forceinline__ uint64_t op_token_key(float x, int id) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.f);          // (-0 and +0 are equal logits)
    return (uint64_t)(b >> 31 ? ~b : b | 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float op_key_logit(uint64_t key) { const uint32_t o = (uint32_t)(key >> 32); return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ int op_key_id(uint64_t key) { return (int)~(uint32_t)key; }

// What a part of a row adds to its distribution: s = sum e^(x - m), t = sum e^(x - m) (x - m), over its logits; m its largest.
struct OpPart { float m, s, t; };
__device__ __forceinline__ OpPart op_join(const OpPart& a, const OpPart& b) {
    if (b.s == 0.f) return a;          // (nothing but -inf; a NaN is kept)
    if (a.s == 0.f) return b;
    const float m = fmaxf(a.m, b.m), da = a.m - m, db = b.m - m, ea = __expf(da), eb = __expf(db);
    return OpPart{m, a.s * ea + b.s * eb, (a.t + a.s * da) * ea + (b.t + b.s * db) * eb};
}

template <typename T>
static __global__ __launch_bounds__(256) void op_logprobs_kernel(const T* __restrict__ logits, int vocab, int64_t ld, const int32_t* __restrict__ targets, int top,
                                                                 float* __restrict__ logprob, int32_t* __restrict__ rank, float* __restrict__ entropy, int32_t* __restrict__ top_ids,
                                                                 float* __restrict__ top_logprobs) {
    __shared__ float rm[4], rs[4], rt[4];
    __shared__ int rc[4], rn[4];
    __shared__ uint64_t rk[4];
    const int64_t row = blockIdx.x;
    const T* x = logits + row * ld;
    const int t = targets ? targets[row] : -1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float xt = t >= 0 && t < vocab ? op_f32<T>(x[t]) : 0.f;
    float mx = -INFINITY;
    int bad = 0, front = 0;
    for (int i = threadIdx.x; i < vocab; i += 256) {
        const float v = op_f32<T>(x[i]);
        mx = fmaxf(mx, v);
        bad |= !(v < INFINITY);
        front += v > xt || (v == xt && i < t);
    }
    for (int d = 32; d; d >>= 1) { mx = fmaxf(mx, __shfl_xor(mx, d)); bad |= __shfl_xor(bad, d); front += __shfl_xor(front, d); }
    if (lane == 0) { rm[wave] = mx; rc[wave] = bad; rn[wave] = front; }
    __syncthreads();
    mx = fmaxf(fmaxf(rm[0], rm[1]), fmaxf(rm[2], rm[3]));
    bad = rc[0] | rc[1] | rc[2] | rc[3];
    front = rn[0] + rn[1] + rn[2] + rn[3];
    float s = 0.f, u = 0.f;
    if (!bad && mx > -INFINITY)
        for (int i = threadIdx.x; i < vocab; i += 256) {
            const float d = op_f32<T>(x[i]) - mx, e = expf(d);
            s += e;
            if (e > 0.f) u += e * d;
        }
    for (int d = 32; d; d >>= 1) { s += __shfl_xor(s, d); u += __shfl_xor(u, d); }
    if (lane == 0) { rs[wave] = s; rt[wave] = u; }
    __syncthreads();
    s = rs[0] + rs[1] + rs[2] + rs[3];
    u = rt[0] + rt[1] + rt[2] + rt[3];
    const bool none = !bad && mx == -INFINITY;
    const float nan = __uint_as_float(0x7fc00000u), ls = logf(s);
    auto lp = [&](float v) { return bad ? nan : none ? -INFINITY : (v - mx) - ls; };
    if (threadIdx.x == 0) {
        if (targets) {
            logprob[row] = t < 0 ? 0.f : t >= vocab ? nan : lp(xt);
            rank[row] = t < 0 || t >= vocab || xt != xt ? 0 : front + 1;
        }
        if (entropy) entropy[row] = bad ? nan : none ? 0.f : ls - u / s;
    }
    uint64_t last = ~0ull;
    for (int j = 0; j < top; ++j) {
        uint64_t best = 0;
        for (int i = threadIdx.x; i < vocab; i += 256) {
            const uint64_t key = op_token_key(op_f32<T>(x[i]), i);
            if (key < last && key > best) best = key;
        }
        for (int d = 32; d; d >>= 1) { const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)best, d); best = o > best ? o : best; }
        __syncthreads();
        if (lane == 0) rk[wave] = best;
        __syncthreads();
        for (int q = 0; q < 4; ++q) best = rk[q] > best ? rk[q] : best;
        if (threadIdx.x == 0) {
            top_ids[row * top + j] = best ? op_key_id(best) : -1;
            top_logprobs[row * top + j] = best ? lp(op_key_logit(best)) : -INFINITY;
        }
        last = best;
    }
}
