// gl3_ops_logprobs.h — log probabilities of given tokens, entropy and the most probable tokens of rows of logits (include/gpullama3_hip.h).
//
// One pass over the logits.  A wavefront keeps, for what it has seen of a row: the largest logit m (one value, all lanes), per lane
// s = sum e^(x - m) and t = sum e^(x - m) (x - m) (a new maximum scales both, once per batch of 32 logits a lane at most), how many logits stand
// in front of the given one, and the best 64 tokens, one a lane, sorted.  A batch touches the list only if one of its logits reaches the smallest
// of the `top` kept (lo): such logits are collected in LDS, 64 at a time are sorted (bitonic network) and merged.  lo comes from the
// largest logits of the lanes (behind batch 1, 2, 4, ...), so the first batch adds about `top` candidates and not all it holds.
// What bounds it (us): float32 reads (512 x 128256: 46 without alternatives, 5.7 TB/s); 16-bit logits arithmetic, 10 vector instructions a logit, of them four or
// five for entropy and rank, asked for or not (1500 x 32064 bfloat16 22, 13.8 for the bytes), alternatives on top of it: bounds 3.5, candidates 4.5 (5 of them) .. 7.5 (20).  A row alone: the launches.
// Tried: bounds behind batch 1, 4, 16 (2 % less), at every half more (5 % more); candidates found without branches (36 -> 40); maxima of three by hand (same).
// With P = sum p (x - m) = t / s:  lse = m + ln s,  logprob = (x_t - m) - ln s,  entropy = ln s - P: both terms >= 0, nothing cancels.
// e^d is the hardware's power of two of d log2 e, whose product is rounded once more than a library's argument: |d| half steps of a term.  Against 64 bits at
// 512 x 128256 float32 the entropies are off by 1.5e-7 (the same sums from torch's functions in float32 8e-8), the log probabilities by 5.1e-8 (5.5e-8).
#pragma once
#include "gl3_ops_int8.h"          // element types

// A token of a row as one whole number that orders like (logit, lower id first); 0: nothing.  A NaN orders as nothing.
__device__ __forceinline__ uint64_t op_token_key(float x, int id) {
    const uint32_t b = __float_as_uint(x + 0.f);          // (-0 and +0 are equal logits)
    return (uint64_t)(b >> 31 ? ~b : b | 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float op_key_logit(uint64_t key) { const uint32_t o = (uint32_t)(key >> 32); return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ int op_key_id(uint64_t key) { return (int)~(uint32_t)key; }
// the next float32 above x (NaN above +inf and NaN: nothing is)
__device__ __forceinline__ float op_above(float x) {
    if (!(x < INFINITY)) return __uint_as_float(0x7fc00000u);
    if (x == 0.f) return __uint_as_float(1u);
    const uint32_t b = __float_as_uint(x);
    return __uint_as_float(b >> 31 ? b - 1 : b + 1);
}

// ---- lanes ----------------------------------------------------------------------------------------------------------------------------
template <int M> __device__ __forceinline__ uint32_t op_xor_lane(uint32_t v) {          // the value of lane (lane ^ M)
    if constexpr (M == 1) return __builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, true);
    else if constexpr (M == 2) return __builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, true);
    else if constexpr (M == 4) return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, true), 0x1B, 0xf, 0xf, true);          // 7 - i, then i ^ 3
    else if constexpr (M == 8) return __builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, true);          // rows of 16, turned by 8
    else {          // the instruction swaps odd rows (halves) of its first register with even ones of its second: of one value, both neighbours
        const auto r = [&] { if constexpr (M == 16) return __builtin_amdgcn_permlane16_swap(v, v, false, false); else return __builtin_amdgcn_permlane32_swap(v, v, false, false); }();
        return threadIdx.x & M ? r[0] : r[1];
    }
}
template <int M> __device__ __forceinline__ float op_xor_lane(float v) { return __uint_as_float(op_xor_lane<M>(__float_as_uint(v))); }
template <int M> __device__ __forceinline__ uint64_t op_xor_lane(uint64_t v) { return (uint64_t)op_xor_lane<M>((uint32_t)(v >> 32)) << 32 | op_xor_lane<M>((uint32_t)v); }
template <typename V, typename F> __device__ __forceinline__ V op_all_lanes(V v, F f) {
    v = f(v, op_xor_lane<1>(v)); v = f(v, op_xor_lane<2>(v)); v = f(v, op_xor_lane<4>(v));
    v = f(v, op_xor_lane<8>(v)); v = f(v, op_xor_lane<16>(v)); return f(v, op_xor_lane<32>(v));
}
__device__ __forceinline__ float op_wave_max(float v) { return op_all_lanes(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float op_wave_sum(float v) { return op_all_lanes(v, [](float a, float b) { return a + b; }); }
// One step of a bitonic network: of two lanes M apart the one with (lane & M) == 0 gets the larger value where DOWN has its bit, else the smaller.
// Which lane takes what is a constant of the step, so a step is the exchange, one comparison and a select by a mask that the scalar unit makes.
constexpr uint64_t op_low_lanes(int m) { return m == 1 ? 0x5555555555555555ull : m == 2 ? 0x3333333333333333ull : m == 4 ? 0x0f0f0f0f0f0f0f0full : m == 8 ? 0x00ff00ff00ff00ffull : m == 16 ? 0x0000ffff0000ffffull : m == 32 ? 0x00000000ffffffffull : ~0ull; }
template <int M, uint64_t DOWN, typename V> __device__ __forceinline__ V op_exchange(V v) {
    const V o = op_xor_lane<M>(v);
    constexpr uint64_t larger = ~(op_low_lanes(M) ^ DOWN);          // lanes that keep the larger value
    return __builtin_amdgcn_inverse_ballot_w64(~(__builtin_amdgcn_ballot_w64(o > v) ^ larger)) ? o : v;
}
template <int M, uint64_t DOWN, typename V> __device__ __forceinline__ V op_clean(V v) {          // bitonic runs of 2 M values, sorted
    v = op_exchange<M, DOWN>(v);
    if constexpr (M > 1) v = op_clean<M / 2, DOWN>(v);
    return v;
}
template <bool FALLING, typename V> __device__ __forceinline__ V op_sort64(V v) {          // FALLING: largest in lane 0, else in lane 63
    v = op_clean<1, op_low_lanes(2)>(v); v = op_clean<2, op_low_lanes(4)>(v); v = op_clean<4, op_low_lanes(8)>(v);
    v = op_clean<8, op_low_lanes(16)>(v); v = op_clean<16, op_low_lanes(32)>(v); return op_clean<32, FALLING ? ~0ull : 0ull>(v);
}
// the 64 largest of two sorted lists of 64, one falling and one rising with the lane
__device__ __forceinline__ uint64_t op_merge64(uint64_t falling, uint64_t rising) { return op_clean<32, ~0ull>(rising > falling ? rising : falling); }
__device__ __forceinline__ float op_uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// ---- what a wavefront knows of a row -----------------------------------------------------------------------------------------------------
constexpr int OP_LP_THREADS = 256, OP_LP_WAVES = OP_LP_THREADS / 64;

struct OpSums { float m, s, t; };          // m = -inf: no logit above -inf so far (s is 0, or NaN)
__device__ __forceinline__ OpSums op_rescale(OpSums a, float m) {          // to a larger maximum
    if (a.m == m || a.m == -INFINITY) { a.m = m; return a; }
    const float d = a.m - m, e = __expf(d);
    // (d = -inf: nothing of a is left)
    return OpSums{m, a.s * e, fmaf(a.s, fmaxf(d, -200.f), a.t) * e};
}
__device__ __forceinline__ OpSums op_join(const OpSums& a, const OpSums& b) {
    const float m = fmaxf(a.m, b.m);
    const OpSums x = op_rescale(a, m), y = op_rescale(b, m);
    return OpSums{m, x.s + y.s, x.t + y.t};
}

struct OpTop {
    uint64_t key;            // the list: lane i holds the i-th best token so far (0: none)
    float lo;                // a logit below it cannot enter
    int n;                   // collected candidates
    bool any_key;
    float mine;              // the largest logit this lane has seen
    int seen, next;          // batches; lo is put up behind batch 1, 2, 4, ...
    __device__ __forceinline__ void init() { key = 0; lo = -3.402823466e38f; n = 0; any_key = false; mine = -INFINITY; seen = 0; next = 1; }
    static __device__ __forceinline__ float logit(uint32_t ord) { return __uint_as_float(ord >> 31 ? ord & 0x7fffffffu : ~ord); }
    // Nothing below the top-th largest of what this wavefront's lanes have seen at most can enter: `top` of them have seen as much.  Nor below what a quarter of
    // `top` lanes of each of the four wavefronts have seen.  (All wavefronts come here together.)
    __device__ __forceinline__ void batch_max(float mx, int top, uint32_t (*bound)[OP_LP_WAVES], int wave) {
        mine = fmaxf(mine, mx);
        if (++seen < next) return;
        next = 2 * seen;
        const uint32_t k = __float_as_uint(mine), ord = op_sort64<true>(k >> 31 ? ~k : k | 0x80000000u);
        uint32_t* b = bound[__builtin_ctz(seen) & 1];          // (the last bounds may still be read)
        if ((threadIdx.x & 63) == 0) b[wave] = __builtin_amdgcn_readlane(ord, (top + OP_LP_WAVES - 1) / OP_LP_WAVES - 1);
        __syncthreads();
        uint32_t least = b[0];
#pragma unroll
        for (int w = 1; w < OP_LP_WAVES; ++w) least = min(least, b[w]);
        lo = fmaxf(lo, fmaxf(logit(__builtin_amdgcn_readlane(ord, top - 1)), logit(__builtin_amdgcn_readfirstlane(least))));
    }
    // 64 of the collected candidates, or what is left of them, into the list
    __device__ __forceinline__ void merge(uint64_t* buf, int lane) {
        const int first = max(0, n - 64);
        const uint64_t c = first + lane < n ? buf[first + lane] : 0;
        n = first;
        key = any_key ? op_merge64(key, op_sort64<false>(c)) : op_sort64<true>(c);
        any_key = true;
    }
    // logits behind the ones in the list (higher ids) have to exceed its last one
    __device__ __forceinline__ void raise(int top, int lane) {
        const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(key >> 32), top - 1);
        if (hi) lo = fmaxf(lo, op_above(op_key_logit((uint64_t)hi << 32)));
    }
    __device__ __forceinline__ void collect(uint64_t* buf, float x, int id, bool ok) {
        const uint64_t pass = __ballot(ok);
        if (!pass) return;
        asm volatile("" : "+v"(x), "+v"(id));          // (or the keys of all logits are made ahead of the loop around this: 104 instructions a batch)
        if (ok) buf[n + __popcll(pass & ((1ull << (threadIdx.x & 63)) - 1ull))] = op_token_key(x, id);
        n += __popcll(pass);
    }
};

// One vector of 16 bytes of logits
template <typename T> struct OpVec { static constexpr int N = 16 / (int)sizeof(T); };
template <typename T> __device__ __forceinline__ void op_unpack(const uint4& v, float* x) {
    if constexpr (sizeof(T) == 4) { x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w); }
    else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = op_f32<T>(__builtin_bit_cast(T, (uint16_t)w[i]));
            x[2 * i + 1] = op_f32<T>(__builtin_bit_cast(T, (uint16_t)(w[i] >> 16)));
        }
    }
}

// What a part of a row leaves for the join: OpPartHead, then `top` keys.
struct OpPartHead { float m, s, t; int front; };
static inline __host__ __device__ uint64_t op_part_bytes(int top) { return sizeof(OpPartHead) + 8ull * top; }

struct OpRowOut { const int32_t* targets; int top; float *logprob; int32_t* rank; float* entropy; int32_t* top_ids; float* top_logprobs; };

// One wavefront writes a row's results; k: lane i holds the i-th best token.
__device__ __forceinline__ void op_row_results(const OpRowOut& o, int64_t row, int vocab, float xt, const OpSums& a, int front, uint64_t k, int lane) {
    const float nan = __uint_as_float(0x7fc00000u);
    const bool bad = !(a.s < INFINITY) || a.m == INFINITY, none = !bad && a.m == -INFINITY;
    const float ls = logf(a.s);
    auto lp = [&](float v) { return bad ? nan : none ? -INFINITY : (v - a.m) - ls; };
    if (lane == 0) {
        if (o.targets) {
            const int t = o.targets[row];
            o.logprob[row] = t < 0 ? 0.f : t >= vocab ? nan : lp(xt);
            o.rank[row] = t < 0 || t >= vocab || xt != xt ? 0 : front + 1;
        }
        if (o.entropy) o.entropy[row] = bad ? nan : none ? 0.f : ls - a.t / a.s;
    }
    if (lane < o.top) {
        o.top_ids[row * o.top + lane] = k ? op_key_id(k) : -1;
        o.top_logprobs[row * o.top + lane] = k ? lp(op_key_logit(k)) : -INFINITY;
    }
}

// Grid: x = parts of a row, y = rows (row0 + blockIdx.y).  A part is `per` vectors, a multiple of a workgroup's batch of 256 U; the fewer than
// 2 x 16 bytes of a row in front of its first whole vector and behind its last one belong to part 0.  parts == 1: the row's results; else a record.
template <typename T, int U, bool TOP>
static __global__ __launch_bounds__(OP_LP_THREADS, 5) void op_logprobs_kernel(const T* __restrict__ logits, int vocab, int64_t ld, int64_t row0, int per, OpRowOut o, uint8_t* __restrict__ parts) {
    constexpr int V = OpVec<T>::N, NT = OP_LP_THREADS;
    __shared__ uint64_t buf_s[TOP ? OP_LP_WAVES : 1][TOP ? 64 * V + 64 : 1];
    __shared__ OpSums sums_s[OP_LP_WAVES];
    __shared__ uint32_t bound_s[2][OP_LP_WAVES];
    __shared__ int got_s[OP_LP_WAVES];          // a wavefront's candidates that are in no list, and whether it has a list (at its buffer's 64)
    __shared__ int front_s[OP_LP_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = row0 + blockIdx.y;
    const T* x = logits + row * ld;
    uint64_t* buf = buf_s[TOP ? wave : 0];
    const int head = min(vocab, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T)), nv = (vocab - head) / V, tail = vocab - head - nv * V;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    const int v0 = blockIdx.x * per, v1 = min(nv, v0 + per);
    const int t = o.targets ? o.targets[row] : -1;
    const bool given = t >= 0 && t < vocab;
    const float nan = __uint_as_float(0x7fc00000u), xt = given ? op_f32<T>(x[t]) : nan, xt_above = op_above(xt);          // (NaN: no logit is counted)

    float m = -INFINITY, s[2] = {0.f, 0.f}, u[2] = {0.f, 0.f};
    int front = 0;
    OpTop best;
    best.init();
    auto load = [&](uint4* raw, int b) {          // vectors b + 256 i + thread of the row (behind the part's end: its last one again)
#pragma unroll
        for (int i = 0; i < U; ++i) { const op_v4i q = __builtin_nontemporal_load(reinterpret_cast<const op_v4i*>(xv) + min(b + NT * i + (int)threadIdx.x, v1 - 1)); raw[i] = __builtin_bit_cast(uint4, q); }
    };
    auto batch = [&](const uint4* raw, int b, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        float a[U][V], vm[U];
        bool in[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            in[i] = WHOLE || b + NT * i + (int)threadIdx.x < v1;
            op_unpack<T>(raw[i], a[i]);
            if (!WHOLE && !in[i])
#pragma unroll
                for (int e = 0; e < V; ++e) a[i][e] = -INFINITY;
            vm[i] = a[i][0];
#pragma unroll
            for (int e = 1; e < V; ++e) vm[i] = fmaxf(vm[i], a[i][e]);
        }
        float mx = vm[0];
#pragma unroll
        for (int i = 1; i < U; ++i) mx = fmaxf(mx, vm[i]);
        if (__any(mx > m)) {
            const OpSums n0 = op_rescale(OpSums{m, s[0], u[0]}, op_wave_max(fmaxf(mx, m))), n1 = op_rescale(OpSums{m, s[1], u[1]}, n0.m);
            s[0] = n0.s; u[0] = n0.t; s[1] = n1.s; u[1] = n1.t;
            m = op_uniform(n0.m);
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int id = head + (b + NT * i + (int)threadIdx.x) * V;
            const float th = t >= id + V ? xt : xt_above;          // (the vector that holds t is put right below)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = a[i][e] - ref, p = __builtin_amdgcn_exp2f(d * 1.44269504f);
                s[e & 1] += p;
                u[e & 1] = fmaf(p, fmaxf(d, -200.f), u[e & 1]);          // (0 x -inf stays out; e^-200 is 0)
                front += __popcll(__ballot(a[i][e] >= th && (WHOLE || in[i])));
            }
        }
        if constexpr (TOP) {
            best.batch_max(mx, o.top, bound_s, wave);
            int i0 = 0;
            while (i0 < U && __any(mx >= best.lo)) {          // from vector i0 on: until 64 are together
                int next = U;
#pragma unroll
                for (int i = 0; i < U; ++i)
                    if (i >= i0 && i < next && __any(vm[i] >= best.lo)) {
                        const int id = head + (b + NT * i + (int)threadIdx.x) * V;
#pragma unroll
                        for (int e = 0; e < V; ++e) best.collect(buf, a[i][e], id + e, a[i][e] >= best.lo);
                        if (best.n >= 64) next = i + 1;
                    }
                i0 = next;
                if (best.n >= 64) {
                    do best.merge(buf, lane); while (best.n >= 64);
                    best.raise(o.top, lane);
                }
            }
        }
    };
    // the next batch is on its way while this one is worked on
    if (v0 < v1) {
        uint4 r0[U], r1[U];
        int b = v0;
        load(r0, b);
        for (; b + 2 * NT * U <= v1; b += 2 * NT * U) {
            load(r1, b + NT * U);
            batch(r0, b, std::true_type{});
            if (b + 2 * NT * U < v1) load(r0, b + 2 * NT * U);
            batch(r1, b + NT * U, std::true_type{});
        }
        if (b + NT * U <= v1) {
            if (b + NT * U < v1) load(r1, b + NT * U);
            batch(r0, b, std::true_type{});
            b += NT * U;
#pragma unroll
            for (int i = 0; i < U; ++i) r0[i] = r1[i];
        }
        if (b < v1) batch(r0, b, std::false_type{});
    }
    if (blockIdx.x == 0 && wave == 0) {          // the row's ends, one logit a lane
        const int id = lane < 32 ? lane : head + nv * V + lane - 32;
        const bool in = lane < 32 ? lane < head : lane - 32 < tail;
        const float v = in ? op_f32<T>(x[id]) : -INFINITY;
        if (__any(v > m)) {
            const OpSums n0 = op_rescale(OpSums{m, s[0], u[0]}, op_wave_max(fmaxf(v, m))), n1 = op_rescale(OpSums{m, s[1], u[1]}, n0.m);
            s[0] = n0.s; u[0] = n0.t; s[1] = n1.s; u[1] = n1.t;
            m = op_uniform(n0.m);
        }
        const float d = v - (m == -INFINITY ? 0.f : m), p = __expf(d);
        s[0] += p;
        u[0] = fmaf(p, fmaxf(d, -200.f), u[0]);
        front += __popcll(__ballot(in && (v > xt || (v == xt && id < t))));
        if constexpr (TOP) {
            // ids of the head are lower than the list's: equal to its last one is enough
            best.collect(buf, v, id, in && v > -INFINITY);
        }
    }
    if constexpr (TOP) {
        while (best.n >= 64) best.merge(buf, lane);
        if (best.any_key) buf[64 + lane] = best.key;
        if (lane == 0) got_s[wave] = best.n | (best.any_key ? 256 : 0);
    }
    // logits of t's own vector that stand in front of it with the same value
    if (given && t >= head && t < head + nv * V && (t - head) / V >= v0 && (t - head) / V < v1 && wave == 0) {
        const int first = head + (t - head) / V * V;
        front += __popcll(__ballot(lane < t - first && op_f32<T>(x[first + min(lane, t - first)]) == xt));
    }
    const OpSums mine{m, op_wave_sum(s[0] + s[1]), op_wave_sum(u[0] + u[1])};
    if (lane == 0) { sums_s[wave] = mine; front_s[wave] = front; }
    __syncthreads();
    if (wave) return;
    OpSums all = mine;
#pragma unroll
    for (int w = 1; w < OP_LP_WAVES; ++w) {
        all = op_join(all, sums_s[w]);
        front += front_s[w];
    }
    if constexpr (TOP) {          // one list of all: the candidates 64 at a time, then the lists there are
        int end[OP_LP_WAVES], n = 0;
#pragma unroll
        for (int w = 0; w < OP_LP_WAVES; ++w) end[w] = n += got_s[w] & 255;
        uint64_t key = 0;
        for (int i = 0; i < n; i += 64) {
            const int at = i + lane, w = (at >= end[0]) + (at >= end[1]) + (at >= end[2]);
            const uint64_t c = at < n ? buf_s[w][at - (w == 0 ? 0 : w == 1 ? end[0] : w == 2 ? end[1] : end[2])] : 0;
            key = i == 0 ? op_sort64<true>(c) : op_merge64(key, op_sort64<false>(c));
        }
#pragma unroll
        for (int w = 0; w < OP_LP_WAVES; ++w) if (got_s[w] & 256) key = op_merge64(key, buf_s[w][64 + 63 - lane]);
        best.key = key;
    }
    if (gridDim.x == 1) op_row_results(o, row, vocab, xt, all, front, best.key, lane);
    else {
        uint8_t* rec = parts + ((uint64_t)row * gridDim.x + blockIdx.x) * op_part_bytes(o.top);
        if (lane == 0) *reinterpret_cast<OpPartHead*>(rec) = OpPartHead{all.m, all.s, all.t, front};
        if (TOP && lane < o.top) reinterpret_cast<uint64_t*>(rec + sizeof(OpPartHead))[lane] = best.key;
    }
}

// The parts of a row (at most 64), joined by one workgroup: lane i of every wavefront holds part i's sums, wavefront w the lists of parts w, w + 8, ...;
// all are on their way before the first is looked at (63 parts of 20 tokens one after the other: 18.2 us).
constexpr int OP_LP_JOIN_WAVES = 8;
template <typename T>
static __global__ __launch_bounds__(64 * OP_LP_JOIN_WAVES) void op_logprobs_join_kernel(const T* __restrict__ logits, int vocab, int64_t ld, int n, OpRowOut o, const uint8_t* __restrict__ parts) {
    constexpr int LISTS = 64 / OP_LP_JOIN_WAVES;
    __shared__ uint64_t buf[64 * 64];
    __shared__ int count;
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), top = o.top;
    const uint64_t bytes = op_part_bytes(top);
    const uint8_t* rec = parts + (uint64_t)row * n * bytes;
    const bool in = lane < n;
    OpPartHead h{-INFINITY, 0.f, 0.f, 0};
    uint64_t some = 0, k[LISTS];
    if (wave == 0 && in) h = *reinterpret_cast<const OpPartHead*>(rec + lane * bytes);
    const int t = o.targets ? o.targets[row] : -1;
    const float xt = t >= 0 && t < vocab ? op_f32<T>(logits[row * ld + t]) : 0.f;
    OpTop best;
    best.init();
    if (top > 0) {
        // q of the parts have j tokens each that are no worse than the q-th best of their j-th ones: with j q >= top nothing below that is among the first `top`
        const int j = (top + n - 1) / n;
        if (in) some = reinterpret_cast<const uint64_t*>(rec + lane * bytes + sizeof(OpPartHead))[j - 1];
#pragma unroll
        for (int i = 0; i < LISTS; ++i) {
            const int p = wave + OP_LP_JOIN_WAVES * i;
            k[i] = p < n && lane < top ? reinterpret_cast<const uint64_t*>(rec + p * bytes + sizeof(OpPartHead))[lane] : 0;
        }
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        const int q = (top + j - 1) / j;
        some = op_sort64<true>(some);
        const uint64_t least = (uint64_t)__builtin_amdgcn_readlane((uint32_t)(some >> 32), q - 1) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)some, q - 1);
#pragma unroll
        for (int i = 0; i < LISTS; ++i) {
            const bool ok = k[i] != 0 && k[i] >= least;
            const uint64_t pass = __ballot(ok);
            if (pass) {          // (any order: they are sorted)
                int first = 0;
                if (lane == 0) first = atomicAdd(&count, (int)__popcll(pass));
                first = __builtin_amdgcn_readfirstlane(first);
                if (ok) buf[first + __popcll(pass & ((1ull << lane) - 1ull))] = k[i];
            }
        }
        __syncthreads();
        if (wave == 0) {
            best.n = count;
            while (best.n) best.merge(buf, lane);
        }
    }
    if (wave) return;
    const float m = op_wave_max(h.m);
    const OpSums mine = op_rescale(OpSums{h.m, h.s, h.t}, m);
    const OpSums all{m, op_wave_sum(mine.s), op_wave_sum(mine.t)};
    const int front = op_all_lanes((uint32_t)h.front, [](uint32_t a, uint32_t b) { return a + b; });
    op_row_results(o, row, vocab, xt, all, front, best.key, lane);
}
