// gl3_ops_int8.h — rows in 8-bit integers with a scale each, and their products (include/gpullama3_hip.h: gl3_quantize_rows, gl3_int8_matmul).
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

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

// A thread's share of a row in registers: NV pieces of 16 bytes, nt (the threads of a row) pieces apart; zeros behind the row's end.
template <typename T, int NV> struct OpRowPart {
    static constexpr int V = 16 / (int)sizeof(T);
    T x[NV][V];
    __device__ __forceinline__ void load(const T* row, int k, int t, int nt) {
        if (((uintptr_t)row & 15) == 0) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (t + nt * i) * V;
                if (c + V <= k) *reinterpret_cast<uint4*>(x[i]) = *reinterpret_cast<const uint4*>(row + c);
                else
#pragma unroll
                    for (int e = 0; e < V; ++e) x[i][e] = c + e < k ? row[c + e] : op_cast<T>(0.f);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < V; ++e) { const int c = (t + nt * i) * V + e; x[i][e] = c < k ? row[c] : op_cast<T>(0.f); }
        }
    }
    __device__ __forceinline__ uint32_t largest() const {          // of the wavefront
        uint32_t mag = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) mag = max(mag, op_mag(op_f32<T>(x[i][e])));
        for (int d = 32; d; d >>= 1) mag = max(mag, (uint32_t)__shfl_xor((int)mag, d));
        return mag;
    }
    __device__ __forceinline__ void store(int8_t* codes, int kp, int t, int nt, float to_code) const {          // kp: the row's end with its zeros
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (t + nt * i) * V;
            if (c >= kp) continue;
            uint32_t w[V / 4];
#pragma unroll
            for (int e = 0; e < V; ++e) w[e / 4] = (e % 4 ? w[e / 4] : 0u) | (uint32_t)(uint8_t)op_code(op_f32<T>(x[i][e]), to_code) << 8 * (e % 4);
#pragma unroll
            for (int e = 0; e < V / 4; ++e) reinterpret_cast<uint32_t*>(codes + c)[e] = w[e];
        }
    }
};
// W wavefronts a row, 4 / W rows a workgroup (one where W > 4); the row stays in registers between its largest value and its codes: one read, one write.
// kp <= OP_ROW_E x 64 W.  2041 x 4096 bfloat16 9.4 us, a few rows 4 .. 5: little more than a launch.  (Two passes over memory, one element a thread and step: 8192 columns of one row 11.5 us in front of a product, 2041 x 4096 bfloat16 12.8.)
constexpr int OP_ROW_E = 32;
template <typename T, int W>
static __global__ __launch_bounds__(W > 4 ? 64 * W : 256) void op_quantize_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t ldx, int8_t* __restrict__ codes, int64_t ldq, float* __restrict__ scale) {
    __shared__ uint32_t red[W > 4 ? W : 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = threadIdx.x & (64 * W - 1);
    const int64_t row = (int64_t)blockIdx.x * (W > 4 ? 1 : 4 / W) + wave / W;
    const bool live = row < rows;
    OpRowPart<T, OP_ROW_E * (int)sizeof(T) / 16> part;
    uint32_t mag = 0;
    if (live) {
        part.load(x + row * ldx, cols, t, 64 * W);
        mag = part.largest();
    }
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) red[wave] = mag;
        __syncthreads();
        mag = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) mag = max(mag, red[wave / W * W + i]);
    }
    if (!live) return;
    float s, r;
    op_row_scale(mag, s, r);
    if (t == 0) scale[row] = s;
    part.store(codes + row * ldq, (cols + GL3_CODE_BLOCK - 1) / GL3_CODE_BLOCK * GL3_CODE_BLOCK, t, 64 * W, r);
}
// longer rows: read twice
template <typename T>
static __global__ __launch_bounds__(1024) void op_quantize_long_kernel(const T* __restrict__ x, int cols, int64_t ldx, int8_t* __restrict__ codes, int64_t ldq, float* __restrict__ scale) {
    __shared__ uint32_t red[16];
    constexpr int STEP = OP_ROW_E / 2 * 1024;
    const T* row = x + (int64_t)blockIdx.x * ldx;
    const int kp = (cols + GL3_CODE_BLOCK - 1) / GL3_CODE_BLOCK * GL3_CODE_BLOCK;
    OpRowPart<T, OP_ROW_E / 2 * (int)sizeof(T) / 16> part;
    uint32_t mag = 0;
    for (int c = 0; c < cols; c += STEP) { part.load(row + c, cols - c, threadIdx.x, 1024); mag = max(mag, part.largest()); }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mag;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i) mag = max(mag, red[i]);
    float s, r;
    op_row_scale(mag, s, r);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    for (int c = 0; c < kp; c += STEP) { part.load(row + c, cols - c, threadIdx.x, 1024); part.store(codes + (int64_t)blockIdx.x * ldq + c, kp - c, threadIdx.x, 1024, r); }
}

// ---- products -------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float op_result(int acc, float as, float ws) { return ((float)acc * as) * ws; }
// Results in whole lines of 128 bytes go past the caches: in them they push out weights on their way (64 tokens, 151936 x 2560 float32, us: through / past them
// 100 / 86; none stored 81).  Other rows need the caches, where the halves of a line meet (2000 x 39171, k = 275, float32 96 / 155, bfloat16 76 / 109).
template <typename TY> __device__ __forceinline__ void op_store_past(TY* p, TY v) {
    if constexpr (sizeof(TY) == 4) __builtin_nontemporal_store(v, p);
    else __builtin_nontemporal_store(__builtin_bit_cast(uint16_t, v), reinterpret_cast<uint16_t*>(p));
}
template <typename TY> struct OpProductArgs {
    const int8_t* a; int64_t lda; const float* as;
    const int8_t* w; int64_t ldw; const float* ws; const float* bias;
    int m, n, kp;            // kp: k rounded up to a multiple of 128
    TY* y; int64_t ldy;
};

// A few tokens: the weights' bytes are what it costs, and they go from memory to the matrix cores' registers directly.  A wavefront has 16 channels
// x 16 MT tokens (v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive k of row l % 16) and a ring of D steps of 64 k on their way; the KS wavefronts of a
// workgroup share the channels and split k (their int32 sums meet in LDS: exact in any order).  The tokens' codes come from the caches again in every
// strip, which costs 4 % of the weights' time a token (128256 x 4096, us, the least of many: 1 token 83 = 6.3 TB/s, 4 95, 16 144, 32 197; tiles 88, 92, 96, 96): op_streams compares.
// A short k starts no loads that it does not need (100000 x 256, a step a wavefront: 31 -> 13).  (Loads past the caches fetch the 128-byte lines twice, half by half: 85 -> 95.  32 or 64 channels a wavefront: 92, 97.)
template <int KS> struct OpStrip {          // the wavefront's part of a strip of 16 channels
    int lane, wave, r16, kg, n0, s0, cnt;
    const int8_t* wb;
    uint32_t wo;
    __device__ __forceinline__ OpStrip(const int8_t* w, int64_t ldw, int n, int kp) {
        lane = threadIdx.x & 63; wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); r16 = lane & 15; kg = lane >> 4;
        const int steps = kp / 64;
        s0 = steps * wave / KS; cnt = steps * (wave + 1) / KS - s0;
        n0 = (int)blockIdx.x * 16;
        wb = w + n0 * ldw + s0 * 64;          // (uniform; the lane's part fits 32 bits; rows past the end repeat the last one)
        wo = (uint32_t)(min(n0 + r16, n - 1) - n0) * (uint32_t)ldw + 16 * kg;
    }
    __device__ __forceinline__ op_v4i load(int s) const { return *reinterpret_cast<const op_v4i*>(wb + s * 64 + wo); }
};
// lane: token r16 of tile j, channels 4 kg .. of the strip
template <typename TY> __device__ __forceinline__ void op_store4(const OpProductArgs<TY>& p, const op_v4i& v, int row, int col, float sa) {
    if (row >= p.m) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (col + r < p.n) {
            const float x = op_result(v[r], sa, p.ws[col + r]);
            p.y[(int64_t)row * p.ldy + col + r] = op_cast<TY>(p.bias ? x + p.bias[col + r] : x);
        }
}
template <typename TY, int MT, int KS, int D>
static __global__ __launch_bounds__(64 * KS) void op_stream_kernel(OpProductArgs<TY> p) {
    __shared__ op_v4i part[KS][MT][64];
    const OpStrip<KS> st(p.w, p.ldw, p.n, p.kp);
    const int8_t* ab = p.a + st.s0 * 64;
    uint32_t ao[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) ao[j] = (uint32_t)min(16 * j + st.r16, p.m - 1) * (uint32_t)p.lda + 16 * st.kg;
    op_v4i acc[MT], fw[D], fa[D][MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[j] = op_v4i{0, 0, 0, 0};
    auto load = [&](int d, int s) {
        fw[d] = st.load(s);
#pragma unroll
        for (int j = 0; j < MT; ++j) fa[d][j] = *reinterpret_cast<const op_v4i*>(ab + s * 64 + ao[j]);
    };
    auto mma = [&](int d) {
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[d], fa[d][j], acc[j], 0, 0, 0);
    };
    if (st.cnt > 0) {
#pragma unroll
        for (int d = 0; d < D; ++d) if (d == 0 || d < st.cnt) load(d, d);
        int s = 0;
        for (; s + D < st.cnt; s += D)
#pragma unroll
            for (int d = 0; d < D; ++d) { mma(d); load(d, min(s + D + d, st.cnt - 1)); }
#pragma unroll
        for (int d = 0; d < D; ++d) if (s + d < st.cnt) mma(d);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j) part[st.wave][j][st.lane] = acc[j];
    __syncthreads();
    if (st.wave >= MT) return;
    op_v4i v = part[0][st.wave][st.lane];
#pragma unroll
    for (int q = 1; q < KS; ++q) v += part[q][st.wave][st.lane];
    const int row = 16 * st.wave + st.r16;
    op_store4(p, v, row, st.n0 + 4 * st.kg, p.as[min(row, p.m - 1)]);
}

// A few tokens of a linear (at most 8): every workgroup quantises the rows for itself (LDS) while its first weights are on their way, and one launch is all.  That
// costs each of them about a microsecond, more than the launch where they run in many rounds (us, this / a launch of its own for the codes; 1 token: 2048 x 2048 5.0 / 8.0,
// 14336 x 4096 15.2 / 18.0, 32000 x 2048 15.7 / 16.9, 128256 x 4096 95 / 89; 2: 4096 x 4096 8.0 / 10.7, 32000 x 4096 27.1 / 29.7; 4: 16000 x 2048 10.6 / 12.4,
// 32000 x 4096 32.4 / 31.3; 8: 8192 x 2048 8.3 / 11.3, 32000 x 2048 20.8 / 17.6; several strips a workgroup 100).  KS >> lg wavefronts have a row each, in registers: k <= OP_ROW_E x their threads.
constexpr int OP_TOKENS = 8;
template <typename TX, typename TY, int KS, int D, bool ONE>          // ONE: lg = 0
static __global__ __launch_bounds__(64 * KS) void op_token_kernel(OpProductArgs<TY> p, const TX* __restrict__ x, int64_t ldx, int k, int lg_) {
    const int lg = ONE ? 0 : lg_;
    __shared__ __attribute__((aligned(16))) int8_t codes[OP_ROW_E * 64 * KS + OP_TOKENS * 16];          // rows kp + 16 apart
    __shared__ op_v4i sums[KS][64];
    __shared__ uint32_t red[KS];
    __shared__ float scales[OP_TOKENS];
    const OpStrip<KS> st(p.w, p.ldw, p.n, p.kp);
    constexpr int LOG = KS == 8 ? 3 : 2;
    static_assert(KS == 1 << LOG, "wavefronts");
    const int row = st.wave >> (LOG - lg), nt = 64 * KS >> lg, t = threadIdx.x & (nt - 1);
    const bool live = ONE || row < p.m;
    // the rows first: loads come back in order, and the weights behind them do not hold them up
    OpRowPart<TX, OP_ROW_E * (int)sizeof(TX) / 16> part;
    if (live) part.load(x + row * ldx, k, t, nt);
    op_v4i acc = {0, 0, 0, 0}, fw[D];
#pragma unroll
    for (int d = 0; d < D; ++d) fw[d] = st.load(max(0, min(d, st.cnt - 1)));          // (branches around them hold everything up: 32000 x 2048 15.5 -> 33)
    uint32_t mag = live ? part.largest() : 0;
    if (st.lane == 0) red[st.wave] = mag;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < KS; ++q) { const uint32_t v = red[q]; mag = q >> (LOG - lg) == row ? max(mag, v) : mag; }
    if (live) {
        float scale, to_code;
        op_row_scale(mag, scale, to_code);
        if (t == 0) scales[row] = scale;
        part.store(codes + row * (p.kp + 16), p.kp, t, nt, to_code);
    }
    __syncthreads();
    const int mine = ONE ? 0 : min(st.r16, p.m - 1);
    const int8_t* cb = codes + mine * (p.kp + 16) + st.s0 * 64 + 16 * st.kg;
    if (st.cnt > 0) {
        int s = 0;
        for (; s + D < st.cnt; s += D)
#pragma unroll
            for (int d = 0; d < D; ++d) {
                acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[d], *reinterpret_cast<const op_v4i*>(cb + (s + d) * 64), acc, 0, 0, 0);
                fw[d] = st.load(min(s + D + d, st.cnt - 1));
            }
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (s + d < st.cnt) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[d], *reinterpret_cast<const op_v4i*>(cb + (s + d) * 64), acc, 0, 0, 0);
    }
    sums[st.wave][st.lane] = acc;
    __syncthreads();
    if (st.wave) return;
    op_v4i v = sums[0][st.lane];
#pragma unroll
    for (int q = 1; q < KS; ++q) v += sums[q][st.lane];
    op_store4(p, v, st.r16, st.n0 + 4 * st.kg, scales[mine]);
}

// More tokens: BM tokens x BN channels per workgroup of WM x WN wavefronts, v_mfma_i32_32x32x32_i8.  The operands go straight to LDS (16 bytes a lane, no
// registers in between) into rings of SA stages of a and SW of w, a stage being 128 k of every row; the barrier of a stage stands in front of its last
// quarter, so the matrix cores have that quarter while the next stage's first fragments are read, and it waits for all loads but those that have a
// stage left to travel.  16-byte chunk c of row r stands at chunk c ^ (r / 2 % 8): the 16 lanes of a read cover the banks once.  Workgroups go to the
// 8 XCDs in turn; the token tiles of one channel tile run on one XCD, so its weights leave HBM once.
// What bounds it: 32 x 128 and 64 x 128 tiles the weights' way through LDS (32 tokens, 151936 x 2560: 76 us, 5.1 TB/s).  256 x 256 tiles: 512 x 128256 x 4096 takes
// 255 - 310 us from card to card, 2.0 POP/s, as fast as the library's product (a short loop of nothing but these MFMAs 4.0; 8192 x 8192 x 8192 554 us, the library's 533).
// The matrix cores are busy for 62 % of the launch's cycles (256.5 k of 413 k at 1.4 GHz; 2041 x 14336 x 4096 61 %).  Stamps in one workgroup gave 2030 MFMA cycles
// of 2048 - 2080 a stage, 1.5 - 4 us in front of a tile's first stage and 3.3 (bfloat16) - 4.8 us (float32) for its results: four rounds of tiles make that a
// fifth to a third of the idle cycles, and what takes the others is not known.
// Tried: 64 k a stage with a longer ring of weights, loads by some wavefronts and MFMAs by others (62 -> 85 us at 512 x 28672 x 4096); four wavefronts of
// 128 x 128 (same); one workgroup a CU that goes through its tiles without a pause (same); priorities, one or three reads behind an MFMA (same).
__device__ __forceinline__ void op_dma16(const void* src, void* lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}
template <int I, int N, typename F> __device__ __forceinline__ void op_static_for(F f) { if constexpr (I < N) { f(std::integral_constant<int, I>{}); op_static_for<I + 1, N>(f); } }
// all but the newest N loads of this wavefront have landed, its LDS reads are done, and so are everybody's
template <int N> __device__ __forceinline__ void op_wait_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory"); }

// TY = int: part blockIdx.y of gridDim.y of the sum over k, y[part][m][ldy] (op_parts_kernel adds them up).
template <typename TY, int BM, int BN, int WM, int WN, int SA, int SW>
static __global__ __launch_bounds__(WM * WN * 64, 1) void op_ring_kernel(OpProductArgs<TY> p, int mt, int nt) {
    constexpr bool PART = std::is_same<TY, int>::value;
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int PA = BM / 8, PW = BN / 8, NPA = (PA + NW - 1) / NW, NPW = (PW + NW - 1) / NW, NP = NPA + NPW;          // 1 KB pieces (8 rows) of a stage, per wavefront
    constexpr int SZA = BM * 128, SZW = BN * 128, OW = SA * SZA;
    static_assert(SW >= SA + 1 && SA >= 2 && TM * WM * 32 == BM && TN * WN * 32 == BN, "tile layout");
    static_assert(SA * SZA + SW * SZW <= 160 * 1024 && BM <= NW * 64 && BN <= NW * 64, "LDS; a scale per thread");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[SA * SZA + SW * SZW];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    const int total = mt * nt, per_xcd = (total + 7) >> 3, J = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (J >= total) return;
    const int m0 = (J % mt) * BM, n0 = (J / mt) * BN, stages = p.kp / 128;
    const int it0 = PART ? stages * (int)blockIdx.y / (int)gridDim.y : 0, n_it = PART ? stages * ((int)blockIdx.y + 1) / (int)gridDim.y - it0 : stages;
    const int8_t *ab = p.a + m0 * p.lda + it0 * 128, *wb = p.w + n0 * p.ldw + it0 * 128;
    if constexpr (PART) p.y += (int64_t)blockIdx.y * p.m * p.ldy;
    // this wavefront's pieces (rows past the end repeat the last one: their results are not stored; wavefronts without a piece of their own load one again)
    uint32_t offa[NPA], offw[NPW];
    int pa[NPA], pw[NPW];
#pragma unroll
    for (int u = 0; u < NPA; ++u) {
        const int q = (wave + NW * u) % PA, row = 8 * q + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
        pa[u] = q * 1024;
        offa[u] = (uint32_t)(min(m0 + row, p.m - 1) - m0) * (uint32_t)p.lda + 16 * c;
    }
#pragma unroll
    for (int u = 0; u < NPW; ++u) {
        const int q = (wave + NW * u) % PW, row = 8 * q + (lane >> 3), c = (lane & 7) ^ ((row >> 1) & 7);
        pw[u] = OW + q * 1024;
        offw[u] = (uint32_t)(min(n0 + row, p.n - 1) - n0) * (uint32_t)p.ldw + 16 * c;
    }
    // scales of the tile's rows and columns, one a thread: needed at the end, in LDS
    const int my_m = min(m0 + (tid < BM ? tid : 0), p.m - 1), my_n = min(n0 + (tid < BN ? tid : 0), p.n - 1);
    const float my_as = PART ? 0.f : p.as[my_m], my_ws = PART ? 0.f : p.ws[my_n], my_b = !PART && p.bias ? p.bias[my_n] : 0.f;
    constexpr int WH = (NPW + 1) / 2;
    auto issue_a = [&](int it, int slot) {
        const int8_t* a = ab + (int64_t)it * 128;
#pragma unroll
        for (int u = 0; u < NPA; ++u) op_dma16(a + offa[u], smem + slot * SZA + pa[u]);
    };
    auto issue_w = [&](int it, int slot, int u0, int u1) {
        const int8_t* w = wb + (int64_t)it * 128;
#pragma unroll
        for (int u = 0; u < NPW; ++u)
            if (u >= u0 && u < u1) op_dma16(w + offw[u], smem + slot * SZW + pw[u]);
    };
    op_v16i acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
    const int r32 = lane & 31, kh = lane >> 5;
    uint32_t ca[4];          // a stage is four quarters of 32 k: a lane reads row lane % 32, chunk 2 quarter + lane / 32
#pragma unroll
    for (int q = 0; q < 4; ++q) ca[q] = ((2 * q + kh) ^ ((r32 >> 1) & 7)) * 16;
    const uint32_t aw = (wm * (BM / WM) + r32) * 128, ww = OW + (wn * (BN / WN) + r32) * 128;
    // step s (behind barrier s) starts the loads of a's stage s + SA (into the slot the barrier freed) and, in the two quarters after it, of w's stage
    // s + SW; the steps before 0 are the prologue, the last one's w belongs to the loop's first round
    constexpr int LEFT = (SA - 2) * NP + NPW;          // loads started behind a's stage s + 1 when barrier s waits for it
#pragma unroll
    for (int s = -SW; s < 0; ++s) {
        if (s + SA >= 0 && s + SA < n_it) issue_a(s + SA, s + SA);
        if (s < -1 && s + SW < n_it) issue_w(s + SW, s + SW, 0, NPW);
    }
    if (n_it >= SW) op_wait_barrier<(SA - 1) * NP>(); else op_wait_barrier<0>();
    int sa = 0, sw = 0, sp = SW - 1, it = 0;          // slots of the current stage; sp: the w slot that the step before fills
    op_v4i fa[2][TM], fw[2][TN];
    constexpr int NR = TM + TN, NM = TM * TN;
    auto rd1 = [&](int set, int q, int f) {          // fragment f of a quarter: TM of a, TN of w
        if (f < TM) fa[set][f] = *reinterpret_cast<const op_v4i*>(smem + sa * SZA + aw + f * 4096 + ca[q]);
        else fw[set][f - TM] = *reinterpret_cast<const op_v4i*>(smem + sw * SZW + ww + (f - TM) * 4096 + ca[q]);
    };
    // A quarter: its MFMAs with the next quarter's fragment reads (RPM behind each of the first ones) and then ND loads between them, in this very order
    // (all reads have to stand in front of the loads: both are in LDS, and nobody tells the compiler that they are apart).  The reads are waited for at its
    // end, where the compiler sees it (else it waits in front of the next quarter's first MFMA for a read that has just been started as well).
    constexpr int RPM = 2, NRM = (NR + RPM - 1) / RPM;
    auto quarter = [&](auto set_, auto q_, bool more, auto nd_, auto load) {
        constexpr int set = decltype(set_)::value, q = decltype(q_)::value, ND = decltype(nd_)::value, ROOM = NM > NRM ? NM - NRM : 1;
        op_static_for<0, NM>([&](auto c_) {
            constexpr int c = decltype(c_)::value;
            acc[c / TN][c % TN] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[set][c / TN], fw[set][c % TN], acc[c / TN][c % TN], 0, 0, 0);
            if constexpr (c < NRM || c == NM - 1) {
                if (more)
                    op_static_for<0, (c == NM - 1 && c < NRM ? NR : RPM)>([&](auto f) { constexpr int fr = c * RPM + decltype(f)::value; if constexpr (fr < NR) rd1(1 - set, q, fr); });
            }
            if constexpr (NM <= NRM) { if constexpr (c == NM - 1) op_static_for<0, ND>([&](auto u) { load(u); }); }
            else if constexpr (c >= NRM) op_static_for<(c - NRM) * ND / ROOM, (c - NRM + 1) * ND / ROOM>([&](auto u) { load(u); });
            __builtin_amdgcn_sched_barrier(0);
        });
        __builtin_amdgcn_s_waitcnt(0xc07f);
    };
    constexpr std::integral_constant<int, 0> I0{};
    constexpr std::integral_constant<int, 1> I1{};
    constexpr std::integral_constant<int, 2> I2{};
    constexpr std::integral_constant<int, 3> I3{};
    constexpr std::integral_constant<int, WH> IW0{};
    constexpr std::integral_constant<int, NPW - WH> IW1{};
    constexpr std::integral_constant<int, NPA> IA{};
    auto nothing = [](auto) {};
    op_static_for<0, NR>([&](auto f) { rd1(0, 0, decltype(f)::value); });
    __builtin_amdgcn_s_waitcnt(0xc07f);
    for (; it < n_it - SW; ++it) {
        const int8_t* gw = wb + (int64_t)(it - 1 + SW) * 128;
        uint8_t* dw = smem + sp * SZW;
        quarter(I0, I1, true, IW0, [&](auto u) { constexpr int v = decltype(u)::value; op_dma16(gw + offw[v], dw + pw[v]); });
        quarter(I1, I2, true, IW1, [&](auto u) { constexpr int v = WH + decltype(u)::value; op_dma16(gw + offw[v], dw + pw[v]); });
        quarter(I0, I3, true, I0, nothing);
        op_wait_barrier<LEFT>();
        const int8_t* ga = ab + (int64_t)(it + SA) * 128;
        uint8_t* da = smem + sa * SZA;
        sp = sw;
        if (++sa == SA) sa = 0;
        if (++sw == SW) sw = 0;
        quarter(I1, I0, true, IA, [&](auto u) { constexpr int v = decltype(u)::value; op_dma16(ga + offa[v], da + pa[v]); });
    }
    if (it - 1 + SW < n_it) issue_w(it - 1 + SW, sp, 0, NPW);
    for (; it < n_it; ++it) {          // the last SW stages: nothing (a: little) left to load
        quarter(I0, I1, true, I0, nothing);
        quarter(I1, I2, true, I0, nothing);
        quarter(I0, I3, true, I0, nothing);
        op_wait_barrier<0>();
        if (it + SA < n_it) issue_a(it + SA, sa);
        if (++sa == SA) sa = 0;
        if (++sw == SW) sw = 0;
        quarter(I1, I0, it + 1 < n_it, I0, nothing);
    }
    // Lane holds channel lane % 32 and tokens 8 (r / 4) + 4 (lane / 32) + r % 4 of every 32 x 32 tile.  A store's row comes from the scalar unit, the lane's
    // part is one 32-bit offset.  (Behind the last barrier nobody reads the rings and no load is on its way.)
    float *las = reinterpret_cast<float*>(smem), *lws = las + BM, *lb = lws + BN;
    if constexpr (!PART) {
        if (tid < BM) las[tid] = my_as;
        if (tid < BN) { lws[tid] = my_ws; lb[tid] = my_b; }
        __syncthreads();
    }
    const int mb = m0 + wm * (BM / WM), nb = n0 + wn * (BN / WN);
    const bool whole = m0 + BM <= p.m && n0 + BN <= p.n, biased = p.bias != nullptr;
    const uint32_t lo = ((uint32_t)(4 * kh) * (uint32_t)p.ldy + r32) * (uint32_t)sizeof(TY);
    auto store = [&](auto all, auto past) {
        constexpr bool ALL = decltype(all)::value, PAST = decltype(past)::value;
        float w_[TN], b_[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) { const int c = wn * (BN / WN) + j * 32 + r32; w_[j] = PART ? 0.f : lws[c]; b_[j] = PART ? 0.f : lb[c]; }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float* s4 = las + wm * (BM / WM) + i * 32 + 8 * g + 4 * kh;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = mb + i * 32 + 8 * g + r;          // (of lanes 0 .. 31)
                    uint8_t* y = reinterpret_cast<uint8_t*>(p.y + row * p.ldy + nb);
#pragma unroll
                    for (int j = 0; j < TN; ++j) {          // (a row's columns one behind the other: with the rows inside, 13.4 us a float32 tile of 256 x 256 instead of 5)
                        const bool in = ALL || (row + 4 * kh < p.m && nb + j * 32 + r32 < p.n);
                        TY* at = reinterpret_cast<TY*>(y + j * 32 * sizeof(TY) + lo);
                        if constexpr (PART) { if (in) *at = acc[i][j][4 * g + r]; }
                        else {
                            const float x = op_result(acc[i][j][4 * g + r], s4[r], w_[j]);
                            const TY r_ = op_cast<TY>(biased ? x + b_[j] : x);
                            if constexpr (PAST) { if (in) op_store_past(at, r_); }
                            else { if (in) *at = r_; }
                        }
                    }
                }
            }
    };
    if constexpr (PART) { if (whole) store(std::true_type{}, std::false_type{}); else store(std::false_type{}, std::false_type{}); }
    else if (((uintptr_t)p.y | (uintptr_t)(p.ldy * (int)sizeof(TY))) & 127) { if (whole) store(std::true_type{}, std::false_type{}); else store(std::false_type{}, std::false_type{}); }
    else { if (whole) store(std::true_type{}, std::true_type{}); else store(std::false_type{}, std::true_type{}); }
}

// The parts of a product's sums, added up: grid (n / 256, m), a result a thread.
constexpr int OP_MAX_PARTS = 16;
template <typename TY>
static __global__ __launch_bounds__(256) void op_parts_kernel(const int* __restrict__ parts, int count, OpProductArgs<TY> p) {
    const int col = (int)blockIdx.x * 256 + threadIdx.x, row = blockIdx.y;
    if (col >= p.n) return;
    int v[OP_MAX_PARTS];
#pragma unroll
    for (int i = 0; i < OP_MAX_PARTS; ++i) v[i] = i < count ? parts[((int64_t)i * p.m + row) * p.n + col] : 0;
    int sum = 0;
#pragma unroll
    for (int i = 0; i < OP_MAX_PARTS; ++i) sum += v[i];
    const float x = op_result(sum, p.as[row], p.ws[col]);
    p.y[(int64_t)row * p.ldy + col] = op_cast<TY>(p.bias ? x + p.bias[col] : x);
}
