// gl3_ops.hip — operators on the caller's device memory: int8 rows, their products, log probabilities of tokens.  Argument checks, launches.
#include "gl3_ops.h"

#include <algorithm>
#include <climits>
#include <tuple>
#include <type_traits>
#include <utility>

#include "gl3_ops_int8.h"
#include "gl3_ops_logprobs.h"

void gl3_set_op_error(const char* msg);          // gl3_create_err.h
void gl3_no_error();

static inline int64_t op_cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int64_t OP_GRID = 1 << 21;          // workgroups of one launch, at most (a launch has fewer than 2^32 threads: 1024 of them a workgroup)
template <typename F> static hipError_t op_with_type(int32_t type, F&& f) {
    return type == GL3_TYPE_F32 ? f(float{}) : type == GL3_TYPE_F16 ? f(__half{}) : f(op_bf16{});
}
// A launch and its own error: what hipGetLastError() holds may be another call's, which the caller has dealt with.  Nothing is launched behind one that failed.
template <typename... P, size_t... I> static hipError_t op_launch_args(const void* kernel, dim3 grid, dim3 block, hipStream_t s, std::tuple<P...>& v, std::index_sequence<I...>) {
    void* args[] = {&std::get<I>(v)...};
    return hipLaunchKernel(kernel, grid, block, args, 0, s);
}
template <typename... P, typename... A> static hipError_t op_launch(void (*kernel)(P...), dim3 grid, dim3 block, hipStream_t s, A&&... a) {
    std::tuple<P...> v(std::forward<A>(a)...);
    return op_launch_args((const void*)kernel, grid, block, s, v, std::index_sequence_for<P...>{});
}
#define OP_TRY(call) do { const hipError_t e_ = (call); if (e_ != hipSuccess) return e_; } while (0)

// ---- launches -------------------------------------------------------------------------------------------------------------------------
hipError_t op_quantize(hipStream_t s, const void* x, int32_t type, int64_t rows, int32_t cols, int64_t ldx, int8_t* codes, int64_t ldq, float* scale) {
    return op_with_type(type, [&](auto t) {
        typedef decltype(t) T;
        const int64_t kp = op_code_ld(cols);
        for (int64_t r = 0; r < rows; r += OP_GRID) {
            const int64_t n = std::min<int64_t>(OP_GRID, rows - r);
            const T* xr = (const T*)x + r * ldx;
#define OP_Q(W) OP_TRY(op_launch(op_quantize_kernel<T, W>, dim3((unsigned)(W > 4 ? n : op_cdiv(n * W, 4))), dim3(W > 4 ? 64 * W : 256), s, xr, n, cols, ldx, codes + r * ldq, ldq, scale + r))
            // as many wavefronts a row as it needs; of a few rows more, so that a thread has 16 bytes or so
            if (kp <= 512 || (kp <= OP_ROW_E * 64 && rows > 2048)) OP_Q(1);
            else if (kp <= OP_ROW_E * 256 && (kp <= 2048 || rows > 64)) OP_Q(4);
            else if (kp <= OP_ROW_E * 1024) OP_Q(16);
            else OP_TRY(op_launch(op_quantize_long_kernel<T>, dim3((unsigned)n), dim3(1024), s, xr, cols, ldx, codes + r * ldq, ldq, scale + r));
#undef OP_Q
        }
        return hipSuccess;
    });
}

// Which tile, and into how many parts its sum over k goes: the ones with the least estimated time.  A stage of a BM x BN tile takes a CU 0.00164 (BM + BN) us for
// its operands' bytes + 0.0000101 BM BN us for its MFMAs (256 x 256 1.5, 128 x 256 0.96, 128 x 128 0.59, 64 x 128 0.40, 32 x 128 0.30, 64 x 64 0.25), a tile 3 us and its results'
// bytes at 37 GB/s besides.  256 CUs take the workgroups in rounds; two workgroups of a small tile share a CU; the weights leave memory at 5.4 TB/s.  Tiles that are
// too few for the CUs get their sums in parts of at least OP_PART_STAGES stages; a launch of its own adds them up, 2.5 us (on the host another 3: 4.5 here)
// and what it reads (us, in parts / whole,
// m tokens, n x k: 40, 4096 x 4096 10.9 / 12.3 (parts of 8 stages 12.5); 64, 4096 x 14336 17.7 / 36.1; 256 29.5 / 36.0; 64, 1024 x 4096 7.8 / 10.1; 64, 256 x 131000 24 / 254).
enum { OP_T256x256, OP_T128x256, OP_T128x128, OP_T64x128, OP_T64x64, OP_T32x128, OP_T_COUNT };
static const struct { int bm, bn, share; } OP_TILES[OP_T_COUNT] = {{256, 256, 1}, {128, 256, 1}, {128, 128, 2}, {64, 128, 2}, {64, 64, 2}, {32, 128, 2}};
constexpr int OP_PART_STAGES = 4;
struct OpRingPlan { int tile, parts; double us; };
static OpRingPlan op_ring_plan(int m, int n, int kp, int size) {
    OpRingPlan best{0, 1, 1e300};
    const int stages = kp / 128;
    const double memory = (double)n * kp / 5.4e6 + 4.0;
    for (int t = 0; t < OP_T_COUNT; ++t) {
        const int bm = OP_TILES[t].bm, bn = OP_TILES[t].bn, slots = 256 * OP_TILES[t].share;
        const double stage = 0.00164 * (bm + bn) + 0.0000101 * bm * bn;
        const int64_t tiles = op_cdiv(m, bm) * op_cdiv(n, bn), rest = tiles % slots;
        const double rounds = (double)(tiles / slots * OP_TILES[t].share + (rest == 0 ? 0 : rest <= 256 ? 1 : 2));
        const double busy = rounds * (stages * stage + 3.0 + (double)bm * bn * size / 37e3), whole = std::max(memory, busy) + 1e-3 * busy;          // (of several that memory holds up, the least busy)
        if (whole < best.us) best = OpRingPlan{t, 1, whole};
        const int parts = (int)std::min<int64_t>(std::min(256 / tiles, (int64_t)stages / OP_PART_STAGES), OP_MAX_PARTS);
        if (parts < 2 || bn > 128) continue;          // (parts of the larger tiles: 45.2 us, whole 46.1, at 142 tokens, 11037 x 9472)
        const double part = (double)op_cdiv(stages, parts) * stage + 3.0 + bm * bn * 4 / 37e3, split = std::max(memory, part) + 1e-3 * part + 4.5 + (double)m * n * 4 * parts / 2.5e6;
        if (split < best.us) best = OpRingPlan{t, parts, split};
    }
    return best;
}
template <typename TY, int BM, int BN, int WM, int WN, int SA, int SW>
static hipError_t op_ring_launch(hipStream_t s, const OpProductArgs<TY>& p, int parts) {
    const int mt = (int)op_cdiv(p.m, BM), nt = (int)op_cdiv(p.n, BN);
    return op_launch(op_ring_kernel<TY, BM, BN, WM, WN, SA, SW>, dim3((unsigned)op_cdiv((int64_t)mt * nt, 8) * 8, (unsigned)parts), dim3(WM * WN * 64), s, p, mt, nt);
}
template <typename TY>
static hipError_t op_ring(hipStream_t s, const OpProductArgs<TY>& p, int tile, int parts) {
    if constexpr (!std::is_same<TY, int>::value) {          // (tiles that are never in parts)
        if (tile == OP_T256x256) return op_ring_launch<TY, 256, 256, 4, 2, 2, 3>(s, p, parts);
        if (tile == OP_T128x256) return op_ring_launch<TY, 128, 256, 2, 4, 2, 4>(s, p, parts);
    }
    switch (tile) {
        case OP_T128x128: return op_ring_launch<TY, 128, 128, 2, 2, 2, 3>(s, p, parts);
        case OP_T64x128: return op_ring_launch<TY, 64, 128, 2, 2, 2, 4>(s, p, parts);
        case OP_T64x64: return op_ring_launch<TY, 64, 64, 2, 2, 4, 5>(s, p, parts);
        default: return op_ring_launch<TY, 32, 128, 1, 4, 3, 4>(s, p, parts);          // (rings of 2 and 4: 81 us instead of 77 at 32 tokens, 151936 x 2560)
    }
}
// Up to 32 tokens (16 where there are many strips: tiles win beyond) may be streamed: 6.6 TB/s of weights, 4.2 % more time a token (us, streamed / tiles; m tokens, n x k: 1, 4096 x 4096 6.5 / 10.3; 16 8.0 / 10.8;
// 24 9.1 / 11.6; 8, 4096 x 14336 14.6 / 15.9; 16 18.4 / 16.0; 4, 14336 x 4096 15.0 / 14.8; 8 16.5 / 14.8; 8, 32000 x 2048 16.2 / 14.0), and a strip alone takes
// 26.6 KB a us, 3 % more time a token (16, 2560 x 9728 14.0 / 11.2; 16, 256 x 131000 117 / 21), and 0.5 (more than 16 tokens: 1.5) ns of the whole card's time beside
// its bytes (1, 100000 x 256 13.3 / 10.3; 20 20.7 / 11.6).  Eight wavefronts share the k of a strip where there are few strips (4096 x 14336 12.6, four of them
// 14.5), four where they fill the chip (128256 x 4096 85.3, eight 86.5).
constexpr int OP_FEW_STRIPS = 512;
static bool op_streams(int m, int n, int kp, const OpRingPlan& ring) {
    return m <= (n <= 16 * OP_FEW_STRIPS ? 32 : 16) && std::max(4.0 + (double)n * kp / 6.6e6 * (1.0 + 0.042 * m) + n * (m <= 16 ? 3e-5 : 9e-5), 3.2 + kp / 1660.0 * (1.0 + 0.03 * m)) <= ring.us;
}
template <typename TY>
static hipError_t op_product_piece(hipStream_t s, const OpProductArgs<TY>& p, void* workspace) {
    const OpRingPlan ring = op_ring_plan(p.m, p.n, p.kp, sizeof(TY));
    if (op_streams(p.m, p.n, p.kp, ring)) {
        const unsigned strips = (unsigned)op_cdiv(p.n, 16);
#define OP_STREAM(MT, KS, D) return op_launch(op_stream_kernel<TY, MT, KS, D>, dim3(strips), dim3(64 * KS), s, p)
        if (strips <= OP_FEW_STRIPS) { if (p.m <= 16) OP_STREAM(1, 8, 4); else OP_STREAM(2, 8, 4); }
        else OP_STREAM(1, 4, 8);
#undef OP_STREAM
    }
    if (ring.parts == 1) return op_ring<TY>(s, p, ring.tile, 1);
    OP_TRY(op_ring<int>(s, OpProductArgs<int>{p.a, p.lda, nullptr, p.w, p.ldw, nullptr, nullptr, p.m, p.n, p.kp, (int*)workspace, p.n}, ring.tile, ring.parts));
    return op_launch(op_parts_kernel<TY>, dim3((unsigned)op_cdiv(p.n, 256), (unsigned)p.m), dim3(256), s, (const int*)workspace, ring.parts, p);
}
constexpr int64_t OP_PM = 1 << 16, OP_PN = 1 << 18;          // a launch's rows and channels: its tiles have 32-bit numbers
hipError_t op_product(hipStream_t s, const OpProduct& p, void* workspace) {
    return op_with_type(p.y_type, [&](auto t) {
        typedef decltype(t) TY;
        for (int64_t n = 0; n < p.n; n += OP_PN)
            for (int64_t m = 0; m < p.m; m += OP_PM)
                OP_TRY(op_product_piece(s, OpProductArgs<TY>{p.a + m * p.lda, p.lda, p.a_scale + m, p.w + n * p.ldw, p.ldw, p.w_scale + n, p.bias ? p.bias + n : nullptr, (int)std::min(OP_PM, p.m - m),
                                                      (int)std::min(OP_PN, p.n - n), (int)op_code_ld(p.k), (TY*)p.y + m * p.ldy + n, p.ldy}, workspace));
        return hipSuccess;
    });
}
// the parts of the piece that needs most (whatever the results' type); pieces run one after the other
uint64_t op_product_workspace(int64_t m, int64_t n, int32_t k) {
    const int kp = (int)op_code_ld(k);
    uint64_t most = 0;
    const int64_t ms[2] = {std::min(m, OP_PM), m > OP_PM ? m % OP_PM : 0}, ns[2] = {std::min(n, OP_PN), n > OP_PN ? n % OP_PN : 0};
    for (int64_t pm : ms)
        for (int64_t pn : ns)
            for (int size = 2; pm && pn && size <= 4; size += 2) {
                const OpRingPlan ring = op_ring_plan((int)pm, (int)pn, kp, size);
                if (ring.parts > 1 && !op_streams((int)pm, (int)pn, kp, ring)) most = std::max<uint64_t>(most, (uint64_t)pm * pn * ring.parts * 4);
            }
    return most;
}

constexpr int OP_TOKEN_STRIPS = 2048;          // of one or two tokens; of four half as many, of eight a quarter
// workspace of a linear: codes of the rows, their scales, then what the product needs
static uint64_t op_linear_codes(int64_t m, int32_t k) { return (uint64_t)m * op_code_ld(k); }
static uint64_t op_linear_rows(int64_t m, int32_t k) { return op_linear_codes(m, k) + (uint64_t)op_cdiv(m, 4) * 16; }
// a few tokens whose rows every workgroup quantises for itself: no workspace.  lg: 2^lg rows at least
static int op_token_lg(int64_t m) { return m <= 1 ? 0 : m <= 2 ? 1 : m <= 4 ? 2 : 3; }
static bool op_token(int64_t m, int64_t n, int32_t k) {
    const int lg = op_token_lg(m);
    return m <= OP_TOKENS && n <= 16 * (OP_TOKEN_STRIPS >> std::max(0, lg - 1)) && op_code_ld(k) <= OP_ROW_E * 512 >> lg;
}
uint64_t op_linear_workspace(int64_t m, int64_t n, int32_t k) { return op_token(m, n, k) ? 0 : op_linear_rows(m, k) + op_product_workspace(m, n, k); }
hipError_t op_linear(hipStream_t s, const void* x, int32_t x_type, int64_t ldx, const OpProduct& p, void* workspace) {
    if (op_token(p.m, p.n, p.k)) {
        return op_with_type(x_type, [&](auto tx) {
            return op_with_type(p.y_type, [&](auto ty) {
                typedef decltype(tx) TX; typedef decltype(ty) TY;
                const OpProductArgs<TY> a{nullptr, 0, nullptr, p.w, p.ldw, p.w_scale, p.bias, (int)p.m, (int)p.n, (int)op_code_ld(p.k), (TY*)p.y, p.ldy};
                const dim3 grid((unsigned)op_cdiv(p.n, 16));
                const int lg = op_token_lg(p.m);
#define OP_TOKEN(KS, D, ONE) return op_launch(op_token_kernel<TX, TY, KS, D, ONE>, grid, dim3(64 * KS), s, a, (const TX*)x, ldx, p.k, lg)
                if (grid.x <= OP_FEW_STRIPS || 4 >> lg == 0 || a.kp > OP_ROW_E * 256 >> lg) { if (lg) OP_TOKEN(8, 4, false); else OP_TOKEN(8, 4, true); }
                else { if (lg) OP_TOKEN(4, 8, false); else OP_TOKEN(4, 8, true); }
#undef OP_TOKEN
            });
        });
    }
    OpProduct q = p;
    int8_t* codes = (int8_t*)workspace;
    float* scale = (float*)(codes + op_linear_codes(p.m, p.k));
    q.a = codes; q.lda = op_code_ld(p.k); q.a_scale = scale;
    OP_TRY(op_quantize(s, x, x_type, p.m, p.k, ldx, codes, q.lda, scale));
    return op_product(s, q, (uint8_t*)workspace + op_linear_rows(p.m, p.k));
}

// Parts of a row: as many as give the launch OP_LP_WGS workgroups, none shorter than a small batch, at most 64 (one lane each joins them).
constexpr int OP_LP_WGS = 1280, OP_LP_SMALL = 2048, OP_LP_BIG = 4096;          // logits of a workgroup's batch
struct OpLpPlan { int parts, per; bool big; };          // per: logits of a part
static OpLpPlan op_lp_plan(int64_t rows, int32_t vocab) {
    const int64_t want = std::min<int64_t>(64, std::max<int64_t>(1, OP_LP_WGS / rows));
    int64_t per = op_cdiv(op_cdiv(vocab, want), OP_LP_SMALL) * OP_LP_SMALL;
    const bool big = per >= OP_LP_BIG;
    if (big) per = op_cdiv(per, OP_LP_BIG) * OP_LP_BIG;
    return OpLpPlan{(int)op_cdiv(vocab, per), (int)std::min<int64_t>(per, INT32_MAX - OP_LP_BIG + 1), big};
}
uint64_t op_logprobs_workspace(int64_t rows, int32_t vocab, int32_t top) {
    const OpLpPlan pl = op_lp_plan(rows, vocab);
    return pl.parts == 1 ? 0 : (uint64_t)rows * pl.parts * op_part_bytes(top);
}
hipError_t op_logprobs(hipStream_t s, const OpLogprobs& p, void* workspace) {
    const OpRowOut o{p.targets, p.top, p.logprob, p.rank, p.entropy, p.top_ids, p.top_logprobs};
    const OpLpPlan pl = op_lp_plan(p.rows, p.vocab);
    return op_with_type(p.type, [&](auto t) {
        typedef decltype(t) T;
        constexpr int V = 16 / (int)sizeof(T), NT = OP_LP_THREADS;
        for (int64_t r = 0; r < p.rows; r += 65535) {          // (a grid's y)
            const dim3 grid((unsigned)pl.parts, (unsigned)std::min<int64_t>(65535, p.rows - r));
#define OP_LP(U, TOP) OP_TRY(op_launch(op_logprobs_kernel<T, U, TOP>, grid, dim3(NT), s, (const T*)p.logits, p.vocab, p.ld, r, pl.per / V, o, (uint8_t*)workspace))
            if (pl.big) { if (p.top) OP_LP(OP_LP_BIG / NT / V, true); else OP_LP(OP_LP_BIG / NT / V, false); }
            else { if (p.top) OP_LP(OP_LP_SMALL / NT / V, true); else OP_LP(OP_LP_SMALL / NT / V, false); }
#undef OP_LP
        }
        if (pl.parts == 1) return hipSuccess;
        return op_launch(op_logprobs_join_kernel<T>, dim3((unsigned)p.rows), dim3(64 * OP_LP_JOIN_WAVES), s, (const T*)p.logits, p.vocab, p.ld, pl.parts, o, (const uint8_t*)workspace);
    });
}

// ---- entry points ---------------------------------------------------------------------------------------------------------------------
namespace {
int32_t refuse(int32_t code, const char* msg) { gl3_set_op_error(msg); return code; }
#define OP_ARG(cond, msg) do { if (!(cond)) return refuse(GL3_E_ARG, msg); } while (0)

constexpr int32_t MAX_VOCAB = 1 << 30;
bool float_type(int32_t t) { return t == GL3_TYPE_F32 || t == GL3_TYPE_F16 || t == GL3_TYPE_BF16; }
int type_size(int32_t t) { return t == GL3_TYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
// rows of `cols` elements, `ld` apart (one row: any ld): whether their bytes fit an address
constexpr int64_t MAX_Y_LD = 1 << 26;
constexpr int64_t MAX_CODE_LD = 1 << 23;          // (a tile's rows are reached with 32-bit offsets)
bool rows_ok(int64_t rows, int64_t cols, int64_t ld) { return rows <= 1 || (ld >= cols && ld <= (INT64_MAX >> 4) / rows); }

// the caller's device for the length of a call
struct OnDevice {
    int before = -1;
    bool changed = false;
    const char* enter(int32_t device, hipStream_t s) {
        if (device < 0 || hipGetDevice(&before) != hipSuccess) { (void)hipGetLastError(); return "no such device"; }
        if (before != device) {
            if (hipSetDevice(device) != hipSuccess) { (void)hipGetLastError(); return "no such device"; }
            changed = true;
        }
        int on = device;
        if (s && hipStreamGetDevice(s, &on) != hipSuccess) { (void)hipGetLastError(); return "the stream is not valid"; }
        return on == device ? nullptr : "the stream belongs to another device";
    }
    ~OnDevice() { if (changed) (void)hipSetDevice(before); }
};
int32_t launched(hipError_t e) {
    if (e == hipSuccess) return GL3_OK;
    (void)hipGetLastError();          // (it is told here)
    return refuse(e == hipErrorOutOfMemory ? GL3_E_OOM : GL3_E_HIP, hipGetErrorString(e));
}
int32_t check_product(const OpProduct& p) {
    OP_ARG(p.k >= 1 && p.k <= GL3_INT8_MAX_K, "k out of range (1 .. GL3_INT8_MAX_K)");
    OP_ARG(p.m >= 0 && p.n >= 0 && p.m <= INT32_MAX && p.n <= INT32_MAX, "m or n out of range");
    OP_ARG(float_type(p.y_type), "results are GL3_TYPE_F32, F16 or BF16");
    if (p.m == 0 || p.n == 0) return GL3_OK;
    OP_ARG(p.w && p.w_scale && p.y, "null pointer");
    OP_ARG(aligned(p.w, 16) && p.ldw % 16 == 0, "codes start on 16 bytes, and so does every row of them");
    OP_ARG(rows_ok(p.n, op_code_ld(p.k), p.ldw) && p.ldw <= MAX_CODE_LD, "ldw: a row of codes is k columns and zeros up to a multiple of GL3_CODE_BLOCK");
    OP_ARG(aligned(p.w_scale, 4) && aligned(p.bias, 4) && aligned(p.y, type_size(p.y_type)), "misaligned pointer");
    OP_ARG(rows_ok(p.m, p.n, p.ldy) && (p.m <= 1 || p.ldy <= MAX_Y_LD), "ldy out of range (n .. 2^26)");
    return GL3_OK;
}
int32_t check_workspace(const void* workspace, uint64_t have, uint64_t need) {
    OP_ARG(have >= need && (workspace || need == 0), "workspace too small");
    OP_ARG(need == 0 || aligned(workspace, 16), "the workspace starts on 16 bytes");
    return GL3_OK;
}
}  // namespace

extern "C" {

int32_t gl3_quantize_rows(int32_t device, void* stream, const void* x, int32_t x_type, int64_t rows, int32_t cols, int64_t ldx, int8_t* codes, int64_t ldq, float* scale) {
    gl3_no_error();
    OP_ARG(float_type(x_type), "rows are GL3_TYPE_F32, F16 or BF16");
    OP_ARG(rows >= 0 && rows <= INT32_MAX, "rows out of range");
    OP_ARG(cols >= 1 && cols <= GL3_INT8_MAX_K, "cols out of range (1 .. GL3_INT8_MAX_K)");
    if (rows == 0) return GL3_OK;
    OP_ARG(x && codes && scale, "null pointer");
    OP_ARG(aligned(x, type_size(x_type)) && aligned(scale, 4), "misaligned pointer");
    OP_ARG(rows_ok(rows, cols, ldx), "ldx is less than cols, or rows end past what an address holds");
    OP_ARG(aligned(codes, 16) && ldq % 16 == 0, "codes start on 16 bytes, and so does every row of them");
    OP_ARG(rows_ok(rows, op_code_ld(cols), ldq), "ldq: a row of codes is cols columns and zeros up to a multiple of GL3_CODE_BLOCK");
    OnDevice on;
    if (const char* why = on.enter(device, (hipStream_t)stream)) return refuse(GL3_E_ARG, why);
    return launched(op_quantize((hipStream_t)stream, x, x_type, rows, cols, ldx, codes, ldq, scale));
}

int32_t gl3_int8_workspace(int64_t m, int64_t n, int32_t k, uint64_t* matmul_bytes, uint64_t* linear_bytes) {
    gl3_no_error();
    OP_ARG(k >= 1 && k <= GL3_INT8_MAX_K && m >= 0 && n >= 0 && m <= INT32_MAX && n <= INT32_MAX, "sizes out of range");
    const bool none = m == 0 || n == 0;
    if (matmul_bytes) *matmul_bytes = none ? 0 : op_product_workspace(m, n, k);
    if (linear_bytes) *linear_bytes = none ? 0 : op_linear_workspace(m, n, k);
    return GL3_OK;
}

int32_t gl3_int8_matmul(int32_t device, void* stream, const int8_t* a, int64_t lda, const float* a_scale, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias, int64_t m,
                        int64_t n, int32_t k, void* y, int32_t y_type, int64_t ldy, void* workspace, uint64_t workspace_bytes) {
    gl3_no_error();
    const OpProduct p{a, lda, a_scale, w, ldw, w_scale, bias, m, n, k, y, y_type, ldy};
    int32_t r = check_product(p);
    if (r != GL3_OK || m == 0 || n == 0) return r;
    OP_ARG(a && a_scale, "null pointer");
    OP_ARG(aligned(a, 16) && lda % 16 == 0, "codes start on 16 bytes, and so does every row of them");
    OP_ARG(aligned(a_scale, 4), "misaligned pointer");
    OP_ARG(rows_ok(m, op_code_ld(k), lda) && lda <= MAX_CODE_LD, "lda: a row of codes is k columns and zeros up to a multiple of GL3_CODE_BLOCK");
    if ((r = check_workspace(workspace, workspace_bytes, op_product_workspace(m, n, k))) != GL3_OK) return r;
    OnDevice on;
    if (const char* why = on.enter(device, (hipStream_t)stream)) return refuse(GL3_E_ARG, why);
    return launched(op_product((hipStream_t)stream, p, workspace));
}

int32_t gl3_int8_linear(int32_t device, void* stream, const void* x, int32_t x_type, int64_t ldx, const int8_t* w, int64_t ldw, const float* w_scale, const float* bias, int64_t m, int64_t n,
                        int32_t k, void* y, int32_t y_type, int64_t ldy, void* workspace, uint64_t workspace_bytes) {
    gl3_no_error();
    const OpProduct p{nullptr, 0, nullptr, w, ldw, w_scale, bias, m, n, k, y, y_type, ldy};
    OP_ARG(float_type(x_type), "rows are GL3_TYPE_F32, F16 or BF16");
    int32_t r = check_product(p);
    if (r != GL3_OK || m == 0 || n == 0) return r;
    OP_ARG(x && aligned(x, type_size(x_type)), "x is null or misaligned");
    OP_ARG(rows_ok(m, k, ldx), "ldx is less than k, or rows end past what an address holds");
    if ((r = check_workspace(workspace, workspace_bytes, op_linear_workspace(m, n, k))) != GL3_OK) return r;
    OnDevice on;
    if (const char* why = on.enter(device, (hipStream_t)stream)) return refuse(GL3_E_ARG, why);
    return launched(op_linear((hipStream_t)stream, x, x_type, ldx, p, workspace));
}

int32_t gl3_logprobs_workspace(int64_t rows, int32_t vocab, int32_t top, uint64_t* bytes) {
    gl3_no_error();
    OP_ARG(bytes, "null pointer");
    OP_ARG(rows >= 0 && rows <= INT32_MAX && vocab >= 1 && vocab <= MAX_VOCAB && top >= 0 && top <= GL3_LOGPROBS_MAX_TOP, "sizes out of range");
    *bytes = rows == 0 ? 0 : op_logprobs_workspace(rows, vocab, top);
    return GL3_OK;
}

int32_t gl3_token_logprobs(int32_t device, void* stream, const void* logits, int32_t type, int64_t rows, int32_t vocab, int64_t ld, const int32_t* targets, int32_t top, float* logprob,
                           int32_t* rank, float* entropy, int32_t* top_ids, float* top_logprobs, void* workspace, uint64_t workspace_bytes) {
    gl3_no_error();
    OP_ARG(float_type(type), "logits are GL3_TYPE_F32, F16 or BF16");
    OP_ARG(rows >= 0 && rows <= INT32_MAX && vocab >= 1 && vocab <= MAX_VOCAB, "rows or vocab out of range");
    OP_ARG(top >= 0 && top <= GL3_LOGPROBS_MAX_TOP, "top out of range (0 .. GL3_LOGPROBS_MAX_TOP)");
    OP_ARG((targets != nullptr) == (logprob != nullptr) && (targets != nullptr) == (rank != nullptr), "targets, logprob and rank: all or none");
    if (rows == 0) return GL3_OK;
    OP_ARG(logits && aligned(logits, type_size(type)), "logits are null or misaligned");
    OP_ARG(rows_ok(rows, vocab, ld), "ld is less than vocab, or rows end past what an address holds");
    OP_ARG(top == 0 || (top_ids && top_logprobs), "top > 0 needs top_ids and top_logprobs");
    OP_ARG(aligned(targets, 4) && aligned(logprob, 4) && aligned(rank, 4) && aligned(entropy, 4) && aligned(top_ids, 4) && aligned(top_logprobs, 4), "misaligned pointer");
    int32_t r = check_workspace(workspace, workspace_bytes, op_logprobs_workspace(rows, vocab, top));
    if (r != GL3_OK) return r;
    if (!targets && !entropy && top == 0) return GL3_OK;
    OnDevice on;
    if (const char* why = on.enter(device, (hipStream_t)stream)) return refuse(GL3_E_ARG, why);
    return launched(op_logprobs((hipStream_t)stream, OpLogprobs{logits, type, rows, vocab, ld, targets, top, logprob, rank, entropy, top_ids, top_logprobs}, workspace));
}

}  // extern "C"
