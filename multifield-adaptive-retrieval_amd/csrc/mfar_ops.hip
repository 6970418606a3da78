// mfar_ops.hip -- host side of the encoder / training operators of libmfar_hip.so (include/mfar_hip.h, last section).
// gfx950 only.  Every entry point returns an error code; nothing throws across the ABI.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdio>

#include "mfar_hip.h"
#include "mfar_error.h"
#include "mfar_attention.h"
#include "mfar_distill.h"
#include "mfar_int8.h"

namespace {

int bad(const char* msg) { return mfar_report(MFAR_ERR_INVALID, msg); }
int hip_failed(const char* what, hipError_t e) {
    (void)hipGetLastError();     // reported here: not left behind for the next call
    char msg[256];
    std::snprintf(msg, sizeof msg, "%s: %s", what, hipGetErrorString(e));
    return mfar_report(MFAR_ERR_HIP, msg);
}

// makes `device` current for a scope
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else if (err == hipSuccess) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
#define ON_DEVICE(device)                                                              \
    OnDevice on_device_(device);                                                       \
    if (on_device_.err != hipSuccess) return hip_failed("hipSetDevice", on_device_.err)
#define LAUNCHED(what)                                                \
    do {                                                              \
        const hipError_t e_ = hipGetLastError();                      \
        if (e_ != hipSuccess) return hip_failed(what, e_);            \
    } while (0)

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr int64_t MAX_BLOCKS = 1 << 24;       // of 256 threads: a launch counts its threads in 32 bits
int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
int type_size(int dtype) { return dtype == MFAR_DTYPE_F32 ? 4 : (dtype == MFAR_DTYPE_BF16 || dtype == MFAR_DTYPE_F16) ? 2 : 0; }

// a kernel that may need more than the default 64 KB of dynamic LDS: allowed once per device and kernel
template <typename F> hipError_t allow_lds(F kernel, std::atomic<uint32_t>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint32_t bit = dev < 32 ? 1u << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return hipSuccess;
    e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 156 * 1024);   // (some have a few static bytes)
    if (e == hipSuccess && bit) done.fetch_or(bit, std::memory_order_release);
    return e;
}
// (kernels that share a type have a flag each: the address of one instance is a template argument)
template <auto KERNEL, typename... P> int launch(const char* name, dim3 grid, size_t lds, hipStream_t st, const P&... p) {
    if (lds > 64 * 1024) {
        static std::atomic<uint32_t> done{0};
        const hipError_t e = allow_lds(KERNEL, done);
        if (e != hipSuccess) return hip_failed(name, e);
    }
    KERNEL<<<grid, dim3(256), lds, st>>>(p...);
    LAUNCHED(name);
    return MFAR_OK;
}

// ---- attention --------------------------------------------------------------------------------------------------------------------------
int check_attention(const mfar_attention* a, bool backward) {
    if (!a) return bad("NULL arguments");
    const int es = type_size(a->dtype);
    if (!es) return bad("dtype must be F32, BF16 or F16");
    if (a->B < 0 || a->Lq < 0 || a->Lk < 0 || a->H < 1 || a->B > 65535 || a->H > 65535) return bad("B, Lq, Lk must be >= 0, H >= 1, B and H <= 65535");
    if (a->D < 8 || a->D > 128 || a->D % 8) return bad("D must be a multiple of 8, at most 128");
    if (a->Lq > (1 << 30) - 256 || a->Lk > (1 << 30) - 256) return bad("at most 2^30 - 256 queries and keys");     // positions and their differences fit 32 bits
    if (cdiv((int64_t)a->B * a->H, 8) * 8 * cdiv(std::max(a->Lq, a->Lk), AT_COLS) >= MAX_BLOCKS) return bad("batch, heads and tiles of 128 queries or keys: under 2^24 blocks");
    if (a->q_start < -(1 << 30) || a->q_start > (1 << 30)) return bad("q_start out of range");
    if (a->n_buckets < 2 || a->n_buckets > 256 || (!a->causal && (a->n_buckets % 2 || a->n_buckets < 4))) return bad("n_buckets must be 2..256, even and >= 4 unless causal");
    const int side = a->causal ? a->n_buckets : a->n_buckets / 2, each = side / 2;
    if (a->n_borders != side - each - 1 || (a->n_borders && !a->borders)) return bad("n_borders must be side - side / 2 - 1");
    for (int j = 0; j < a->n_borders; ++j)
        if (a->borders[j] < each || (j && a->borders[j] < a->borders[j - 1])) return bad("borders must ascend from the first shared distance");
    if ((a->n_borders ? a->borders[a->n_borders - 1] : each) > 1023) return bad("the last bucket must begin at a distance <= 1023");
    if (a->B == 0 || a->Lq == 0) return MFAR_OK;
    if (!a->q || !a->out || !a->table || (a->Lk && (!a->k || !a->v))) return bad("NULL tensor");
    const int64_t strides[] = {a->q_b, a->q_l, a->q_h, a->k_b, a->k_l, a->k_h, a->v_b, a->v_l, a->v_h};
    for (int64_t s : strides)
        if (s * es % 16) return bad("strides must be multiples of 16 bytes");
    for (int64_t s : {a->q_l, a->k_l, a->v_l, backward ? a->do_l : 0})
        if (s < 0 || s > AT_MAX_STRIDE) return bad("row strides must be 0..2^22 elements");
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) || !aligned16(a->out_lo)) return bad("tensors must be 16-byte aligned");
    if (backward) {
        if (!a->dout || !a->dq || !a->lse || (a->Lk && (!a->dk || !a->dv))) return bad("NULL gradient or lse");
        if (a->do_b * es % 16 || a->do_l * es % 16 || a->do_h * es % 16) return bad("strides must be multiples of 16 bytes");
        if (!aligned16(a->dout) || !aligned16(a->dq) || !aligned16(a->dk) || !aligned16(a->dv)) return bad("tensors must be 16-byte aligned");
    }
    return MFAR_OK;
}
AttnParams attention_params(const mfar_attention* a) {
    AttnParams p = {};
    p.q = a->q, p.k = a->k, p.v = a->v, p.o = a->out, p.dout = a->dout;
    p.out = a->out, p.dq = a->dq, p.dk = a->dk, p.dv = a->dv;
    p.o_lo = p.out_lo = a->dtype == MFAR_DTYPE_F32 ? nullptr : a->out_lo;
    p.q_b = a->q_b, p.q_l = a->q_l, p.q_h = a->q_h, p.k_b = a->k_b, p.k_l = a->k_l, p.k_h = a->k_h, p.v_b = a->v_b, p.v_l = a->v_l, p.v_h = a->v_h;
    p.do_b = a->do_b, p.do_l = a->do_l, p.do_h = a->do_h;
    p.table = a->table, p.mask = a->key_mask, p.mask_b = a->mask_b, p.start_ptr = a->q_start_each, p.start = a->q_start, p.lse = a->lse;
    p.B = a->B, p.Lq = a->Lq, p.Lk = a->Lk, p.H = a->H, p.D = a->D, p.causal = a->causal != 0, p.scale = a->scale;
    p.n_buckets = a->n_buckets, p.n_side = a->causal ? a->n_buckets : a->n_buckets / 2;
    const int each = p.n_side / 2;
    p.sat = a->n_borders ? a->borders[a->n_borders - 1] : each;
    for (int m = 0; m < p.n_side; ++m) p.first[m] = (short)(m <= each ? m : a->borders[m - each - 1]);
    for (int d = 0, m = 0; d <= p.sat; ++d) {
        while (m + 1 < p.n_side && d >= p.first[m + 1]) ++m;
        p.bucket[d] = (unsigned char)m;
    }
    return p;
}
int64_t drow_bytes(const mfar_attention* a) { return ((int64_t)a->B * a->H * a->Lq * 4 + 15) / 16 * 16; }
// (behind the loop the tiles' memory takes the results on their way out)
template <typename T, int DP> constexpr size_t tile_bytes(bool backward) {
    const size_t n = at_stages(sizeof(T), DP, backward) * 2ull * AT_TILE * DP * sizeof(T);
    static_assert(at_stages(sizeof(T), DP, true) * 2ull * AT_TILE * DP * sizeof(T) >= 4 * at_out_bytes<T, DP>());
    return n;
}
size_t lut_bytes(const AttnParams& p) { return (size_t)(2 * (p.sat + AT_EDGE) + 1) * 4; }

// Up to 32 queries, and batches of fewer than 128 blocks of 128 queries, take the kernel that divides the keys over waves and blocks (7 x 4 heads x 213
// fp32, 56 blocks: 12.4 us against 25.3; about even at 192: 1 x 12 x 2048 fp16 42 against 49, 4 x 12 x 512 17.5 against 15.4).  A block gets at least
// 8 tiles of 32 keys, and there are no more than about two blocks per CU (16 x 12 heads over ragged caches of 4097: 32.9 us; three 33.8, four
// 36.6, eight 39.9; full caches: 47, 44, 47, 51).
bool few_queries(const mfar_attention* a) { return a->Lq <= 32 || cdiv(a->Lq, AT_COLS) * a->B * a->H < 128; }
int key_splits(const mfar_attention* a) {
    return (int)std::max<int64_t>(1, std::min(cdiv(512, cdiv(a->Lq, 32) * a->B * a->H), cdiv(a->Lk, 8 * 32)));
}
int64_t split_rows(const mfar_attention* a) { return (int64_t)a->B * a->Lq * a->H * key_splits(a); }
int64_t split_bytes(const mfar_attention* a) { return few_queries(a) && key_splits(a) > 1 ? split_rows(a) * (a->D + 2) * 4 : 0; }

template <typename T, int DP, bool KEEP> int attention_few(const AttnParams& p, const AttnSplit& sp, hipStream_t st) {
    const size_t lds = at_few_bytes<T, DP>() + 4 * 64 * 4 + lut_bytes(p);
    int rc = launch<mfar_attn_few_kernel<T, DP, KEEP>>("mfar_attn_few_kernel", dim3(cdiv(p.Lq, 32) * sp.splits, p.H, p.B), lds, st, p, sp);
    if (rc == MFAR_OK && sp.splits > 1)
        rc = launch<mfar_attn_join_kernel<T, KEEP>>("mfar_attn_join_kernel", dim3(cdiv((int64_t)p.B * p.Lq * p.H, 4)), 0, st, p, sp);
    return rc;
}
// blocks of 128 columns for every (batch, head), in groups of 8 (at_place)
unsigned at_grid(const AttnParams& p, int64_t columns) { return (unsigned)(cdiv((int64_t)p.B * p.H, 8) * 8 * cdiv(columns, AT_COLS)); }

template <typename T, int DP> int attention_forward(const AttnParams& p, const AttnSplit& sp, hipStream_t st) {
    if (sp.splits) {
        if constexpr (sizeof(T) == 2)
            if (p.out_lo) return attention_few<T, DP, true>(p, sp, st);
        return attention_few<T, DP, false>(p, sp, st);
    }
    const size_t lds = tile_bytes<T, DP>(false) + lut_bytes(p);
    const dim3 grid(at_grid(p, p.Lq));
    if constexpr (sizeof(T) == 2)
        if (p.out_lo) return launch<mfar_attn_forward_kernel<T, DP, true>>("mfar_attn_forward_kernel", grid, lds, st, p);
    return launch<mfar_attn_forward_kernel<T, DP, false>>("mfar_attn_forward_kernel", grid, lds, st, p);
}
template <typename T, int DP> int attention_backward(const AttnParams& p, float* dtable, hipStream_t st) {
    constexpr int S = at_stages(sizeof(T), DP, true);
    const size_t tiles = tile_bytes<T, DP>(true);
    const dim3 grid(at_grid(p, p.Lq));
    int rc = launch<mfar_attn_dq_kernel<T, DP>>("mfar_attn_dq_kernel", grid, tiles + lut_bytes(p) * (p.dpart ? 5 : 1) + (p.dpart ? 4 * AT_SKEW * 4 : 0), st, p);
    if (rc != MFAR_OK) return rc;
    if (p.Lk) {
        rc = launch<mfar_attn_dkv_kernel<T, DP>>("mfar_attn_dkv_kernel", dim3(at_grid(p, p.Lk)), tiles + S * 2 * AT_TILE * 4 + lut_bytes(p), st, p);
        if (rc != MFAR_OK) return rc;
    }
    if (p.dpart) {
        mfar_attn_dtable_kernel<<<p.H * p.n_buckets, AT_BLOCK, 0, st>>>(p.dpart, (int)(cdiv(p.Lq, AT_COLS) * p.B), p.H, p.n_buckets, dtable);
        LAUNCHED("mfar_attn_dtable_kernel");
    }
    return MFAR_OK;
}
#define FOR_TYPE_AND_DIM(FN, ...)                                                                                                     \
    (a->dtype == MFAR_DTYPE_F32    ? (a->D <= 32 ? FN<float, 32>(__VA_ARGS__) : a->D <= 64 ? FN<float, 64>(__VA_ARGS__) : FN<float, 128>(__VA_ARGS__)) \
     : a->dtype == MFAR_DTYPE_BF16 ? (a->D <= 32 ? FN<__bf16, 32>(__VA_ARGS__) : a->D <= 64 ? FN<__bf16, 64>(__VA_ARGS__) : FN<__bf16, 128>(__VA_ARGS__)) \
                                   : (a->D <= 32 ? FN<_Float16, 32>(__VA_ARGS__) : a->D <= 64 ? FN<_Float16, 64>(__VA_ARGS__) : FN<_Float16, 128>(__VA_ARGS__)))
#define FOR_TYPE(dtype, FN, ...) ((dtype) == MFAR_DTYPE_F32 ? FN<float>(__VA_ARGS__) : (dtype) == MFAR_DTYPE_BF16 ? FN<__bf16>(__VA_ARGS__) : FN<_Float16>(__VA_ARGS__))

// ---- distillation -----------------------------------------------------------------------------------------------------------------------
// A row is cut into pieces of at least 4096 columns while there are fewer than 2048 blocks (8 per CU).
int distill_chunk(int64_t T, int64_t N) {
    const int64_t splits = std::max<int64_t>(1, std::min(cdiv(2048, std::max<int64_t>(1, T)), cdiv(N, 4096)));
    return (int)(cdiv(cdiv(N, splits), 64) * 64);
}
template <typename T> int distill_forward(const DistillParams& p, hipStream_t st) {
    int rc = launch<mfar_distill_forward_kernel<T>>("mfar_distill_forward_kernel", dim3(p.T, p.splits), 0, st, p);
    if (rc == MFAR_OK && p.splits > 1) rc = launch<mfar_distill_join_kernel<T>>("mfar_distill_join_kernel", dim3(p.T), 0, st, p);
    return rc;
}
template <typename T> int distill_backward(const DistillParams& p, hipStream_t st) {
    return launch<mfar_distill_backward_kernel<T>>("mfar_distill_backward_kernel", dim3(p.T, p.splits), 0, st, p);
}
int check_distill(const void* x, int dtype, int64_t ld, int64_t T, int64_t N, const int64_t* ids, int K, float tau) {
    if (!type_size(dtype)) return bad("dtype must be F32, BF16 or F16");
    if (T < 0 || T >= MAX_BLOCKS || N < 1 || N > (1 << 30)) return bad("T must be 0..2^24 - 1, N 1..2^30");
    if (K < 1 || K > DI_MAX_K) return bad("K must be 1..1024");
    if (!(tau >= 1e-18f && tau <= 1e18f)) return bad("the temperature must be 1e-18..1e18");                 // its square and log2(e) over it are fp32 numbers
    if (T && (!x || !ids)) return bad("NULL tensor");
    if (T > 1 && ld < 0) return bad("rows must not run backwards");
    return MFAR_OK;
}

// ---- 8-bit linear -----------------------------------------------------------------------------------------------------------------------
template <typename T>
int quantize_rows(const void* x, int64_t ldx, int64_t M, int K, int8_t* q, int64_t ldq, float* scale, int pad, const Int8Copy& cp, hipStream_t st) {
    const int64_t blocks = cdiv(M, 4) + std::min<int64_t>(256, cdiv(cp.rows, 4));
    mfar_quantize_rows_kernel<T><<<blocks, 256, 0, st>>>((const T*)x, ldx, (int)M, K, (signed char*)q, ldq, scale, pad, cp);
    LAUNCHED("mfar_quantize_rows_kernel");
    return MFAR_OK;
}
// Tiles of 128 x 128 need about a block per CU to pay; fewer take 32 x 32 tiles, whose blocks divide k.
bool small_product(int64_t M, int64_t N) { return cdiv(M, 128) * cdiv(N, 128) < 128; }
template <typename T, int WN, int WM, int I, int J> int int8_gemm(const Int8Params& p, hipStream_t st) {
    typedef Int8Shape<WN, WM, I, J> S;
    static std::atomic<uint32_t> done{0};
    auto kernel = mfar_int8_gemm_kernel<T, WN, WM, I, J>;
    if (S::LDS > 64 * 1024) {
        const hipError_t e = allow_lds(kernel, done);
        if (e != hipSuccess) return hip_failed("mfar_int8_gemm_kernel", e);
    }
    kernel<<<cdiv(p.N, S::TN) * cdiv(p.M, S::TM), S::THREADS, S::LDS, st>>>(p);
    LAUNCHED("mfar_int8_gemm_kernel");
    return MFAR_OK;
}
template <typename T> int int8_product(const Int8Params& p, hipStream_t st) {
    if (small_product(p.M, p.N)) return launch<mfar_int8_tile_kernel<T>>("mfar_int8_tile_kernel", dim3(cdiv(p.N, 32), cdiv(p.M, 32)), 0, st, p);
    // Tiles of 256 x 256 move half the bytes per product but take a CU each: with a tile for every CU they win (16384 x 4096 x 4096: 287 us against 335;
    // 32768 x 768 x 1536: 54 against 62), with half as many they lose (8192 x 4096 x 1024: 84 us against 70, quantising included).
    if (cdiv(p.M, 256) * cdiv(p.N, 256) >= 256) return int8_gemm<T, 2, 4, 4, 2>(p, st);
    return int8_gemm<T, 2, 2, 2, 2>(p, st);
}
template <typename T, typename X> int int8_few(const Int8Params& p, const void* x, int64_t ldx, hipStream_t st) {
    const size_t lds = std::max<size_t>(Q8_FEW_ROWS * (size_t)(p.Kp + 16), 3 * 64 * 17 * 4);
    return launch<mfar_int8_few_kernel<T, X>>("mfar_int8_few_kernel", dim3(cdiv(p.N, 32)), lds, st, p, (const X*)x, (long long)ldx);
}
template <typename T> int int8_few_f32(const Int8Params& p, const void* x, int64_t ldx, hipStream_t st) { return int8_few<T, float>(p, x, ldx, st); }
template <typename T> int int8_few_bf16(const Int8Params& p, const void* x, int64_t ldx, hipStream_t st) { return int8_few<T, __bf16>(p, x, ldx, st); }
template <typename T> int int8_few_f16(const Int8Params& p, const void* x, int64_t ldx, hipStream_t st) { return int8_few<T, _Float16>(p, x, ldx, st); }
int check_rows(const void* x, int dtype, int64_t ldx, int64_t M, int K) {
    if (!type_size(dtype)) return bad("dtype must be F32, BF16 or F16");
    if (M < 0 || M > (1 << 23) || K < 1 || K > Q8_MAX_K) return bad("M must be 0..2^23, K 1..131072");
    if (M && !x) return bad("NULL tensor");
    if (M > 1 && ldx < 0) return bad("rows must not run backwards");
    return MFAR_OK;
}
int64_t padded_k(int K) { return cdiv(K, Q8_STEP) * Q8_STEP; }
// Few enough rows for every block to quantise them all.
bool few_rows(int64_t M, int K) { return M <= Q8_FEW_ROWS && K <= Q8_FEW_K; }
bool copies_weights(int64_t M, int64_t N, int K) { return K % 16 && !small_product(M, N); }   // rows have to start on 16 bytes
int64_t int8_scales_at(int64_t M, int K) { return M * padded_k(K); }
int64_t int8_weights_at(int64_t M, int K) { return int8_scales_at(M, K) + cdiv(M * 4, 16) * 16; }

}  // namespace

extern "C" int64_t mfar_attention_workspace_bytes(const mfar_attention* a, int backward) {
    const int rc = check_attention(a, false);
    if (rc != MFAR_OK) return rc;
    if (a->B == 0 || a->Lq == 0) return 0;
    if (!backward) return split_bytes(a);
    return drow_bytes(a) + (a->dtable ? cdiv(a->Lq, AT_COLS) * a->B * a->H * a->n_buckets * 4 : 0);
}
extern "C" int mfar_attention_forward(int device, const mfar_attention* a, void* stream) {
    int rc = check_attention(a, false);
    if (rc != MFAR_OK || a->B == 0 || a->Lq == 0) return rc;
    if (split_bytes(a) && (!a->workspace || a->workspace_bytes < split_bytes(a))) return bad("workspace too small");
    ON_DEVICE(device);
    const AttnParams p = attention_params(a);
    AttnSplit sp = {};
    if (few_queries(a)) sp = {(float*)a->workspace, (float*)a->workspace + split_rows(a) * a->D, key_splits(a)};
    return FOR_TYPE_AND_DIM(attention_forward, p, sp, (hipStream_t)stream);
}
extern "C" int mfar_attention_backward(int device, const mfar_attention* a, void* stream) {
    int rc = check_attention(a, true);
    if (rc != MFAR_OK) return rc;
    if (a->B == 0 || a->Lq == 0) return bad("an empty batch has no backward pass");
    if (!a->workspace || a->workspace_bytes < mfar_attention_workspace_bytes(a, 1)) return bad("workspace too small");
    ON_DEVICE(device);
    AttnParams p = attention_params(a);
    p.drow = (float*)a->workspace;
    p.dpart = a->dtable ? (float*)((char*)a->workspace + drow_bytes(a)) : nullptr;
    return FOR_TYPE_AND_DIM(attention_backward, p, a->dtable, (hipStream_t)stream);
}

extern "C" int mfar_quantize_rows(int device, const void* x, int dtype, int64_t ldx, int64_t M, int K, int8_t* q, int64_t ldq, float* scale, void* stream) {
    const int rc = check_rows(x, dtype, ldx, M, K);
    if (rc != MFAR_OK || M == 0) return rc;
    if (!q || !scale) return bad("NULL output");
    if (ldq < K) return bad("ldq must be at least K");
    ON_DEVICE(device);
    return FOR_TYPE(dtype, quantize_rows, x, ldx, M, K, q, ldq, scale, 0, Int8Copy{}, (hipStream_t)stream);
}
extern "C" int64_t mfar_int8_linear_workspace_bytes(int64_t M, int K, int N) {
    if (M < 0 || K < 1 || N < 0) return bad("M and N must be >= 0, K >= 1");
    if (few_rows(M, K)) return 0;
    return int8_weights_at(M, K) + (copies_weights(M, N, K) ? (int64_t)N * padded_k(K) : 0);
}
extern "C" int mfar_int8_linear(int device, const void* x, int dtype, int64_t ldx, int64_t M, int K, int N, const int8_t* wq, const float* w_scale,
                                const float* bias, void* y, int y_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    int rc = check_rows(x, dtype, ldx, M, K);
    if (rc != MFAR_OK) return rc;
    if (N < 0 || N > (1 << 23)) return bad("N must be 0..2^23");
    if (!type_size(y_dtype)) return bad("y_dtype must be F32, BF16 or F16");
    if (M == 0 || N == 0) return MFAR_OK;
    if (!wq || !w_scale || !y) return bad("NULL tensor");
    if (!aligned16(wq)) return bad("the weights must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    if (few_rows(M, K)) {
        ON_DEVICE(device);
        const Int8Params p = {nullptr, (const signed char*)wq, nullptr, w_scale, bias, y, 0, (long long)K, false, (int)M, N, K, (int)padded_k(K)};
        return dtype == MFAR_DTYPE_F32    ? FOR_TYPE(y_dtype, int8_few_f32, p, x, ldx, st)
               : dtype == MFAR_DTYPE_BF16 ? FOR_TYPE(y_dtype, int8_few_bf16, p, x, ldx, st)
                                          : FOR_TYPE(y_dtype, int8_few_f16, p, x, ldx, st);
    }
    if (!workspace || !aligned16(workspace) || workspace_bytes < mfar_int8_linear_workspace_bytes(M, K, N)) return bad("workspace too small or not 16-byte aligned");
    ON_DEVICE(device);
    const int64_t Kp = padded_k(K);
    int8_t* xq = (int8_t*)workspace;
    float* xs = (float*)((char*)workspace + int8_scales_at(M, K));
    Int8Copy cp = {};
    const signed char* w = (const signed char*)wq;
    int64_t ldw = K;
    if (copies_weights(M, N, K)) {
        cp = {w, (signed char*)workspace + int8_weights_at(M, K), (long long)Kp, N, K};
        w = cp.to, ldw = Kp;
    }
    rc = FOR_TYPE(dtype, quantize_rows, x, ldx, M, K, xq, Kp, xs, 1, cp, st);
    if (rc != MFAR_OK) return rc;
    const Int8Params p = {(const signed char*)xq, w, xs, w_scale, bias, y, (long long)Kp, (long long)ldw,
                          (int64_t)N * type_size(y_dtype) % 16 == 0 && aligned16(y), (int)M, N, K, (int)Kp};
    return FOR_TYPE(y_dtype, int8_product, p, st);
}

extern "C" int64_t mfar_distill_workspace_bytes(int64_t T, int64_t N) {
    if (T < 0 || N < 1 || N > (1 << 30)) return bad("T must be >= 0, N 1..2^30");
    const int64_t splits = cdiv(N, distill_chunk(T, N));
    return splits > 1 ? T * splits * 8 : 0;
}
extern "C" int mfar_distill_forward(int device, const void* student, int dtype, int64_t ld, int64_t T, int64_t N, const int64_t* ids, const float* scores,
                                    int K, float tau, float* loss, float* prob, float* stat, void* workspace, int64_t workspace_bytes, void* stream) {
    const int rc = check_distill(student, dtype, ld, T, N, ids, K, tau);
    if (rc != MFAR_OK || T == 0) return rc;
    if (!scores || !loss || !prob || !stat) return bad("NULL tensor");
    const int64_t need = mfar_distill_workspace_bytes(T, N);
    if (need && (!workspace || workspace_bytes < need)) return bad("workspace too small");
    ON_DEVICE(device);
    DistillParams p = {};
    p.x = student, p.x_row = ld, p.ids = (const long long*)ids, p.scores = scores, p.loss = loss, p.prob = prob, p.stat = stat, p.part = (float*)workspace;
    p.T = (int)T, p.N = (int)N, p.K = K, p.chunk = distill_chunk(T, N), p.splits = (int)cdiv(N, p.chunk), p.tau = tau;
    return FOR_TYPE(dtype, distill_forward, p, (hipStream_t)stream);
}
extern "C" int mfar_distill_backward(int device, const void* student, int dtype, int64_t ld, int64_t T, int64_t N, const int64_t* ids, int K, float tau,
                                     const float* prob, const float* stat, const float* dloss, void* dstudent, void* stream) {
    const int rc = check_distill(student, dtype, ld, T, N, ids, K, tau);
    if (rc != MFAR_OK || T == 0) return rc;
    if (!prob || !stat || !dloss || !dstudent) return bad("NULL tensor");
    ON_DEVICE(device);
    DistillParams p = {};
    p.x = student, p.x_row = ld, p.ids = (const long long*)ids, p.g = dloss, p.prob = (float*)prob, p.stat = (float*)stat, p.dx = dstudent;
    p.T = (int)T, p.N = (int)N, p.K = K, p.chunk = distill_chunk(T, N), p.splits = (int)cdiv(N, p.chunk), p.tau = tau;
    return FOR_TYPE(dtype, distill_backward, p, (hipStream_t)stream);
}
