// mfar_int8.h -- 8-bit linear layer: y[m][n] = (sum_k xq[m][k] wq[n][k]) * xs[m] * ws[n] + bias[n]
//
//   xs[m] = max_k |x[m][k]| / 127, xq = rint(x / xs) (ties to even)          one scale per token, computed on the fly
//   ws[n], wq: one scale per output channel, laid out once by the caller
// The integer sums are exact (|sum| <= 127^2 K < 2^31 for K <= 131072); rounding happens in the scales and once at the end.
// A row of zeros has scale 0 and gives the bias; a row with an infinity or NaN has scale NaN and gives NaN.
//
// The product is computed as W X' (rows: channels, columns: tokens): a lane of a result tile then holds runs of 4 channels of one token and stores
// them together.  Fragments of v_mfma_i32_32x32x32_i8: lane l holds row l % 32 and the 16 bytes k = 16 (l / 32) .. + 15 of a step of 32.
#pragma once
#include "mfar_ops_device.h"

#define Q8_MAX_K 131072
#define Q8_KEPT 8                // chunks of 8 elements a lane keeps in registers while its row's maximum is found: rows up to 4096
#define Q8_STEP 128              // bytes of k per staged step

typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// rows of `n` bytes at their places in a padded copy (weights whose rows do not start on 16 bytes)
struct Int8Copy {
    const signed char* from;
    signed char* to;
    long long ld;
    int rows, n;
};

template <typename T> __device__ __forceinline__ V8<T> q8_load(const T* row, int c, int K) {
    V8<T> x = {};
    if (8 * c + 8 <= K) __builtin_memcpy(&x, row + 8 * c, sizeof x);       // (rows may start anywhere: unaligned vector loads)
    else
        for (int j = 0; j < 8; ++j)
            if (8 * c + j < K) x[j] = row[8 * c + j];
    return x;
}
// |x| with NaN as infinity, so that a maximum keeps it
__device__ __forceinline__ float q8_size(float x) {
    const float a = __builtin_fabsf(x);
    return a <= 3.4028234e38f ? a : __builtin_inff();
}
// rint(x / s) as a byte, the quotient rounded to fp32 first.  quick: y = 1 / s rounded, then one step of the remainder gives the correctly rounded
// quotient (Markstein; not for divisors of an all-ones mantissa, nor where 1 / s or the remainder would leave the normal range); adding 1.5 * 2^23
// leaves the whole number in the low byte.
__device__ __forceinline__ u32 q8_byte(float x, float s, float y, bool quick) {
    if (quick) {
        const float q = x * y;
        return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, s, x), y, q) + 12582912.0f) & 0xffu;
    }
    return (u32)(int)fminf(fmaxf(__builtin_rintf(x / s), -127.0f), 127.0f) & 0xffu;
}
template <typename T> __device__ __forceinline__ u64 q8_pack(const V8<T>& x, float s, float y, bool quick) {
    u64 w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) w |= (u64)q8_byte((float)x[j], s, y, quick) << (8 * j);
    return w;
}

// Rows of x -> 8-bit rows (ldq bytes apart; pad: bytes [K, ldq) become zeros) and their scales.  One wave per row; a row is read once while it fits
// the registers.  Bound by reading x: 32768 x 768 fp16 (75 MB) 16 us.
// The blocks behind the rows' copy weights (launch count: one).
template <typename T>
__global__ __launch_bounds__(256) void mfar_quantize_rows_kernel(const T* x, long long ldx, int M, int K, signed char* q, long long ldq, float* scale, int pad, const Int8Copy cp) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, row = blockIdx.x * 4 + wave;
    const int row_blocks = (M + 3) / 4;
    if ((int)blockIdx.x >= row_blocks) {
        for (int r = ((int)blockIdx.x - row_blocks) * 4 + wave; r < cp.rows; r += ((int)gridDim.x - row_blocks) * 4) {
            const signed char* from = cp.from + (long long)r * cp.n;
            for (int k = l * 8; k < cp.n; k += 512) {
                u64 w = 0;
                if (k + 8 <= cp.n) __builtin_memcpy(&w, from + k, 8);
                else
                    for (int j = 0; k + j < cp.n; ++j) w |= (u64)(unsigned char)from[k + j] << (8 * j);
                *(u64*)(cp.to + (long long)r * cp.ld + k) = w;
            }
        }
        return;
    }
    if (row >= M) return;
    const T* xr = x + (long long)row * ldx;
    signed char* qr = q + (long long)row * ldq;
    const int chunks = (K + 7) / 8;
    V8<T> kept[Q8_KEPT];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < Q8_KEPT; ++i)
        if (i * 64 < chunks) {
            const int c = i * 64 + l;
            kept[i] = c < chunks ? q8_load<T>(xr, c, K) : V8<T>{};
        }
#pragma unroll
    for (int i = 0; i < Q8_KEPT; ++i)
        if (i * 64 < chunks) {
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, q8_size((float)kept[i][j]));
        }
    for (int c = Q8_KEPT * 64 + l; c < chunks; c += 64) {
        const V8<T> v = q8_load<T>(xr, c, K);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, q8_size((float)v[j]));
    }
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float s = top == __builtin_inff() ? __builtin_nanf("") : top / 127.0f;
    if (l == 0) scale[row] = s;
    const bool live = s > 0.0f, quick = s > 1e-30f && (__float_as_uint(s) & 0x7fffff) != 0x7fffff;
    const float y = 1.0f / s;
    auto put = [&](int c, const V8<T>& v) {
        const u64 w = live ? q8_pack<T>(v, s, y, quick) : 0;
        if (8 * c + 8 <= K || pad) __builtin_memcpy(qr + 8 * c, &w, 8);      // (what lies behind the row's end quantises from zeros)
        else
            for (int j = 0; 8 * c + j < K; ++j) qr[8 * c + j] = (signed char)(w >> (8 * j));
    };
#pragma unroll
    for (int i = 0; i < Q8_KEPT; ++i)
        if (i * 64 + l < chunks) put(i * 64 + l, kept[i]);
    for (int c = Q8_KEPT * 64 + l; c < chunks; c += 64) put(c, q8_load<T>(xr, c, K));
    if (pad)
        for (long long c = chunks + l; c < ldq / 8; c += 64) *(u64*)(qr + 8 * c) = 0;
}

struct Int8Params {
    const signed char *xq, *wq;
    const float *xs, *ws, *bias;
    void* y;
    long long ldx, ldw;
    int M, N, K, Kp;             // Kp: K rounded up to Q8_STEP; xq rows hold zeros in [K, Kp)
};

// one lane's column of a 32 x 32 tile: channels n0 + crow(i), token m
template <typename T> __device__ __forceinline__ void q8_store(const Int8Params& p, const i32x16& acc, int n0, int m) {
    if (m >= p.M) return;
    const int half = (threadIdx.x & 63) >> 5;
    const float xs = p.xs[m];
    T* y = (T*)p.y + (long long)m * p.N;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const int n = n0 + 8 * g + 4 * half;
        V4<T> o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = min(n + j, p.N - 1);
            const float v = (float)acc[4 * g + j] * xs * p.ws[at];
            o[j] = (T)(p.bias ? v + p.bias[at] : v);
        }
        if (n + 4 <= p.N) __builtin_memcpy(y + n, &o, sizeof o);
        else
            for (int j = 0; j < 4; ++j)
                if (n + j < p.N) y[n + j] = o[j];
    }
}

// ---- few tiles: one 32 x 32 tile per block, its k divided over the 4 waves, fragments straight from memory -------------------------------------
// Bound by latency: every load of a wave's share is in flight at once.  Rows of the weights may start anywhere.
template <typename T>
__global__ __launch_bounds__(256) void mfar_int8_tile_kernel(const Int8Params p) {
    __shared__ int part[3][64][17];
    const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, half = l >> 5;
    const signed char* x = p.xq + (long long)min(m0 + (l & 31), p.M - 1) * p.ldx;
    const long long w0 = (long long)min(n0 + (l & 31), p.N - 1) * p.ldw, w_end = (long long)(p.N - 1) * p.ldw + p.K;
    i32x16 acc = {};
    auto weights = [&](int k) {
        // past a row's end the weights may be anything (x holds zeros there), but past the last row's end nothing is read
        i32x4 w = {};
        if (k < p.K) {
            const long long at = w0 + k;
            if (at + 16 <= w_end) {
                __builtin_memcpy(&w, p.wq + at, 16);
            } else {
                signed char tail[16];
                for (int j = 0; j < 16; ++j) tail[j] = at + j < w_end ? p.wq[at + j] : (signed char)0;
                __builtin_memcpy(&w, tail, 16);
            }
        }
        return w;
    };
    for (int k0 = wave * 32; k0 < p.K; k0 += 4 * 128) {
        i32x4 a[4], b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = k0 + u * 128 + 16 * half;
            a[u] = weights(k);
            b[u] = k < p.Kp ? *(const i32x4*)(x + k) : i32x4{};
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[u], b[u], acc, 0, 0, 0);
    }
    if (wave) {
#pragma unroll
        for (int i = 0; i < 16; ++i) part[wave - 1][l][i] = acc[i];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] += part[0][l][i] + part[1][l][i] + part[2][l][i];
    q8_store<T>(p, acc, n0, m0 + (l & 31));
}

// ---- many tiles: 128 channels x 128 tokens per block, 4 waves of 64 x 64, k steps of 128 bytes ---------------------------------------------------
// Both operands go straight from memory to LDS, two steps' buffers in turn, one barrier a step.  A wave's load instruction fills 8 rows of 128 bytes
// in lane order; the swizzle (chunk c of row r at place c ^ (r / 2 % 8): 16 rows at one chunk meet 64 different banks) is applied on the
// addresses the lanes load from.  Rows of both operands start on 16 bytes.
__device__ __forceinline__ int q8_swz(int r) { return (r >> 1) & 7; }
#define Q8_TILE 128
#define Q8_TILE_BYTES (Q8_TILE * Q8_STEP)

__device__ __forceinline__ void q8_to_lds(const signed char* base, u32 off, u32 lds) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
}

template <typename T>
__global__ __launch_bounds__(256, 2) void mfar_int8_gemm_kernel(const Int8Params p) {
    extern __shared__ __align__(16) signed char q8_lds[];                  // [2][weights, tokens][128][128]
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, half = l >> 5;
    // consecutive blocks go to the 8 XCDs in turn: an XCD takes a run of tiles, walked in groups of 4 token tiles, so that its L2 sees rows again
    const int tn = (p.N + Q8_TILE - 1) / Q8_TILE, tm = (p.M + Q8_TILE - 1) / Q8_TILE, total = tn * tm, id = blockIdx.x;
    const int per = total / 8, rest = total % 8, xcd = id % 8;
    const int at = xcd * per + min(xcd, rest) + id / 8;
    const int group = at / (4 * tn), rows = min(4, tm - group * 4), in = at - group * 4 * tn;
    const int m0 = (group * 4 + in % rows) * Q8_TILE, n0 = in / rows * Q8_TILE;
    const signed char* xb = p.xq + (long long)m0 * p.ldx;
    const signed char* wb = p.wq + (long long)n0 * p.ldw;
    u32 xo[4], wo[4], wl[4];
    const int steps = p.Kp / Q8_STEP, cut = p.K - (steps - 1) * Q8_STEP;    // bytes of the last step that the weights have
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int r = (wave * 4 + t) * 8 + (l >> 3), c = (l & 7) ^ q8_swz(r);
        const int wr = min(r, p.N - 1 - n0) * (int)p.ldw;
        xo[t] = (u32)(min(r, p.M - 1 - m0) * (int)p.ldx + c * 16);
        wo[t] = (u32)(wr + c * 16);
        wl[t] = (u32)(wr + (c * 16 < cut ? c * 16 : 0));                   // past the row's end: any bytes, x holds zeros there
    }
    const u32 lds = (u32)(uintptr_t)q8_lds;
    auto load = [&](int s) {
        const u32 to = lds + (s & 1) * 2 * Q8_TILE_BYTES + wave * 4096;
        const signed char *x = xb + s * Q8_STEP, *w = wb + s * Q8_STEP;
        const bool last = s == steps - 1;
#pragma unroll
        for (int t = 0; t < 4; ++t) q8_to_lds(w, last ? wl[t] : wo[t], to + t * 1024);
#pragma unroll
        for (int t = 0; t < 4; ++t) q8_to_lds(x, xo[t], to + Q8_TILE_BYTES + t * 1024);
    };
    const int wn = (wave & 1) * 64, wm = (wave >> 1) * 64;
    i32x16 acc[2][2] = {};
    load(0);
    for (int s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                    // this wave's loads of step s
        __syncthreads();                                                   // everyone's; and step s - 1 has been read
        if (s + 1 < steps) load(s + 1);
        const signed char* wt = q8_lds + (s & 1) * 2 * Q8_TILE_BYTES;
        const signed char* xt = wt + Q8_TILE_BYTES;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            i32x4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int rn = wn + 32 * i + (l & 31), rm = wm + 32 * i + (l & 31), c = 2 * u + half;
                a[i] = *(const i32x4*)(wt + rn * 128 + ((c ^ q8_swz(rn)) << 4));
                b[i] = *(const i32x4*)(xt + rm * 128 + ((c ^ q8_swz(rm)) << 4));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) q8_store<T>(p, acc[i][j], n0 + wn + 32 * i, m0 + wm + 32 * j + (l & 31));
}
