// mfar_int8.h -- 8-bit linear layer: y[m][n] = (sum_k xq[m][k] wq[n][k]) * xs[m] * ws[n] + bias[n]
//
//   xs[m] = max_k |x[m][k]| (1 / 127), xq = rint(x / xs) (ties to even)          one scale per token, computed on the fly
// (1 / 127 rounded to fp32, which is 2^-28 off, then the product: within 1.07 half steps of max / 127, and what a division by a constant number gives in
// torch, so that the elementary operations there find the same bytes.  Of 4e7 random numbers 59 (fp32), 341 (fp16), 1832 (bf16) get another byte than
// under the scale in 64 bits, all next to a half; 61, 727 and 4577 would under the correctly rounded quotient.)
//   ws[n], wq: one scale per output channel, laid out once by the caller
// The integer sums are exact (|sum| <= 127^2 K < 2^31 for K <= 131072); a sum's conversion, the two products with the scales and the sum with the bias
// round to fp32, the result to its type.
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

// chunk c (8 elements) of a row that may start anywhere: an unaligned vector load
template <typename T> __device__ __forceinline__ V8<T> q8_load(const T* row, int c) {
    V8<T> x;
    __builtin_memcpy(&x, row + 8 * c, sizeof x);
    return x;
}
// the chunk that the row's end cuts, zeros behind it
template <typename T> __device__ __forceinline__ V8<T> q8_load_cut(const T* row, int c, int K) {
    V8<T> x = {};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (8 * c + j < K) x[j] = row[8 * c + j];
    return x;
}
// |x| with NaN as infinity, so that a maximum keeps it
__device__ __forceinline__ float q8_size(float x) {
    const float a = __builtin_fabsf(x);
    return a <= 3.4028234e38f ? a : __builtin_inff();
}
// A row's scale and the bytes under it: rint(x / s), the quotient rounded to fp32 first.  quick: y = 1 / s rounded, then one step of the remainder gives
// the correctly rounded quotient (Markstein; not for divisors of an all-ones mantissa, nor where 1 / s or the remainder would leave the normal
// range); adding 1.5 * 2^23 leaves the whole number in the low byte.
struct Q8Divisor {
    float s, y;
    bool live, quick;
    __device__ __forceinline__ explicit Q8Divisor(float top) {
        s = top == __builtin_inff() ? __builtin_nanf("") : top * (1.0f / 127.0f);
        live = s > 0.0f;
        quick = s > 1e-30f && (__float_as_uint(s) & 0x7fffff) != 0x7fffff;
        y = 1.0f / s;
    }
    template <typename T> __device__ __forceinline__ u64 pack(const V8<T>& x) const {
        u64 w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float v = (float)x[j], q = v * y;
            w |= (u64)(__float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, s, v), y, q) + 12582912.0f) & 0xffu) << (8 * j);
        }
        return w;
    }
    template <typename T> __device__ __forceinline__ u64 pack_slowly(const V8<T>& x) const {
        u64 w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= (u64)((u32)(int)fminf(fmaxf(__builtin_rintf((float)x[j] / s), -127.0f), 127.0f) & 0xffu) << (8 * j);
        return live ? w : 0;
    }
};

// One row by LANES lanes (`i`: this lane's place among them): K elements of xr -> bytes at qr, of which [K, ldq) become zeros with pad; returns the scale.
// Up to KEPT chunks a lane stay in registers between the row's maximum and its bytes; longer rows are read again.  Whole chunks, the cut one and
// the divisors that need a true division take paths of their own: unrolled together they did not fit the instruction cache.
template <typename T, int LANES, int KEPT> __device__ __forceinline__ float q8_row(const T* xr, int K, signed char* qr, long long ldq, bool pad, int i) {
    const int whole = K / 8, cut = K % 8 && whole % LANES == i ? whole : -1;
    V8<T> kept[KEPT], end = {};
    float top = 0.0f;
    auto larger = [&](const V8<T>& v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, q8_size((float)v[j]));
    };
#pragma unroll
    for (int t = 0; t < KEPT; ++t)
        if (t * LANES < whole) kept[t] = t * LANES + i < whole ? q8_load<T>(xr, t * LANES + i) : V8<T>{};
    if (cut >= 0) {
        end = q8_load_cut<T>(xr, cut, K);
        larger(end);
    }
#pragma unroll
    for (int t = 0; t < KEPT; ++t)
        if (t * LANES < whole) larger(kept[t]);
#pragma unroll 1
    for (int c = KEPT * LANES + i; c < whole; c += LANES) larger(q8_load<T>(xr, c));
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const Q8Divisor d(top);
    auto put = [&](int c, u64 w) { __builtin_memcpy(qr + 8 * c, &w, 8); };
    int from = i;
    if (d.quick) {
#pragma unroll
        for (int t = 0; t < KEPT; ++t)
            if (t * LANES + i < whole) put(t * LANES + i, d.pack<T>(kept[t]));
        from = KEPT * LANES + i;
    }
#pragma unroll 1
    for (int c = from; c < whole; c += LANES) {
        const V8<T> v = q8_load<T>(xr, c);
        put(c, d.quick ? d.pack<T>(v) : d.pack_slowly<T>(v));
    }
    if (cut >= 0) {
        const u64 w = d.pack_slowly<T>(end);                               // (what lies behind the row's end quantises from zeros)
        if (pad) put(cut, w);
        else
            for (int j = 0; 8 * cut + j < K; ++j) qr[8 * cut + j] = (signed char)(w >> (8 * j));
    }
    if (pad)
        for (long long c = (K + 7) / 8 + i; c < ldq / 8; c += LANES) put((int)c, 0);
    return d.s;
}

// Rows of x -> 8-bit rows (ldq bytes apart; pad: bytes [K, ldq) become zeros) and their scales.  One wave per row.
// Bound by reading x: 32768 x 768 fp16 (75 MB) 20 us, 16384 x 4096 bf16 (201 MB) 46 us.
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
    const float s = q8_row<T, 64, Q8_KEPT>(x + (long long)row * ldx, K, q + (long long)row * ldq, ldq, pad != 0, l);
    if (l == 0) scale[row] = s;
}

struct Int8Params {
    const signed char *xq, *wq;
    const float *xs, *ws, *bias;
    void* y;
    long long ldx, ldw;
    bool whole_rows;             // rows of y start on 16 bytes
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
            o[j] = (T)(v + (p.bias ? p.bias[at] : 0.0f));
        }
        if (n + 4 <= p.N) __builtin_memcpy(y + n, &o, sizeof o);
        else
            for (int j = 0; j < 4; ++j)
                if (n + j < p.N) y[n + j] = o[j];
    }
}

// 16 bytes of a channel's weights.  Past a row's end they may be anything (x holds zeros there), but past the last row's end nothing is read.
__device__ __forceinline__ i32x4 q8_weights(const Int8Params& p, int n, int k) {
    i32x4 w = {};
    if (k < p.K) {
        const long long at = (long long)min(n, p.N - 1) * p.ldw + k, end = (long long)(p.N - 1) * p.ldw + p.K;
        if (at + 16 <= end) {
            __builtin_memcpy(&w, p.wq + at, 16);
        } else {
            u64 part[2] = {0, 0};
#pragma unroll 1
            for (long long j = end - 1; j >= at; --j) {                     // from the last byte down, each pushing the others up
                part[1] = part[1] << 8 | part[0] >> 56;
                part[0] = part[0] << 8 | (unsigned char)p.wq[j];
            }
            __builtin_memcpy(&w, part, 16);
        }
    }
    return w;
}

// ---- up to 32 tokens: quantising and product in one launch ------------------------------------------------------------------------------------
// Every block quantises all rows into LDS (they are few) while its first weights are on their way, then multiplies 32 channels by them, k divided over
// the waves.  12 x 768 x 768: one launch of 8 us for two of 9 together.
#define Q8_FEW_ROWS 32
#define Q8_FEW_K 2048
template <typename T, typename X>
__global__ __launch_bounds__(256) void mfar_int8_few_kernel(const Int8Params p, const X* x, long long ldx) {
    extern __shared__ __align__(16) signed char q8_lds[];                  // [32][Kp + 16] rows, then partial sums
    __shared__ float scales[Q8_FEW_ROWS];
    const int n0 = blockIdx.x * 32, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, half = l >> 5;
    const int pitch = p.Kp + 16;
    i32x4 a[4];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) a[u] = q8_weights(p, n0 + (l & 31), k0 + u * 128 + 16 * half);
    };
    fetch(wave * 32);
    // 16 lanes a row, 16 rows at a time
    for (int r0 = 0; r0 < p.M; r0 += 16) {
        const int r = r0 + (int)threadIdx.x / 16;
        if (r < p.M) {
            const float s = q8_row<X, 16, 8>(x + (long long)r * ldx, p.K, q8_lds + r * pitch, p.Kp, true, threadIdx.x & 15);
            if ((threadIdx.x & 15) == 0) scales[r] = s;
        }
    }
    __syncthreads();
    const signed char* row = q8_lds + min(l & 31, p.M - 1) * pitch + 16 * half;
    i32x16 acc = {};
    for (int k0 = wave * 32; k0 < p.K; k0 += 4 * 128) {
        i32x4 b[4], now[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            now[u] = a[u];
            b[u] = k0 + u * 128 + 16 * half < p.Kp ? *(const i32x4*)(row + k0 + u * 128) : i32x4{};
        }
        if (k0 + 4 * 128 < p.K) fetch(k0 + 4 * 128);
#pragma unroll
        for (int u = 0; u < 4; ++u) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(now[u], b[u], acc, 0, 0, 0);
    }
    __syncthreads();                                                       // (the rows' memory takes the partial sums)
    int* part = (int*)q8_lds;                                              // [3][64][17]
    if (wave) {
#pragma unroll
        for (int i = 0; i < 16; ++i) part[((wave - 1) * 64 + l) * 17 + i] = acc[i];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] += part[l * 17 + i] + part[(64 + l) * 17 + i] + part[(128 + l) * 17 + i];
    Int8Params o = p;
    o.xs = scales;
    q8_store<T>(o, acc, n0, l & 31);
}

// ---- few tiles: one 32 x 32 tile per block, its k divided over the 4 waves, fragments straight from memory -------------------------------------
// Bound by latency: every load of a wave's share is in flight at once.  1003 x 1001 x 519: 11 us.  Rows of the weights may start anywhere.
template <typename T>
__global__ __launch_bounds__(256) void mfar_int8_tile_kernel(const Int8Params p) {
    __shared__ int part[3][64][17];
    const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, half = l >> 5;
    const signed char* x = p.xq + (long long)min(m0 + (l & 31), p.M - 1) * p.ldx;
    i32x16 acc = {};
    for (int k0 = wave * 32; k0 < p.K; k0 += 4 * 128) {
        i32x4 a[4], b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = k0 + u * 128 + 16 * half;
            a[u] = q8_weights(p, n0 + (l & 31), k);
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

// ---- many tiles ------------------------------------------------------------------------------------------------------------------------------------
// Bound by the matrix units at long k (16384 x 4096 x 4096: 248 to 291 us, 1.9 to 2.2 10^15 operations a second), by filling and storing a tile at short
// (32768 x 768 x 1536: 53 us).
// A block computes TN channels x TM tokens with WN x WM waves of I x J tiles each, in k steps of 128 bytes (whole cache lines: steps of 64 bytes in a
// deeper ring were 15 % slower).  Both operands go straight from memory to LDS, two steps' buffers in turn, one barrier a step.  A load
// instruction of a wave fills 8 rows of 128 bytes in lane order; the swizzle (chunk c of row r at place c ^ (r / 2 % 8): 16 rows at one chunk meet
// 64 different banks) is applied on the addresses the lanes load from.  Rows of both operands start on 16 bytes.
__device__ __forceinline__ int q8_swz(int r) { return (r >> 1) & 7; }
__device__ __forceinline__ void q8_to_lds(const signed char* base, u32 off, u32 lds) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
}

template <int WN, int WM, int I, int J> struct Int8Shape {
    static constexpr int WAVES = WN * WM, THREADS = 64 * WAVES, TN = WN * I * 32, TM = WM * J * 32, BYTES = (TN + TM) * Q8_STEP;
    static constexpr int LDS = 2 * BYTES + (2 * TN + TM) * 4;
    static_assert(TN * Q8_STEP % (1024 * WAVES) == 0 && TM * Q8_STEP % (1024 * WAVES) == 0);
    static_assert(WAVES * 32 * (64 * 4 + 16) <= 2 * BYTES && I % 2 == 0);
};
template <int I, int J> struct Int8Frags { i32x4 a[I], b[J]; };

template <typename T, int WN, int WM, int I, int J>
__global__ __launch_bounds__(64 * WN * WM, 2) void mfar_int8_gemm_kernel(const Int8Params p) {
    typedef Int8Shape<WN, WM, I, J> S;
    extern __shared__ __align__(16) signed char q8_lds[];                  // [2][weights TN, tokens TM][Q8_STEP]
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), l = threadIdx.x & 63, half = l >> 5;
    // consecutive blocks go to the 8 XCDs in turn: an XCD takes a run of tiles, walked in groups of 4 token tiles, so that its L2 sees rows again
    const int tn = (p.N + S::TN - 1) / S::TN, tm = (p.M + S::TM - 1) / S::TM, total = tn * tm, id = blockIdx.x;
    const int xcd = id % 8, at = xcd * (total / 8) + min(xcd, total % 8) + id / 8;
    const int group = at / (4 * tn), rows = min(4, tm - group * 4), in = at - group * 4 * tn;
    const int m0 = (group * 4 + in % rows) * S::TM, n0 = in / rows * S::TN;
    const signed char* xb = p.xq + (long long)m0 * p.ldx;
    const signed char* wb = p.wq + (long long)n0 * p.ldw;
    constexpr int PW = S::TN * Q8_STEP / 1024 / S::WAVES, PX = S::TM * Q8_STEP / 1024 / S::WAVES;
    u32 xo[PX], wo[PW], wl[PW];
    const int steps = p.Kp / Q8_STEP, cut = p.K - (steps - 1) * Q8_STEP;    // bytes of the last step that the weights have
#pragma unroll
    for (int t = 0; t < PW; ++t) {
        const int r = (wave * PW + t) * 8 + (l >> 3), c = (l & 7) ^ q8_swz(r), row = min(r, p.N - 1 - n0) * (int)p.ldw;
        wo[t] = (u32)(row + c * 16);
        wl[t] = (u32)(row + (c * 16 < cut ? c * 16 : 0));                  // past the row's end: any bytes, x holds zeros there
    }
#pragma unroll
    for (int t = 0; t < PX; ++t) {
        const int r = (wave * PX + t) * 8 + (l >> 3), c = (l & 7) ^ q8_swz(r);
        xo[t] = (u32)(min(r, p.M - 1 - m0) * (int)p.ldx + c * 16);
    }
    const u32 lds = (u32)(uintptr_t)q8_lds;
    auto load = [&](int s) {
        const u32 to = lds + (s & 1) * S::BYTES + wave * PW * 1024, tx = lds + (s & 1) * S::BYTES + S::TN * Q8_STEP + wave * PX * 1024;
        const signed char *x = xb + s * Q8_STEP, *w = wb + s * Q8_STEP;
        const bool last = s == steps - 1;
#pragma unroll
        for (int t = 0; t < PW; ++t) q8_to_lds(w, last ? wl[t] : wo[t], to + t * 1024);
#pragma unroll
        for (int t = 0; t < PX; ++t) q8_to_lds(x, xo[t], tx + t * 1024);
    };
    // the tile's scales and bias, for the epilogue
    float* channels = (float*)(q8_lds + 2 * S::BYTES);                // [2][TN] scales, bias
    float* tokens = channels + 2 * S::TN;                                  // [TM] scales
    for (int i = threadIdx.x; i < S::TN; i += S::THREADS) {
        const int n = min(n0 + i, p.N - 1);
        channels[i] = p.ws[n];
        channels[S::TN + i] = p.bias ? p.bias[n] : 0.0f;
    }
    for (int i = threadIdx.x; i < S::TM; i += S::THREADS) tokens[i] = p.xs[min(m0 + i, p.M - 1)];

    const int wn = wave % WN * I * 32, wm = wave / WN * J * 32;
    i32x16 acc[I][J] = {};
    // Fragments are read a quarter step ahead of their products: while the matrix units work on one quarter, the next (of this step, or the first of the
    // next step, behind its wait and barrier) comes from LDS.
    Int8Frags<I, J> f[2];
    auto read = [&](Int8Frags<I, J>& to, int s, int u) {
        const signed char* wt = q8_lds + (s & 1) * S::BYTES;
        const signed char* xt = wt + S::TN * Q8_STEP;
        const int c = 2 * u + half;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int r = wn + 32 * i + (l & 31);
            to.a[i] = *(const i32x4*)(wt + r * Q8_STEP + ((c ^ q8_swz(r)) << 4));
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int r = wm + 32 * j + (l & 31);
            to.b[j] = *(const i32x4*)(xt + r * Q8_STEP + ((c ^ q8_swz(r)) << 4));
        }
    };
    auto multiply = [&](const Int8Frags<I, J>& g) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(g.a[i], g.b[j], acc[i][j], 0, 0, 0);
    };
    // a step is there once every wave has waited for its own loads; by then every wave also holds its last fragments of the step before
    auto arrive = [&]() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
    };
    load(0);
    arrive();
    if (steps > 1) load(1);
    read(f[0], 0, 0);
    for (int s = 0; s < steps; ++s) {
        read(f[1], s, 1);
        multiply(f[0]);
        read(f[0], s, 2);
        multiply(f[1]);
        read(f[1], s, 3);
        multiply(f[0]);
        if (s + 1 < steps) {
            arrive();
            if (s + 2 < steps) load(s + 2);
            read(f[0], s + 1, 0);
        }
        multiply(f[1]);
    }
    if (!p.whole_rows) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < I; ++i) q8_store<T>(p, acc[i][j], n0 + wn + 32 * i, m0 + wm + 32 * j + (l & 31));
        return;
    }
    // Scaled results through LDS of the wave's own, 32 tokens x 64 channels at a time, so that a token's channels leave in runs of 16 bytes a lane
    // (8 bytes a lane of 32 different tokens straight from the registers: twice the time at 32768 x 768 x 1536)
    constexpr int PITCH = 64 * sizeof(T) + 16, LANES = 64 * sizeof(T) / 16, EACH = 16 / sizeof(T);
    __syncthreads();
    signed char* mine = q8_lds + wave * 32 * PITCH;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const float xs = tokens[wm + 32 * j + (l & 31)];
#pragma unroll
        for (int i0 = 0; i0 < I; i0 += 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int n = 32 * i + 8 * g + 4 * half;
                    const f32x4 ws = *(const f32x4*)(channels + wn + 32 * i0 + n), bias = *(const f32x4*)(channels + S::TN + wn + 32 * i0 + n);
                    V4<T> o;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = (T)((float)acc[i0 + i][j][4 * g + e] * xs * ws[e] + bias[e]);
                    *(V4<T>*)(mine + (l & 31) * PITCH + n * sizeof(T)) = o;
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += 64 / LANES) {
                const int r = r0 + l / LANES, c = l % LANES, m = m0 + wm + 32 * j + r, n = n0 + wn + 32 * i0 + c * EACH;
                const i32x4 x = *(const i32x4*)(mine + r * PITCH + c * 16);
                if (m < p.M && n < p.N) *(i32x4*)((T*)p.y + (long long)m * p.N + n) = x;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}
