// mfar_int8.h -- 8-bit linear layer: y[m][n] = (sum_k xq[m][k] wq[n][k]) * xs[m] * ws[n] + bias[n]
//
//   xs[m] = max_k |x[m][k]| / 127, xq = rint(x / xs) (ties to even)          one scale per token, computed on the fly
//   ws[n], wq: one scale per output channel, laid out once by the caller
// The integer sums are exact (|sum| <= 127^2 K < 2^31 for K <= 131072); rounding happens in the scales and once at the end.
// A row of zeros has scale 0 and gives the bias; a row with an infinity or NaN has scale NaN and gives NaN.
#pragma once
#include "mfar_ops_device.h"

#define Q8_TILE 128
#define Q8_MAX_K 131072

typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// rows of x -> 8-bit rows (ldq bytes apart, bytes [K, ldq) zero when pad != 0) and their scales; one wave per row
template <typename T>
__global__ __launch_bounds__(256) void mfar_quantize_rows_kernel(const T* x, long long ldx, int M, int K, signed char* q, long long ldq, float* scale, int pad) {
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
    if (row >= M) return;
    const T* xr = x + (long long)row * ldx;
    float top = 0.0f;
    for (int k = l; k < K; k += 64) {
        const float a = __builtin_fabsf((float)xr[k]);
        top = a <= 3.4028234e38f ? fmaxf(top, a) : __builtin_inff();        // (NaN and inf: the row is poisoned below)
    }
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const bool bad = top == __builtin_inff();
    const float s = bad ? __builtin_nanf("") : top / 127.0f;
    signed char* qr = q + (long long)row * ldq;
    const bool live = s > 0.0f;
    for (int k = l; k < K; k += 64) {
        const float n = live ? __builtin_rintf((float)xr[k] / s) : 0.0f;
        qr[k] = (signed char)(int)fminf(fmaxf(n, -127.0f), 127.0f);
    }
    if (pad)
        for (long long k = K + l; k < ldq; k += 64) qr[k] = 0;
    if (l == 0) scale[row] = s;
}

struct Int8Params {
    const signed char *xq, *wq;
    const float *xs, *ws, *bias;
    void* y;
    long long ldx, ldw;
    int M, N, K, Kp;             // Kp: K rounded up to 128; xq rows hold zeros in [K, Kp)
};

__device__ __forceinline__ int q8_swz(int r) { return (r >> 1) & 7; }

// Tiles of 128 x 128, k steps of 128 bytes; 4 waves of 64 x 64.  The product is computed as W X' (rows: channels, columns: tokens), so that a
// lane holds runs of 4 channels of one token and stores them together.
template <typename T>
__global__ __launch_bounds__(256) void mfar_int8_gemm_kernel(const Int8Params p) {
    __shared__ __align__(16) signed char xt[Q8_TILE * 128], wt[Q8_TILE * 128];
    const int n0 = blockIdx.x * Q8_TILE, m0 = blockIdx.y * Q8_TILE, wave = threadIdx.x >> 6, l = threadIdx.x & 63, half = l >> 5;
    const int wn = (wave & 1) * 64, wm = (wave >> 1) * 64;
    i32x16 acc[2][2] = {};
    const long long w_end = (long long)(p.N - 1) * p.ldw + p.K;             // one past the weights' last byte
    for (int k0 = 0; k0 < p.Kp; k0 += 128) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int e = t * 256 + (int)threadIdx.x, r = e >> 3, c = e & 7;
            const int m = min(m0 + r, p.M - 1), n = min(n0 + r, p.N - 1), k = k0 + c * 16;
            *(i32x4*)(xt + r * 128 + ((c ^ q8_swz(r)) << 4)) = *(const i32x4*)(p.xq + (long long)m * p.ldx + k);
            // past a row's end the weights may be anything: x holds zeros there.  Past the last row's end nothing is read.
            const long long at = (long long)n * p.ldw + k;
            i32x4 w = {};
            if (k < p.K) {
                if (at + 16 <= w_end) {
                    __builtin_memcpy(&w, p.wq + at, 16);
                } else {
                    signed char tail[16];
                    for (int j = 0; j < 16; ++j) tail[j] = at + j < w_end ? p.wq[at + j] : (signed char)0;
                    __builtin_memcpy(&w, tail, 16);
                }
            }
            *(i32x4*)(wt + r * 128 + ((c ^ q8_swz(r)) << 4)) = w;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            i32x4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int rn = wn + 32 * i + (l & 31), rm = wm + 32 * i + (l & 31), c = 2 * s + half;
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
    for (int j = 0; j < 2; ++j) {
        const int m = m0 + wm + 32 * j + (l & 31);
        if (m >= p.M) continue;
        const float xs = p.xs[m];
        T* y = (T*)p.y + (long long)m * p.N;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int n = n0 + wn + 32 * i + crow(e, half);
                if (n < p.N) {
                    const float v = (float)acc[i][j][e] * xs * p.ws[n];
                    y[n] = (T)(p.bias ? v + p.bias[n] : v);
                }
            }
    }
}
