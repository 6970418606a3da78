// mfar_attention.h -- attention with a learned relative position bias by buckets, forward and backward.
//
//   S[q][k] = scale <Q[q], K[k]> + table[bucket(k - pos(q))][head]      over the keys the mask (and causality) leaves
//   P = softmax_k(S),  O = P V
//   D[q] = <dO[q], O[q]>,  dP = dO V',  dS = P (dP - D)
//   dQ = scale dS K,  dK = scale dS' Q,  dV = P' dO,  dtable[b] = sum of the dS whose (q, k) fall into bucket b
//
// One pass over the keys with the running maximum and sum of the softmax, in the log2 domain (scale and bias are multiplied by log2 e).
// The tiles are computed TRANSPOSED, S' = K Q': a lane then owns one query (column l % 32) and 16 of a tile's 32 keys, so row statistics are
// in-lane plus one swap of the wave's halves, and the rounded P' is, register for register, the B operand of O' += V' P' (the order of the
// summed index is free, mfar_ops_device.h).  The backward pass uses the same trick twice: queries in lanes for dQ (and the bias gradient),
// keys in lanes for dK / dV; each recomputes P from the stored log2-sum of the forward pass.  No float atomics on shared addresses: results
// do not change from run to run.
//
// The bias of a (query, key) pair depends on k - pos(q) alone and is constant beyond `sat` (the first distance of the last bucket): a table
// of 2 sat + 1 values per head lives in LDS, and a tile whose distances all lie beyond sat adds one constant.
#pragma once
#include "mfar_ops_device.h"

#define AT_BLOCK 256      // 4 waves, 32 query (key) columns each
#define AT_COLS 128
#define AT_TILE 64        // keys (queries) staged in LDS per step
#define AT_MAX_BORDERS 128

struct AttnParams {
    const void *q, *k, *v, *o, *o_lo, *dout;
    void *out, *out_lo, *dq, *dk, *dv;
    long long q_b, q_l, q_h, k_b, k_l, k_h, v_b, v_l, v_h, do_b, do_l, do_h;      // strides in elements; out, out_lo, dq, dk, dv: contiguous
    const float* table;          // [n_buckets, H]
    const unsigned char* mask;   // [B, Lk] rows mask_b apart, or NULL
    long long mask_b;
    const int* start_ptr;        // [B] position of the first query among the keys, or NULL
    float *lse, *drow;           // [B, H, Lq], log2 units
    float* dpart;                // [blocks, H, n_buckets] partial bias gradients, or NULL
    int start, B, Lq, Lk, H, D, causal, n_buckets, n_side, each, n_borders, sat;
    float scale;
    int borders[AT_MAX_BORDERS]; // first distance of each shared bucket after the first
};

__device__ __forceinline__ int attn_bucket(const AttnParams& p, int delta) {
    int far = p.causal ? (delta < 0 ? -delta : 0) : (delta < 0 ? -delta : delta);
    int b = far;
    if (far >= p.each) {
        b = p.each;
        for (int j = 0; j < p.n_borders; ++j) b += far >= p.borders[j] ? 1 : 0;
    }
    return b + ((delta > 0 && !p.causal) ? p.n_side : 0);
}

// (a position from device memory is kept where sums of positions fit 32 bits)
__device__ __forceinline__ int at_start(const AttnParams& p, int b) { return p.start_ptr ? min(max(p.start_ptr[b], -(1 << 30)), 1 << 30) : p.start; }

// LDS image of a tile: rows of DP elements, chunk c of 8 elements of row r at position c ^ at_swz(r).  Conflict-free for both readers: 16
// consecutive rows at one chunk (row fragments), and 4 consecutive rows x 4 consecutive chunks (transposed fragments).
template <int DP> __device__ __forceinline__ int at_swz(int r) {
    if (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    if (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return (r >> 2) & 3;
}
template <typename T, int DP> __device__ __forceinline__ T* at_at(T* tile, int r, int c) { return tile + r * DP + ((c ^ at_swz<DP>(r)) << 3); }

// rows [r0, r0 + AT_TILE) of one (batch, head) -> LDS; rows whose bit of `bits` is 0 and dims >= D become zeros (a masked row may hold
// anything, also NaN: it must not reach a product)
template <typename T, int DP>
__device__ __forceinline__ void at_stage(T* tile, const T* src, long long stride, int r0, u64 bits, int D) {
    constexpr int CH = DP / 8;
#pragma unroll
    for (int t = 0; t < AT_TILE * CH / AT_BLOCK; ++t) {
        const int e = t * AT_BLOCK + (int)threadIdx.x, r = e / CH, c = e % CH;
        V8<T> x = {};
        if (((bits >> r) & 1) && c * 8 < D) x = *(const V8<T>*)(src + (long long)(r0 + r) * stride + c * 8);
        *(V8<T>*)at_at<T, DP>(tile, r, c) = x;
    }
}
// A fragment: rows row0 + l % 32, dims 16 s + 8 (l / 32) + j
template <typename T, int DP> __device__ __forceinline__ V8<T> at_rows(T* tile, int row0, int s) {
    const int l = threadIdx.x & 63;
    return *(const V8<T>*)at_at<T, DP>(tile, row0 + (l & 31), 2 * s + (l >> 5));
}
// A fragment of the transposed tile: row = dim 32 dt + l % 32, places j = tile rows row0 + 16 m + 8 (j / 4) + 4 (l / 32) + j % 4: the rows
// that half l / 32 of a result tile holds in its registers 8 m + j
template <typename T, int DP> __device__ __forceinline__ V8<T> at_cols(T* tile, int row0, int m, int dt) {
    const int l = threadIdx.x & 63, d = 32 * dt + (l & 31);
    V8<T> x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = at_at<T, DP>(tile, row0 + 16 * m + 8 * (j >> 2) + 4 * (l >> 5) + (j & 3), d >> 3)[d & 7];
    return x;
}
// B fragment straight from memory: column = row `row` of the matrix, dims 16 s + 8 half + j
template <typename T> __device__ __forceinline__ V8<T> at_load(const T* row, bool live, int s, int D) {
    const int d = 16 * s + 8 * ((threadIdx.x & 63) >> 5);
    V8<T> x = {};
    if (live && d < D) x = *(const V8<T>*)(row + d);
    return x;
}
template <typename T> __device__ __forceinline__ V8<T> at_pack(const f32x16& t, int m) {
    V8<T> x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (T)t[8 * m + j];
    return x;
}
// what at_pack dropped
template <typename T> __device__ __forceinline__ V8<T> at_pack_lo(const f32x16& t, int m) {
    V8<T> x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (T)(t[8 * m + j] - (float)(T)t[8 * m + j]);
    return x;
}
// O' tile (lane: column, rows = dims) -> the column's row of a [.., D] matrix
template <typename T, int DP> __device__ __forceinline__ void at_store(T* row, const f32x16* acc, float f, int D) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * half;
            if (d < D) {
                V4<T> x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = (T)(acc[dt][4 * g + j] * f);
                *(V4<T>*)(row + d) = x;
            }
        }
}

// visibility of keys [k0, k0 + 64) as bits: the key mask and the end of the keys
__device__ __forceinline__ u64 at_word(const AttnParams& p, int b, int k0, int end) {
    const int k = k0 + (int)(threadIdx.x & 63);
    bool on = k < end;
    if (on && p.mask) on = p.mask[(long long)b * p.mask_b + k] != 0;
    return __ballot(on);
}

// bias of this lane's 16 elements of a 32 x 32 tile whose first key is k0 (queries in lanes): s2 = s * c + bias, masked places -inf.
// sign = +1: the lane's column is a query at position `col`, rows are keys; sign = -1: the column is a key, rows are queries.
template <int SIGN>
__device__ __forceinline__ void at_bias(f32x16& s, const float* lut, int sat, float c, int row0, int col, int col_lo, int col_hi, bool causal) {
    const int half = (threadIdx.x & 63) >> 5;
    const int lo = SIGN > 0 ? row0 - col_hi : col_lo - (row0 + 31), hi = SIGN > 0 ? row0 + 31 - col_lo : col_hi - row0;   // key - query over the tile
    if (lo >= sat || hi <= -sat) {
        const float add = lut[lo >= sat ? 2 * sat : 0];
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], c, add);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = row0 + crow(i, half);
            int d = SIGN > 0 ? r - col : col - r;
            d = d < -sat ? -sat : (d > sat ? sat : d);
            s[i] = __builtin_fmaf(s[i], c, lut[d + sat]);
        }
    }
    if (causal && hi > 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int r = row0 + crow(i, half);
            if ((SIGN > 0 ? r - col : col - r) > 0) s[i] = -__builtin_inff();
        }
    }
}
__device__ __forceinline__ void at_lut(const AttnParams& p, float* lut, int h) {
    for (int i = threadIdx.x; i <= 2 * p.sat; i += AT_BLOCK) lut[i] = p.table[(long long)attn_bucket(p, i - p.sat) * p.H + h] * LOG2E;
}

// ---- forward ------------------------------------------------------------------------------------------------------------------------------
// KEEP (training, 16-bit types): D = <dO, O> of the backward pass enters the bias table's fp32 gradient, a difference of large sums.  P V takes
// P in two parts (value and what its rounding dropped, error u^2) and out_lo keeps what the output's rounding dropped.
template <typename T, int DP, bool KEEP>
__global__ __launch_bounds__(AT_BLOCK) void mfar_attn_forward_kernel(const AttnParams p) {
    extern __shared__ __align__(16) unsigned char at_lds[];
    T* kt = (T*)at_lds;
    T* vt = kt + AT_TILE * DP;
    u64* words = (u64*)(vt + AT_TILE * DP);
    float* lut = (float*)(words + 64);
    const int b = blockIdx.z, h = blockIdx.y, wave = threadIdx.x >> 6, l = threadIdx.x & 63, half = l >> 5;
    const int start = at_start(p, b);
    const int q = blockIdx.x * AT_COLS + wave * 32 + (l & 31);
    const bool live = q < p.Lq;
    const int col = start + q, col_lo = start + (int)blockIdx.x * AT_COLS + wave * 32, col_hi = col_lo + 31;
    int end = p.Lk;
    if (p.causal) {
        const int last = start + min(p.Lq, ((int)blockIdx.x + 1) * AT_COLS);      // one past the last query's position
        end = min(end, max(last, 0));
    }
    at_lut(p, lut, h);
    const T* qrow = (const T*)p.q + b * p.q_b + (long long)q * p.q_l + h * p.q_h;
    V8<T> qf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = at_load<T>(qrow, live, s, p.D);
    f32x16 acc[DP / 32] = {};
    float m = -__builtin_inff(), sum = 0.0f;
    const float c = p.scale * LOG2E;
    const T* kb = (const T*)p.k + b * p.k_b + h * p.k_h;
    const T* vb = (const T*)p.v + b * p.v_b + h * p.v_h;
    for (int k0 = 0; k0 < end; k0 += AT_TILE) {
        const int tile = k0 / AT_TILE;
        if ((tile & 63) == 0) {                                            // the visibility of the next 64 tiles
            __syncthreads();
            for (int t = wave; t < 64; t += 4) {
                const u64 w = at_word(p, b, k0 + t * AT_TILE, end);
                if (l == 0) words[t] = w;
            }
            __syncthreads();
        }
        const u64 bits = words[tile & 63];
        if (!bits) continue;                                               // (the same for the whole block)
        __syncthreads();
        at_stage<T, DP>(kt, kb, p.k_l, k0, bits, p.D);
        at_stage<T, DP>(vt, vb, p.v_l, k0, bits, p.D);
        __syncthreads();
        f32x16 s[2];
        float top = m;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = f32x16{};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) s[t] = mma(at_rows<T, DP>(kt, 32 * t, d), qf[d], s[t]);
            at_bias<1>(s[t], lut, p.sat, c, k0 + 32 * t, col, col_lo, col_hi, p.causal != 0);
            if (bits != ~0ull) {
                const u32 mine = (u32)(bits >> (32 * t)) >> (4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (!((mine >> crow(i, 0)) & 1)) s[t][i] = -__builtin_inff();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
        }
        top = fmaxf(top, swap_halves(top));
        const float base = top == -__builtin_inff() ? 0.0f : top;           // nothing visible so far: exp2(-inf - 0) = 0
        const float keep = exp2_fast(m - base);
        m = top;
        sum *= keep;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[t][i] = exp2_fast(s[t][i] - base);
                sum += s[t][i];
            }
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) {
            acc[dt] *= keep;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const V8<T> vf = at_cols<T, DP>(vt, 32 * t, g, dt);
                    acc[dt] = mma(vf, at_pack<T>(s[t], g), acc[dt]);
                    if (KEEP) acc[dt] = mma(vf, at_pack_lo<T>(s[t], g), acc[dt]);
                }
        }
    }
    sum += swap_halves(sum);
    if (!live) return;
    const float f = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);    // a row without keys: zeros; NaN stays NaN
    const long long row = ((long long)b * p.Lq + q) * p.H + h;
    at_store<T, DP>((T*)p.out + row * p.D, acc, f, p.D);
    if (KEEP) {
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] = acc[dt][i] * f - (float)(T)(acc[dt][i] * f);
        at_store<T, DP>((T*)p.out_lo + row * p.D, acc, 1.0f, p.D);
    }
    if (p.lse && half == 0) p.lse[((long long)b * p.H + h) * p.Lq + q] = sum == 0.0f ? -__builtin_inff() : m + __log2f(sum);
}

// ---- backward: dQ, the bias gradient, D ---------------------------------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(AT_BLOCK) void mfar_attn_dq_kernel(const AttnParams p) {
    extern __shared__ __align__(16) unsigned char at_lds[];
    T* kt = (T*)at_lds;
    T* vt = kt + AT_TILE * DP;
    u64* words = (u64*)(vt + AT_TILE * DP);
    float* lut = (float*)(words + 64);
    const int n_lut = 2 * p.sat + 1;
    float* hist = lut + n_lut;                                             // [4 waves][2 halves][n_lut]: a lane meets no other at an address
    const int b = blockIdx.z, h = blockIdx.y, wave = threadIdx.x >> 6, l = threadIdx.x & 63, half = l >> 5;
    const int start = at_start(p, b);
    const int q = blockIdx.x * AT_COLS + wave * 32 + (l & 31);
    const bool live = q < p.Lq;
    const int col = start + q, col_lo = start + (int)blockIdx.x * AT_COLS + wave * 32, col_hi = col_lo + 31;
    int end = p.Lk;
    if (p.causal) end = min(end, max(start + min(p.Lq, ((int)blockIdx.x + 1) * AT_COLS), 0));
    at_lut(p, lut, h);
    if (p.dpart)
        for (int i = threadIdx.x; i < 8 * n_lut; i += AT_BLOCK) hist[i] = 0.0f;
    float* mine_hist = hist + (wave * 2 + half) * n_lut;
    const T* qrow = (const T*)p.q + b * p.q_b + (long long)q * p.q_l + h * p.q_h;
    const T* grow = (const T*)p.dout + b * p.do_b + (long long)q * p.do_l + h * p.do_h;
    const long long orow = (((long long)b * p.Lq + q) * p.H + h) * p.D;
    V8<T> qf[DP / 16], gf[DP / 16];
    float dsum = 0.0f;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        qf[s] = at_load<T>(qrow, live, s, p.D);
        gf[s] = at_load<T>(grow, live, s, p.D);
        const V8<T> o = at_load<T>((const T*)p.o + orow, live, s, p.D), lo = at_load<T>((const T*)p.o_lo + orow, live && p.o_lo, s, p.D);
#pragma unroll
        for (int j = 0; j < 8; ++j) dsum = __builtin_fmaf((float)gf[s][j], (float)o[j] + (float)lo[j], dsum);
    }
    dsum += swap_halves(dsum);
    const long long srow = ((long long)b * p.H + h) * p.Lq + q;
    float lse = live ? p.lse[srow] : 0.0f;
    if (!live || lse == -__builtin_inff()) lse = __builtin_inff();          // no keys: P = exp2(-inf) = 0 everywhere
    if (live && half == 0) p.drow[srow] = dsum;
    f32x16 acc[DP / 32] = {};
    float far_lo = 0.0f, far_hi = 0.0f;
    const float c = p.scale * LOG2E;
    const T* kb = (const T*)p.k + b * p.k_b + h * p.k_h;
    const T* vb = (const T*)p.v + b * p.v_b + h * p.v_h;
    for (int k0 = 0; k0 < end; k0 += AT_TILE) {
        const int tile = k0 / AT_TILE;
        if ((tile & 63) == 0) {
            __syncthreads();
            for (int t = wave; t < 64; t += 4) {
                const u64 w = at_word(p, b, k0 + t * AT_TILE, end);
                if (l == 0) words[t] = w;
            }
            __syncthreads();
        }
        const u64 bits = words[tile & 63];
        if (!bits) continue;
        __syncthreads();
        at_stage<T, DP>(kt, kb, p.k_l, k0, bits, p.D);
        at_stage<T, DP>(vt, vb, p.v_l, k0, bits, p.D);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int row0 = k0 + 32 * t;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                s = mma(at_rows<T, DP>(kt, 32 * t, d), qf[d], s);
                dp = mma(at_rows<T, DP>(vt, 32 * t, d), gf[d], dp);
            }
            at_bias<1>(s, lut, p.sat, c, row0, col, col_lo, col_hi, p.causal != 0);
            const u32 mine = (u32)(bits >> (32 * t)) >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float pr = exp2_fast(s[i] - lse);
                s[i] = ((mine >> crow(i, 0)) & 1) ? pr * (dp[i] - dsum) : 0.0f;
            }
            if (p.dpart) {
                if (row0 - col_hi >= p.sat) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) far_hi += s[i];
                } else if (row0 + 31 - col_lo <= -p.sat) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) far_lo += s[i];
                } else {
                    // 32 lanes of a half hold 32 neighbouring distances: one address each; distances beyond sat go to the lane's own sums
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int d = row0 + crow(i, half) - col;
                        if (d >= p.sat) far_hi += s[i];
                        else if (d <= -p.sat) far_lo += s[i];
                        else mine_hist[d + p.sat] += s[i];
                    }
                }
            }
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int g = 0; g < 2; ++g) acc[dt] = mma(at_cols<T, DP>(kt, 32 * t, g, dt), at_pack<T>(s, g), acc[dt]);
        }
    }
    if (live) at_store<T, DP>((T*)p.dq + orow, acc, p.scale, p.D);
    if (p.dpart) {
        for (int o = 1; o < 64; o <<= 1) {
            far_lo += __shfl_xor(far_lo, o);
            far_hi += __shfl_xor(far_hi, o);
        }
        __syncthreads();
        if (l == 0) {
            hist[wave * 2 * n_lut] = far_lo;                               // places 0 and 2 sat of the wave's first row
            hist[wave * 2 * n_lut + 2 * p.sat] += far_hi;                  // (sat = 0 cannot be: the first bucket holds distance 0 alone)
        }
        __syncthreads();
        float* to = p.dpart + ((long long)(b * gridDim.x + blockIdx.x) * p.H + h) * p.n_buckets;
        for (int n = threadIdx.x; n < p.n_buckets; n += AT_BLOCK) {
            float t = 0.0f;
            for (int i = 0; i < n_lut; ++i)
                if (attn_bucket(p, i - p.sat) == n)
                    for (int w = 0; w < 8; ++w) t += hist[w * n_lut + i];
            to[n] = t;
        }
    }
}
// partial bias gradients [n][H * n_buckets] -> their sum, in the order of the blocks
__global__ __launch_bounds__(AT_BLOCK) void mfar_attn_dtable_kernel(const float* part, int n, int H, int nb, float* dtable) {
    __shared__ float sh[AT_BLOCK];
    const int at = blockIdx.x;                                             // head * nb + bucket
    float t = 0.0f;
    for (int i = threadIdx.x; i < n; i += AT_BLOCK) t += part[(long long)i * H * nb + at];
    sh[threadIdx.x] = t;
    __syncthreads();
    for (int o = AT_BLOCK / 2; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) dtable[(long long)(at % nb) * H + at / nb] = sh[0];
}

// ---- backward: dK, dV (keys in lanes) -------------------------------------------------------------------------------------------------------
template <typename T, int DP>
__global__ __launch_bounds__(AT_BLOCK) void mfar_attn_dkv_kernel(const AttnParams p) {
    extern __shared__ __align__(16) unsigned char at_lds[];
    T* qt = (T*)at_lds;
    T* gt = qt + AT_TILE * DP;
    float* rows = (float*)(gt + AT_TILE * DP);                             // [2][AT_TILE]: log2-sum, D
    float* lut = rows + 2 * AT_TILE;
    const int b = blockIdx.z, h = blockIdx.y, wave = threadIdx.x >> 6, l = threadIdx.x & 63, half = l >> 5;
    const int start = at_start(p, b);
    const int key0 = blockIdx.x * AT_COLS, key = key0 + wave * 32 + (l & 31);
    const bool live = key < p.Lk;
    const bool seen = live && (!p.mask || p.mask[(long long)b * p.mask_b + key] != 0);
    const int col_lo = key0 + wave * 32, col_hi = col_lo + 31;
    at_lut(p, lut, h);
    const T* krow = (const T*)p.k + b * p.k_b + (long long)key * p.k_l + h * p.k_h;
    const T* vrow = (const T*)p.v + b * p.v_b + (long long)key * p.v_l + h * p.v_h;
    V8<T> kf[DP / 16], vf[DP / 16];
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        kf[s] = at_load<T>(krow, seen, s, p.D);
        vf[s] = at_load<T>(vrow, seen, s, p.D);
    }
    f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
    const float c = p.scale * LOG2E;
    const T* qb = (const T*)p.q + b * p.q_b + h * p.q_h;
    const T* gb = (const T*)p.dout + b * p.do_b + h * p.do_h;
    const long long srow = ((long long)b * p.H + h) * p.Lq;
    int first = p.causal ? max(0, key0 - start) : 0;                       // the first query that sees the block's first key
    const bool any = __syncthreads_or(seen);                               // (also the barrier behind at_lut)
    if (!any) first = p.Lq;
    for (int q0 = first / AT_TILE * AT_TILE; q0 < p.Lq; q0 += AT_TILE) {
        const int n = min(AT_TILE, p.Lq - q0);
        const u64 bits = n == 64 ? ~0ull : ((1ull << n) - 1);
        __syncthreads();
        at_stage<T, DP>(qt, qb, p.q_l, q0, bits, p.D);
        at_stage<T, DP>(gt, gb, p.do_l, q0, bits, p.D);
        if (threadIdx.x < AT_TILE) {
            const bool in = (int)threadIdx.x < n;
            const float e = in ? p.lse[srow + q0 + threadIdx.x] : -__builtin_inff();
            rows[threadIdx.x] = e == -__builtin_inff() ? __builtin_inff() : e;
            rows[AT_TILE + threadIdx.x] = in ? p.drow[srow + q0 + threadIdx.x] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                s = mma(at_rows<T, DP>(qt, 32 * t, d), kf[d], s);
                dp = mma(at_rows<T, DP>(gt, 32 * t, d), vf[d], dp);
            }
            at_bias<-1>(s, lut, p.sat, c, start + q0 + 32 * t, key, col_lo, col_hi, p.causal != 0);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = 32 * t + crow(i, half);
                const float pr = seen ? exp2_fast(s[i] - rows[r]) : 0.0f;
                s[i] = pr;
                dp[i] = seen ? pr * (dp[i] - rows[AT_TILE + r]) : 0.0f;
            }
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    dv[dt] = mma(at_cols<T, DP>(gt, 32 * t, g, dt), at_pack<T>(s, g), dv[dt]);
                    dk[dt] = mma(at_cols<T, DP>(qt, 32 * t, g, dt), at_pack<T>(dp, g), dk[dt]);
                }
        }
    }
    if (!live) return;
    const long long row = (((long long)b * p.Lk + key) * p.H + h) * p.D;
    at_store<T, DP>((T*)p.dk + row, dk, p.scale, p.D);
    at_store<T, DP>((T*)p.dv + row, dv, 1.0f, p.D);
}
