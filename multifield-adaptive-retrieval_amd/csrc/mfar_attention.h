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
// P and dS are rounded to the inputs' type on their way into a product (the matrix unit takes nothing wider at its rate): half a step each, in fp16
// whatever their size (AtFit), independent from key to key, which adds to dQ and dK about what the rounding of those results does (2.9e-4 from the
// 64-bit gradient for 2.1e-4 in fp16; bf16 over two keys 2.9e-3 for 1.7e-3) and to the outputs of large batches a quarter of it (2.6e-4 for 2.1e-4).
// Where there is time, and where a backward pass follows, P goes in two parts.  Sums stay in fp32, the table's gradient takes dS unrounded.
//
// The bias of a (query, key) pair depends on k - pos(q) alone and is constant beyond `sat` (the first distance of the last bucket): a table
// of 2 sat + 1 values per head lives in LDS, and a tile whose distances all lie beyond sat adds one constant.
#pragma once
#include <type_traits>

#include "mfar_ops_device.h"

#define AT_BLOCK 256      // 4 waves, 32 query (key) columns each
#define AT_COLS 128
#define AT_TILE 64        // keys (queries) staged in LDS per step
#define AT_MAX_SAT 1023
#define AT_MAX_STRIDE (1 << 22)
// The running maximum of the softmax follows a tile's only when that is 2^8 over it: probabilities stay under 2^14 (fp16 holds them as exactly as
// those under 1), and the accumulated output is hardly ever rescaled.
#define AT_SLACK 8.0f
// ... and the base lies 2^6 under the maximum it was set from, so that fp16 still holds what its rounding of a middling probability dropped (at_pack_lo).
#define AT_SHIFT 6.0f

// Waves per SIMD the register budget is set for.  From 2 on (256 registers) the compiler keeps accumulators where the vector unit reaches them;
// with the whole file for one wave it parks them in accumulation registers and copies every score back and forth.
constexpr int at_waves(int size, int dp, int want) { return size == 2 && dp <= 64 ? want : (size == 2 ? 2 : (dp <= 64 ? 2 : 1)); }

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
    int start, B, Lq, Lk, H, D, causal, n_buckets, n_side, sat;
    float scale;
    short first[129 * 2];        // first distance of each bucket of a side
    unsigned char bucket[AT_MAX_SAT + 1];   // of the distances 0 .. sat
};

__device__ __forceinline__ int attn_bucket(const AttnParams& p, int delta) {
    const int far = p.causal ? max(-delta, 0) : abs(delta);
    return p.bucket[min(far, p.sat)] + ((delta > 0 && !p.causal) ? p.n_side : 0);
}
// Consecutive blocks go to the 8 XCDs in turn, each with an L2 of its own: the blocks of one (batch, head), which read the same keys (queries), are
// numbered 8 apart.  A 1-D grid of at_grid blocks; false: this block has nothing to do.
struct AtPlace { int tile, h, b; };
__device__ __forceinline__ bool at_place(const AttnParams& p, int tiles, AtPlace& at) {
    const int j = blockIdx.x / 8, g = j / tiles * 8 + blockIdx.x % 8;
    at.tile = j % tiles, at.h = g % p.H, at.b = g / p.H;
    return at.b < p.B;
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

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// Steps of tiles held in LDS: two, so that one loads while the other is multiplied; one where two would leave a CU a single block (the backward pass
// holds more beside them).
constexpr int at_stages(int size, int dp, bool backward) { return size * dp >= (backward ? 256 : 512) ? 1 : 2; }

// Tiles of AT_TILE rows of one (batch, head) straight from memory to LDS: a wave's load instruction fills 1 KB in lane order, the swizzle of at_at is
// applied on the addresses the lanes load from.  Rows >= n are not read (the last row stands in), nor are dims >= D (the row's first chunk stands in:
// the other operand of every product holds zeros there, and results of those dims are dropped).  Row strides fit 22 bits, so a lane's place in a
// tile is a 32-bit offset from a scalar address.
template <typename T, int DP> struct AtStream {
    static constexpr int ROW = DP * sizeof(T), N = AT_TILE * ROW / 1024 / 4, PIECES = ROW / 16, EACH = sizeof(T) / 2;   // EACH: 16-byte pieces a chunk
    const T* base;
    long long stride;
    int n;
    u32 off[N];
    __device__ __forceinline__ AtStream(const T* base_, long long stride_, int n_, int D) : base(base_), stride(stride_), n(n_) {
        const int piece = (threadIdx.x & 63) % PIECES;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const int c = (piece / EACH) ^ at_swz<DP>(row(t));
            off[t] = (u32)(row(t) * (int)stride + (c * 8 < D ? c * 8 : 0)) * (u32)sizeof(T) + (piece % EACH) * 16;
        }
    }
    static __device__ __forceinline__ int row(int t) { return (wave_index() * N + t) * (64 / PIECES) + (int)(threadIdx.x & 63) / PIECES; }
    __device__ __forceinline__ void load(int r0, T* tile) const {
        const u64 address = (u64)(uintptr_t)(base + (long long)r0 * stride);
        const u64 at = ((u64)(u32)__builtin_amdgcn_readfirstlane((int)(address >> 32)) << 32) | (u32)__builtin_amdgcn_readfirstlane((int)address);
        const u32 to = (u32)__builtin_amdgcn_readfirstlane((int)((u32)(uintptr_t)tile + wave_index() * N * 1024));
        auto go = [&](u32 from, int t) {
            asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(from), "s"(at), "s"(to + t * 1024) : "memory");
        };
        if (r0 + AT_TILE <= n) {
#pragma unroll
            for (int t = 0; t < N; ++t) go(off[t], t);
        } else {
#pragma unroll
            for (int t = 0; t < N; ++t) go(off[t] - (u32)__mul24(max(0, r0 + row(t) - (n - 1)), (int)stride) * (u32)sizeof(T), t);
        }
    }
};
// this wave's loads have arrived, then everyone's
__device__ __forceinline__ void at_arrive() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}
// Rows of a tile that nobody may see become zeros: a masked row may hold anything, also NaN, and must not reach a product.
template <typename T, int DP> __device__ __forceinline__ void at_blank(T* tile, u64 bits) {
    constexpr int CH = DP / 8;
    for (int e = threadIdx.x; e < AT_TILE * CH; e += AT_BLOCK)
        if (!((bits >> (e / CH)) & 1)) *(V8<T>*)(tile + e * 8) = V8<T>{};
}
__device__ __forceinline__ u64 read_lane(u64 x, int lane) {
    return ((u64)(u32)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32) | (u32)__builtin_amdgcn_readlane((int)x, lane);
}
// A fragment: rows row0 + l % 32, dims 16 s + 8 (l / 32) + j
template <typename T, int DP> __device__ __forceinline__ V8<T> at_rows(T* tile, int row0, int s) {
    const int l = threadIdx.x & 63;
    return *(const V8<T>*)at_at<T, DP>(tile, row0 + (l & 31), 2 * s + (l >> 5));
}
// A fragment of the transposed tile: row = dim 32 dt + l % 32, places j = tile rows row0 + 16 m + 8 (j / 4) + 4 (l / 32) + j % 4: the rows
// that half l / 32 of a result tile holds in its registers 8 m + j
// (16-bit types: two transposing reads of 4 rows x 16 dims per group of 16 lanes; lane i of a group points at dims 4 (i % 4).. of row i / 4 and
// receives dim i of the 4 rows)
template <typename T, int DP> __device__ __forceinline__ V8<T> at_cols(T* tile, int row0, int m, int dt) {
    const int l = threadIdx.x & 63;
    V8<T> x;
    if constexpr (sizeof(T) == 2) {
        const int d = 32 * dt + 16 * ((l >> 4) & 1) + 4 * (l & 3);
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
            T* from = at_at<T, DP>(tile, row0 + 16 * m + 8 * jj + 4 * (l >> 5) + ((l & 15) >> 2), d >> 3) + (d & 7);
            const s16x4 w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)from);
            const V4<T> y = __builtin_bit_cast(V4<T>, w);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * jj + j] = y[j];
        }
    } else {
        const int d = 32 * dt + (l & 31);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = at_at<T, DP>(tile, row0 + 16 * m + 8 * (j >> 2) + 4 * (l >> 5) + (j & 3), d >> 3)[d & 7];
    }
    return x;
}
// B fragment straight from memory: column = row `row` of the matrix, dims 16 s + 8 half + j; zeros where the row is not live or has no such dim.
// (`row` may be read in any case: loads without branches are all in flight at once)
template <typename T> __device__ __forceinline__ V8<T> at_load(const T* row, bool live, int s, int D) {
    const int d = 16 * s + 8 * ((threadIdx.x & 63) >> 5);
    const V8<T> x = *(const V8<T>*)(row + (d < D ? d : 0));
    return live && d < D ? x : V8<T>{};
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
// O' tiles of a wave (lane: one of 32 rows of the result, registers: dims) -> n rows of a [.., D] matrix `stride` elements apart, through LDS of the
// wave's own (at_out_bytes), 128 bytes of a row at a time, so that a row leaves in runs of whole cache lines (8 bytes a lane of 32 rows
// straight from the registers: 5 us more for the encode's 73).
template <typename T, int DP> constexpr int at_out_dims() { return DP * (int)sizeof(T) < 128 ? DP : 128 / (int)sizeof(T); }
template <typename T, int DP> constexpr int at_out_bytes() { return 32 * (at_out_dims<T, DP>() * (int)sizeof(T) + 16); }
template <typename T, int DP> __device__ __forceinline__ void at_store(T* out, long long stride, int n, const f32x16* acc, float f, int D, void* lds) {
    constexpr int W = at_out_dims<T, DP>(), PITCH = W * sizeof(T) + 16, LANES = W * sizeof(T) / 16, EACH = 16 / sizeof(T);
    const int l = threadIdx.x & 63, half = l >> 5;
    unsigned char* mine = (unsigned char*)lds;
#pragma unroll
    for (int d0 = 0; d0 < DP; d0 += W) {
#pragma unroll
        for (int dt = 0; dt < W / 32; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                V4<T> x;
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = (T)(acc[d0 / 32 + dt][4 * g + j] * f);
                *(V4<T>*)(mine + (l & 31) * PITCH + (32 * dt + 8 * g + 4 * half) * sizeof(T)) = x;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += 64 / LANES) {
            const int r = r0 + l / LANES, d = d0 + l % LANES * EACH;
            if (r < n && d < D) *(u32x4*)(out + (long long)r * stride + d) = *(const u32x4*)(mine + r * PITCH + l % LANES * 16);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Visibility of the 4096 keys from `base`: lane t gets the 64 bits of tile t (key mask, and keys < end).  A lane packs its whole tile from eight
// 8-byte loads; the tile that `end` cuts is read a byte per lane.
__device__ __forceinline__ u64 at_words(const AttnParams& p, int b, int base, int end) {
    const int l = threadIdx.x & 63, n = end - base, mine = n - l * AT_TILE;        // keys left from this lane's tile on
    u64 w = mine >= 64 ? ~0ull : (mine > 0 ? (1ull << mine) - 1 : 0ull);
    if (p.mask) {
        const unsigned char* m = p.mask + (long long)b * p.mask_b + base;
        if (mine >= 64) {
            w = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                u64 x;
                __builtin_memcpy(&x, m + l * AT_TILE + j * 8, 8);
                x = ((((x & 0x7f7f7f7f7f7f7f7full) + 0x7f7f7f7f7f7f7f7full) | x) >> 7) & 0x0101010101010101ull;   // 1 for every byte that is not 0
                w |= ((x * 0x0102040810204080ull) >> 56) << (8 * j);
            }
        }
        if (n < 64 * AT_TILE && (n & 63)) {
            const int at = (n & ~63) + l;
            const u64 cut = __ballot(at < n && m[at < n ? at : 0] != 0);
            if (l == n >> 6) w = cut;
        }
    }
    return w;
}

// hidden keys of a 32 x 32 tile (bit per row) -> -inf
__device__ __forceinline__ void at_hide(f32x16& s, u32 seen) {
    seen >>= 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (!((seen >> crow(i, 0)) & 1)) s[i] = -__builtin_inff();
}

// Runs `step(k0, bits, K, V)` for every tile of 64 keys in [0, end) that shows any key, with the tile's K and V in LDS; by the whole block.
// tiles: at_stages of [K, V][AT_TILE][DP].  `ahead()` is run once, while the first tile is on its way.
template <typename T, int DP, bool BACKWARD, typename A, typename F>
__device__ __forceinline__ void at_for_tiles(const AttnParams& p, int b, int h, int end, T* tiles, A&& ahead, F&& step) {
    constexpr int S = at_stages(sizeof(T), DP, BACKWARD), SIZE = AT_TILE * DP;
    const AtStream<T, DP> ks((const T*)p.k + b * p.k_b + h * p.k_h, p.k_l, end, p.D), vs((const T*)p.v + b * p.v_b + h * p.v_h, p.v_l, end, p.D);
    u64 words = 0, left = 0;                                               // left: the same in every wave
    int t = 0, slot = 0;
    auto begin = [&](int base) {
        words = at_words(p, b, base, end);
        left = __ballot(words != 0);
        if (!left) return;
        t = __builtin_ctzll(left), slot = 0;
        ks.load(base + t * AT_TILE, tiles);
        vs.load(base + t * AT_TILE, tiles + SIZE);
    };
    if (end > 0) begin(0);
    ahead();
    for (int base = 0; base < end; ) {
        while (left) {
            const int k0 = base + t * AT_TILE;
            const u64 bits = read_lane(words, t);
            T *kt = tiles + slot * 2 * SIZE, *vt = kt + SIZE;
            left &= left - 1;
            at_arrive();                                                   // (also: the other slot has been read by every wave)
            auto next = [&]() {
                if (!left) return;
                t = __builtin_ctzll(left);
                if (S == 2) slot ^= 1;
                ks.load(base + t * AT_TILE, tiles + slot * 2 * SIZE);
                vs.load(base + t * AT_TILE, tiles + slot * 2 * SIZE + SIZE);
            };
            if (S == 2) next();
            if (bits != ~0ull) {
                at_blank<T, DP>(kt, bits);
                at_blank<T, DP>(vt, bits);
                __syncthreads();
            }
            const bool last = S == 2 ? k0 == base + t * AT_TILE : !left;
            step(k0, bits, kt, vt);
            if (last) break;
            if (S == 1) {
                __syncthreads();
                next();
            }
        }
        base += 64 * AT_TILE;
        if (base < end) {
            __syncthreads();                                               // (the readers of the 4096 keys before are done)
            begin(base);
        }
    }
}

// The bias table in LDS: distances -(sat + 63) .. sat + 63, so that a 32 x 32 tile which holds any distance inside (-sat, sat) stays inside it and
// is read without clamping, at fixed offsets from one address per lane.
#define AT_EDGE 63
__device__ __forceinline__ int at_lut_size(int sat) { return 2 * (sat + AT_EDGE) + 1; }
__device__ __forceinline__ void at_lut(const AttnParams& p, float* lut, int h) {
    for (int i = threadIdx.x; i < at_lut_size(p.sat); i += AT_BLOCK)
        lut[i] = p.table[(long long)attn_bucket(p, i - p.sat - AT_EDGE) * p.H + h] * LOG2E;
}
// s2 - off = s * c + bias - off for this lane's 16 elements of a 32 x 32 tile, places behind the query -inf when causal.
// SIGN = +1: the lane's column is a query at position `col`, rows are keys from row0; -1: the column is a key, rows are query positions from row0.
template <int SIGN>
__device__ __forceinline__ void at_bias(f32x16& s, const float* lut, int sat, float c, int row0, int col, int col_lo, bool causal, float off) {
    const int half = (threadIdx.x & 63) >> 5;
    const int lo = SIGN > 0 ? row0 - col_lo - 31 : col_lo - row0 - 31, hi = lo + 62;      // key - query over the tile
    if (lo >= sat || hi <= -sat) {
        const float add = lut[lo >= sat ? 2 * (sat + AT_EDGE) : 0] - off;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], c, add);
    } else {
        const float* at = lut + (SIGN > 0 ? row0 + 4 * half - col : col - row0 - 4 * half) + sat + AT_EDGE;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], c, at[SIGN * crow(i, 0)] - off);
    }
    if (causal && hi > 0) {
        const int edge = SIGN > 0 ? col - row0 - 4 * half : row0 + 4 * half - col;         // the last visible row / minus the first
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (SIGN > 0 ? crow(i, 0) > edge : crow(i, 0) + edge < 0) s[i] = -__builtin_inff();
    }
}

// Running softmax of a lane's query.  Scores arrive as x = s2 - base (at_bias takes the base off with the bias); the base moves to the tile's maximum only
// when that is 2^AT_SLACK over it, and at the first visible key (limit = -inf until then).
struct AtSoftmax {
    float base = 0.0f, limit = -__builtin_inff(), sum = 0.0f;               // sum: this half's part
};
// N tiles of 32 x 32 scores into the softmax and O' += V' P' with the rows of vt.  The sum is of the probabilities as they are multiplied: what rounding
// added to one that stands far ahead of the rest cancels in the quotient (summed unrounded, such a query's output was off by a half step more than its
// own rounding).  TWO multiplies them in two parts, exact to u^2, and sums them unrounded.
template <typename T, int DP, bool TWO, int N>
__device__ __forceinline__ void at_softmax(f32x16 (&s)[N], T* vt, AtSoftmax& m, f32x16* acc) {
    float top = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
    top = max_halves(top);
    if (__any(top > m.limit)) {
        const float up = top > m.limit ? top - AT_SHIFT : 0.0f, keep = m.limit > 0.0f ? exp2_fast(-up) : 0.0f;   // (before the first key there is nothing to keep)
        m.base += up;
        if (top > m.limit) m.limit = AT_SHIFT + AT_SLACK;
        m.sum *= keep;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= keep;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] -= up;
    }
#pragma unroll
    for (int t = 0; t < N; ++t) {
        float part[2] = {};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[t][i] = exp2_fast(s[t][i]);
            if (TWO || sizeof(T) == 4) part[i & 1] += s[t][i];
        }
        if constexpr (!TWO && sizeof(T) == 2)
#pragma unroll
            for (int g = 0; g < 2; ++g) part[g] = add_up(at_pack<T>(s[t], g), 0.0f);
        m.sum += part[0] + part[1];
        if (sizeof(T) == 2) __builtin_amdgcn_s_setprio(1);                 // (matrix work first: the other waves' exponentials fill the gaps; 3 % at 8 x 4096)
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const V8<T> vf = at_cols<T, DP>(vt, 32 * t, g, dt);
                acc[dt] = mma(vf, at_pack<T>(s[t], g), acc[dt]);
                if (TWO) acc[dt] = mma(vf, at_pack_lo<T>(s[t], g), acc[dt]);
            }
        if (sizeof(T) == 2) __builtin_amdgcn_s_setprio(0);
    }
}
// log2-sum of a query: -inf if it saw nothing
__device__ __forceinline__ float at_lse(float base, float sum) { return sum == 0.0f ? -__builtin_inff() : base + __log2f(sum); }

// x as fp32 rounded it: a product that is converted to fp16 in the same instruction rounds once, and what is left of x would be taken from another
// rounding than the one that was stored
__device__ __forceinline__ float at_rounded(float x) {
    asm volatile("" : "+v"(x));
    return x;
}
__device__ __forceinline__ float at_norm(float sum) { return sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum); }   // no keys: zeros; NaN stays

// ---- forward ------------------------------------------------------------------------------------------------------------------------------
// At long lengths bound by the vector unit: an exponential, the bias, a maximum, a sum and half a conversion a score, beside 8 matrix instructions a tile of
// 32 x 32 (8 x 4096 x 12 heads x 64 fp16: 530 us, 780 TFLOP/s; keeping what the backward pass needs, 4 x 4096: 366 us).  At 512 keys a block lives for up to 8
// tiles, and about half of its time is what lies before and behind them: the first loads, mask, bias table, results (64 x 512, padded: 74 us, 400
// TFLOP/s; 32 x 512 keeping: 53 us ragged, 60 full).
// KEEP (training, 16-bit types): D = <dO, O> of the backward pass enters every score gradient as the part that P dP is reduced by, and so dQ, dK and, in
// fp32, the bias table's gradient, all differences of large sums.  P V takes P in two parts (value and what its rounding dropped, error u^2) and out_lo keeps what the output's rounding dropped.
template <typename T, int DP, bool KEEP>
__global__ __launch_bounds__(AT_BLOCK, at_waves(sizeof(T), DP, 3)) void mfar_attn_forward_kernel(const AttnParams p) {
    AtPlace place;
    if (!at_place(p, (p.Lq + AT_COLS - 1) / AT_COLS, place)) return;
    extern __shared__ __align__(16) unsigned char at_lds[];
    T* tiles = (T*)at_lds;
    float* lut = (float*)(tiles + at_stages(sizeof(T), DP, false) * 2 * AT_TILE * DP);
    const int b = place.b, h = place.h, wave = wave_index(), l = threadIdx.x & 63, half = l >> 5;
    const int start = at_start(p, b);
    const int q = place.tile * AT_COLS + wave * 32 + (l & 31);
    const bool live = q < p.Lq;
    const int col = start + q, col_lo = start + place.tile * AT_COLS + wave * 32;
    int end = p.Lk;
    if (p.causal) {
        const int last = start + min(p.Lq, (place.tile + 1) * AT_COLS);      // one past the last query's position
        end = min(end, max(last, 0));
    }
    const T* qrow = (const T*)p.q + b * p.q_b + (long long)(live ? q : 0) * p.q_l + h * p.q_h;
    V8<T> qf[DP / 16];
    f32x16 acc[DP / 32] = {};
    AtSoftmax m;
    const float c = p.scale * LOG2E;
    at_for_tiles<T, DP, false>(p, b, h, end, tiles, [&]() {
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) qf[s] = at_load<T>(qrow, live, s, p.D);
        at_lut(p, lut, h);
    }, [&](int k0, u64 bits, T* kt, T* vt) {
        f32x16 s[2] = {};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[t] = mma(at_rows<T, DP>(kt, 32 * t, d), qf[d], s[t]);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            at_bias<1>(s[t], lut, p.sat, c, k0 + 32 * t, col, col_lo, p.causal != 0, m.base);
            if ((u32)(bits >> (32 * t)) != ~0u) at_hide(s[t], (u32)(bits >> (32 * t)));
        }
        at_softmax<T, DP, KEEP, 2>(s, vt, m, acc);
    });
    const float sum = sum_halves(m.sum), f = at_norm(sum);
    __syncthreads();                                                       // (the tiles' memory is free)
    const int q0 = place.tile * AT_COLS + wave * 32;
    const long long at = (((long long)b * p.Lq + q0) * p.H + h) * p.D;
    void* lds = at_lds + wave * at_out_bytes<T, DP>();
    if (!KEEP) {
        at_store<T, DP>((T*)p.out + at, (long long)p.H * p.D, p.Lq - q0, acc, f, p.D, lds);
    } else {
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] = at_rounded(acc[dt][i] * f);
        at_store<T, DP>((T*)p.out + at, (long long)p.H * p.D, p.Lq - q0, acc, 1.0f, p.D, lds);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[dt][i] -= (float)(T)acc[dt][i];
        at_store<T, DP>((T*)p.out_lo + at, (long long)p.H * p.D, p.Lq - q0, acc, 1.0f, p.D, lds);
    }
    if (p.lse && live && half == 0) p.lse[((long long)b * p.H + h) * p.Lq + q] = at_lse(m.base, sum);
}

// ---- forward, few queries (short texts, a decoder's next token, small batches): the work of 32 queries is divided over the keys --------------------
// Tiles of 32 keys go to the waves in turn, 4 waves a block and `splits` blocks per (batch, head): K and V in whole rows through LDS of the
// wave's own, no barrier in the loop, the next tile's loads in flight.  The waves' partial softmaxes are joined in LDS, the blocks' in a second
// launch, both in a fixed order.  The matrix unit has time for P in two parts (serving alone: 16 caches of 4097 25.1 -> 25.7 us, a short text 6.2 -> 6.3), so
// outputs are as exact as from an fp32 P.  Bound by reading K and V (16 ragged caches of 4097 x 12 heads x 64 bf16, 113 MB:
// 29 us, and 4 to join) and, for a short text, by latency (12 x 12 heads x 64: 6 us).
struct AttnSplit {
    float *o, *ml;               // [rows, splits, D], [rows, splits, 2] (maximum, sum); row = (batch * Lq + query) * H + head
    int splits;
};
template <typename T> __device__ __forceinline__ void at_write(const AttnParams& p, bool keep, long long at, float x) {
    x = at_rounded(x);
    const T y = (T)x;
    ((T*)p.out)[at] = y;
    if (keep) ((T*)p.out_lo)[at] = (T)(x - (float)y);
}

// LDS of the waves' tiles, and behind the loop of their partial outputs
template <typename T, int DP> constexpr int at_few_bytes() { return 4 * DP * 32 * (sizeof(T) == 4 ? 8 : 4); }

template <typename T, int DP, bool KEEP>
__global__ __launch_bounds__(AT_BLOCK, at_waves(sizeof(T), DP, 3)) void mfar_attn_few_kernel(const AttnParams p, const AttnSplit sp) {
    extern __shared__ __align__(16) unsigned char at_lds[];
    T* vt = (T*)at_lds + wave_index() * 64 * DP;                           // the wave's V and K tiles
    T* kt = vt + 32 * DP;
    float* part = (float*)at_lds;                                          // [4 waves][DP][32], behind the loop
    float* stat = (float*)(at_lds + at_few_bytes<T, DP>());                // [4 waves][2][32]
    float* lut = stat + 4 * 64;
    const int b = blockIdx.z, h = blockIdx.y, wave = wave_index(), l = threadIdx.x & 63, half = l >> 5, qi = l & 31;
    const int q0 = (int)blockIdx.x / sp.splits * 32, part_of = (int)blockIdx.x % sp.splits, q = q0 + qi;
    const int start = at_start(p, b);
    const bool live = q < p.Lq;
    const int col = start + q;
    const int end = p.causal ? min(p.Lk, max(start + min(p.Lq, q0 + 32), 0)) : p.Lk;
    constexpr int CH = DP / 8, NV = DP / 16;                               // chunks a row; chunks of V a lane
    const T* kb = (const T*)p.k + b * p.k_b + h * p.k_h;
    const T* vb = (const T*)p.v + b * p.v_b + h * p.v_h;
    const unsigned char* mask = p.mask ? p.mask + (long long)b * p.mask_b : nullptr;
    const T* qrow = (const T*)p.q + b * p.q_b + (long long)(live ? q : 0) * p.q_l + h * p.q_h;
    V8<T> qf[DP / 16], kr[NV], vr[NV];
    bool on = false;
    const int step = sp.splits * 4 * 32;
    int k0 = (part_of * 4 + wave) * 32;
    const bool vin = (l % CH) * 8 < p.D;
    auto fetch = [&]() {
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            const int r = min(k0 + (t * 64 + l) / CH, end - 1), d = vin ? (l % CH) * 8 : 0;
            kr[t] = *(const V8<T>*)(kb + (long long)r * p.k_l + d);
            vr[t] = *(const V8<T>*)(vb + (long long)r * p.v_l + d);
        }
        on = k0 + (l & 31) < end && (!mask || mask[min(k0 + (l & 31), end - 1)] != 0);
    };
    if (k0 < end) fetch();
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) qf[s] = at_load<T>(qrow, live, s, p.D);
    at_lut(p, lut, h);
    __syncthreads();
    f32x16 acc[DP / 32] = {};
    AtSoftmax run;
    const float c = p.scale * LOG2E;
    while (k0 < end) {
        const u32 seen = (u32)__ballot(on);
        const int row0 = k0;
#pragma unroll
        for (int t = 0; t < NV; ++t) {
            const int r = (t * 64 + l) / CH;
            const bool shown = vin && ((seen >> r) & 1);
            *(V8<T>*)at_at<T, DP>(kt, r, l % CH) = shown ? kr[t] : V8<T>{};
            *(V8<T>*)at_at<T, DP>(vt, r, l % CH) = shown ? vr[t] : V8<T>{};
        }
        k0 += step;
        if (k0 < end) fetch();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        f32x16 s[1] = {};
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) s[0] = mma(at_rows<T, DP>(kt, 0, d), qf[d], s[0]);
        if (seen) {
            at_bias<1>(s[0], lut, p.sat, c, row0, col, start + q0, p.causal != 0, run.base);
            if (seen != ~0u) at_hide(s[0], seen);
            at_softmax<T, DP, sizeof(T) == 2, 1>(s, vt, run, acc);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    float m = run.limit > 0.0f ? run.base : -__builtin_inff(), sum = sum_halves(run.sum);
    __syncthreads();                                                       // (part lies where the V tiles were)
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(wave * DP + 32 * dt + crow(i, half)) * 32 + qi] = acc[dt][i];
    if (half == 0) {
        stat[wave * 64 + qi] = m;
        stat[wave * 64 + 32 + qi] = sum;
    }
    __syncthreads();
    if (!live) return;
    float f[4], all = 0.0f;
    m = fmaxf(fmaxf(stat[qi], stat[64 + qi]), fmaxf(stat[128 + qi], stat[192 + qi]));
    const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        f[w] = exp2_fast(stat[w * 64 + qi] - base);
        all += f[w] * stat[w * 64 + 32 + qi];
    }
    const long long row = ((long long)b * p.Lq + q) * p.H + h;
    const float norm = sp.splits == 1 ? at_norm(all) : 1.0f;
    for (int d = threadIdx.x >> 5; d < p.D; d += 8) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) x += f[w] * part[(w * DP + d) * 32 + qi];
        if (sp.splits == 1) at_write<T>(p, KEEP, row * p.D + d, x * norm);
        else sp.o[(row * sp.splits + part_of) * p.D + d] = x;
    }
    if (threadIdx.x < 32) {
        if (sp.splits > 1) {
            float* to = sp.ml + (row * sp.splits + part_of) * 2;
            to[0] = m, to[1] = all;
        } else if (p.lse) {
            p.lse[((long long)b * p.H + h) * p.Lq + q] = all == 0.0f ? -__builtin_inff() : m + __log2f(all);
        }
    }
}
// joins the blocks of mfar_attn_few_kernel: one wave per row
template <typename T, bool KEEP> __global__ __launch_bounds__(AT_BLOCK) void mfar_attn_join_kernel(const AttnParams p, const AttnSplit sp) {
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (long long)p.B * p.Lq * p.H;
    const int l = threadIdx.x & 63;
    if (row >= rows) return;
    const float* ml = sp.ml + row * sp.splits * 2;
    float m = -__builtin_inff(), sum = 0.0f;
    for (int s = 0; s < sp.splits; ++s) m = fmaxf(m, ml[2 * s]);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float x[2] = {};
    for (int s = 0; s < sp.splits; ++s) {
        const float f = exp2_fast(ml[2 * s] - base);
        sum += f * ml[2 * s + 1];
        const float* o = sp.o + (row * sp.splits + s) * p.D;
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (l + 64 * j < p.D) x[j] += f * o[l + 64 * j];
    }
    const float norm = at_norm(sum);
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (l + 64 * j < p.D) at_write<T>(p, KEEP, row * p.D + l + 64 * j, x[j] * norm);
    if (p.lse && l == 0) {
        const long long h = row % p.H, q = row / p.H % p.Lq, b = row / p.H / p.Lq;
        p.lse[(b * p.H + h) * p.Lq + q] = sum == 0.0f ? -__builtin_inff() : m + __log2f(sum);
    }
}

// Sums along the diagonals of a 32 x 32 tile (lanes: queries, registers: keys) times the lane's f, added to sums[key - query]; by one wave, in memory of
// its own.  A lane's registers come in runs of 4 rows: from the last row of a run up, the sum so far moves on by a query (a lane) and the next row is
// added.  What leaves the run's half of the wave by that (query 0) enters the other half's upper end, at distances past the run's own, and is
// kept apart (`off`).  The 8 runs of a tile, their distances in columns, lie in a buffer of 8 x 64 (what no run reaches stays the zero it was set to
// once); every lane adds up a column and adds the sum to its distance's place.  No atomics (LDS float atomics took 205 cycles a wave here).
#define AT_SKEW (8 * 64)
__device__ __forceinline__ float at_next_lane(float x) {                    // lane n: lane n + 1's, the last lane: 0
    return __uint_as_float((u32)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x130, 0xf, 0xf, true));
}
__device__ __forceinline__ float at_next_lane_around(float x) {             // lane n: lane n + 1's, the last lane: the first's
    return __uint_as_float((u32)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x134, 0xf, 0xf, true));
}
__device__ __forceinline__ void at_diagonals(const f32x16& s, float f, float* skew, float* sums) {
    const int l = threadIdx.x & 63, half = l >> 5, q = l & 31;
    float *own = skew + 68 * half + 31 - q, *other = skew + 68 * (1 - half) + 63 - q;     // run g of a half: row 2 g + half, first key 8 g + 4 half
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float sum = s[4 * g + 3] * f, off = 0.0f;
#pragma unroll
        for (int i = 2; i >= 0; --i) {
            off = at_next_lane_around(q == 0 ? sum : off);
            sum = s[4 * g + i] * f + at_next_lane(l == 32 ? 0.0f : sum);
        }
        own[136 * g] = sum;
        if (q >= 29) other[136 * g] = off;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float t[2] = {};
#pragma unroll
    for (int r = 0; r < 8; ++r) t[r & 1] += skew[r * 64 + l];
    if (l < 63) sums[l - 31] += t[0] + t[1];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// What the backward pass multiplies in fp16 does not stay within its range: dS is dO times V times P, and the P of a key that is unlikely for every
// query is small throughout (fp16: exact from 2^-14, nothing under 2^-25).  So each lane's column (dQ: a query's dS; dK, dV: a key's dS and P)
// goes into its product times a power of two of its own, taken back behind the sums.  The column's first tile sets it, its largest entry
// to 2^6; when an entry passes 2^15 it is set anew and the sums so far move with it.  What then lies under fp16's normal numbers is under 2^-20 of the
// column's largest.  (32 x 512 x 12 heads x 64, ragged: dQ 71 -> 75 us, dK / dV 78 -> 81; 4 x 4096: 390 -> 407 and 500 -> 530.)
struct AtFit {
    float scale = 1.0f, cap = 0.0f;                                         // cap: 2^15; 0 until an entry is met
    __device__ __forceinline__ float back() const { return __uint_as_float(0x7f000000u - __float_as_uint(scale)); }   // 1 / scale
    __device__ __forceinline__ float power() const { return (float)((int)(__float_as_uint(scale) >> 23) - 127); }     // log2 of it
};
__device__ __forceinline__ float at_pow2(int e) { return __uint_as_float((u32)(e + 127) << 23); }
__device__ __forceinline__ float at_largest(const f32x16& s) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, __builtin_fabsf(s[i]));
    return top;
}
// what a column whose tile has `top` as its largest is to be multiplied by, the sums so far with it
__device__ __forceinline__ float at_refit(float top, AtFit& m) {
    const int e = (int)(__float_as_uint(top) >> 23) - 127;                  // infinite: left as it is; under 2^-60 the results are zeros
    const float keep = top > m.cap && e < 128 ? at_pow2(6 - max(e, -60)) : 1.0f;
    m.scale *= keep;
    if (top > m.cap) m.cap = 0x1p15f;
    return keep;
}

// ---- backward: dQ, the bias gradient, D ---------------------------------------------------------------------------------------------------
// Bound by the vector unit (exponentials, bias, diagonal sums) with the matrix unit behind it at long lengths, by the first loads of a block at short ones:
// three blocks a CU (32 x 512 x 12 heads x 64 fp16, no mask: 87 us; before dS had a factor for each query 84, and with two blocks a CU 94; of it the bias
// gradient 16; ragged from 1 / 8 of the length 75; 4 x 4096: 405 us, 760 TFLOP/s).
template <typename T, int DP>
__global__ __launch_bounds__(AT_BLOCK, at_waves(sizeof(T), DP, 3)) void mfar_attn_dq_kernel(const AttnParams p) {
    AtPlace place;
    if (!at_place(p, (p.Lq + AT_COLS - 1) / AT_COLS, place)) return;
    extern __shared__ __align__(16) unsigned char at_lds[];
    T* tiles = (T*)at_lds;
    float* lut = (float*)(tiles + at_stages(sizeof(T), DP, true) * 2 * AT_TILE * DP);
    const int n_lut = at_lut_size(p.sat);
    float* hist = lut + n_lut;                                             // [4 waves][n_lut] sums of dS by distance
    float* skew = hist + 4 * n_lut;                                        // [4 waves][AT_SKEW]
    const int b = place.b, h = place.h, wave = wave_index(), l = threadIdx.x & 63, half = l >> 5;
    const int start = at_start(p, b);
    const int q = place.tile * AT_COLS + wave * 32 + (l & 31);
    const bool live = q < p.Lq;
    const int col = start + q, col_lo = start + place.tile * AT_COLS + wave * 32;
    int end = p.Lk;
    if (p.causal) end = min(end, max(start + min(p.Lq, (place.tile + 1) * AT_COLS), 0));
    const T* qrow = (const T*)p.q + b * p.q_b + (long long)(live ? q : 0) * p.q_l + h * p.q_h;
    const T* grow = (const T*)p.dout + b * p.do_b + (long long)(live ? q : 0) * p.do_l + h * p.do_h;
    const long long orow = (((long long)b * p.Lq + (live ? q : 0)) * p.H + h) * p.D, srow = ((long long)b * p.H + h) * p.Lq + q;
    V8<T> qf[DP / 16], gf[DP / 16];
    float dsum = 0.0f, lse = 0.0f;
    constexpr bool FIT = std::is_same<T, _Float16>::value;
    AtFit fit;
    f32x16 acc[DP / 32] = {};
    float far_lo = 0.0f, far_hi = 0.0f;
    const float c = p.scale * LOG2E;
    at_for_tiles<T, DP, true>(p, b, h, end, tiles, [&]() {
        if (live) lse = p.lse[srow];
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            qf[s] = at_load<T>(qrow, live, s, p.D);
            gf[s] = at_load<T>(grow, live, s, p.D);
            const V8<T> o = at_load<T>((const T*)p.o + orow, live, s, p.D);
            const V8<T> lo = sizeof(T) == 2 ? at_load<T>((const T*)(p.o_lo ? p.o_lo : p.o) + orow, live && p.o_lo, s, p.D) : V8<T>{};
#pragma unroll
            for (int j = 0; j < 8; ++j) dsum = __builtin_fmaf((float)gf[s][j], (float)o[j] + (float)lo[j], dsum);
        }
        at_lut(p, lut, h);
        if (p.dpart)
            for (int i = threadIdx.x; i < 4 * (n_lut + AT_SKEW); i += AT_BLOCK) hist[i] = 0.0f;
        dsum = sum_halves(dsum);
        if (live && half == 0) p.drow[srow] = dsum;
        if (!live || lse == -__builtin_inff()) lse = __builtin_inff();      // no keys: P = exp2(-inf) = 0 everywhere
    }, [&](int k0, u64 bits, T* kt, T* vt) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int row0 = k0 + 32 * t;
            f32x16 s = {}, dp = {};
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                s = mma(at_rows<T, DP>(kt, 32 * t, d), qf[d], s);
                dp = mma(at_rows<T, DP>(vt, 32 * t, d), gf[d], dp);
            }
            at_bias<1>(s, lut, p.sat, c, row0, col, col_lo, p.causal != 0, lse);
            const u32 shown = (u32)(bits >> (32 * t));
            if (shown != ~0u) at_hide(s, shown);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = exp2_fast(s[i]) * (FIT ? __builtin_fmaf(dp[i], fit.scale, -dsum * fit.scale) : dp[i] - dsum);
            if (FIT) {
                const float top = at_largest(s);
                if (__any(top > fit.cap)) {
                    const float keep = at_refit(max_halves(top), fit);      // (a column lies in both halves)
                    s *= keep, far_lo *= keep, far_hi *= keep;
#pragma unroll
                    for (int dt = 0; dt < DP / 32; ++dt) acc[dt] *= keep;
                }
            }
            if (p.dpart) {
                if (row0 - col_lo - 31 >= p.sat) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) far_hi += s[i];
                } else if (row0 + 31 - col_lo <= -p.sat) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) far_lo += s[i];
                } else {
                    at_diagonals(s, FIT ? fit.back() : 1.0f, skew + wave * AT_SKEW, hist + wave * n_lut + (row0 - col_lo) + p.sat + AT_EDGE);
                }
            }
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int g = 0; g < 2; ++g) acc[dt] = mma(at_cols<T, DP>(kt, 32 * t, g, dt), at_pack<T>(s, g), acc[dt]);
        }
    });
    __syncthreads();                                                       // (the tiles' memory is free)
    const int q0 = place.tile * AT_COLS + wave * 32;
    at_store<T, DP>((T*)p.dq + (((long long)b * p.Lq + q0) * p.H + h) * p.D, (long long)p.H * p.D, p.Lq - q0, acc, p.scale * (FIT ? fit.back() : 1.0f), p.D, at_lds + wave * at_out_bytes<T, DP>());
    if (p.dpart) {
        if (FIT) far_lo *= fit.back(), far_hi *= fit.back();
        for (int o = 1; o < 64; o <<= 1) {
            far_lo += __shfl_xor(far_lo, o);
            far_hi += __shfl_xor(far_hi, o);
        }
        __syncthreads();
        if (l == 0) {
            hist[wave * n_lut] += far_lo;                                  // the outermost distances: both in a last bucket
            hist[wave * n_lut + n_lut - 1] += far_hi;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n_lut; i += AT_BLOCK) {
            float t = 0.0f;
            for (int w = 0; w < 4; ++w) t += hist[w * n_lut + i];
            hist[i] = t;
        }
        __syncthreads();
        // a bucket holds the distances [lo, hi) of one side; 8 lanes add them up
        const int q_tiles = (p.Lq + AT_COLS - 1) / AT_COLS;
        float* to = p.dpart + ((long long)(b * q_tiles + place.tile) * p.H + h) * p.n_buckets;
        for (int n = threadIdx.x / 8; n < p.n_buckets; n += AT_BLOCK / 8) {
            const bool front = n >= p.n_side;
            const int m = n - (front ? p.n_side : 0);
            const int lo = max((int)p.first[m], front ? 1 : 0), hi = m == p.n_side - 1 ? p.sat + AT_EDGE + 1 : p.first[m + 1];   // (distance 0 counts as behind)
            float t = 0.0f;
            for (int d = lo + (threadIdx.x & 7); d < hi; d += 8) t += hist[(front ? d : -d) + p.sat + AT_EDGE];
            for (int o = 1; o < 8; o <<= 1) t += __shfl_xor(t, o);
            if ((threadIdx.x & 7) == 0) to[n] = t;
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
// Two blocks a CU: what a third would leave of the registers does not hold two accumulators, K and V (32 x 512 x 12 heads x 64 fp16, no mask, before P and dS had
// factors: 83 us against 95 to 103; with them 86, ragged from 1 / 8 of the length 81; 4 x 4096: 530 us, 780 TFLOP/s).  Head size 128 spills 53 to 62
// registers (152 to 212 bytes of scratch).
template <typename T, int DP>
__global__ __launch_bounds__(AT_BLOCK, at_waves(sizeof(T), DP, 2)) void mfar_attn_dkv_kernel(const AttnParams p) {
    AtPlace place;
    if (!at_place(p, (p.Lk + AT_COLS - 1) / AT_COLS, place)) return;
    extern __shared__ __align__(16) unsigned char at_lds[];
    constexpr int S = at_stages(sizeof(T), DP, true), SIZE = AT_TILE * DP;
    T* tiles = (T*)at_lds;                                                 // [S][Q, dO][AT_TILE][DP]
    float* stats = (float*)(tiles + S * 2 * SIZE);                          // [S][log2-sum, -D][AT_TILE]
    float* lut = stats + S * 2 * AT_TILE;
    const int b = place.b, h = place.h, wave = wave_index(), l = threadIdx.x & 63, half = l >> 5;
    const int start = at_start(p, b);
    const int key0 = place.tile * AT_COLS, key = key0 + wave * 32 + (l & 31);
    const bool live = key < p.Lk;
    const bool seen = live && (!p.causal || key < start + p.Lq) && (!p.mask || p.mask[(long long)b * p.mask_b + key] != 0);
    const int col_lo = key0 + wave * 32;
    f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
    const float c = p.scale * LOG2E;
    const T* qb = (const T*)p.q + b * p.q_b + h * p.q_h;
    const T* gb = (const T*)p.dout + b * p.do_b + h * p.do_h;
    const long long srow = ((long long)b * p.H + h) * p.Lq;
    int first = p.causal ? max(0, key0 - start) : 0;                       // the first query that sees the block's first key
    if (!__syncthreads_or(seen)) first = p.Lq;
    first = first / AT_TILE * AT_TILE;
    const AtStream<T, DP> qs(qb, p.q_l, p.Lq, p.D), gs(gb, p.do_l, p.Lq, p.D);
    float mine = 0.0f;                                                     // thread i: entry i of the next tile's statistics
    constexpr bool FIT = std::is_same<T, _Float16>::value;
    AtFit fit, raise;                                                      // of dS; of P, which is small alone for a key that is unlikely for every query
    auto fetch = [&](int q0, int slot) {
        qs.load(q0, tiles + slot * 2 * SIZE);
        gs.load(q0, tiles + slot * 2 * SIZE + SIZE);
        if (threadIdx.x < 2 * AT_TILE) {
            const int i = threadIdx.x % AT_TILE;
            const bool in = q0 + i < p.Lq, d = threadIdx.x >= AT_TILE;
            mine = in ? (d ? -p.drow[srow + q0 + i] : p.lse[srow + q0 + i]) : 0.0f;
            // rows behind the last and rows that saw nothing: P = exp2(s - inf) = 0
            if (!d && (!in || mine == -__builtin_inff())) mine = __builtin_inff();
            stats[slot * 2 * AT_TILE + threadIdx.x] = mine;
        }
    };
    int slot = 0;
    if (first < p.Lq) fetch(first, 0);
    const T* krow = (const T*)p.k + b * p.k_b + (long long)key * p.k_l + h * p.k_h;
    const T* vrow = (const T*)p.v + b * p.v_b + (long long)key * p.v_l + h * p.v_h;
    V8<T> kf[DP / 16], vf[DP / 16];                                         // (hidden keys' rows are not read)
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = 16 * s + 8 * half;
        kf[s] = vf[s] = V8<T>{};
        if (seen && d < p.D) kf[s] = *(const V8<T>*)(krow + d), vf[s] = *(const V8<T>*)(vrow + d);
    }
    at_lut(p, lut, h);
    for (int q0 = first; q0 < p.Lq; q0 += AT_TILE) {
        T *qt = tiles + slot * 2 * SIZE, *gt = qt + SIZE;
        const float* rows = stats + slot * 2 * AT_TILE;
        at_arrive();
        if (S == 2 && q0 + AT_TILE < p.Lq) fetch(q0 + AT_TILE, slot ^ 1);
        if (q0 + AT_TILE > p.Lq) {
            at_blank<T, DP>(qt, (1ull << (p.Lq - q0)) - 1);
            at_blank<T, DP>(gt, (1ull << (p.Lq - q0)) - 1);
            __syncthreads();
        }
        if (S == 2) slot ^= 1;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x16 s = {}, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] = rows[AT_TILE + 32 * t + crow(i, half)];      // -D: dP - D out of the product
#pragma unroll
            for (int d = 0; d < DP / 16; ++d) {
                s = mma(at_rows<T, DP>(qt, 32 * t, d), kf[d], s);
                dp = mma(at_rows<T, DP>(gt, 32 * t, d), vf[d], dp);
            }
            at_bias<-1>(s, lut, p.sat, c, start + q0 + 32 * t, key, col_lo, p.causal != 0, FIT ? -raise.power() : 0.0f);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = exp2_fast(s[i] - rows[32 * t + crow(i, half)]);
                dp[i] *= FIT ? s[i] * fit.scale : s[i];
            }
            if (FIT) {
                const float top_p = at_largest(s), top = at_largest(dp);
                if (__any(top_p > raise.cap || top > fit.cap)) {
                    const float up = at_refit(max_halves(top_p), raise), keep = at_refit(max_halves(top) * up, fit) * up;
                    s *= up, dp *= keep;
#pragma unroll
                    for (int dt = 0; dt < DP / 32; ++dt) dv[dt] *= up, dk[dt] *= keep;
                }
            }
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    dv[dt] = mma(at_cols<T, DP>(gt, 32 * t, g, dt), at_pack<T>(s, g), dv[dt]);
                    dk[dt] = mma(at_cols<T, DP>(qt, 32 * t, g, dt), at_pack<T>(dp, g), dk[dt]);
                }
        }
        if (S == 1) {
            __syncthreads();
            if (q0 + AT_TILE < p.Lq) fetch(q0 + AT_TILE, 0);
        }
    }
    if (!seen) {                                                           // a hidden key's column met no other: its sums are dropped here
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt) dk[dt] = f32x16{}, dv[dt] = f32x16{};
    }
    __syncthreads();                                                       // (the tiles' memory is free)
    const int k0 = key0 + wave * 32;
    const long long at = (((long long)b * p.Lk + k0) * p.H + h) * p.D;
    void* lds = at_lds + wave * at_out_bytes<T, DP>();
    const float lower = FIT ? raise.back() : 1.0f;
    at_store<T, DP>((T*)p.dk + at, (long long)p.H * p.D, p.Lk - k0, dk, p.scale * (FIT ? fit.back() * lower : 1.0f), p.D, lds);
    at_store<T, DP>((T*)p.dv + at, (long long)p.H * p.D, p.Lk - k0, dv, lower, p.D, lds);
}
