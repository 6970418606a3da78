// mfar_distill.h -- distillation from a teacher's top scores, forward and backward.
//
//   p = softmax(teacher / tau) over a row's listed columns (absent entries: id < 0), q = softmax(student / tau) over all N columns
//   loss = tau^2 sum_k p_k (log p_k - log q[id_k]),      d student[j] = g tau (q_j - sum over k with id_k = j of p_k)
//
// Bound by memory: the forward pass reads the student's scores once (running maximum and sum, in the log2 domain), the backward pass reads
// them again and writes the gradient.  A row is split over blocks when there are few rows; partial (maximum, sum) pairs are joined in a
// second launch, in block order.  A listed column's gradient is written once, from its sum over the list in list order: no atomics.
// An id >= N makes the row's loss and gradient NaN.
#pragma once
#include "mfar_ops_device.h"

#define DI_BLOCK 256
#define DI_MAX_K 1024

struct DistillParams {
    const void* x;               // [T, N] student scores, rows x_row apart
    long long x_row;
    const long long* ids;        // [T, K]
    const float* scores;         // [T, K] teacher scores
    const float* g;              // [T] gradient of the losses
    float *loss, *prob, *lse;    // [T], [T, K], [T] (log2 units of student / tau)
    float* part;                 // [T, splits, 2]
    void* dx;                    // [T, N] contiguous
    int T, N, K, splits, chunk;
    float tau;
};

__device__ __forceinline__ void di_join(float& m, float& s, float m2, float s2) {
    const float top = fmaxf(m, m2), base = top == -__builtin_inff() ? 0.0f : top;
    s = s * exp2_fast(m - base) + s2 * exp2_fast(m2 - base);
    m = top;
}
__device__ __forceinline__ void di_join_wave(float& m, float& s) {
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
        di_join(m, s, m2, s2);
    }
}
// the block's (m, s), valid in thread 0
__device__ __forceinline__ void di_join_block(float& m, float& s) {
    __shared__ float sh[2 * DI_BLOCK / 64];
    di_join_wave(m, s);
    if ((threadIdx.x & 63) == 0) {
        sh[threadIdx.x >> 6] = m;
        sh[4 + (threadIdx.x >> 6)] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < DI_BLOCK / 64; ++w) di_join(m, s, sh[w], sh[4 + w]);
}

// the row's loss from its log2-sum: run by the whole block
template <typename T> __device__ void di_row_loss(const DistillParams& p, int row, float lse) {
    __shared__ float red[DI_BLOCK / 64];
    const float c = LOG2E / p.tau;
    const long long at = (long long)row * p.K;
    float top = -__builtin_inff(), bad = 0.0f;
    for (int k = threadIdx.x; k < p.K; k += DI_BLOCK) {
        const long long id = p.ids[at + k];
        if (id >= p.N) bad = __builtin_nanf("");
        if (id >= 0) top = fmaxf(top, p.scores[at + k] * c);
    }
    for (int o = 32; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor(top, o));
        bad += __shfl_xor(bad, o);
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float sum = bad;
    for (int k = threadIdx.x; k < p.K; k += DI_BLOCK)
        if (p.ids[at + k] >= 0) sum += exp2_fast(p.scores[at + k] * c - base);
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    const float norm = sum == 0.0f ? 0.0f : 1.0f / sum, lsum = __log2f(sum);
    float t = 0.0f;
    for (int k = threadIdx.x; k < p.K; k += DI_BLOCK) {
        const long long id = p.ids[at + k];
        float pr = 0.0f;
        if (id >= 0) {
            const float z = p.scores[at + k] * c - base;
            pr = exp2_fast(z) * norm;
            const float xs = id < p.N ? (float)((const T*)p.x)[(long long)row * p.x_row + id] * c : 0.0f;
            if (pr != 0.0f) t += pr * ((z - lsum) - (xs - lse));            // (0 log 0 = 0; NaN != 0 stays)
        }
        p.prob[at + k] = pr;
    }
    for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = t;
    __syncthreads();
    if (threadIdx.x == 0) {
        p.loss[row] = p.tau * p.tau * LN2 * ((red[0] + red[1]) + (red[2] + red[3]));
        p.lse[row] = lse;
    }
}

// A piece [lo, hi) of a row, as wide loads see it: `step(i, v, n)` is called by one thread for each run of up to EACH elements, of which the first n
// (EACH but at the row's ends) are real.  Rows may start anywhere; the runs start on 16 bytes.
template <typename T> struct DiRun {
    static constexpr int EACH = 16 / sizeof(T);
    typedef T V __attribute__((ext_vector_type(EACH)));
};
// elements before the first 16-byte border at or behind `at`
template <typename T> __device__ __forceinline__ int di_head(const T* at) { return (int)((16 - ((uintptr_t)at & 15)) & 15) / (int)sizeof(T); }

template <typename T>
__global__ __launch_bounds__(DI_BLOCK) void mfar_distill_forward_kernel(const DistillParams p) {
    const int row = blockIdx.x, lo = blockIdx.y * p.chunk, hi = min(p.N, lo + p.chunk);
    const T* x = (const T*)p.x + (long long)row * p.x_row;
    const float c = LOG2E / p.tau;
    constexpr int E = DiRun<T>::EACH, U = 16 / E;                           // 16 elements a thread and turn
    typedef typename DiRun<T>::V V;
    const int first = min(hi, lo + di_head(x + lo)), runs = (hi - first) / E, last = first + runs * E;
    const V* xv = (const V*)(x + first);
    float m = -__builtin_inff(), s = 0.0f;
    for (int i = threadIdx.x; i < runs; i += U * DI_BLOCK) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = xv[min(i + u * DI_BLOCK, runs - 1)];
        float t[16], top = m;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                t[u * E + e] = i + u * DI_BLOCK < runs ? (float)v[u][e] * c : -__builtin_inff();
                top = fmaxf(top, t[u * E + e]);
            }
        const float base = top == -__builtin_inff() ? 0.0f : top;
        s *= exp2_fast(m - base);
        m = top;
#pragma unroll
        for (int e = 0; e < 16; ++e) s += exp2_fast(t[e] - base);
    }
    // what lies before the first and behind the last whole run: at most 2 (E - 1) elements
    {
        const int k = threadIdx.x, j = k < first - lo ? lo + k : last + k - (first - lo);
        if (j < hi && (j < first || j >= last)) di_join(m, s, (float)x[j] * c, 1.0f);
    }
    di_join_block(m, s);
    if (p.splits > 1) {
        if (threadIdx.x == 0) {
            float* to = p.part + ((long long)row * p.splits + blockIdx.y) * 2;
            to[0] = m;
            to[1] = s;
        }
        return;
    }
    __shared__ float all;
    if (threadIdx.x == 0) all = m + __log2f(s);
    __syncthreads();
    di_row_loss<T>(p, row, all);
}
template <typename T>
__global__ __launch_bounds__(DI_BLOCK) void mfar_distill_join_kernel(const DistillParams p) {
    const int row = blockIdx.x;
    float m = -__builtin_inff(), s = 0.0f;
    for (int i = threadIdx.x; i < p.splits; i += DI_BLOCK) {
        const float* at = p.part + ((long long)row * p.splits + i) * 2;
        di_join(m, s, at[0], at[1]);
    }
    di_join_block(m, s);
    __shared__ float all;
    if (threadIdx.x == 0) all = m + __log2f(s);
    __syncthreads();
    di_row_loss<T>(p, row, all);
}
template <typename T>
__global__ __launch_bounds__(DI_BLOCK) void mfar_distill_backward_kernel(const DistillParams p) {
    __shared__ int ids[DI_MAX_K];
    __shared__ float prob[DI_MAX_K];
    const int row = blockIdx.x, lo = blockIdx.y * p.chunk, hi = min(p.N, lo + p.chunk);
    const T* x = (const T*)p.x + (long long)row * p.x_row;
    T* dx = (T*)p.dx + (long long)row * p.N;
    const float c = LOG2E / p.tau, lse = p.lse[row], g = p.g[row] * p.tau;
    float mass = 0.0f;                                                      // 1, 0 for a row without a teacher, NaN for a bad one
    for (int k = threadIdx.x; k < p.K; k += DI_BLOCK) {
        const long long id = p.ids[(long long)row * p.K + k];
        ids[k] = id >= 0 && id < p.N ? (int)id : -1;
        prob[k] = p.prob[(long long)row * p.K + k];
    }
    __syncthreads();
    for (int k = 0; k < p.K; ++k) mass += prob[k];
    mass = mass > 0.5f ? 1.0f : (mass == 0.0f ? 0.0f : mass);
    const float scale = mass == 0.0f ? 0.0f : g * mass;
    auto grad = [&](float v) { return (T)(mass == 0.0f ? 0.0f : scale * exp2_fast(v * c - lse)); };
    constexpr int E = DiRun<T>::EACH;
    typedef typename DiRun<T>::V V;
    // runs start where dx has a 16-byte border; x is read wherever that falls
    const int first = min(hi, lo + di_head(dx + lo)), runs = (hi - first) / E, last = first + runs * E;
    for (int i = threadIdx.x; i < runs; i += 2 * DI_BLOCK) {
        V v[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) __builtin_memcpy(&v[u], x + first + min(i + u * DI_BLOCK, runs - 1) * E, sizeof(V));
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (i + u * DI_BLOCK < runs) {
                V o;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = grad((float)v[u][e]);
                *(V*)(dx + first + (i + u * DI_BLOCK) * E) = o;
            }
    }
    {
        const int k = threadIdx.x, j = k < first - lo ? lo + k : last + k - (first - lo);
        if (j < hi && (j < first || j >= last)) dx[j] = grad((float)x[j]);
    }
    __threadfence_block();
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += DI_BLOCK) {
        const int id = ids[k];
        if (id < lo || id >= hi) continue;
        float t = 0.0f;
        bool first = true;
        for (int i = 0; i < p.K; ++i)
            if (ids[i] == id) {
                if (i < k) first = false;
                t += prob[i];
            }
        if (first) dx[id] = (T)(g * (mass * exp2_fast((float)x[id] * c - lse) - t));
    }
}
