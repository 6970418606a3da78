// mfar_distill.h -- distillation from a teacher's top scores, forward and backward.
//
//   p = softmax(teacher / tau) over a row's listed columns (absent entries: id < 0), q = softmax(student / tau) over all N columns
//   loss = tau^2 sum_k p_k (log p_k - log q[id_k]),      d student[j] = g tau (q_j - sum over k with id_k = j of p_k)
//
// Bound by memory: the forward pass reads the student's scores once (running maximum and sum, in the log2 domain), the backward pass reads
// them again and writes the gradient (64 x 500009 fp32: 31 us, 4.1 TB/s, and 47, 5.4 TB/s; 4096 x 32005 bf16: 94, 2.8 TB/s, and 98.  There a row is 4
// turns of a block, and the teacher's fetch and four reductions over the block around them overlap with nothing; the arithmetic itself comes to some 30 us).  A row is split over blocks when there are few rows; partial (maximum, sum) pairs are joined in a
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
    float *loss, *prob, *stat;   // [T], [T, K], [T, 2]: the row's largest score, log2 of the sum of 2^((score - largest) c)
    float* part;                 // [T, splits, 2]
    void* dx;                    // [T, N] contiguous
    int T, N, K, splits, chunk;
    float tau;
};

// Scores of any size: differences from the largest are taken before they are scaled to log2 units (c = log2(e) / tau), and the largest score and the
// logarithm of the sum are kept apart.
__device__ __forceinline__ void di_join(float& m, float& s, float m2, float s2, float c) {
    const float top = fmaxf(m, m2), base = top == -__builtin_inff() ? 0.0f : top;
    s = s * exp2_fast((m - base) * c) + s2 * exp2_fast((m2 - base) * c);
    m = top;
}
// the block's (m, s), valid in thread 0
__device__ __forceinline__ void di_join_block(float& m, float& s, float c) {
    __shared__ float sh[2 * DI_BLOCK / 64];
    for (int o = 32; o > 0; o >>= 1) {
        const float m2 = __shfl_xor(m, o), s2 = __shfl_xor(s, o);
        di_join(m, s, m2, s2, c);
    }
    if ((threadIdx.x & 63) == 0) {
        sh[threadIdx.x >> 6] = m;
        sh[4 + (threadIdx.x >> 6)] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < DI_BLOCK / 64; ++w) di_join(m, s, sh[w], sh[4 + w], c);
}

__device__ __forceinline__ float di_sum_block(float x, float* red) {
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return x;
}
__device__ __forceinline__ float di_max_block(float x, float* red) {
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    return x;
}
// A row's teacher, up to four entries a thread: fetched (with the student's scores of the same columns) ahead of the pass over the row, so that only
// arithmetic is left behind it.
template <typename T> struct DiTeacher {
    static constexpr int N = DI_MAX_K / DI_BLOCK;
    float z[N], xs[N];           // scores of teacher and student; z = -inf: no entry
    float bad;                   // NaN: an id past the last column
    __device__ __forceinline__ void fetch(const DistillParams& p, int row) {
        bad = 0.0f;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const int k = t * DI_BLOCK + (int)threadIdx.x;
            z[t] = -__builtin_inff(), xs[t] = 0.0f;
            if (k < p.K) {
                const long long id = p.ids[(long long)row * p.K + k];
                if (id >= 0) z[t] = p.scores[(long long)row * p.K + k];
                if (id >= p.N) bad = __builtin_nanf("");
                if (id >= 0 && id < p.N) xs[t] = (float)((const T*)p.x)[(long long)row * p.x_row + id];
            }
        }
    }
    // loss, probabilities and statistics of the row (m, s: its largest score and sum, in thread 0); without a teacher the logarithm is +inf, in a bad
    // row NaN
    __device__ __forceinline__ void finish(const DistillParams& p, int row, float m, float s) {
        __shared__ float all[2];
        if (threadIdx.x == 0) {
            all[0] = m;
            all[1] = __log2f(s);
        }
        __syncthreads();
        m = all[0];
        const float l2s = all[1], c = LOG2E / p.tau;
        __shared__ float red[DI_BLOCK / 64];
        float top = -__builtin_inff(), sum = bad;
#pragma unroll
        for (int t = 0; t < N; ++t) top = fmaxf(top, z[t]);
        top = di_max_block(top, red);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float e[N];
#pragma unroll
        for (int t = 0; t < N; ++t) {
            z[t] = (z[t] - base) * c;
            e[t] = exp2_fast(z[t]);
            sum += e[t];
        }
        sum = di_sum_block(sum, red);
        const float norm = sum == 0.0f ? 0.0f : 1.0f / sum, lsum = __log2f(sum);
        float loss = 0.0f;
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const int k = t * DI_BLOCK + (int)threadIdx.x;
            const float pr = e[t] * norm;
            if (pr != 0.0f) loss += pr * ((z[t] - lsum) - ((xs[t] - m) * c - l2s));   // (0 log 0 = 0; NaN != 0 stays)
            if (k < p.K) p.prob[(long long)row * p.K + k] = pr;
        }
        loss = di_sum_block(loss, red);
        if (threadIdx.x == 0) {
            p.loss[row] = p.tau * p.tau * LN2 * loss;
            p.stat[2 * row] = m;
            p.stat[2 * row + 1] = sum == 0.0f ? __builtin_inff() : (sum == sum ? l2s : sum);
        }
    }
};

// Runs of 16 bytes of a row's piece [lo, hi): they start where `at` has a 16-byte border; before the first and behind the last lie at most
// EACH - 1 elements each, taken one by thread (di_rest).
template <typename T> struct DiRuns {
    static constexpr int EACH = 16 / sizeof(T);
    typedef T V __attribute__((ext_vector_type(EACH)));
    int lo, hi, first, n, last;
    __device__ __forceinline__ DiRuns(const T* at, int lo_, int hi_) : lo(lo_), hi(hi_) {
        first = min(hi, lo + (int)((16 - ((uintptr_t)(at + lo) & 15)) & 15) / (int)sizeof(T));
        n = (hi - first) / EACH;
        last = first + n * EACH;
    }
    // this thread's element outside the runs, or -1
    __device__ __forceinline__ int rest() const {
        const int k = threadIdx.x, j = k < first - lo ? lo + k : last + k - (first - lo);
        return j < hi && (j < first || j >= last) ? j : -1;
    }
};

template <typename T>
__global__ __launch_bounds__(DI_BLOCK) void mfar_distill_forward_kernel(const DistillParams p) {
    const int row = blockIdx.x, lo = blockIdx.y * p.chunk, hi = min(p.N, lo + p.chunk);
    const T* x = (const T*)p.x + (long long)row * p.x_row;
    const float c = LOG2E / p.tau;
    typedef typename DiRuns<T>::V V;
    constexpr int E = DiRuns<T>::EACH, U = 4;                               // 64 bytes a thread and turn, the next turn's in flight
    const int n = (hi - lo) / E;                                            // runs of 16 bytes, wherever they start: the sum's order goes by columns alone
    const T* xl = x + lo;
    V next[U];
    auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&next[u], xl + min(i + u * DI_BLOCK, n - 1) * E, sizeof(V));
    };
    if ((int)threadIdx.x < n) fetch(threadIdx.x);
    DiTeacher<T> teacher;
    if (p.splits == 1) teacher.fetch(p, row);
    const int rest = lo + n * E + (int)threadIdx.x < hi ? lo + n * E + (int)threadIdx.x : -1;   // (fewer than E of them)
    const float one = rest >= 0 ? (float)x[rest] : -__builtin_inff();
    float m = -__builtin_inff(), s = 0.0f;
    for (int i = threadIdx.x; i < n; i += U * DI_BLOCK) {
        float t[U * E], top = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) t[u * E + e] = (float)next[u][e];
        const int have = (n - 1 - i) / DI_BLOCK;                       // of the U runs, 0..have are this thread's
        if (i + U * DI_BLOCK < n) fetch(i + U * DI_BLOCK);
        if (have < U - 1) {
#pragma unroll
            for (int u = 1; u < U; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) t[u * E + e] = u <= have ? t[u * E + e] : -__builtin_inff();
        }
#pragma unroll
        for (int e = 0; e < U * E; ++e) top = fmaxf(top, t[e]);
        top = fmaxf(m, top);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        s *= exp2_fast((m - base) * c);
        m = top;
        float s2 = 0.0f;
#pragma unroll
        for (int e = 0; e < U * E; e += 2) {
            s += exp2_fast((t[e] - base) * c);
            s2 += exp2_fast((t[e + 1] - base) * c);
        }
        s += s2;
    }
    if (rest >= 0) di_join(m, s, one, 1.0f, c);
    di_join_block(m, s, c);
    if (p.splits > 1) {
        if (threadIdx.x == 0) {
            float* to = p.part + ((long long)row * p.splits + blockIdx.y) * 2;
            to[0] = m;
            to[1] = s;
        }
        return;
    }
    teacher.finish(p, row, m, s);
}
template <typename T>
__global__ __launch_bounds__(DI_BLOCK) void mfar_distill_join_kernel(const DistillParams p) {
    const int row = blockIdx.x;
    DiTeacher<T> teacher;
    teacher.fetch(p, row);
    const float c = LOG2E / p.tau;
    float m = -__builtin_inff(), s = 0.0f;
    for (int i = threadIdx.x; i < p.splits; i += DI_BLOCK) {
        const float* at = p.part + ((long long)row * p.splits + i) * 2;
        di_join(m, s, at[0], at[1], c);
    }
    di_join_block(m, s, c);
    teacher.finish(p, row, m, s);
}
template <typename T>
__global__ __launch_bounds__(DI_BLOCK) void mfar_distill_backward_kernel(const DistillParams p) {
    __shared__ int ids[DI_MAX_K];
    __shared__ float prob[DI_MAX_K];
    const int row = blockIdx.x, lo = blockIdx.y * p.chunk, hi = min(p.N, lo + p.chunk);
    const T* x = (const T*)p.x + (long long)row * p.x_row;
    T* dx = (T*)p.dx + (long long)row * p.N;
    const float c = LOG2E / p.tau, m = p.stat[2 * row], l2s = p.stat[2 * row + 1], g = p.g[row] * p.tau;
    const bool none = l2s == __builtin_inff();                              // no teacher: zeros, whatever the scores
    auto prob_of = [&](T v) { return none ? 0.0f : exp2_fast(((float)v - m) * c - l2s); };
    auto grad = [&](T v) { return (T)(g * prob_of(v)); };
    typedef typename DiRuns<T>::V V;
    constexpr int E = DiRuns<T>::EACH, U = 2;
    const DiRuns<T> runs(dx, lo, hi);                                       // (x is read wherever dx has its borders)
    const int rest = runs.rest();
    for (int i = threadIdx.x; i < runs.n; i += U * DI_BLOCK) {
        V v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(&v[u], x + runs.first + min(i + u * DI_BLOCK, runs.n - 1) * E, sizeof(V));
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i + u * DI_BLOCK < runs.n) {
                V o;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = grad(v[u][e]);
                *(V*)(dx + runs.first + (i + u * DI_BLOCK) * E) = o;
            }
    }
    if (rest >= 0) dx[rest] = grad(x[rest]);
    for (int k = threadIdx.x; k < p.K; k += DI_BLOCK) {
        const long long id = p.ids[(long long)row * p.K + k];
        ids[k] = id >= lo && id < hi ? (int)id : -1;
        prob[k] = p.prob[(long long)row * p.K + k];
    }
    __threadfence_block();                                                 // the listed columns are written again, behind what was written above
    __syncthreads();
    for (int k = threadIdx.x; k < p.K; k += DI_BLOCK) {
        const int id = ids[k];
        if (id < 0) continue;
        float t = 0.0f;
        bool first = true;
        for (int i = 0; i < p.K; ++i)
            if (ids[i] == id) {
                if (i < k) first = false;
                t += prob[i];
            }
        if (first) dx[id] = (T)(g * (prob_of(x[id]) - t));
    }
}
