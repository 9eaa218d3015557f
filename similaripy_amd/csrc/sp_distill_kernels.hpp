// sp_distill_kernels.hpp — divergence of a student's dense scores from a teacher's top-k lists, and its gradient.
//
//   p_j = softmax of t_j / tau over the list (or exp(t_j / tau - teacher_lse)),   q = softmax of z / tau over all columns
//   loss = tau^2 sum_j p_j (log p_j - log q[c_j]),     dz_v = g tau (P q_v - sum_{c_j = v} p_j),   P = sum_j p_j
//
// One reading of the row gives its maximum and the sum of exp2((z - max) c), c = log2(e) / tau, in a single pass: every thread
// keeps a running maximum and rescales its sum when a vector raises it.  Between forward and backward a row keeps both, not their
// log-sum-exp: one float32 of about 20 would tilt all of q by its rounding, and for scores near the type's lowest value (masks) it
// would lose the sum altogether.  The list is one wave's work.
#pragma once
#include "sp_dense_common.hpp"

namespace {

struct DistillParams {
    const void *student;
    void *grad;
    i64 n_rows, n_cols, ld_student, ld_grad;
    int k, cols64, values_dtype;
    float tau, inv_tau, c;             // c = log2(e) / tau
    const void *cols, *values;
    const int *counts;
    const float *teacher_lse;
    float *loss;
    float *stats;                      // [n_rows, 2] maximum of z, sum of exp((z - maximum) / tau)
    const float *grad_loss;
    int splits;                        // workgroups of a row
    i64 chunk;                         // columns of one of them (a multiple of the vector)
    float *part;                       // [n_rows, splits, 2] maximum, sum
    int stage;                         // vectors of a row that the one-call kernel keeps in LDS
};

// maximum and sum of exp2((z - max) c) of some columns
struct MaxSum {
    float m, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c) {
    const float m = fmaxf(a.m, b.m);
    return {m, a.s * (a.m == m ? 1.f : exp2_fast((a.m - m) * c)) + b.s * (b.m == m ? 1.f : exp2_fast((b.m - m) * c))};
}
__device__ __forceinline__ MaxSum wave_join(MaxSum a, float c) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) a = join(a, MaxSum{__shfl_xor(a.m, d, 64), __shfl_xor(a.s, d, 64)}, c);
    return a;
}

// exp2((z - m) c) is taken as exp2(z c - off) 2^-r, one fused operation per score with off = m c rounded and r = m c - off what the
// rounding left (exact as a fused operation, the same for the whole row): scores far from 0 lose nothing.  Up to |m c| = 2^31 r is at most
// 64.  Beyond (a row masked with -1e10, -1e30, the type's lowest value) 2^r would leave float32, and every score that is not m itself lies
// at least 2^-24 |m| below it, 128 in the exponent: its q is below 2^-126 and counts as 0.  A power of two in the place of c, the one that makes
// that distance at least 256, then keeps z c - off exactly 0 for the scores that are m.
constexpr float OFF_MAX = 2147483648.f;
struct Exponent {
    float c, off;
};
__device__ __forceinline__ bool off_fits(float m, float c) { return fabsf(m * c) <= OFF_MAX || m == NEG_INF; }
__device__ __forceinline__ Exponent exponent_of(float m, float c) {
    if (m == NEG_INF) return {c, 0.f};
    if (off_fits(m, c)) return {c, m * c};
    if (fabsf(m) > 3.402823466e38f) return {c, m};              // +inf, NaN: every q is NaN or 0
    int e;
    (void)frexpf(m, &e);                                       // -69 <= e <= 128: temperatures are at least 1e-30
    const float pow2 = ldexpf(1.f, 33 - e);
    return {pow2, m * pow2};
}
__device__ __forceinline__ float correction_of(float m, Exponent x) { return m == NEG_INF ? 1.f : exp2_fast(-__fmaf_rn(m, x.c, -x.off)); }      // 2^-r
// (sh: one slot per wave; the result is everybody's)
template <int NT> __device__ __forceinline__ MaxSum block_join(MaxSum a, float c, MaxSum *sh) {
    a = wave_join(a, c);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    constexpr int W = NT / 64;
    a = sh[threadIdx.x & (W - 1)];
#pragma unroll
    for (int d = W / 2; d > 0; d >>= 1) a = join(a, MaxSum{__shfl_xor(a.m, d, 64), __shfl_xor(a.s, d, 64)}, c);
    return a;
}

// a thread's running sum, relative to 2^off
struct Running {
    float m, off, s;
};
template <int N> __device__ __forceinline__ void add_vec(Running &a, const float *z, float c) {
    float m = a.m;
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, z[j]);
    const float off = fminf(fmaxf(m * c, -OFF_MAX), OFF_MAX);      // (below, the sum stays as it is, relative to 2^-OFF_MAX; above, it is not used)
    float s = a.s * exp2_fast(a.off - off);
#pragma unroll
    for (int j = 0; j < N; ++j) s += exp2_fast(__fmaf_rn(z[j], c, -off));
    a = {m, off, s};
}

// (a maximum whose m c is beyond OFF_MAX has no sum here: it is nothing next to a larger one, and the row is summed again otherwise)
__device__ __forceinline__ MaxSum finish(const Running &a, float c) {
    return {a.m, a.m == NEG_INF || !off_fits(a.m, c) ? (a.s != a.s ? a.s : 0.f) : a.s * exp2_fast(-__fmaf_rn(a.m, c, -a.off))};
}

// maximum and sum over columns [c0, c1) of a row, by the NT threads of the workgroup (each its share)
template <typename T, int NT> __device__ __forceinline__ MaxSum thread_columns(const T *z, i64 c0, i64 c1, float c) {
    constexpr int N = VecOf<T>::N, U = 4;
    Running a{NEG_INF, NEG_INF, 0.f};
    i64 i = c0 + (i64)threadIdx.x * N;
    for (; i + (U - 1) * NT * N + N <= c1; i += U * NT * N) {
        RawVec<T, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = vec_load<T, N>(z + i + u * NT * N);
        float v[U * N];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) v[u * N + j] = up(x[u].v[j]);
        add_vec<U * N>(a, v, c);
    }
    for (; i + N <= c1; i += NT * N) {
        const RawVec<T, N> x = vec_load<T, N>(z + i);
        float v[N];
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = up(x.v[j]);
        add_vec<N>(a, v, c);
    }
    for (int j = 0; j < N; ++j)
        if (i + j < c1) {
            const float v = up(z[i + j]);
            add_vec<1>(a, &v, c);
        }
    return finish(a, c);
}

// columns summed once more, with an exponent that fits; a.m is their maximum
template <typename T, int NT> __device__ __forceinline__ MaxSum rescan(const T *z, i64 c0, i64 c1, MaxSum a, float c, MaxSum *sh) {
    const Exponent x = exponent_of(a.m, c);
    a.s = 0.f;
    for (i64 i = c0 + threadIdx.x; i < c1; i += NT) a.s += exp2_fast(__fmaf_rn(up(z[i]), x.c, -x.off));
    __syncthreads();
    return block_join<NT>(a, c, sh);
}
// thread_columns for the workgroup: the result is everybody's
template <typename T, int NT> __device__ __forceinline__ MaxSum scan_columns(const T *z, i64 c0, i64 c1, float c, MaxSum *sh) {
    MaxSum a = block_join<NT>(thread_columns<T, NT>(z, c0, c1, c), c, sh);
    if (!off_fits(a.m, c)) a = rescan<T, NT>(z, c0, c1, a, c, sh);      // (uniform)
    return a;
}

// A row's list in LDS: columns (-1: not in the list), probabilities, the student's scores there; for the gradient also the entries of
// every thread, those whose columns it writes, as a chain from head[thread] over next.
struct ListLds {
    int *col;
    float *prob, *z;
    int *next, *head;
    __device__ __forceinline__ ListLds(int *mem, int k) : col(mem), prob((float *)(mem + room(k))), z((float *)(mem + 2 * room(k))), next(mem + 3 * room(k)), head(mem + 4 * room(k)) {}
    static __host__ __device__ constexpr int room(int k) { return (k + 3) / 4 * 4; }
    static __host__ __device__ constexpr int loss_bytes(int k) { return 12 * room(k); }
    static __host__ __device__ constexpr int grad_bytes(int k, int threads) { return 16 * room(k) + 4 * threads; }
};
// The teacher's list of a row, by the 64 lanes of one wave, with S = sum p_j log p_j and P = sum p_j.  Nothing here depends on the row's
// maximum and sum.  256 entries are requested at once, then the student's scores at all of their columns.
struct ListSums {
    float mass, plogp;
};
template <typename T> __device__ __forceinline__ ListSums list_sums(const DistillParams &p, i64 row, const T *z, const ListLds &list) {
    constexpr int R = 4;
    const int lane = threadIdx.x & 63;
    int n = p.counts ? p.counts[row] : p.k;
    n = n < 0 ? 0 : n > p.k ? p.k : n;
    const i64 base = row * p.k;
    float top = NEG_INF;
    for (int j0 = lane; j0 < p.k; j0 += 64 * R) {
        i64 col[R];
        float t[R], zc[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int j = j0 + 64 * u;
            col[u] = -1;
            t[u] = NEG_INF;
            if (j < n) {
                col[u] = load_index(p.cols, p.cols64, base + j);
                t[u] = load_scalar(p.values, p.values_dtype, base + j);
            }
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const bool in = col[u] >= 0 && col[u] < p.n_cols;
            zc[u] = 0.f;
            if (in) zc[u] = up(z[col[u]]);
            else {
                col[u] = -1;
                t[u] = NEG_INF;
            }
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int j = j0 + 64 * u;
            if (j < p.k) {
                list.col[j] = (int)col[u];
                list.prob[j] = t[u];
                list.z[j] = zc[u];
            }
            top = fmaxf(top, t[u]);
        }
    }
    float shift;
    if (p.teacher_lse) {
        shift = -p.teacher_lse[row];
        top = 0.f;
    } else {
        top = wave_max(top);
        float sum = 0.f;
        for (int j = lane; j < p.k; j += 64)
            if (list.col[j] >= 0 && top != NEG_INF) sum += exp2_fast((list.prob[j] - top) * p.inv_tau * LOG2E);
        sum = wave_sum(sum);
        shift = sum > 0.f || sum != sum ? -logf(sum) : NEG_INF;       // (nothing in the list, or -inf only: all p_j are 0)
    }
    ListSums r{0.f, 0.f};
    for (int j = lane; j < p.k; j += 64) {
        float prob = 0.f;
        if (list.col[j] >= 0) {
            // (a value of -inf has no mass, also where all of the teacher's are -inf and teacher_lse with them)
            const float logp = top == NEG_INF || list.prob[j] == NEG_INF ? NEG_INF : __fmaf_rn(list.prob[j] - top, p.inv_tau, shift);
            prob = exp2_fast(logp * LOG2E);
            r.mass += prob;
            if (prob != 0.f) r.plogp += prob * logp;
        }
        list.prob[j] = prob;
    }
    r.mass = wave_sum(r.mass);
    r.plogp = wave_sum(r.plogp);
    return r;
}
// tau^2 sum p_j (log p_j - log q[c_j]) by the same wave, log q = (z - m) / tau - log s: taken from score - maximum, so that the type's lowest
// value as a mask stays finite
__device__ __forceinline__ float list_loss(const DistillParams &p, ListSums l, MaxSum a, const ListLds &list) {
    const float high = a.m == NEG_INF ? 0.f : a.m, logs = logf(a.s);
    float cross = 0.f;
    for (int j = threadIdx.x & 63; j < p.k; j += 64)
        if (list.prob[j] != 0.f) cross += list.prob[j] * (list.z[j] == NEG_INF ? NEG_INF : __fmaf_rn(list.z[j] - high, p.inv_tau, -logs));
    return p.tau * (p.tau * (l.plogp - wave_sum(cross)));      // (tau^2 alone may leave float32: 0 * inf for an empty list)
}
// The chains, by the wave that has made the list: column c of [c0, c1) is in the chain of the thread that writes it with the row, vector by
// vector ((c - c0) / N) % NT, from column `tail` on one by one.  (What a thread writes twice ends as the later of its two stores: no barrier
// lies between the row's vectors and the listed columns.)
template <int NT, int N> __device__ __forceinline__ void chain_listed(int k, i64 c0, i64 c1, i64 tail, const ListLds &list) {
    const int lane = threadIdx.x & 63;
    for (int i = lane; i < NT; i += 64) list.head[i] = -1;
    for (int j = lane; j < k; j += 64) {
        const int c = list.col[j];
        if (c >= c0 && c < c1) list.next[j] = atomicExch(&list.head[c >= tail ? (int)(c - tail) : (int)((unsigned)(c - c0) / N % NT)], j);
    }
}
// The listed columns of this thread once more, with their probabilities taken off.  Entries of the same column are in the same chain; the
// first one of the list writes their sum, added up in the order of the list.
template <typename T, typename F> __device__ __forceinline__ void write_listed(int k, T *d, F one, float gt, const ListLds &list) {
    const int head = list.head[threadIdx.x];
    for (int j = head; j >= 0; j = list.next[j]) {
        const int c = list.col[j];
        bool first = true, again = false;
        for (int i = list.next[j]; i >= 0 && first; i = list.next[i])
            if (list.col[i] == c) {
                again = true;
                first = i > j;
            }
        for (int i = head; i != j && first; i = list.next[i])
            if (list.col[i] == c) {
                again = true;
                first = i > j;
            }
        if (!first) continue;
        float prob = list.prob[j];
        if (again) {
            prob = 0.f;
            for (int i = j; i < k; ++i)
                if (list.col[i] == c) prob += list.prob[i];
        }
        d[c] = (T)(one(list.z[j]) - gt * prob);
    }
}

// (16 bytes aligned: the one-call kernel's vectors are read as such)
extern __shared__ __align__(16) int distill_list[];

template <typename T> __device__ __forceinline__ void finish_loss(const DistillParams &p, i64 row, MaxSum a) {
    if (p.loss) {
        const ListLds list(distill_list, p.k);
        const ListSums l = list_sums<T>(p, row, (const T *)p.student + row * p.ld_student, list);
        const float loss = list_loss(p, l, a, list);
        if ((threadIdx.x & 63) == 0) p.loss[row] = loss;
    }
    if (p.stats && (threadIdx.x & 63) == 0) {
        p.stats[2 * row] = a.m;
        p.stats[2 * row + 1] = a.s;
    }
}

// one workgroup per row and split; a row in one piece is finished here
template <typename T, int NT> __global__ __launch_bounds__(NT) void sp_distill_scan_kernel(DistillParams p) {
    __shared__ MaxSum sh[NT / 64];
    const i64 row = blockIdx.x / p.splits, c0 = (blockIdx.x % p.splits) * p.chunk, c1 = min(p.n_cols, c0 + p.chunk);
    const T *z = (const T *)p.student + row * p.ld_student;
    const MaxSum a = scan_columns<T, NT>(z, c0, c1, p.c, sh);
    if (p.splits == 1) {
        if (threadIdx.x < 64) finish_loss<T>(p, row, a);
    } else if (threadIdx.x == 0) {
        p.part[2 * blockIdx.x] = a.m;
        p.part[2 * blockIdx.x + 1] = a.s;
    }
}

__device__ __forceinline__ MaxSum join_parts(const DistillParams &p, i64 row) {
    MaxSum a{NEG_INF, 0.f};
    for (int i = threadIdx.x & 63; i < p.splits; i += 64) a = join(a, MaxSum{p.part[2 * (row * p.splits + i)], p.part[2 * (row * p.splits + i) + 1]}, p.c);
    return wave_join(a, p.c);
}

// rows in several pieces: one wave joins them
template <typename T> __global__ __launch_bounds__(64) void sp_distill_join_kernel(DistillParams p) { finish_loss<T>(p, blockIdx.x, join_parts(p, blockIdx.x)); }

// The gradient of columns [c0, c1) of a row by the NT threads of a workgroup: g tau P q everywhere, then the listed columns once
// more with their probabilities taken off.  The list keeps the scores at its columns: they have been read before
// anything is written, so `grad` may be `student`.  A row whose list
// has no mass gets zeros, whatever its scores hold (a padded row of a batch).
template <typename T, int NT>
__device__ __forceinline__ void grad_columns(const DistillParams &p, i64 row, i64 c0, i64 c1, MaxSum a, float mass, float gt, const ListLds &list) {
    constexpr int N = VecOf<T>::N, U = 4;
    const int tid = threadIdx.x;
    const T *z = (const T *)p.student + row * p.ld_student;
    T *d = (T *)p.grad + row * p.ld_grad;
    if (mass == 0.f) {
        RawVec<T, N> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = (T)0.f;
        i64 i = c0 + (i64)tid * N;
        for (; i + N <= c1; i += NT * N) vec_store<T, N>(d + i, o);
        for (int j = 0; j < N; ++j)
            if (i + j < c1) d[i + j] = (T)0.f;
        return;
    }
    const Exponent x = exponent_of(a.m, p.c);
    const float coef = a.s == 0.f ? 0.f : gt * mass / a.s * correction_of(a.m, x);       // (a row of -inf only has q = 0)
    auto one = [&](float v) { return coef * exp2_fast(__fmaf_rn(v, x.c, -x.off)); };
    i64 i = c0 + (i64)tid * N;
    for (; i + (U - 1) * NT * N + N <= c1; i += U * NT * N) {
        RawVec<T, N> y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) y[u] = vec_load<T, N>(z + i + u * NT * N);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            RawVec<T, N> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.v[j] = (T)one(up(y[u].v[j]));
            vec_store<T, N>(d + i + u * NT * N, o);
        }
    }
    for (; i + N <= c1; i += NT * N) {
        const RawVec<T, N> y = vec_load<T, N>(z + i);
        RawVec<T, N> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = (T)one(up(y.v[j]));
        vec_store<T, N>(d + i, o);
    }
    for (int j = 0; j < N; ++j)
        if (i + j < c1) d[i + j] = (T)one(up(z[i + j]));
    write_listed(p.k, d, one, gt, list);
}

template <typename T, int NT> __global__ __launch_bounds__(NT) void sp_distill_grad_kernel(DistillParams p) {
    __shared__ float mass;
    const ListLds list(distill_list, p.k);
    const i64 row = blockIdx.x / p.splits, c0 = (blockIdx.x % p.splits) * p.chunk, c1 = min(p.n_cols, c0 + p.chunk);
    if (threadIdx.x < 64) {
        const ListSums l = list_sums<T>(p, row, (const T *)p.student + row * p.ld_student, list);
        chain_listed<NT, VecOf<T>::N>(p.k, c0, c1, c1, list);
        if (threadIdx.x == 0) mass = l.mass;
    }
    const MaxSum a{p.stats[2 * row], p.stats[2 * row + 1]};
    const float gt = (p.grad_loss ? p.grad_loss[row] : 1.f) * p.tau;
    __syncthreads();                                           // (every listed score has been read: `grad` may be `student`)
    grad_columns<T, NT>(p, row, c0, c1, a, mass, gt, list);
}

// what the compiler has derived from a vector is to be derived again
template <typename T, int N> __device__ __forceinline__ void forget(RawVec<T, N> &x) {
    typedef unsigned Quad __attribute__((ext_vector_type(4)));
    Quad q;
    __builtin_memcpy(&q, &x, 16);
    asm volatile("" : "+v"(q));
    __builtin_memcpy(&x, &q, 16);
}

// Loss and gradient of a row by one workgroup that keeps the row: RV vectors of 16 bytes per thread in registers, `stage` more per
// workgroup in LDS; only what is left of a still longer row is read a second time.  The sums are formed while vectors arrive, the gradient
// while they leave; several workgroups share a CU where the row allows it, so that one loads while another stores.
template <typename T, int NT, int RV> __global__ __launch_bounds__(NT, RV <= 4 ? 8 : 4) void sp_distill_loss_grad_kernel(DistillParams p) {
    constexpr int N = VecOf<T>::N, M = 16 / N;                 // M vectors, 16 scores, are added at once
    __shared__ MaxSum sh[NT / 64];
    __shared__ float mass_of_row;
    const ListLds list(distill_list, p.k);
    RawVec<T, N> *stage = (RawVec<T, N> *)(distill_list + 4 * ListLds::room(p.k) + NT);
    const i64 row = blockIdx.x;
    const int tid = threadIdx.x, n_cols = (int)p.n_cols, vecs = n_cols / N;
    const int kept = min(vecs, RV * NT + p.stage);             // vectors that are not read again
    const T *z = (const T *)p.student + row * p.ld_student;
    T *d = (T *)p.grad + row * p.ld_grad;

    ListSums l{0.f, 0.f};
    if (tid < 64) {                                            // (one wave is a little late; what it does is in nobody's way then)
        l = list_sums<T>(p, row, z, list);
        chain_listed<NT, N>(p.k, 0, n_cols, (i64)vecs * N, list);
        if (tid == 0) mass_of_row = l.mass;
    }
    RawVec<T, N> x[RV];
#pragma unroll
    for (int q = 0; q < RV; ++q) {
        const int j = q * NT + tid;
        if (j < vecs) x[q] = vec_load<T, N>(z + (i64)j * N);
        else {
#pragma unroll
            for (int e = 0; e < N; ++e) x[q].v[e] = (T)NEG_INF;          // (adds nothing)
        }
    }
    Running run{NEG_INF, NEG_INF, 0.f};
    for (int j = RV * NT + tid; j < vecs; j += NT) {
        const RawVec<T, N> y = vec_load<T, N>(z + (i64)j * N);
        if (j < kept) stage[j - RV * NT] = y;
        float v[N];
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = up(y.v[e]);
        add_vec<N>(run, v, p.c);
    }
    const int end = vecs * N + tid;                            // fewer than N columns behind the last vector
    const float lone = end < n_cols ? up(z[end]) : NEG_INF;
    add_vec<1>(run, &lone, p.c);
#pragma unroll
    for (int q = 0; q < RV; q += M) {
        if (q * NT >= vecs) break;
        float v[16];
#pragma unroll
        for (int u = 0; u < M; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) v[u * N + e] = up(x[q + u].v[e]);
        add_vec<16>(run, v, p.c);
    }
    MaxSum a = block_join<NT>(finish(run, p.c), p.c, sh);
    if (!off_fits(a.m, p.c)) a = rescan<T, NT>(z, 0, n_cols, a, p.c, sh);
    // (the barrier in block_join: the row and the listed scores have been read; from here on `grad` is written, which may be `student`)
#pragma unroll
    for (int q = 0; q < RV; ++q) forget(x[q]);                 // (or the scores stay unpacked in registers, which there are not enough of)
    const float mass = mass_of_row, gt = (p.grad_loss ? p.grad_loss[row] : 1.f) * p.tau;
    const Exponent ex = exponent_of(a.m, p.c);
    const bool some = mass != 0.f;                             // (a row whose list has no mass gets zeros, whatever its scores hold)
    const float coef = a.s == 0.f || !some ? 0.f : gt * mass / a.s * correction_of(a.m, ex);
    auto one = [&](float v) { return some ? coef * exp2_fast(__fmaf_rn(v, ex.c, -ex.off)) : 0.f; };
    auto put = [&](int j, const RawVec<T, N> &y) {
        RawVec<T, N> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = (T)one(up(y.v[e]));
        vec_store<T, N>(d + (i64)j * N, o);
    };
    // (what has to be read again goes first: nothing of it has been written yet)
    for (int j = RV * NT + tid; j < vecs; j += NT)
        if (j >= kept) put(j, vec_load<T, N>(z + (i64)j * N));
#pragma unroll
    for (int q = 0; q < RV; ++q)
        if (q * NT + tid < vecs) put(q * NT + tid, x[q]);
    for (int j = RV * NT + tid; j < kept; j += NT) put(j, stage[j - RV * NT]);
    if (end < n_cols) d[end] = (T)one(lone);
    write_listed(p.k, d, one, gt, list);
    if (tid < 64 && p.loss) {
        const float loss = list_loss(p, l, a, list);
        if (tid == 0) p.loss[row] = loss;
    }
}

}  // namespace
