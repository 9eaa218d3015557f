// sp_adjust_kernel.hpp — penalties for repeated ids, biases and masks on rows of dense scores.
//
//   y = s;  listed c > 0 times in the history: y = (y > 0 ? y / r : y * r) - presence - frequency * c
//   y += bias;  y = -inf in masked columns
// The lists are the sparse product's selectors (similaripy/cython_code/s_plus.h:159-188 looks every candidate up in its row's
// list); here the row is dense, so the lookup is turned round: the workgroup of a tile of columns writes what the row's lists
// say about its columns into LDS (a counter, a bit) and then streams the tile past it.  Lists need no order, and a column
// listed several times is counted exactly (integer LDS adds: their order does not matter).
#pragma once
#include "sp_dense_common.hpp"

namespace {

struct CsrPattern {
    const void *indptr, *indices;
    i64 n_rows, nnz;
    int index64;
};

struct AdjustParams {
    const void *scores;
    void *out;
    i64 n_rows, n_cols, ld_scores, ld_out;
    const void *targets;
    int targets64, bias_dtype;
    CsrPattern history, filter, target;
    const float *repetition, *presence, *frequency;
    float repetition_all, presence_all, frequency_all;
    const void *bias;
    i64 ld_bias;
    const uint32_t *allowed;
    i64 ld_allowed;
    int tiles;                 // tiles of a row
};

constexpr int AD_NT = 256;     // threads of a workgroup

// calls f(column - c0) for the ids of row r that lie in [c0, c0 + width)
template <typename F> __device__ __forceinline__ void scan_list(const CsrPattern &m, i64 r, i64 c0, int width, F f) {
    if (r < 0 || r >= m.n_rows) return;
    i64 b = load_index(m.indptr, m.index64, r), e = load_index(m.indptr, m.index64, r + 1);
    b = b < 0 ? 0 : b;
    e = e > m.nnz ? m.nnz : e;
    for (i64 i = b + threadIdx.x; i < e; i += AD_NT) {
        const i64 c = load_index(m.indices, m.index64, i) - c0;
        if (c >= 0 && c < width) f((int)c);
    }
}

// One workgroup per tile of AD_NT * N * U columns of a row (N elements of 16 bytes, U vectors per thread).  The tile's scores are
// requested before the lists are looked at: their latency covers the lists'.
template <typename T, int U, bool COUNTS>
__global__ __launch_bounds__(AD_NT) void sp_adjust_kernel(AdjustParams p) {
    constexpr int N = VecOf<T>::N, TILE = AD_NT * N * U;
    __shared__ unsigned count[COUNTS ? TILE : 1];
    __shared__ unsigned gone[TILE / 32];                       // masked by filter or target lists
    const i64 row = blockIdx.x / p.tiles, c0 = (i64)(blockIdx.x % p.tiles) * TILE;
    const int width = (int)min((i64)TILE, p.n_cols - c0), tid = threadIdx.x;
    const T *in = (const T *)p.scores + row * p.ld_scores + c0;
    T *out = (T *)p.out + row * p.ld_out + c0;
    RawVec<T, N> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = (u * AD_NT + tid) * N;
        if (c + N <= width) x[u] = vec_load<T, N>(in + c);
        else
            for (int j = 0; j < N; ++j) x[u].v[j] = c + j < width ? in[c + j] : (T)0.f;
    }
    const bool lists = p.filter.indptr != nullptr || p.target.indptr != nullptr;
    const i64 r = p.targets ? load_index(p.targets, p.targets64, row) : row;
    if (COUNTS)
        for (int i = tid; i < TILE; i += AD_NT) count[i] = 0;
    if (lists)
        for (int i = tid; i < TILE / 32; i += AD_NT) gone[i] = p.target.indptr ? ~0u : 0u;
    __syncthreads();
    if (COUNTS) scan_list(p.history, r, c0, width, [&](int c) { atomicAdd(&count[c], 1u); });
    if (p.target.indptr) {
        scan_list(p.target, r, c0, width, [&](int c) { atomicAnd(&gone[c >> 5], ~(1u << (c & 31))); });
        __syncthreads();
    }
    if (p.filter.indptr) scan_list(p.filter, r, c0, width, [&](int c) { atomicOr(&gone[c >> 5], 1u << (c & 31)); });
    __syncthreads();
    const float rep = p.repetition ? p.repetition[row] : p.repetition_all;
    const float pres = p.presence ? p.presence[row] : p.presence_all;
    const float freq = p.frequency ? p.frequency[row] : p.frequency_all;
    const unsigned char *bits = p.allowed ? (const unsigned char *)(p.allowed + row * p.ld_allowed) + c0 / 8 : nullptr;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = (u * AD_NT + tid) * N;
        if (c >= width) continue;
        float y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = up(x[u].v[j]);
        if (COUNTS) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const unsigned n = count[c + j];
                if (n) y[j] = (y[j] > 0.f ? y[j] / rep : y[j] * rep) - (pres + freq * (float)n);
            }
        }
        if (p.bias) {
            const i64 b = row * p.ld_bias + c0 + c;
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (c + j < width) y[j] += load_scalar(p.bias, p.bias_dtype, b + j);
        }
        unsigned drop = 0;
        if (lists) drop = (gone[c >> 5] >> (c & 31)) & ((1u << N) - 1u);
        if (bits) drop |= ~((unsigned)bits[c >> 3] >> (c & 7));
        RawVec<T, N> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = (T)((drop >> j) & 1u ? NEG_INF : y[j]);
        if (c + N <= width) vec_store<T, N>(out + c, o);
        else
            for (int j = 0; j < N; ++j)
                if (c + j < width) out[c + j] = o.v[j];
    }
}

}  // namespace
