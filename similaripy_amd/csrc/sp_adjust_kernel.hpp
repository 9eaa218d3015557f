// sp_adjust_kernel.hpp — penalties for repeated ids, biases and masks on rows of dense scores.
//
//   y = s;  listed c > 0 times in the history: y = (y > 0 ? y / r : y * r) - presence - frequency * c
//   y += bias;  y = -inf in masked columns
// The lists are the sparse product's selectors (similaripy/cython_code/s_plus.h:159-188 looks every candidate up in its row's
// list); here the row is dense, so the lookup is turned round: a workgroup first writes what the row's lists say about its segment
// of columns into LDS and then streams the segment past it without a barrier.  Two bits per column (masked, listed in the history) are
// all that most columns need; the count of a listed column is in a hash table.  A history with more entries in the segment than the
// table holds is counted column by column instead, a tile at a time in the table's memory.  Lists need no order, and a column
// listed several times is counted exactly (integer LDS adds: their order does not matter).
#pragma once
#include <type_traits>

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
    int segs, seg;             // segments of a row, their columns
};

constexpr int AD_NT = 256;     // threads of a workgroup

__device__ __forceinline__ i64 list_length(const CsrPattern &m, i64 r) {
    return r < 0 || r >= m.n_rows ? 0 : load_index(m.indptr, m.index64, r + 1) - load_index(m.indptr, m.index64, r);
}
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

constexpr int AD_SEG = 32768;      // most columns of a segment: 4 KB of LDS for each kind of bit
constexpr int AD_SLOTS = 2048;     // slots of the hash table {column, count}: 16 KB
constexpr int AD_HASHED = 1536;    // entries it takes; more are counted in tiles of 2 * AD_SLOTS columns

__device__ __forceinline__ unsigned ad_slot(int c) { return ((unsigned)c * 2654435761u) >> (32 - 11); }
static_assert(AD_SLOTS == 1 << 11, "ad_slot");

template <typename T, int N> __device__ __forceinline__ void add_bias(float *y, const void *p, i64 at) {
    const RawVec<T, N> r = vec_load<T, N>((const T *)p + at);
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] += up(r.v[j]);
}

// One workgroup per segment of a row
template <typename T, bool COUNTS> __global__ __launch_bounds__(AD_NT) void sp_adjust_kernel(AdjustParams p) {
    constexpr int N = VecOf<T>::N, U = 4;
    __shared__ unsigned gone[AD_SEG / 32];                     // masked by filter or target lists
    __shared__ unsigned hit[COUNTS ? AD_SEG / 32 : 1];         // listed in the history
    __shared__ unsigned table[COUNTS ? 2 * AD_SLOTS : 1];      // hash: columns, then counts; tiles: counts
    __shared__ int n_hits;
    const i64 row = blockIdx.x / p.segs, c0 = (i64)(blockIdx.x % p.segs) * p.seg;
    const int width = (int)min((i64)p.seg, p.n_cols - c0), tid = threadIdx.x;
    const T *in = (const T *)p.scores + row * p.ld_scores + c0;
    T *out = (T *)p.out + row * p.ld_out + c0;
    // the segment's first scores are requested before the lists are looked at: their latency covers the lists'
    RawVec<T, N> first[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if ((u * AD_NT + tid) * N + N <= width) first[u] = vec_load<T, N>(in + (u * AD_NT + tid) * N);
    const bool lists = p.filter.indptr != nullptr || p.target.indptr != nullptr;
    const i64 r = p.targets ? load_index(p.targets, p.targets64, row) : row;
    for (int i = tid; i < p.seg / 32; i += AD_NT) {
        if (lists) gone[i] = p.target.indptr ? ~0u : 0u;
        if (COUNTS) hit[i] = 0u;
    }
    if (COUNTS) {
        for (int i = tid; i < AD_SLOTS; i += AD_NT) {
            table[i] = ~0u;
            table[AD_SLOTS + i] = 0u;
        }
        if (tid == 0) n_hits = 0;
    }
    __syncthreads();
    if (p.target.indptr) {
        scan_list(p.target, r, c0, width, [&](int c) { atomicAnd(&gone[c >> 5], ~(1u << (c & 31))); });
        if (p.filter.indptr) __syncthreads();
    }
    if (p.filter.indptr) scan_list(p.filter, r, c0, width, [&](int c) { atomicOr(&gone[c >> 5], 1u << (c & 31)); });
    bool hashed = true;
    if (COUNTS) {
        auto insert = [&](int c) {
            unsigned h = ad_slot(c);
            for (;;) {                                         // (at most AD_HASHED of AD_SLOTS are taken: there is a free one)
                const unsigned was = atomicCAS(&table[h], ~0u, (unsigned)c);
                if (was == ~0u || was == (unsigned)c) break;
                h = (h + 1) & (AD_SLOTS - 1);
            }
            atomicAdd(&table[AD_SLOTS + h], 1u);
        };
        if (list_length(p.history, r) <= AD_HASHED)
            scan_list(p.history, r, c0, width, [&](int c) { atomicOr(&hit[c >> 5], 1u << (c & 31)); insert(c); });
        else {                                                 // a long history: how much of it lies in this segment decides
            int mine = 0;
            scan_list(p.history, r, c0, width, [&](int c) { atomicOr(&hit[c >> 5], 1u << (c & 31)); ++mine; });
            if (mine) atomicAdd(&n_hits, mine);
            __syncthreads();
            hashed = n_hits <= AD_HASHED;
            if (hashed) scan_list(p.history, r, c0, width, insert);
        }
    }
    __syncthreads();
    const float rep = COUNTS && p.repetition ? p.repetition[row] : p.repetition_all;
    const float pres = COUNTS && p.presence ? p.presence[row] : p.presence_all;
    const float freq = COUNTS && p.frequency ? p.frequency[row] : p.frequency_all;
    const unsigned char *bits = p.allowed ? (const unsigned char *)(p.allowed + row * p.ld_allowed) + c0 / 8 : nullptr;
    const i64 bias0 = row * p.ld_bias + c0;

    // N columns from c on: what becomes of their scores.  tile >= 0: the count of column c is table[c - tile]
    auto adjust = [&](auto nc, float *y, int c, int tile) {
        constexpr int M = decltype(nc)::value;
        if (COUNTS) {
            const unsigned listed = (hit[c >> 5] >> (c & 31)) & ((1u << M) - 1u);
            if (listed) {
#pragma unroll
                for (int j = 0; j < M; ++j)
                    if ((listed >> j) & 1u) {
                        unsigned n;
                        if (tile >= 0) n = table[c + j - tile];
                        else {
                            unsigned h = ad_slot(c + j);
                            while (table[h] != (unsigned)(c + j)) h = (h + 1) & (AD_SLOTS - 1);       // (it is there)
                            n = table[AD_SLOTS + h];
                        }
                        y[j] = (y[j] > 0.f ? y[j] / rep : y[j] * rep) - (pres + freq * (float)n);
                    }
            }
        }
        if (p.bias) {
            if (p.bias_dtype == 0) add_bias<float, M>(y, p.bias, bias0 + c);
            else if (p.bias_dtype == 1) add_bias<__bf16, M>(y, p.bias, bias0 + c);
            else add_bias<_Float16, M>(y, p.bias, bias0 + c);
        }
        unsigned drop = 0;
        if (lists) drop = gone[c >> 5] >> (c & 31);
        if (bits) drop |= ~((unsigned)bits[c >> 3] >> (c & 7));
#pragma unroll
        for (int j = 0; j < M; ++j) y[j] = (drop >> j) & 1u ? NEG_INF : y[j];
    };
    auto stream = [&](int from, int to, int tile) {
        const int whole = to - (to - from) % N;
        RawVec<T, N> x[U];
        for (int base = from + tid * N; base < whole; base += AD_NT * N * U) {
            if (base != tid * N)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (base + u * AD_NT * N < whole) x[u] = vec_load<T, N>(in + base + u * AD_NT * N);
            if (base == tid * N)
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = first[u];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = base + u * AD_NT * N;
                if (c >= whole) break;
                float y[N];
#pragma unroll
                for (int j = 0; j < N; ++j) y[j] = up(x[u].v[j]);
                adjust(std::integral_constant<int, N>(), y, c, tile);
                RawVec<T, N> o;
#pragma unroll
                for (int j = 0; j < N; ++j) o.v[j] = (T)y[j];
                vec_store<T, N>(out + c, o);
            }
        }
        if (whole + tid < to) {                                // fewer than N columns at the end of the row
            float y = up(in[whole + tid]);
            adjust(std::integral_constant<int, 1>(), &y, whole + tid, tile);
            out[whole + tid] = (T)y;
        }
    };
    if (!COUNTS || hashed) {
        stream(0, width, -1);
        return;
    }
    for (int from = 0; from < width; from += 2 * AD_SLOTS) {
        const int n = min(2 * AD_SLOTS, width - from);
        __syncthreads();                                       // (the tile before has been read)
        for (int i = tid; i < n; i += AD_NT) table[i] = 0u;
        __syncthreads();
        scan_list(p.history, r, c0 + from, n, [&](int c) { atomicAdd(&table[c], 1u); });
        __syncthreads();
        stream(from, from + n, from);
    }
}

}  // namespace
