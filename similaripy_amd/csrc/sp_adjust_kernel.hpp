// sp_adjust_kernel.hpp — penalties for repeated ids, biases and masks on rows of dense scores.
//
//   y = s;  listed c > 0 times in the history: y = (y > 0 ? y / r : y * r) - presence - frequency * c
//   y += bias;  y = -inf in masked columns
// The lists are the sparse product's selectors (similaripy/cython_code/s_plus.h:159-188 looks every candidate up in its row's
// list); here the row is dense, so the lookup is turned round: a workgroup first writes what the row's lists say about its segment
// of columns into LDS and then streams the segment past it without a barrier.  Two bits per column (masked, listed in the history) are
// all that most columns need; the count of a listed column is in a hash table.  A history with more columns in the segment than the
// table holds is counted column by column instead, a tile at a time in the table's memory.  Lists need no order, and a column
// listed several times is counted exactly (integer LDS adds: their order does not matter).
//
// Measured: 512 x 100 000 bf16 with a history and a filter of 144 entries and a float32 bias 52 us; 1021 x 84 431 f16 with 1000 target
// columns, 64 filtered ones and packed bits 86 us.  The same rows without lists and bias move at 5.9 TB/s (34.4 us; torch's copy of them takes 36.1) and
// 5.0 TB/s (69 us):
// the bias costs 11 us (as many bytes again, from L2), the lists the rest, in registers and in the start of every workgroup.  Long histories are
// bound by the instructions of listed columns, which a wave executes for its lane with the most of them: 231 us with 4000 entries a row.  Writing the
// listed columns once more after the stream instead was no faster for 144 entries a row and twice as slow for 1000.
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

__device__ __forceinline__ i64 uniform(i64 v) {                // a value that all lanes share, in scalar registers
    return (i64)((u64)(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)v) | (u64)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}
// a row's entries of a pattern, and this thread's first one as a column of the segment (-1: none, or outside).  Ranges and first entries of
// all lists are requested before any is used.
struct List {
    i64 b, e;
    int first;
};
__device__ __forceinline__ List list_of(const CsrPattern &m, i64 r) {
    List l{0, 0, -1};
    if (m.indptr != nullptr && r >= 0 && r < m.n_rows) {
        l.b = load_index(m.indptr, m.index64, r);
        l.e = load_index(m.indptr, m.index64, r + 1);
    }
    return l;
}
__device__ __forceinline__ void fetch_first(const CsrPattern &m, List &l, i64 c0, int width) {
    l.b = uniform(l.b < 0 ? 0 : l.b);
    l.e = uniform(l.e > m.nnz ? m.nnz : l.e);
    if (l.b + threadIdx.x < l.e) {
        const i64 c = load_index(m.indices, m.index64, l.b + threadIdx.x) - c0;
        l.first = c >= 0 && c < width ? (int)c : -1;
    }
}
// calls f(column - from) for the ids of a list that lie in the columns [from, from + width) of the segment that starts at c0
template <typename F> __device__ __forceinline__ void scan_list(const CsrPattern &m, const List &l, i64 c0, int from, int width, F f) {
    if (l.first >= from && l.first < from + width) f(l.first - from);
    for (i64 i = l.b + threadIdx.x + AD_NT; i < l.e; i += AD_NT) {
        const i64 c = load_index(m.indices, m.index64, i) - c0 - from;
        if (c >= 0 && c < width) f((int)c);
    }
}

constexpr int AD_SEG = 16384;      // most columns of a segment: 2 KB of LDS for each kind of bit
constexpr int AD_SLOTS = 2048;     // slots of the hash table {column, count}: 16 KB
// Columns it takes (and one more for each thread); more are counted in tiles of 4 * AD_SLOTS columns, 16 bits each, or, of a history that 16 bits
// do not count, of 2 * AD_SLOTS.  A fuller table saves readings of the list and costs longer searches.  (512 / 1024 / 1536, 512 x 100 000 bf16: mean
// histories of 1000 entries 92 / 88 / 84 us, of 4000 231 / 231 / 243; 512 x 10 000 with 2000 entries 59 / 63 / 76.)
constexpr int AD_HASHED = 1024;
static_assert(AD_HASHED + 1 + AD_NT < AD_SLOTS, "a free slot is left");

__device__ __forceinline__ unsigned ad_slot(int c) { return ((unsigned)c * 2654435761u) >> (32 - 11); }
static_assert(AD_SLOTS == 1 << 11, "ad_slot");

template <typename T, int N> __device__ __forceinline__ void load_bias(float *b, const void *p, i64 at) {
    const RawVec<T, N> r = vec_load<T, N>((const T *)p + at);
#pragma unroll
    for (int j = 0; j < N; ++j) b[j] = up(r.v[j]);
}
// N elements of a bias of any type
template <int N> __device__ __forceinline__ void any_bias(float *b, const void *p, int dtype, i64 at) {
    if (dtype == 0) load_bias<float, N>(b, p, at);
    else if (dtype == 1) load_bias<__bf16, N>(b, p, at);
    else load_bias<_Float16, N>(b, p, at);
}

struct Penalty {
    float rep, pres, freq;
    __device__ __forceinline__ float of(float y, unsigned n) const { return (y > 0.f ? y / rep : y * rep) - (pres + freq * (float)n); }
};
__device__ __forceinline__ Penalty penalty_of(const AdjustParams &p, i64 row) {
    return {p.repetition ? p.repetition[row] : p.repetition_all, p.presence ? p.presence[row] : p.presence_all, p.frequency ? p.frequency[row] : p.frequency_all};
}

__device__ __forceinline__ void table_clear(unsigned *table) {
    for (int i = threadIdx.x; i < AD_SLOTS; i += AD_NT) {
        table[i] = ~0u;
        table[AD_SLOTS + i] = 0u;
    }
}
__device__ __forceinline__ bool table_count(unsigned *table, int c) {      // true: a column that was not there
    unsigned h = ad_slot(c), was;
    for (;;) {                                                 // (not all of AD_SLOTS are taken)
        was = atomicCAS(&table[h], ~0u, (unsigned)c);
        if (was == ~0u || was == (unsigned)c) break;
        h = (h + 1) & (AD_SLOTS - 1);
    }
    atomicAdd(&table[AD_SLOTS + h], 1u);
    return was == ~0u;
}
__device__ __forceinline__ unsigned table_find(const unsigned *table, int c) {      // 0: not there
    unsigned h = ad_slot(c);
    for (;;) {
        const unsigned at = table[h];
        if (at == (unsigned)c) return table[AD_SLOTS + h];
        if (at == ~0u) return 0u;
        h = (h + 1) & (AD_SLOTS - 1);
    }
}

// One workgroup per segment of a row
template <typename T, bool COUNTS> __global__ __launch_bounds__(AD_NT) void sp_adjust_kernel(AdjustParams p) {
    constexpr int N = VecOf<T>::N, U = 1;      // vectors in flight per thread: occupancy does more than depth (1: 54 / 86 us, 2: 55 / 90, 4: 62 / 115 for the two shapes above, as first measured)
    __shared__ unsigned gone[AD_SEG / 32];                     // masked by filter or target lists
    __shared__ unsigned hit[COUNTS ? AD_SEG / 32 : 1];         // listed in the history
    __shared__ unsigned table[COUNTS ? 2 * AD_SLOTS : 1];      // hash: columns, then counts; tiles: counts
    __shared__ int n_hits;
    const i64 row = blockIdx.x / p.segs, c0 = (i64)(blockIdx.x % p.segs) * p.seg;
    const int width = (int)min((i64)p.seg, p.n_cols - c0), tid = threadIdx.x;
    const T *in = (const T *)p.scores + row * p.ld_scores + c0;
    T *out = (T *)p.out + row * p.ld_out + c0;
    const bool lists = p.filter.indptr != nullptr || p.target.indptr != nullptr, sparse = p.target.indptr != nullptr;
    const i64 r = uniform(p.targets ? load_index(p.targets, p.targets64, row) : row);
    List history, filter = list_of(p.filter, r), target = list_of(p.target, r);
    if (COUNTS) history = list_of(p.history, r);
    fetch_first(p.filter, filter, c0, width);
    fetch_first(p.target, target, c0, width);
    if (COUNTS) fetch_first(p.history, history, c0, width);
    for (int i = tid; i < p.seg / 32; i += AD_NT) {
        if (lists) gone[i] = p.target.indptr ? ~0u : 0u;
        if (COUNTS) hit[i] = 0u;
    }
    if (COUNTS) {
        table_clear(table);
        if (tid == 0) n_hits = 0;
    }
    __syncthreads();
    if (p.target.indptr) {
        scan_list(p.target, target, c0, 0, width, [&](int c) { atomicAnd(&gone[c >> 5], ~(1u << (c & 31))); });
        if (p.filter.indptr) __syncthreads();
    }
    if (p.filter.indptr) scan_list(p.filter, filter, c0, 0, width, [&](int c) { atomicOr(&gone[c >> 5], 1u << (c & 31)); });
    bool hashed = true;                                        // else the counts are taken tile by tile
    const bool narrow = COUNTS && history.e - history.b <= 0xFFFF;
    if (COUNTS) {
        if (history.e - history.b <= AD_HASHED)
            scan_list(p.history, history, c0, 0, width, [&](int c) { atomicOr(&hit[c >> 5], 1u << (c & 31)); table_count(table, c); });
        else {                                                 // a long history: how many columns of this segment are in it decides
            scan_list(p.history, history, c0, 0, width, [&](int c) {
                atomicOr(&hit[c >> 5], 1u << (c & 31));
                if (*(volatile int *)&n_hits <= AD_HASHED && table_count(table, c)) atomicAdd(&n_hits, 1);
            });
            __syncthreads();
            hashed = n_hits <= AD_HASHED;
        }
    }
    __syncthreads();
    const Penalty pen = penalty_of(p, row);
    const unsigned char *bits = p.allowed ? (const unsigned char *)(p.allowed + row * p.ld_allowed) + c0 / 8 : nullptr;
    const i64 bias0 = row * p.ld_bias + c0;

    // N columns from c on: what becomes of their scores, with their biases and the byte of `allowed` that holds column c.  tile >= 0: the counts are those of a tile
    auto adjust = [&](auto nc, float *y, const float *bias, unsigned allow, int c, int tile) {
        constexpr int M = decltype(nc)::value;
        if (COUNTS) {
            // (a loop over the listed columns, hardly ever more than one: written out for each of the M it doubles the kernel's registers)
            for (unsigned listed = (hit[c >> 5] >> (c & 31)) & ((1u << M) - 1u); listed; listed &= listed - 1u) {
                const int at = __builtin_ctz(listed);
                float v = y[0];
#pragma unroll
                for (int j = 1; j < M; ++j) v = at == j ? y[j] : v;
                const int t = c + at - tile;
                v = pen.of(v, tile < 0 ? table_find(table, c + at) : narrow ? table[t >> 1] >> (t & 1) * 16 & 0xFFFFu : table[t]);
#pragma unroll
                for (int j = 0; j < M; ++j) y[j] = at == j ? v : y[j];
            }
        }
        if (p.bias) {
#pragma unroll
            for (int j = 0; j < M; ++j) y[j] += bias[j];
        }
        unsigned drop = ~(allow >> (c & 7));
        if (lists) drop |= gone[c >> 5] >> (c & 31);
#pragma unroll
        for (int j = 0; j < M; ++j) {
            const unsigned all = (unsigned)__builtin_amdgcn_sbfe((int)drop, j, 1);       // the bit, all over the word
            y[j] = __uint_as_float((all & 0xFF800000u) | (~all & __float_as_uint(y[j])));
        }
    };
    auto stream = [&](int from, int to, int tile) {
        const int whole = to - (to - from) % N;
        for (int base = from + tid * N; base < whole; base += AD_NT * N * U) {
            RawVec<T, N> x[U];
            float bias[U][N];
            unsigned allow[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = base + u * AD_NT * N;
                if (c < whole && !(sparse && !((~gone[c >> 5] >> (c & 31)) & ((1u << N) - 1u)))) x[u] = vec_load<T, N>(in + c);
                allow[u] = bits && c < whole ? bits[c >> 3] : 0xFFu;
            }
            if (p.bias)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (base + u * AD_NT * N < whole) any_bias<N>(bias[u], p.bias, p.bias_dtype, bias0 + base + u * AD_NT * N);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = base + u * AD_NT * N;
                if (c >= whole) break;
                float y[N];
#pragma unroll
                for (int j = 0; j < N; ++j) y[j] = up(x[u].v[j]);
                adjust(std::integral_constant<int, N>(), y, bias[u], allow[u], c, tile);
                RawVec<T, N> o;
#pragma unroll
                for (int j = 0; j < N; ++j) o.v[j] = (T)y[j];
                vec_store<T, N>(out + c, o);
            }
        }
        if (whole + tid < to) {                                // fewer than N columns at the end of the row
            const int c = whole + tid;
            float y = up(in[c]), bias = 0.f;
            if (p.bias) any_bias<1>(&bias, p.bias, p.bias_dtype, bias0 + c);
            adjust(std::integral_constant<int, 1>(), &y, &bias, bits ? bits[c >> 3] : 0xFFu, c, tile);
            out[c] = (T)y;
        }
    };
    // one tile, the whole segment, unless the counts of a long history are taken tile by tile
    if (!COUNTS) {
        stream(0, width, -1);
        return;
    }
    const int step = hashed ? AD_SEG : narrow ? 4 * AD_SLOTS : 2 * AD_SLOTS;
    for (int from = 0; from < width; from += step) {
        const int to = min(from + step, width);
        if (!hashed) {
            __syncthreads();                                   // (the tile before has been read)
            for (int i = tid; i < 2 * AD_SLOTS; i += AD_NT) table[i] = 0u;
            __syncthreads();
            if (narrow) scan_list(p.history, history, c0, from, to - from, [&](int c) { atomicAdd(&table[c >> 1], 1u << (c & 1) * 16); });
            else scan_list(p.history, history, c0, from, to - from, [&](int c) { atomicAdd(&table[c], 1u); });
            __syncthreads();
        }
        stream(from, to, hashed ? -1 : from);
    }
}

}  // namespace
