// sp_embed_kernels.hpp — rows of a CSR times an embedding table, and the gradient of the table.
//
//   out[i, :]  = scale * sum_{j in row i} w_j T[id_j, :]            (a lookup: row i holds entry i alone)
//   dT[v, :]   = scale * sum_{j: id_j = v} w_j dO[row of j, :]      in ascending j
//
// Both are gathers of whole rows: a group of lanes takes 16 bytes per lane of one row, so that a row is one coalesced access, and
// requests several rows before it adds the first.  Nothing is added with atomics.
#pragma once
#include "sp_dense_common.hpp"

namespace {

struct EmbedParams {
    const void *in;
    const void *indices, *indptr;
    const float *data;
    void *out;
    i64 n_rows, n_vocab, nnz, ld_in, ld_out;
    int dim, index64, accumulate;
    float scale;
    int slabs;              // column slabs of a row: ceil(dim / (G * N))
};

// N elements at column c of a row of `dim`, in 32 bits; beyond the row 0
template <typename T, int N> struct Piece {
    RawVec<T, N> r;
    __device__ __forceinline__ void load(const T *row, int c, int dim) {
        if (c + N <= dim) r = vec_load<T, N>(row + c);
        else {
#pragma unroll
            for (int j = 0; j < N; ++j) r.v[j] = c + j < dim ? row[c + j] : (T)0.f;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < N; ++j) r.v[j] = (T)0.f;
    }
};
template <typename T, int N> __device__ __forceinline__ void store_piece(T *row, int c, int dim, const float *v) {
    RawVec<T, N> o;
#pragma unroll
    for (int j = 0; j < N; ++j) o.v[j] = (T)v[j];
    if (c + N <= dim) vec_store<T, N>(row + c, o);
    else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < dim) row[c + j] = o.v[j];
    }
}

// One group of G lanes per row and slab of G * N columns.
template <typename T, typename I, int G> __global__ __launch_bounds__(256) void sp_embed_rows_kernel(EmbedParams p) {
    constexpr int N = VecOf<T>::N, U = 4;
    const int lane = threadIdx.x & (G - 1);
    const i64 item = (i64)blockIdx.x * (256 / G) + threadIdx.x / G;
    const i64 row = item / p.slabs;
    if (row >= p.n_rows) return;
    const int c = ((int)(item % p.slabs) * G + lane) * N;
    if (c >= p.dim) return;
    const I *ids = (const I *)p.indices;
    i64 b = row, e = row + 1;
    if (p.indptr) {
        b = max((i64)0, (i64)((const I *)p.indptr)[row]);
        e = min(p.nnz, (i64)((const I *)p.indptr)[row + 1]);
    }
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    for (i64 i = b; i < e; i += U) {
        Piece<T, N> x[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            i64 id = -1;
            if (i + u < e) id = (i64)ids[i + u];
            const bool ok = id >= 0 && id < p.n_vocab;
            w[u] = !ok ? 0.f : p.data ? p.data[i + u] : 1.f;
            if (ok) x[u].load((const T *)p.in + id * p.ld_in, c, p.dim);
            else x[u].zero();
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = __fmaf_rn(w[u], up(x[u].r.v[j]), acc[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] *= p.scale;
    store_piece<T, N>((T *)p.out + row * p.ld_out, c, p.dim, acc);
}

// ---- the gradient: entries sorted by id, stably ------------------------------------------------------------------------------
// A radix sort from the low digit: per pass one launch counts the digits of every workgroup's chunk, one moves the entries.  Every
// wave owns a contiguous part of the chunk and goes through it in order; equal digits of 64 entries are ranked by their lane.
// Ids outside the table take the key n_vocab and end up behind everything else.

constexpr int SORT_NT = 512, SORT_WAVES = SORT_NT / 64, SORT_BINS = 512, SORT_WGS = 256;

struct SortParams {
    i64 n;                       // entries
    int chunk;                   // entries of a workgroup (a multiple of SORT_NT)
    int wgs, shift, bits;
    const unsigned *key_in;      // first pass: NULL, the keys are `indices`
    const unsigned *pay_in;
    const float *w_in;
    unsigned *key_out, *pay_out;
    float *w_out;                // NULL without weights
    unsigned *hist;              // [wgs][SORT_BINS]
    const void *indices, *indptr;
    i64 n_rows, n_vocab;
};

template <typename I> __device__ __forceinline__ unsigned sort_key(const SortParams &p, i64 i) {
    if (p.key_in) return p.key_in[i];
    const i64 id = (i64)((const I *)p.indices)[i];
    return id >= 0 && id < p.n_vocab ? (unsigned)id : (unsigned)p.n_vocab;
}

template <typename I> __global__ __launch_bounds__(SORT_NT) void sp_sort_count_kernel(SortParams p) {
    __shared__ unsigned h[SORT_BINS];
    for (int i = threadIdx.x; i < SORT_BINS; i += SORT_NT) h[i] = 0;
    __syncthreads();
    const i64 b = (i64)blockIdx.x * p.chunk, e = min(p.n, b + p.chunk);
    const unsigned mask = (1u << p.bits) - 1u;
    for (i64 i = b + threadIdx.x; i < e; i += SORT_NT) atomicAdd(&h[(sort_key<I>(p, i) >> p.shift) & mask], 1u);
    __syncthreads();
    for (int i = threadIdx.x; i < SORT_BINS; i += SORT_NT) p.hist[(i64)blockIdx.x * SORT_BINS + i] = h[i];
}

// the CSR row of entry i; n_rows for an entry that no row holds
template <typename I> __device__ __forceinline__ i64 row_of(const void *indptr, i64 n_rows, i64 i) {
    i64 lo = 0, hi = n_rows;                 // first r with indptr[r + 1] > i
    while (lo < hi) {
        const i64 mid = (lo + hi) >> 1;
        if ((i64)((const I *)indptr)[mid + 1] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo < n_rows && (i64)((const I *)indptr)[lo] > i ? n_rows : lo;
}
static_assert(SORT_NT == SORT_BINS, "a thread per digit");

template <typename I> __global__ __launch_bounds__(SORT_NT) void sp_sort_move_kernel(SortParams p) {
    __shared__ unsigned off[SORT_WAVES][SORT_BINS];
    __shared__ unsigned wsum[SORT_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned mask = (1u << p.bits) - 1u;
    for (int w = 0; w < SORT_WAVES; ++w) off[w][tid] = 0;
    // entries of digit `tid` before this workgroup: those of smaller digits anywhere, and of its own in the workgroups before
    unsigned before = 0, all = 0;
    for (int g = 0; g < p.wgs; ++g) {
        const unsigned v = p.hist[(i64)g * SORT_BINS + tid];
        before += g < (int)blockIdx.x ? v : 0u;
        all += v;
    }
    unsigned inc = all;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wsum[wave] = inc;
    __syncthreads();
    unsigned base = before + inc - all;
    for (int w = 0; w < wave; ++w) base += wsum[w];
    // digits of every wave's part
    const int per = p.chunk / SORT_WAVES;
    const i64 b = (i64)blockIdx.x * p.chunk + (i64)wave * per, e = min(p.n, b + per);
    for (i64 i = b + lane; i < e; i += 64) atomicAdd(&off[wave][(sort_key<I>(p, i) >> p.shift) & mask], 1u);
    __syncthreads();
    for (int w = 0; w < SORT_WAVES; ++w) {
        const unsigned n = off[w][tid];
        off[w][tid] = base;
        base += n;
    }
    __syncthreads();
    volatile unsigned *mine = off[wave];
    for (i64 i0 = b; i0 < e; i0 += 64) {
        const i64 i = i0 + lane;
        const bool ok = i < e;
        const unsigned key = ok ? sort_key<I>(p, i) : 0u, digit = (key >> p.shift) & mask;
        u64 same = __ballot(ok);
        for (int k = 0; k < p.bits; ++k) {
            const u64 set = __ballot((digit >> k) & 1u);
            same &= (digit >> k) & 1u ? set : ~set;
        }
        if (ok) {
            const unsigned rank = (unsigned)__popcll(same & ((1ull << lane) - 1ull));
            const unsigned at = mine[digit] + rank;
            if (rank == 0) mine[digit] = at + (unsigned)__popcll(same);       // (a wave's LDS accesses keep their order: everybody has read)
            p.key_out[at] = key;
            if (p.key_in) p.pay_out[at] = p.pay_in[i];
            else p.pay_out[at] = p.indptr ? (unsigned)row_of<I>(p.indptr, p.n_rows, i) : (unsigned)i;
            if (p.w_out) p.w_out[at] = p.w_in[i];
        }
    }
}

// every row of the gradient starts at 0
template <typename T> __global__ __launch_bounds__(256) void sp_fill_rows_kernel(T *out, i64 n_rows, i64 dim, i64 ld) {
    constexpr int N = VecOf<T>::N;
    RawVec<T, N> z;
#pragma unroll
    for (int j = 0; j < N; ++j) z.v[j] = (T)0.f;
    const i64 first = ((i64)blockIdx.x * 256 + threadIdx.x) * N, step = (i64)gridDim.x * 256 * N;
    if (ld == dim || n_rows == 1) {
        const i64 total = n_rows * dim;
        i64 i = first;
        for (; i + N <= total; i += step) vec_store<T, N>(out + i, z);
        for (int j = 0; j < N; ++j)
            if (i + j < total) out[i + j] = (T)0.f;
    } else {
        for (i64 r = blockIdx.x; r < n_rows; r += gridDim.x)
            for (i64 c = threadIdx.x; c < dim; c += 256) out[r * ld + c] = (T)0.f;
    }
}

struct ReduceParams {
    const void *in;
    void *out;
    const unsigned *key, *pay;
    const float *w;             // NULL: ones
    float *part;                // [chunks][2][dim]: sums of the runs that cross a chunk's first and last entry
    i64 n, n_vocab, ld_in, ld_out, n_rows;
    i64 chunks;
    int chunk, dim, slabs, accumulate;
    float scale;
};

template <typename TO, int N> __device__ __forceinline__ void write_row(const ReduceParams &p, unsigned key, int c, float *acc) {
    TO *row = (TO *)p.out + (i64)key * p.ld_out;
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] *= p.scale;
    if (p.accumulate) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < p.dim) acc[j] += up(row[c + j]);
    }
    store_piece<TO, N>(row, c, p.dim, acc);
}

// One group of G lanes per chunk of the sorted entries and slab of columns: runs of equal ids are summed as they come.  A run that
// lies inside the chunk is a row of the gradient and is written; one that began before or goes on behind it leaves its sum in `part`.
template <typename T, typename TO, int G> __global__ __launch_bounds__(256) void sp_embed_reduce_kernel(ReduceParams p) {
    constexpr int N = VecOf<T>::N, U = 4;
    const int lane = threadIdx.x & (G - 1);
    const i64 item = (i64)blockIdx.x * (256 / G) + threadIdx.x / G;
    const i64 ch = item / p.slabs;
    if (ch >= p.chunks) return;
    const int c = ((int)(item % p.slabs) * G + lane) * N;
    if (c >= p.dim) return;
    const i64 b = ch * p.chunk, e = min(p.n, b + p.chunk);
    const unsigned none = (unsigned)p.n_vocab;
    const unsigned prev = b > 0 ? p.key[b - 1] : none, next = e < p.n ? p.key[e] : none;
    unsigned run = p.key[b];
    bool head = b > 0 && run == prev;
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    auto flush = [&](bool last) {
        if (run == none) return;
        float *slot = nullptr;
        if (head) slot = p.part + (2 * ch) * p.dim;
        else if (last && next == run && e < p.n) slot = p.part + (2 * ch + 1) * p.dim;
        if (slot) store_piece<float, N>(slot, c, p.dim, acc);
        else write_row<TO, N>(p, run, c, acc);
    };
    for (i64 i = b; i < e; i += U) {
        Piece<T, N> x[U];
        float w[U];
        unsigned k[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = none;
            w[u] = 0.f;
            if (i + u < e) k[u] = p.key[i + u];
            const unsigned r = k[u] != none ? p.pay[i + u] : 0u;
            const bool ok = k[u] != none && (i64)r < p.n_rows;
            if (ok) {
                w[u] = p.w ? p.w[i + u] : 1.f;
                x[u].load((const T *)p.in + (i64)r * p.ld_in, c, p.dim);
            } else x[u].zero();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= e) break;
            if (k[u] != run) {
                flush(false);
                run = k[u];
                head = false;
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] = __fmaf_rn(w[u], up(x[u].r.v[j]), acc[j]);
        }
    }
    flush(true);
}

// Runs over several chunks: the group of the chunk in which a run begins adds up its parts, in order, and writes the row.
template <typename TO, int N, int G> __global__ __launch_bounds__(256) void sp_embed_join_kernel(ReduceParams p) {
    const int lane = threadIdx.x & (G - 1);
    const i64 item = (i64)blockIdx.x * (256 / G) + threadIdx.x / G;
    const i64 ch = item / p.slabs;
    if (ch + 1 >= p.chunks) return;
    const int c = ((int)(item % p.slabs) * G + lane) * N;
    if (c >= p.dim) return;
    const i64 b = ch * p.chunk, e = b + p.chunk;               // (not the last chunk: it is full, and key[e] exists)
    const unsigned run = p.key[e - 1];
    if (run == (unsigned)p.n_vocab || p.key[e] != run) return;                              // nothing goes on behind it
    if (p.key[b] == run && b > 0 && p.key[b - 1] == run) return;                            // the run began before this chunk
    float acc[N];
    Piece<float, N> x;
    x.load(p.part + (2 * ch + 1) * p.dim, c, p.dim);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = x.r.v[j];
    for (i64 k = ch + 1; k < p.chunks; ++k) {
        x.load(p.part + (2 * k) * p.dim, c, p.dim);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += x.r.v[j];
        const i64 last = min(p.n, (k + 1) * (i64)p.chunk);
        if (p.key[last - 1] != run || last >= p.n || p.key[last] != run) break;
    }
    write_row<TO, N>(p, run, c, acc);
}

}  // namespace
