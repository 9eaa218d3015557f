// sp_embed_kernels.hpp — rows of a CSR times an embedding table, and the gradient of the table.
//
//   out[i, :]  = scale * sum_{j in row i} w_j T[id_j, :]            (a lookup: row i holds entry i alone)
//   dT[v, :]   = scale * sum_{j: id_j = v} w_j dO[row of j, :]
//
// The order of the additions depends on the sizes and the entries alone: bags take theirs by groups of lanes whose sums are added as a tree,
// the gradient adds in ascending j within a chunk of the sorted entries and joins the chunks' sums in their order.
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
    int dim;
    float scale;
    int slabs;              // column slabs of a row: ceil(dim / (G * N))
    int by_xcd;             // bags: slab s is the work of the XCDs s, s + slabs, .. (slabs divides 8)
};

// The columns of a lane: N of them from c on, of rows of at least N.  The last lane of a row moves back to the row's last N columns instead
// of taking fewer (it repeats what the lane before it computes, to the same bits), and lanes beyond it read the same ones: every access is
// a whole vector and none is behind a branch.  Rows shorter than a vector of 16 bytes are served with N = 1.
template <int N> struct Columns {
    int own;           // first column that is this lane's alone
    int c;
    bool active;
    __device__ __forceinline__ Columns(int first, int dim) : own(first), c(first > dim - N ? dim - N : first), active(first < dim) {}
};
template <typename T, int N> __device__ __forceinline__ void put(T *p, const float *v) {
    RawVec<T, N> o;
#pragma unroll
    for (int j = 0; j < N; ++j) o.v[j] = (T)v[j];
    vec_store<T, N>(p, o);
}

// value of lane `at` of the group of G lanes
template <int G> __device__ __forceinline__ int group_lane(int v, int at) { return G == 64 ? __builtin_amdgcn_readlane(v, at) : __shfl(v, at, G); }

// Lookup: one group of G lanes per row and slab of G * N columns; HBM bounds it: 16 384 rows of 2 KB, read and written, take 10.9 us
// (6.2 TB/s, some of the rows being read twice).  More waves beat more loads per wave: with two rows per group it is a third slower, with four 40 %.
template <typename T, typename I, int G, int N> __global__ __launch_bounds__(256) void sp_embed_lookup_kernel(EmbedParams p) {
    const int lane = threadIdx.x & (G - 1);
    const i64 item = (i64)blockIdx.x * (256 / G) + threadIdx.x / G;
    const i64 row = item / p.slabs;
    const Columns<N> cols(((int)(item % p.slabs) * G + lane) * N, p.dim);
    if (row >= p.n_rows || !cols.active) return;
    const i64 id = (i64)((const I *)p.indices)[row];
    float v[N];
    if (id >= 0 && id < p.n_vocab) {
        const RawVec<T, N> x = vec_load<T, N>((const T *)p.in + id * p.ld_in + cols.c);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = up(x.v[j]) * p.scale;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = 0.f;
    }
    put<T, N>((T *)p.out + row * p.ld_out + cols.c, v);
}

// Bags: one wave per row and slab.  65 536 bags of 64 out of 100 000 rows of 512 B (Zipf 0.9) read 2.1 GB in 186 us, 11 TB/s (in bf16 197; of 256 B,
// bf16 and fp16, 99 .. 116).  The L2 of an XCD (4 MB) holds 49 % of the lines.  Misses alone do not bound it: cut into four slabs the L2s hold
// 62 %, which takes a quarter of the misses away, but only 6 % of the time; how much of the rest is the latency of a wave's requests has not been
// shown.  A large table of wide rows is cut by columns, so that each XCD works on one slab only and holds that many times more rows of it, unless a
// launch cannot have as many workgroups; few rows are cut so that there are waves enough.  (16 384 bags, rows of 2 KB: 245 -> 182 us with eight slabs;
// 4000 bags, rows of 512 B: 60 -> 27 with four; 65 536 bags: 512 B 186 -> 179, 256 B 103 -> 106, a table of 10 MB 142 -> 154, which is why those stay
// whole.)
// A wave's 64 / G groups take the row's entries in turn; 64 ids and weights are read at once, a lane each, and
// U rows of the table are on their way per group (an id outside the table reads row 0 and adds nothing).
template <typename T, typename I, int G, int N> __global__ __launch_bounds__(256) void sp_embed_rows_kernel(EmbedParams p) {
    constexpr int S = 64 / G, U = 8;
    static_assert(S * U <= 64, "a round stays inside the 64 entries read at once");
    const int lane = threadIdx.x & 63, sub = lane / G, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    i64 row;
    int slab;
    if (p.by_xcd) {                                            // workgroups are dealt to the eight XCDs in turn
        const int xcd = (int)(blockIdx.x % 8);
        slab = xcd % p.slabs;
        row = ((i64)(blockIdx.x / 8) * (8 / p.slabs) + xcd / p.slabs) * 4 + wave;
    } else {
        slab = (int)(blockIdx.x % p.slabs);
        row = (i64)(blockIdx.x / p.slabs) * 4 + wave;
    }
    if (row >= p.n_rows) return;
    const Columns<N> cols((slab * G + (lane & (G - 1))) * N, p.dim);
    const I *ids = (const I *)p.indices;
    const i64 b = max((i64)0, (i64)((const I *)p.indptr)[row]), e = min(p.nnz, (i64)((const I *)p.indptr)[row + 1]);
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    for (i64 i = b; i < e; i += 64) {
        const int n = (int)min((i64)64, e - i);
        int mine = -1;
        float weight = 0.f;
        if (lane < n) {
            const i64 id = (i64)ids[i + lane];
            mine = id >= 0 && id < p.n_vocab ? (int)id : -1;
            weight = p.data ? p.data[i + lane] : 1.f;
        }
        for (int j = 0; j < n; j += S * U) {
            RawVec<T, N> x[U];
            int id[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                id[u] = S == 1 ? __builtin_amdgcn_readlane(mine, j + u) : __shfl(mine, j + u * S + sub, 64);
                x[u] = vec_load<T, N>((const T *)p.in + (i64)max(id[u], 0) * p.ld_in + cols.c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float w = __int_as_float(S == 1 ? __builtin_amdgcn_readlane(__float_as_int(weight), j + u) : __shfl(__float_as_int(weight), j + u * S + sub, 64));
                if (id[u] >= 0) {
#pragma unroll
                    for (int k = 0; k < N; ++k) acc[k] = __fmaf_rn(w, up(x[u].v[k]), acc[k]);
                }
            }
        }
    }
    // The groups' sums: while a lane holds several columns, two groups share them out (each sends the half it gives up); then they add.
    int first = 0;
    bool mine_alone = true;
#pragma unroll
    for (int d = G, held = N; d < 64; d <<= 1, held = held > 1 ? held / 2 : 1) {
        const bool upper = (lane & d) != 0;
        if (held > 1) {
#pragma unroll
            for (int k = 0; k < held / 2; ++k) {
                const float give = upper ? acc[k] : acc[k + held / 2], keep = upper ? acc[k + held / 2] : acc[k];
                acc[k] = keep + __shfl_xor(give, d, 64);
            }
            first += upper ? held / 2 : 0;
        } else {
            acc[0] += __shfl_xor(acc[0], d, 64);
            mine_alone = mine_alone && !upper;
        }
    }
    if (mine_alone && cols.active) {
        constexpr int LEFT = N > S ? N / S : 1;
#pragma unroll
        for (int k = 0; k < LEFT; ++k) acc[k] *= p.scale;
        put<T, LEFT>((T *)p.out + row * p.ld_out + cols.c + first, acc);
    }
}

// ---- the gradient: entries sorted by id, stably ------------------------------------------------------------------------------
// A radix sort from the low digit: per pass one launch counts the digits of every workgroup's chunk, one moves the entries (with many
// workgroups one more adds the counts up between them).  Every wave owns a contiguous part of the chunk and goes through it in order;
// equal digits of 64 entries are ranked by their lane.  Ids outside the table take the key n_vocab and end up behind everything else.
// An entry carries its row of the gradient and its weight.  The rows of a CSR's entries are written out beside the first count.
// 1.2 M entries: 7 us to count, 5 to add the counts up and 17 to move them, two passes for 2^17 ids: latency of launches with one workgroup on a
// CU, not bandwidth (28 MB a pass).  16 384 lookups into 173 MB: 8.3 + 10.9 us a pass, in which the gradient is cleared as well.

constexpr int SORT_NT = 512, SORT_WAVES = SORT_NT / 64, SORT_BINS = 512;
constexpr int SORT_PER = 9, SORT_CHUNK = SORT_NT * SORT_PER;    // entries of a thread, most of a workgroup: 54 KB of LDS
constexpr int SORT_DIRECT = 32;      // up to so many workgroups the moving launch adds up the counts itself

// The rows of the gradient that no entry names are 0: all of it is cleared, by workgroups behind those of the sort's launches, which leave
// most of the card free.  part / parts: this launch's share of the rows.
struct FillParams {
    void *out;                   // NULL: nothing to clear
    i64 n_rows, dim, ld;         // in elements
    int bytes;                   // of an element
    int part, parts;
};
__device__ __forceinline__ void fill_share(const FillParams &f, int block, int blocks) {
    const i64 r0 = f.n_rows * f.part / f.parts, r1 = f.n_rows * (f.part + 1) / f.parts;
    const i64 width = f.dim * f.bytes, ld = f.ld * f.bytes;
    unsigned char *out = (unsigned char *)f.out + r0 * ld;
    typedef unsigned Quad __attribute__((ext_vector_type(4), aligned(2)));
    const Quad zero = {0, 0, 0, 0};
    if (ld == width) {
        const i64 total = (r1 - r0) * width, step = (i64)blocks * blockDim.x * 16;
        i64 i = ((i64)block * blockDim.x + threadIdx.x) * 16;
        for (; i + 16 <= total; i += step) *(Quad *)(out + i) = zero;
        for (; i < total && i + 16 > total; i += 2) *(unsigned short *)(out + i) = 0;
    } else {
        for (i64 r = block; r < r1 - r0; r += blocks) {
            i64 c = (i64)threadIdx.x * 16;
            for (; c + 16 <= width; c += (i64)blockDim.x * 16) *(Quad *)(out + r * ld + c) = zero;
            for (; c < width && c + 16 > width; c += 2) *(unsigned short *)(out + r * ld + c) = 0;
        }
    }
}
template <int NT> __global__ __launch_bounds__(NT) void sp_fill_kernel(FillParams f) { fill_share(f, blockIdx.x, gridDim.x); }

struct SortParams {
    i64 n;                       // entries
    int chunk;                   // entries of a workgroup (a multiple of SORT_NT)
    int wgs, shift, bits;
    const unsigned *key_in;      // first pass: NULL, the keys are `indices`
    const unsigned *pay_in;
    const float *w_in;
    unsigned *key_out, *pay_out;
    float *w_out;                // NULL without weights
    unsigned *hist;              // [wgs][SORT_BINS] digits of every workgroup's chunk; then, of the workgroups before it
    unsigned *total;             // [SORT_BINS] digits of all
    const void *indices, *indptr;
    unsigned *entry_row;         // [n] rows of a CSR's entries (n_rows: in no row), or NULL: entry i is row i
    i64 n_rows, n_vocab;
    FillParams fill;
};

template <typename I> __device__ __forceinline__ unsigned sort_key(const SortParams &p, i64 i) {
    if (p.key_in) return p.key_in[i];
    const i64 id = (i64)((const I *)p.indices)[i];
    return id >= 0 && id < p.n_vocab ? (unsigned)id : (unsigned)p.n_vocab;
}

// entry_row of every entry, one wave per row; what lies before the first row and behind the last is in none
template <typename I> __device__ __forceinline__ void spread_rows(const SortParams &p, int block, int blocks) {
    const int lane = threadIdx.x & 63;
    const i64 waves = (i64)blocks * SORT_WAVES;
    for (i64 r = (i64)block * SORT_WAVES + threadIdx.x / 64; r < p.n_rows + 2; r += waves) {
        i64 b = r == 0 ? 0 : (i64)((const I *)p.indptr)[r - 1], e = r == p.n_rows + 1 ? p.n : (i64)((const I *)p.indptr)[r];
        b = b < 0 ? 0 : b;
        e = e > p.n ? p.n : e;
        const unsigned row = r == 0 || r == p.n_rows + 1 ? (unsigned)p.n_rows : (unsigned)(r - 1);
        for (i64 i = b + lane; i < e; i += 64) p.entry_row[i] = row;
    }
}

template <typename I> __global__ __launch_bounds__(SORT_NT) void sp_sort_count_kernel(SortParams p) {
    __shared__ unsigned h[SORT_BINS];
    if ((int)blockIdx.x >= p.wgs) {                            // the workgroups behind the sort's: rows of the entries, clearing
        const int block = blockIdx.x - p.wgs, blocks = gridDim.x - p.wgs;
        if (!p.key_in && p.entry_row) spread_rows<I>(p, block, blocks);
        if (p.fill.out) fill_share(p.fill, block, blocks);
        return;
    }
    for (int i = threadIdx.x; i < SORT_BINS; i += SORT_NT) h[i] = 0;
    __syncthreads();
    const i64 b = (i64)blockIdx.x * p.chunk, e = min(p.n, b + p.chunk);
    const unsigned mask = (1u << p.bits) - 1u;
    for (i64 i = b + threadIdx.x; i < e; i += SORT_NT) atomicAdd(&h[(sort_key<I>(p, i) >> p.shift) & mask], 1u);
    __syncthreads();
    for (int i = threadIdx.x; i < SORT_BINS; i += SORT_NT) p.hist[(i64)blockIdx.x * SORT_BINS + i] = h[i];
}

// hist[g][d] becomes the sum over the workgroups before g.  64 digits per workgroup of 16 waves: a wave takes a share of the workgroups, the
// shares' sums are joined in LDS.
__global__ __launch_bounds__(1024) void sp_sort_prefix_kernel(unsigned *hist, unsigned *total, int wgs) {
    __shared__ unsigned sums[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
    const int share = (wgs + 15) / 16, g0 = wave * share, g1 = min(wgs, g0 + share);
    unsigned sum = 0;
    for (int g = g0; g < g1; g += 16) {
        unsigned v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = g + k < g1 ? hist[(i64)(g + k) * SORT_BINS + d] : 0u;
#pragma unroll
        for (int k = 0; k < 16; ++k) sum += v[k];
    }
    sums[wave][lane] = sum;
    __syncthreads();
    unsigned run = 0;
    for (int w = 0; w < wave; ++w) run += sums[w][lane];
    if (wave == 15) total[d] = run + sum;
    for (int g = g0; g < g1; g += 16) {
        unsigned v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = g + k < g1 ? hist[(i64)(g + k) * SORT_BINS + d] : 0u;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            if (g + k < g1) hist[(i64)(g + k) * SORT_BINS + d] = run;
            run += v[k];
        }
    }
}
static_assert(SORT_NT == SORT_BINS, "a thread per digit");

// Entries go to their places by way of LDS, where the chunk is laid out in the order of its digits: neighbours there are neighbours in
// memory, so that what a wave writes are runs (scattered one by one, 1.2 M entries took 24 us a pass).
template <typename I> __global__ __launch_bounds__(SORT_NT) void sp_sort_move_kernel(SortParams p) {
    __shared__ unsigned off[SORT_WAVES][SORT_BINS];
    __shared__ unsigned delta[SORT_BINS];                      // global place - place in the chunk, of a digit
    __shared__ unsigned wsum[2][SORT_WAVES];
    __shared__ unsigned skey[SORT_CHUNK], spay[SORT_CHUNK];
    __shared__ float sweight[SORT_CHUNK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned mask = (1u << p.bits) - 1u;
    // consecutive chunks go to one XCD (workgroups are dealt to the eight in turn): what they write next to each other meets in its L2
    const int per_xcd = (p.wgs + 7) / 8;
    if ((int)blockIdx.x >= 8 * per_xcd) {
        if (p.fill.out) fill_share(p.fill, blockIdx.x - 8 * per_xcd, gridDim.x - 8 * per_xcd);
        return;
    }
    const int wg = (int)(blockIdx.x % 8) * per_xcd + (int)blockIdx.x / 8;
    if (wg >= p.wgs) return;
    // the wave's part, consecutive entries, all of it requested at once
    const int n = (int)min((i64)p.chunk, p.n - (i64)wg * p.chunk), per = p.chunk / SORT_WAVES, rounds = per / 64;
    const int first = wave * per + lane;
    const i64 chunk0 = (i64)wg * p.chunk;
    unsigned key[SORT_PER], pay[SORT_PER];
    float weight[SORT_PER];
#pragma unroll
    for (int q = 0; q < SORT_PER; ++q) {
        const int j = first + q * 64;
        if (q < rounds && j < n) {
            key[q] = sort_key<I>(p, chunk0 + j);
            pay[q] = p.key_in ? p.pay_in[chunk0 + j] : p.entry_row ? p.entry_row[chunk0 + j] : (unsigned)(chunk0 + j);
            if (p.w_out) weight[q] = p.w_in[chunk0 + j];
        }
    }
    for (int w = 0; w < SORT_WAVES; ++w) off[w][tid] = 0;
    // entries of digit `tid` before this workgroup: those of smaller digits anywhere, and of its own in the workgroups before
    unsigned before = 0, all = 0;
    if (p.wgs <= SORT_DIRECT) {
        unsigned v[SORT_DIRECT];
#pragma unroll
        for (int g = 0; g < SORT_DIRECT; ++g) v[g] = g < p.wgs ? p.hist[(i64)g * SORT_BINS + tid] : 0u;
#pragma unroll
        for (int g = 0; g < SORT_DIRECT; ++g) {
            before += g < wg ? v[g] : 0u;
            all += v[g];
        }
    } else {
        before = p.hist[(i64)wg * SORT_BINS + tid];
        all = p.total[tid];
    }
    __syncthreads();
    // digits of every wave's part
#pragma unroll
    for (int q = 0; q < SORT_PER; ++q)
        if (q < rounds && first + q * 64 < n) atomicAdd(&off[wave][(key[q] >> p.shift) & mask], 1u);
    __syncthreads();
    unsigned here = 0;
    for (int w = 0; w < SORT_WAVES; ++w) here += off[w][tid];
    unsigned inc_all = all, inc_here = here;                   // prefix sums over the digits, of all entries and of the chunk's
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(inc_all, d, 64), q = __shfl_up(inc_here, d, 64);
        if (lane >= d) {
            inc_all += o;
            inc_here += q;
        }
    }
    if (lane == 63) {
        wsum[0][wave] = inc_all;
        wsum[1][wave] = inc_here;
    }
    __syncthreads();
    unsigned place = before + inc_all - all, local = inc_here - here;
    for (int w = 0; w < wave; ++w) {
        place += wsum[0][w];
        local += wsum[1][w];
    }
    delta[tid] = place - local;
    for (int w = 0; w < SORT_WAVES; ++w) {
        const unsigned n = off[w][tid];
        off[w][tid] = local;
        local += n;
    }
    __syncthreads();
    volatile unsigned *mine = off[wave];
#pragma unroll
    for (int q = 0; q < SORT_PER; ++q) {
        if (q >= rounds) break;
        const bool ok = first + q * 64 < n;
        const unsigned digit = ok ? (key[q] >> p.shift) & mask : 0u;
        u64 same = __ballot(ok);
        for (int k = 0; k < p.bits; ++k) {
            const u64 set = __ballot((digit >> k) & 1u);
            same &= (digit >> k) & 1u ? set : ~set;
        }
        if (ok) {
            const unsigned rank = (unsigned)__popcll(same & ((1ull << lane) - 1ull));
            const unsigned at = mine[digit] + rank;
            if (rank == 0) mine[digit] = at + (unsigned)__popcll(same);       // (a wave's LDS accesses keep their order: everybody has read)
            skey[at] = key[q];
            spay[at] = pay[q];
            if (p.w_out) sweight[at] = weight[q];
        }
    }
    __syncthreads();
    for (int i = tid; i < n; i += SORT_NT) {
        const unsigned k = skey[i], at = (unsigned)i + delta[(k >> p.shift) & mask];
        p.key_out[at] = k;
        p.pay_out[at] = spay[i];
        if (p.w_out) p.w_out[at] = sweight[i];
    }
}

// the CSR row of entry i; n_rows for an entry that no row holds
template <typename I> __device__ __forceinline__ i64 row_of(const void *indptr, i64 n_rows, i64 i) {
    i64 lo = 0, hi = n_rows;                                   // first r with indptr[r + 1] > i
    while (lo < hi) {
        const i64 mid = (lo + hi) >> 1;
        if ((i64)((const I *)indptr)[mid + 1] > i) hi = mid;
        else lo = mid + 1;
    }
    return lo < n_rows && (i64)((const I *)indptr)[lo] > i ? n_rows : lo;
}

// Up to 8192 entries are sorted by one workgroup, in one launch, while the others clear the gradient: an entry is its key and its index
// in one word, 8 words per thread in registers, moved through LDS once per pass.  The lanes of equal digits are found first; one of them counts
// all of them (a popular id's entries would add to one counter one after the other; 6000 entries 19.6 -> 16.2 us.  In the launches above the same
// costs registers that are missed: 17.2 -> 18.5.)  Gradient of n lookups into 84 433 rows of 1024 bf16, this way / by the launches above:
// n = 4096 35 / 48 us, 8192 37 / 50, 16 384 82 / 54; into 2000 rows, where there is little to clear beside it: 4096 23 / 30 us, 8192 30 / 33.
constexpr int SMALL_NT = 1024, SMALL_WAVES = SMALL_NT / 64, SMALL_PER = 8, SMALL_MAX = SMALL_NT * SMALL_PER, SMALL_INDEX_BITS = 13;
static_assert(SMALL_MAX == 1 << SMALL_INDEX_BITS, "an index fits its bits");

// same[q]: the lanes of the wave whose digit of round q is this lane's, of those that `same` holds on entry.  Bit by bit for all rounds: they do
// not wait for one another.
template <int Q> __device__ __forceinline__ void match_digits(const unsigned (&digit)[Q], u64 (&same)[Q], int rounds, int bits) {
    for (int k = 0; k < bits; ++k) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q >= rounds) break;
            const int bit = __builtin_amdgcn_sbfe((int)digit[q], k, 1);       // 0 or -1
            const u64 set = __ballot(bit != 0);
            const unsigned lo = (unsigned)same[q] & ~((unsigned)set ^ (unsigned)bit), hi = (unsigned)(same[q] >> 32) & ~((unsigned)(set >> 32) ^ (unsigned)bit);
            same[q] = (u64)hi << 32 | lo;
        }
    }
}

template <typename I> __global__ __launch_bounds__(SMALL_NT) void sp_sort_small_kernel(SortParams p, int passes) {
    __shared__ unsigned buf[SMALL_MAX];
    __shared__ unsigned off[SMALL_WAVES][SORT_BINS];
    __shared__ unsigned wsum[SORT_BINS / 64];
    if (blockIdx.x > 0) {
        if (p.fill.out) fill_share(p.fill, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = (int)p.n;
    const int rounds = (n + SMALL_NT - 1) / SMALL_NT, first = wave * rounds * 64 + lane;      // a wave's entries are consecutive
    const unsigned mask = (1u << p.bits) - 1u;
    unsigned v[SMALL_PER];
#pragma unroll
    for (int q = 0; q < SMALL_PER; ++q) {
        const int i = first + q * 64;
        if (q < rounds && i < n) v[q] = sort_key<I>(p, i) << SMALL_INDEX_BITS | (unsigned)i;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = SMALL_INDEX_BITS + pass * p.bits;
        unsigned digit[SMALL_PER];
        u64 same[SMALL_PER];
#pragma unroll
        for (int q = 0; q < SMALL_PER; ++q) {
            const bool ok = q < rounds && first + q * 64 < n;
            digit[q] = ok ? (v[q] >> shift) & mask : 0u;
            same[q] = __ballot(ok);
        }
        match_digits(digit, same, rounds, p.bits);
        for (int i = tid; i < SMALL_WAVES * SORT_BINS; i += SMALL_NT) (&off[0][0])[i] = 0u;
        __syncthreads();
        unsigned rank[SMALL_PER];                              // among the equal digits of its 64 entries
#pragma unroll
        for (int q = 0; q < SMALL_PER; ++q)
            if (q < rounds && first + q * 64 < n) {
                rank[q] = (unsigned)__popcll(same[q] & ((1ull << lane) - 1ull));
                if (rank[q] == 0) atomicAdd(&off[wave][digit[q]], (unsigned)__popcll(same[q]));
            }
        __syncthreads();
        unsigned inc = 0, all = 0;
        if (tid < SORT_BINS) {                                 // a thread per digit: entries of smaller digits, then of the waves before
            for (int w = 0; w < SMALL_WAVES; ++w) all += off[w][tid];
            inc = all;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const unsigned o = __shfl_up(inc, d, 64);
                if (lane >= d) inc += o;
            }
            if (lane == 63) wsum[wave] = inc;
        }
        __syncthreads();
        if (tid < SORT_BINS) {
            unsigned base = inc - all;
            for (int w = 0; w < wave; ++w) base += wsum[w];
            for (int w = 0; w < SMALL_WAVES; ++w) {
                const unsigned c = off[w][tid];
                off[w][tid] = base;
                base += c;
            }
        }
        __syncthreads();
        volatile unsigned *mine = off[wave];
#pragma unroll
        for (int q = 0; q < SMALL_PER; ++q)
            if (q < rounds && first + q * 64 < n) {
                const unsigned at = mine[digit[q]] + rank[q];
                if (rank[q] == 0) mine[digit[q]] = at + (unsigned)__popcll(same[q]);    // (as in the launches above)
                buf[at] = v[q];
            }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < SMALL_PER; ++q)
            if (q < rounds && first + q * 64 < n) v[q] = buf[first + q * 64];
        __syncthreads();
    }
#pragma unroll
    for (int q = 0; q < SMALL_PER; ++q) {
        const int i = first + q * 64;
        if (q < rounds && i < n) {
            const unsigned from = v[q] & (SMALL_MAX - 1);
            p.key_out[i] = v[q] >> SMALL_INDEX_BITS;
            p.pay_out[i] = p.indptr ? (unsigned)row_of<I>(p.indptr, p.n_rows, from) : from;
            if (p.w_out) p.w_out[i] = p.w_in[from];
        }
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
    int by_xcd;                 // slab s is the work of the XCDs s, s + slabs, .. (slabs divides 8)
    float scale;
};

template <typename TO, int N> __device__ __forceinline__ void write_row(const ReduceParams &p, unsigned key, const Columns<N> &cols, float *acc) {
    TO *row = (TO *)p.out + (i64)key * p.ld_out + cols.c;
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] *= p.scale;
    if (p.accumulate) {
        if (cols.c != cols.own) {                              // (columns that another lane writes as well are added to once, by that lane)
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (cols.c + j >= cols.own) row[j] = (TO)(acc[j] + up(row[j]));
            return;
        }
        const RawVec<TO, N> was = vec_load<TO, N>(row);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] += up(was.v[j]);
    }
    put<TO, N>(row, acc);
}

__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0F70); }      // vmcnt(0)

// One group of G lanes per chunk of the sorted entries and slab of columns: runs of equal ids are summed as they come.  A run that
// lies inside the chunk is a row of the gradient and is written; one that began before or goes on behind it leaves its sum in `part`.
// What bounds it is the gather: 1.2 M entries, each a row of 516 bytes, are 0.61 GB in 53 us, 11.5 TB/s out of the L2s (47 us with four times the
// waves, which the joins then lose again).
template <typename T, typename TO, int G, int N> __global__ __launch_bounds__(256) void sp_embed_reduce_kernel(ReduceParams p) {
    constexpr int U = 8;
    const int lane = threadIdx.x & (G - 1);
    const int g = G == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : (int)threadIdx.x / G;
    i64 ch;
    int slab;
    if (p.by_xcd) {                                            // (as in the bags)
        const int xcd = (int)(blockIdx.x % 8);
        slab = xcd % p.slabs;
        ch = ((i64)(blockIdx.x / 8) * (8 / p.slabs) + xcd / p.slabs) * (256 / G) + g;
    } else {
        const i64 item = (i64)blockIdx.x * (256 / G) + g;
        slab = (int)(item % p.slabs);
        ch = item / p.slabs;
    }
    if (ch >= p.chunks) return;
    const Columns<N> cols((slab * G + lane) * N, p.dim);
    const i64 b = ch * p.chunk, e = min(p.n, b + p.chunk);
    const int none = (int)p.n_vocab;
    const int prev = b > 0 ? (int)p.key[b - 1] : none, next = e < p.n ? (int)p.key[e] : none;
    int run = group_lane<G>((int)p.key[b], 0);
    bool head = b > 0 && run == prev;
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    auto flush = [&](bool last) {
        if (run == none || !cols.active) return;
        const bool tail = last && next == run;                 // (next is `none` behind the last entry)
        if (head || tail) put<float, N>(p.part + (2 * ch + (head ? 0 : 1)) * p.dim + cols.c, acc);
        else write_row<TO, N>(p, (unsigned)run, cols, acc);
    };
    for (i64 i = b; i < e; i += G) {                           // G entries at once, a lane each
        const int n = (int)min((i64)G, e - i);
        int key = none, from = -1;
        float weight = 0.f;
        if (lane < n) {
            key = (int)p.key[i + lane];
            const unsigned r = p.pay[i + lane];
            from = ((i64)r < p.n_rows ? (int)r : -1) | (key == none ? -1 : 0);      // (no branch: both are requested at once)
            weight = p.w ? p.w[i + lane] : 1.f;
        }
        for (int j = 0; j < n; j += U) {
            RawVec<T, N> x[U];
            int r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                r[u] = group_lane<G>(from, j + u);
                x[u] = vec_load<T, N>((const T *)p.in + (i64)max(r[u], 0) * p.ld_in + cols.c);
            }
            // Loads and stores of a wave are counted together: once a row has been written behind a branch, waiting for a load that is still
            // on its way means waiting for the store as well.  So all rows of the batch are waited for here.
            loads_done();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j + u >= n) break;
                const int k = group_lane<G>(key, j + u);
                if (k != run) {
                    flush(false);
                    run = k;
                    head = false;
#pragma unroll
                    for (int q = 0; q < N; ++q) acc[q] = 0.f;
                }
                if (r[u] >= 0) {
                    const float w = __int_as_float(group_lane<G>(__float_as_int(weight), j + u));
#pragma unroll
                    for (int q = 0; q < N; ++q) acc[q] = __fmaf_rn(w, up(x[u].v[q]), acc[q]);
                }
            }
        }
    }
    flush(true);
}

// Up to 1024 entries need no sort at all: a workgroup owns DIRECT_IDS ids or fewer (and a slab of columns), looks through all entries, keeps
// those of its ids in their order, sums each id's and clears the rows that have none.  One launch, no workspace.  Gradient of n lookups
// into 84 433 rows of 1024 bf16, this way / by the sort above: n = 64 24 / 33 us, 512 27 / 36, 1024 28 / 33, 2048 36 / 33; into 2000 rows:
// 8.8 / 18, 10 / 19, 16 / 18, 31 / 20 (what a popular id has is summed by one group).
constexpr int DIRECT_MAX = 1024, DIRECT_IDS = 2048, DIRECT_NONE = 0x7FFFFFFF;
struct DirectParams {
    ReduceParams r;              // in, out, n, n_vocab, ld_in, ld_out, n_rows, dim, slabs, accumulate, scale
    const void *indices, *indptr;
    const float *data;
    int per;                     // ids of a workgroup
};
template <typename T, typename TO, typename I, int G, int N> __global__ __launch_bounds__(256) void sp_embed_grad_direct_kernel(DirectParams d) {
    constexpr int GROUPS = 256 / G, U = 8, Q = DIRECT_MAX / 256;
    __shared__ int key[DIRECT_MAX], from[DIRECT_MAX], first[DIRECT_IDS];
    __shared__ float weight[DIRECT_MAX];
    __shared__ int wsum[4];
    const ReduceParams &p = d.r;
    const int tid = threadIdx.x, lane = tid & 63, gl = tid & (G - 1), g = tid / G, n = (int)p.n;
    const i64 v0 = (i64)(blockIdx.x / p.slabs) * d.per;
    const int width = (int)min((i64)d.per, p.n_vocab - v0);
    const Columns<N> cols(((int)(blockIdx.x % p.slabs) * G + gl) * N, p.dim);
    int mine[Q], count = 0;                                    // a thread's entries are consecutive: their order is the threads'
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = tid * Q + q;
        const i64 id = i < n ? (i64)((const I *)d.indices)[i] - v0 : -1;
        mine[q] = id >= 0 && id < width ? (int)id : -1;
        count += mine[q] >= 0;
    }
    for (int i = tid; i < width; i += 256) first[i] = DIRECT_NONE;
    int at = count;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int o = __shfl_up(at, k, 64);
        if (lane >= k) at += o;
    }
    if (lane == 63) wsum[tid >> 6] = at;
    __syncthreads();
    at -= count;
    for (int w = 0; w < (tid >> 6); ++w) at += wsum[w];
    const int m = wsum[0] + wsum[1] + wsum[2] + wsum[3];
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (mine[q] >= 0) {
            key[at] = mine[q];
            from[at] = tid * Q + q;
            atomicMin(&first[mine[q]], at);
            ++at;
        }
    __syncthreads();
    for (int e = tid; e < m; e += 256) {
        const int i = from[e];
        const i64 r = d.indptr ? row_of<I>(d.indptr, p.n_rows, i) : i;
        weight[e] = d.data ? d.data[i] : 1.f;
        from[e] = r < p.n_rows ? (int)r : -1;
    }
    __syncthreads();
    for (int e = g; e < m; e += GROUPS) {
        const int k = key[e];
        if (first[k] != e) continue;
        float acc[N];
#pragma unroll
        for (int q = 0; q < N; ++q) acc[q] = 0.f;
        for (int f0 = e; f0 < m; f0 += G) {                    // G entries looked at together; the id's own ones in their order
            const u64 all = __ballot(f0 + gl < m && key[min(f0 + gl, m - 1)] == k);
            u64 hits = G == 64 ? all : (all >> (lane & ~(G - 1))) & ((1ull << (G & 63)) - 1ull);
            while (hits) {
                RawVec<T, N> x[U];
                int r[U], f[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    f[u] = hits ? f0 + __builtin_ctzll(hits) : f0;
                    r[u] = hits ? from[f[u]] : -1;
                    hits &= hits - 1ull;                       // (0 stays 0)
                    x[u] = vec_load<T, N>((const T *)p.in + (i64)max(r[u], 0) * p.ld_in + cols.c);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r[u] >= 0) {
                        const float w = weight[f[u]];
#pragma unroll
                        for (int q = 0; q < N; ++q) acc[q] = __fmaf_rn(w, up(x[u].v[q]), acc[q]);
                    }
            }
        }
        if (cols.active) write_row<TO, N>(p, (unsigned)(v0 + k), cols, acc);
    }
    if (p.accumulate || !cols.active) return;
    RawVec<TO, N> zero;
#pragma unroll
    for (int q = 0; q < N; ++q) zero.v[q] = (TO)0.f;
    for (int i = g; i < width; i += GROUPS)
        if (first[i] == DIRECT_NONE) vec_store<TO, N>((TO *)p.out + (v0 + i) * p.ld_out + cols.c, zero);
}

// Runs over several chunks: the chunk in which a run begins adds up its parts, in their order, and writes the row.  One group of G lanes per
// chunk and slab: the lanes look how far the run goes; up to JOIN_SHORT more chunks are the group's work, a longer run that of the whole
// workgroup, whose groups sum contiguous shares.  (One workgroup per chunk instead costs 2 ns a chunk, 8 us at 4096 and 33 at 16 384, for the
// launch and the latency of the keys alone.)
constexpr int JOIN_SHORT = 8;
template <typename TO, int G, int N> __device__ __forceinline__ void join_long(const ReduceParams &p, i64 ch, int slab, unsigned run, float (*sums)[G * N], int *ends) {
    constexpr int GROUPS = 256 / G, U = 8;
    const int tid = threadIdx.x, lane = tid & (G - 1), g = tid / G;
    const Columns<N> cols((slab * G + lane) * N, p.dim);
    // chunks ch + 1 .. last hold the rest of it: the first one that does not go on into the next, 256 looked at at once
    i64 last = ch + 1;
    for (;; last += 256) {
        if (tid == 0) *ends = 256;
        __syncthreads();
        const i64 k = last + tid;
        if (k + 1 >= p.chunks || p.key[(k + 1) * p.chunk] != run) atomicMin(ends, tid);
        __syncthreads();
        const int first = *ends;
        __syncthreads();
        if (first < 256) {
            last += first;
            break;
        }
    }
    const i64 count = last - ch, share = (count + GROUPS - 1) / GROUPS;
    const i64 k0 = ch + 1 + g * share, k1 = min(last + 1, k0 + share);
    float acc[N];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = 0.f;
    for (i64 k = k0; k < k1; k += U) {
        RawVec<float, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = vec_load<float, N>(p.part + (2 * min(k + u, k1 - 1)) * p.dim + cols.c);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k + u < k1)
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += x[u].v[j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) sums[g][lane * N + j] = acc[j];
    __syncthreads();
    if (g == 0 && cols.active) {
        const RawVec<float, N> x = vec_load<float, N>(p.part + (2 * ch + 1) * p.dim + cols.c);
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = x.v[j];
        const int parts = (int)min((i64)GROUPS, (count + share - 1) / share);
        for (int q = 0; q < parts; ++q)
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += sums[q][lane * N + j];
        write_row<TO, N>(p, run, cols, acc);
    }
    __syncthreads();
}
template <typename TO, int G, int N> __global__ __launch_bounds__(256) void sp_embed_join_kernel(ReduceParams p) {
    constexpr int GROUPS = 256 / G;
    __shared__ float sums[GROUPS][G * N];
    __shared__ unsigned long_run[GROUPS];                      // n_vocab: none
    __shared__ int ends;
    const int tid = threadIdx.x, lane = tid & (G - 1), g = tid / G;
    const unsigned none = (unsigned)p.n_vocab;
    const int slab = (int)(blockIdx.x % p.slabs);
    const i64 ch0 = (i64)(blockIdx.x / p.slabs) * GROUPS, ch = ch0 + g;
    if (lane == 0) long_run[g] = none;
    if (ch + 1 < p.chunks) {                                   // (the chunk is full then, and there is an entry behind it)
        const i64 e = (ch + 1) * p.chunk, k = ch + 1 + min(lane, JOIN_SHORT - 1);
        const unsigned run = p.key[e - 1], next = p.key[e], before = ch > 0 ? p.key[e - p.chunk - 1] : none;
        const unsigned beyond = k + 1 < p.chunks ? p.key[(k + 1) * p.chunk] : none;
        if (run != none && next == run && before != run) {     // it goes on behind the chunk, and began in it
            const u64 all = __ballot(lane < JOIN_SHORT && beyond != run);
            const unsigned ends_at = (unsigned)((all >> (tid & 63 & ~(G - 1))) & ((1u << JOIN_SHORT) - 1u));
            if (ends_at == 0u) {
                if (lane == 0) long_run[g] = run;
            } else {
                const int more = __builtin_ctz(ends_at) + 1;   // chunks ch + 1 .. ch + more
                const Columns<N> cols((slab * G + lane) * N, p.dim);
                RawVec<float, N> x[JOIN_SHORT], mine = vec_load<float, N>(p.part + (2 * ch + 1) * p.dim + cols.c);
#pragma unroll
                for (int u = 0; u < JOIN_SHORT; ++u) x[u] = vec_load<float, N>(p.part + 2 * (ch + 1 + min(u, more - 1)) * p.dim + cols.c);
                float acc[N];
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] = mine.v[j];
#pragma unroll
                for (int u = 0; u < JOIN_SHORT; ++u)
                    if (u < more)
#pragma unroll
                        for (int j = 0; j < N; ++j) acc[j] += x[u].v[j];
                if (cols.active) write_row<TO, N>(p, run, cols, acc);
            }
        }
    }
    __syncthreads();
    for (int q = 0; q < GROUPS; ++q) {
        const unsigned run = long_run[q];
        if (run != none) join_long<TO, G, N>(p, ch0 + q, slab, run, sums, &ends);
    }
}

}  // namespace
