// sp_dense.hip — the operators on dense tensors (include/sp_dense.h): argument checks, launch shapes, C ABI.
//
// Everything here is device mode: pointers on `device`, launches on the caller's stream, scratch from the caller's workspace, no
// allocation, no synchronisation and no memset (a fill kernel where memory has to be cleared), so that every call can be captured.
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <type_traits>

#include "../../include/sp_dense.h"
#include "../../include/sp_knn.h"
#include "sp_adjust_kernel.hpp"
#include "sp_dense_common.hpp"
#include "sp_distill_kernels.hpp"
#include "sp_embed_kernels.hpp"

__attribute__((visibility("hidden"))) int sp_set_error(int code, const char *text);      // sp_knn.hip

namespace {

int fail(int code, const char *fmt, ...) {
    char text[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    return sp_set_error(code, text);
}

#define TRY(expr) do { int _rc = (expr); if (_rc) return _rc; } while (0)
#define HIP_TRY(expr)                                                                              \
    do {                                                                                           \
        hipError_t _e = (expr);                                                                    \
        if (_e != hipSuccess)                                                                      \
            return fail(SP_EHIP, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(_e), __FILE__, __LINE__); \
    } while (0)

// the call's device while it launches; the thread's own afterwards
struct OnDevice {
    int before = -1;
    bool moved = false;
    int enter(int device) {
        const hipError_t e = hipGetDevice(&before);
        if (e != hipSuccess) { (void)hipGetLastError(); return fail(SP_ENODEVICE, "no HIP device visible: similaripy_amd has no CPU fallback"); }
        if (device == before) return SP_OK;
        int n = 0;
        HIP_TRY(hipGetDeviceCount(&n));
        if (device < 0 || device >= n) return fail(SP_EINVAL, "device %d out of range (have %d)", device, n);
        HIP_TRY(hipSetDevice(device));
        moved = true;
        return SP_OK;
    }
    ~OnDevice() { if (moved) (void)hipSetDevice(before); }
};

i64 ceil_div(i64 a, i64 b) { return (a + b - 1) / b; }
constexpr i64 I32_MAX = 0x7FFFFFFFLL;
constexpr i64 COLS_MAX = I32_MAX - 65536;      // column numbers a workgroup beyond the row's end are still int32
// a launch has fewer than 2^32 threads
bool too_many(i64 blocks, int threads) { return blocks > I32_MAX || blocks * threads > 0xFFFFFFFFLL; }
bool bad_dtype(int d) { return d < SP_DT_F32 || d > SP_DT_F16; }

// calls f with a value of the element type
template <typename F> int with_type(int dtype, F f) {
    if (dtype == SP_DT_F32) return f(float());
    if (dtype == SP_DT_BF16) return f((__bf16)0.f);
    return f((_Float16)0.f);
}

// ---- embedding rows ------------------------------------------------------------------------------------------------------------

int check_embed(const sp_embed_args *a) {
    if (!a || a->struct_size != sizeof(sp_embed_args)) return fail(SP_EINVAL, "sp_embed_args size mismatch");
    if (a->flags) return fail(SP_EINVAL, "flags must be 0");
    if (bad_dtype(a->dtype) || bad_dtype(a->out_dtype)) return fail(SP_EINVAL, "bad dtype");
    if (a->n_rows < 0 || a->n_rows > I32_MAX || a->n_vocab < 0 || a->n_vocab >= I32_MAX || a->dim < 0 || a->dim > I32_MAX / 2 || a->nnz < 0 || a->nnz > I32_MAX)
        return fail(SP_EINVAL, "bad shape / nnz");
    if (!a->indptr && a->nnz != a->n_rows) return fail(SP_EINVAL, "without indptr nnz must equal n_rows");
    if (a->nnz > 0 && !a->indices) return fail(SP_EINVAL, "NULL indices");
    return SP_OK;
}

// Calls f with the lanes of a group and the elements of a lane: 16 bytes a lane, or one element where a row has fewer; the fewest lanes that
// cover a row, 8 .. 64 (columns beyond 64 lanes make further slabs).
template <int N, typename F> auto with_group(i64 dim, F f) {
    using Wide = std::integral_constant<int, N>;
    if (dim < N) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    const i64 lanes = ceil_div(dim, N);
    if (lanes <= 8) return f(std::integral_constant<int, 8>(), Wide());
    if (lanes <= 16) return f(std::integral_constant<int, 16>(), Wide());
    if (lanes <= 32) return f(std::integral_constant<int, 32>(), Wide());
    return f(std::integral_constant<int, 64>(), Wide());
}

EmbedParams embed_params(const sp_embed_args *a) {
    EmbedParams p{};
    p.in = a->src; p.indices = a->indices; p.indptr = a->indptr; p.data = a->data; p.out = a->out;
    p.n_rows = a->n_rows; p.n_vocab = a->n_vocab; p.nnz = a->nnz; p.ld_in = a->ld_src; p.ld_out = a->ld_out;
    p.dim = (int)a->dim; p.scale = a->scale;
    return p;
}

constexpr i64 L2_BYTES = 4 << 20;     // of an XCD
constexpr i64 FEW_BAGS = 8192;        // one wave each does not fill the card
constexpr int FILL_WGS = 512;         // workgroups that clear rows

// A gather of wide rows may be cut by columns into slabs of whole cache lines, each the work of one XCD or of two or four, so that an XCD's L2
// holds that many times more rows of its slab.  Slabs of a row: 8, 4 or 2 where they are equal and their lanes a power of two, 1 otherwise.
template <typename T> int line_slabs(i64 dim, i64 ld) {
    const i64 bytes = dim * (i64)sizeof(T), lanes = dim / VecOf<T>::N;
    if (ld * (i64)sizeof(T) % 128 != 0) return 1;
    for (int slabs = 8; slabs > 1; slabs /= 2)
        if (bytes % (128 * slabs) == 0) {
            const i64 g = lanes / slabs;
            return g <= 64 && (g & (g - 1)) == 0 ? slabs : 1;
        }
    return 1;
}

// Workgroups of 256 threads of a lookup or of bags; `cut`: slabs by XCD, or 1.  Bags: a workgroup takes four rows of a slab.
template <typename T> i64 embed_blocks(const sp_embed_args *a, int cut) {
    return with_group<VecOf<T>::N>(a->dim / cut, [&](auto gc, auto nc) -> i64 {
        const i64 slabs = ceil_div(a->dim, decltype(gc)::value * decltype(nc)::value), fours = ceil_div(a->n_rows, 4);
        if (!a->indptr) return ceil_div(a->n_rows * slabs, 256 / decltype(gc)::value);
        return cut > 1 ? ceil_div(fours, 8 / slabs) * 8 : fours * slabs;
    });
}
// Slabs by XCD of the bags: for a table beyond the L2 of one from which more rows are taken than it has, and for few bags; not where a
// workgroup for every four bags of a slab is more than one launch has.
template <typename T> int bag_slabs(const sp_embed_args *a) {
    const i64 row_bytes = a->dim * (i64)sizeof(T);
    const bool large = a->nnz >= a->n_vocab && a->n_vocab * row_bytes > L2_BYTES && row_bytes >= 1024;
    const int slabs = a->indptr && (large || a->n_rows <= FEW_BAGS) && (uintptr_t)a->src % 128 == 0 ? line_slabs<T>(a->dim, a->ld_src) : 1;
    return slabs > 1 && !too_many(embed_blocks<T>(a, slabs), 256) ? slabs : 1;
}

int check_embed_launch(const sp_embed_args *a) {
    return with_type(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        if (a->n_vocab > 0 && too_many(embed_blocks<T>(a, bag_slabs<T>(a)), 256)) return fail(SP_EINVAL, "too many rows for one launch");
        return (int)SP_OK;
    });
}

int run_embed(const sp_embed_args *a) {
    hipStream_t stream = (hipStream_t)a->stream;
    return with_type(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        if (a->n_vocab == 0) {                                 // every id is outside
            FillParams fill{};
            fill.out = a->out; fill.n_rows = a->n_rows; fill.dim = a->dim; fill.ld = a->n_rows > 1 ? a->ld_out : a->dim; fill.bytes = (int)sizeof(T); fill.parts = 1;
            hipLaunchKernelGGL(sp_fill_kernel<SORT_NT>, dim3(FILL_WGS), dim3(SORT_NT), 0, stream, fill);
            HIP_TRY(hipGetLastError());
            return (int)SP_OK;
        }
        const int cut = bag_slabs<T>(a);
        return with_group<VecOf<T>::N>(a->dim / cut, [&](auto gc, auto nc) {
            constexpr int G = decltype(gc)::value, N = decltype(nc)::value;
            EmbedParams p = embed_params(a);
            p.slabs = (int)ceil_div(a->dim, G * N);
            p.by_xcd = cut > 1;
            const unsigned blocks = (unsigned)embed_blocks<T>(a, cut);
            auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, stream, p); };
            if (a->indptr) a->index64 ? launch(sp_embed_rows_kernel<T, i64, G, N>) : launch(sp_embed_rows_kernel<T, int, G, N>);
            else a->index64 ? launch(sp_embed_lookup_kernel<T, i64, G, N>) : launch(sp_embed_lookup_kernel<T, int, G, N>);
            HIP_TRY(hipGetLastError());
            return (int)SP_OK;
        });
    });
}

// workspace of the gradient: two copies of the sorted entries (the passes alternate), the digit counts, the partial sums
constexpr i64 REDUCE_WAVES = 4096;       // that sum sorted entries, of a slab: four per SIMD; a wave has 64 / G chunks of them
constexpr int DIRECT_WGS = 512;
struct GradLayout {
    int wgs, sort_chunk, passes, bits, chunk;
    int slabs;                                                   // of a row that are cut for the XCDs (1: not cut)
    bool small;                                                  // sorted by one workgroup
    i64 chunks;
    size_t key[2], pay[2], w[2], rows, hist, digits, part, total;
};
GradLayout grad_layout(const sp_embed_args *a) {
    GradLayout L{};
    const i64 n = a->nnz;
    if (n <= DIRECT_MAX) return L;                               // no sort, no workspace
    // chunks for one workgroup per CU, of 1024 .. SORT_CHUNK entries
    i64 chunk = ceil_div(ceil_div(n, 256), SORT_NT) * SORT_NT;
    L.sort_chunk = (int)(chunk < 1024 ? 1024 : chunk > SORT_CHUNK ? SORT_CHUNK : chunk);
    L.wgs = (int)ceil_div(n, L.sort_chunk);
    int kb = 1;                                                  // bits of the keys 0 .. n_vocab
    while (kb < 31 && (1ll << kb) <= a->n_vocab) ++kb;
    L.small = n <= SMALL_MAX && kb + SMALL_INDEX_BITS <= 32;
    L.passes = (kb + 8) / 9;
    L.bits = (kb + L.passes - 1) / L.passes;
    // by XCD: rows of the gradient beyond the L2 of one, each taken many times.  (8192 rows of 144 entries, cut / whole: 4 KB 384 / 595 us, 2 KB
    // 249 / 280, 1 KB 190 / 142; 30 000 rows of 8 entries: 244 / 248, 143 / 138, 90 / 87.)
    const i64 row_bytes = a->dim * (a->dtype == SP_DT_F32 ? 4 : 2);
    const bool large = a->nnz >= 16 * a->n_rows && a->n_rows * row_bytes > L2_BYTES && row_bytes >= 2048;
    L.slabs = !large ? 1 : a->dtype == SP_DT_F32 ? line_slabs<float>(a->dim, a->ld_src) : line_slabs<__bf16>(a->dim, a->ld_src);
    auto group_lanes = [](auto gc, auto) { return (int)decltype(gc)::value; };
    const i64 lanes = a->dtype == SP_DT_F32 ? with_group<4>(a->dim / L.slabs, group_lanes) : with_group<8>(a->dim / L.slabs, group_lanes);
    const i64 per = ceil_div(n, REDUCE_WAVES * 64 / lanes);
    // A chunk is read in batches of 8 rows: with few entries a second batch costs more than twice the chunks do in the joins.  (At least 8 / 16 a
    // chunk: 1206 rows of 64 bf16 19.8 / 20.9 us, 6000 of 256 28.4 / 30.3, 4096 of 1024 33.6 / 35.0, 8192 of 1024 36.9 / 36.2, 16 384 56 / 54.)
    const i64 least = n <= 6144 ? 8 : 16;
    L.chunk = (int)(per < least ? least : per);
    L.chunks = ceil_div(n, L.chunk);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += (bytes + 255) & ~(size_t)255; return o; };
    for (int i = 0; i < 2; ++i) {
        L.key[i] = take((size_t)n * 4);
        L.pay[i] = take((size_t)n * 4);
        L.w[i] = a->data ? take((size_t)n * 4) : 0;
    }
    L.rows = a->indptr ? take((size_t)n * 4) : 0;
    L.hist = take((size_t)L.wgs * SORT_BINS * 4);
    L.digits = take((size_t)SORT_BINS * 4);
    L.part = take((size_t)L.chunks * 2 * (size_t)a->dim * 4);
    L.total = at;
    return L;
}

// ids of a workgroup where nothing is sorted
int direct_ids(const sp_embed_args *a) {
    const i64 per = ceil_div(a->n_vocab, DIRECT_WGS);
    return (int)(per < DIRECT_IDS ? per : DIRECT_IDS);
}
int check_grad_launch(const sp_embed_args *a) {
    if (a->nnz == 0 || a->n_rows == 0) return SP_OK;
    const int cut = a->nnz <= DIRECT_MAX ? 1 : grad_layout(a).slabs;
    auto slabs_of = [&](auto gc, auto nc) { return ceil_div(a->dim, decltype(gc)::value * decltype(nc)::value); };
    const i64 slabs = a->dtype == SP_DT_F32 ? with_group<4>(a->dim / cut, slabs_of) : with_group<8>(a->dim / cut, slabs_of);
    if (a->nnz <= DIRECT_MAX && too_many(ceil_div(a->n_vocab, direct_ids(a)) * slabs, 256)) return fail(SP_EINVAL, "too many rows for one launch");
    if (a->nnz > DIRECT_MAX && too_many(grad_layout(a).chunks * slabs, 256)) return fail(SP_EINVAL, "too many entries for one launch");
    return SP_OK;
}

template <typename T, typename TO> int run_embed_grad_as(const sp_embed_args *a) {
    hipStream_t stream = (hipStream_t)a->stream;
    FillParams fill{};
    if (!a->accumulate) {
        fill.out = a->out;
        fill.n_rows = a->n_vocab; fill.dim = a->dim; fill.ld = a->n_vocab > 1 ? a->ld_out : a->dim; fill.bytes = (int)sizeof(TO);
    }
    const bool entries = a->nnz > 0 && a->n_rows > 0;         // (without rows every entry is in none)
    if (!entries && fill.out) {
        fill.parts = 1;
        hipLaunchKernelGGL(sp_fill_kernel<SORT_NT>, dim3(FILL_WGS * 2), dim3(SORT_NT), 0, stream, fill);
    }
    if (entries && a->nnz <= DIRECT_MAX) {
        DirectParams d{};
        ReduceParams &r = d.r;
        r.in = a->src; r.out = a->out; r.n = a->nnz; r.n_vocab = a->n_vocab; r.n_rows = a->n_rows; r.ld_in = a->ld_src; r.ld_out = a->ld_out;
        r.dim = (int)a->dim; r.accumulate = a->accumulate; r.scale = a->scale;
        d.indices = a->indices; d.indptr = a->indptr; d.data = a->data;
        d.per = direct_ids(a);
        return with_group<VecOf<T>::N>(a->dim, [&](auto gc, auto nc) {
            constexpr int G = decltype(gc)::value, N = decltype(nc)::value;
            r.slabs = (int)ceil_div(a->dim, G * N);
            const i64 blocks = ceil_div(a->n_vocab, d.per) * r.slabs;
            auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, stream, d); };
            a->index64 ? launch(sp_embed_grad_direct_kernel<T, TO, i64, G, N>) : launch(sp_embed_grad_direct_kernel<T, TO, int, G, N>);
            HIP_TRY(hipGetLastError());
            return (int)SP_OK;
        });
    }
    if (entries) {
        const GradLayout L = grad_layout(a);
        unsigned char *ws = (unsigned char *)a->workspace;
        SortParams s{};
        s.n = a->nnz; s.chunk = L.sort_chunk; s.wgs = L.wgs; s.bits = L.bits;
        s.hist = (unsigned *)(ws + L.hist);
        s.total = (unsigned *)(ws + L.digits);
        s.indices = a->indices; s.indptr = a->indptr; s.n_rows = a->n_rows; s.n_vocab = a->n_vocab;
        s.w_in = a->data;
        s.fill = fill;
        s.fill.parts = 2 * L.passes;
        s.entry_row = a->indptr ? (unsigned *)(ws + L.rows) : nullptr;
        if (L.small) {
            s.fill.parts = 1;
            s.key_out = (unsigned *)(ws + L.key[0]);
            s.pay_out = (unsigned *)(ws + L.pay[0]);
            s.w_out = a->data ? (float *)(ws + L.w[0]) : nullptr;
            const dim3 grid(1 + (fill.out ? FILL_WGS : 0));
            if (a->index64) hipLaunchKernelGGL(sp_sort_small_kernel<i64>, grid, dim3(SMALL_NT), 0, stream, s, L.passes);
            else hipLaunchKernelGGL(sp_sort_small_kernel<int>, grid, dim3(SMALL_NT), 0, stream, s, L.passes);
            s.key_in = s.key_out; s.pay_in = s.pay_out; s.w_in = s.w_out;
        }
        for (int pass = 0; pass < (L.small ? 0 : L.passes); ++pass) {
            const int to = pass & 1;
            s.shift = pass * L.bits;
            s.key_out = (unsigned *)(ws + L.key[to]);
            s.pay_out = (unsigned *)(ws + L.pay[to]);
            s.w_out = a->data ? (float *)(ws + L.w[to]) : nullptr;
            auto launch = [&](auto kernel, int wgs, bool more) { hipLaunchKernelGGL(kernel, dim3(wgs + (more ? FILL_WGS : 0)), dim3(SORT_NT), 0, stream, s); ++s.fill.part; };
            const bool more = fill.out || (pass == 0 && s.entry_row);
            a->index64 ? launch(sp_sort_count_kernel<i64>, L.wgs, more) : launch(sp_sort_count_kernel<int>, L.wgs, more);
            if (L.wgs > SORT_DIRECT) hipLaunchKernelGGL(sp_sort_prefix_kernel, dim3(SORT_BINS / 64), dim3(1024), 0, stream, s.hist, s.total, s.wgs);
            a->index64 ? launch(sp_sort_move_kernel<i64>, 8 * (int)ceil_div(L.wgs, 8), fill.out) : launch(sp_sort_move_kernel<int>, 8 * (int)ceil_div(L.wgs, 8), fill.out);
            s.key_in = s.key_out;
            s.pay_in = s.pay_out;
            s.w_in = s.w_out;
        }
        ReduceParams r{};
        r.in = a->src; r.out = a->out; r.key = s.key_in; r.pay = s.pay_in; r.w = s.w_in;
        r.part = (float *)(ws + L.part);
        r.n = a->nnz; r.n_vocab = a->n_vocab; r.n_rows = a->n_rows; r.ld_in = a->ld_src; r.ld_out = a->ld_out;
        r.chunks = L.chunks; r.chunk = L.chunk; r.dim = (int)a->dim; r.accumulate = a->accumulate; r.scale = a->scale;
        TRY(with_group<VecOf<T>::N>(a->dim / L.slabs, [&](auto gc, auto nc) {
            constexpr int G = decltype(gc)::value, N = decltype(nc)::value, GROUPS = 256 / G;
            r.slabs = (int)ceil_div(a->dim, G * N);
            r.by_xcd = L.slabs > 1;
            const i64 blocks = r.by_xcd ? ceil_div(ceil_div(L.chunks, GROUPS), 8 / r.slabs) * 8 : ceil_div(L.chunks * r.slabs, GROUPS);
            hipLaunchKernelGGL((sp_embed_reduce_kernel<T, TO, G, N>), dim3((unsigned)blocks), dim3(256), 0, stream, r);
            if (L.chunks > 1) hipLaunchKernelGGL((sp_embed_join_kernel<TO, G, N>), dim3((unsigned)(ceil_div(L.chunks - 1, GROUPS) * r.slabs)), dim3(256), 0, stream, r);
            return (int)SP_OK;
        }));
    }
    HIP_TRY(hipGetLastError());
    return SP_OK;
}

// ---- score adjustment ------------------------------------------------------------------------------------------------------------

int check_pattern(const sp_csr_pattern &m, const char *what) {
    if (!m.indptr) return SP_OK;
    if (m.n_rows < 0 || m.nnz < 0) return fail(SP_EINVAL, "%s: negative size", what);
    if (m.nnz > 0 && !m.indices) return fail(SP_EINVAL, "%s: NULL indices", what);
    return SP_OK;
}
constexpr i64 AD_WGS = 2048;
CsrPattern pattern_of(const sp_csr_pattern &m) { return {m.indptr, m.indices, m.n_rows, m.nnz, m.index64}; }

template <typename T> int launch_adjust(AdjustParams p, bool counts, hipStream_t stream) {
    // A row in segments of up to AD_SEG columns; few rows in shorter ones, down to 2048, so that about AD_WGS workgroups run.  (512 / 1024 / 2048 / 4096
    // of them: 64 x 100 000 f16 with target lists 21 / 19 / 16.6 / 17.4 us, 512 x 10 000 bf16 with a history, a filter and a bias 18.7 / 15.0 / 13.0 / 14.2.)
    i64 segs = ceil_div(p.n_cols, AD_SEG);
    const i64 want = ceil_div(AD_WGS, p.n_rows), most = ceil_div(p.n_cols, 2048);
    if (segs < want) segs = want < most ? want : most;
    p.seg = (int)(ceil_div(ceil_div(p.n_cols, segs), 2048) * 2048);
    p.segs = (int)ceil_div(p.n_cols, p.seg);
    const i64 blocks = p.n_rows * p.segs;
    if (too_many(blocks, AD_NT)) return fail(SP_EINVAL, "too many rows for one launch");
    if (counts) hipLaunchKernelGGL((sp_adjust_kernel<T, true>), dim3((unsigned)blocks), dim3(AD_NT), 0, stream, p);
    else hipLaunchKernelGGL((sp_adjust_kernel<T, false>), dim3((unsigned)blocks), dim3(AD_NT), 0, stream, p);
    HIP_TRY(hipGetLastError());
    return SP_OK;
}

// ---- distillation ------------------------------------------------------------------------------------------------------------------

enum { DISTILL_LOSS = 1, DISTILL_GRAD = 2 };
constexpr int DI_NT = 512;                               // threads of a workgroup
constexpr i64 SCAN_WGS = 512, GRAD_WGS = 2048;           // workgroups that few rows are cut for
constexpr i64 CACHE_BYTES = 256 << 20;                   // between the L2s and the memory

int check_distill(const sp_distill_args *a, int what) {
    if (!a || a->struct_size != sizeof(sp_distill_args)) return fail(SP_EINVAL, "sp_distill_args size mismatch");
    if (a->flags) return fail(SP_EINVAL, "flags must be 0");
    if (bad_dtype(a->dtype) || bad_dtype(a->values_dtype)) return fail(SP_EINVAL, "bad dtype");
    if (a->n_rows < 0 || a->n_rows > I32_MAX || a->n_cols < 0 || a->n_cols > COLS_MAX) return fail(SP_EINVAL, "bad shape");
    if (a->k < 0 || a->k > SP_DISTILL_KMAX) return fail(SP_EINVAL, "k = %d out of range [0, %d]", a->k, SP_DISTILL_KMAX);
    if (!(a->temperature > 0.f) || a->temperature > 1e30f || a->temperature < 1e-30f) return fail(SP_EINVAL, "temperature must be positive");
    if (a->n_rows == 0) return SP_OK;
    if (too_many(a->n_rows + GRAD_WGS, DI_NT)) return fail(SP_EINVAL, "too many rows for one launch");
    if ((a->n_cols > 0 && !a->student) || (a->k > 0 && (!a->cols || !a->values))) return fail(SP_EINVAL, "NULL pointer");
    if (what & DISTILL_GRAD) {
        if (a->n_cols > 0 && !a->grad) return fail(SP_EINVAL, "grad is NULL");
        if (what == DISTILL_GRAD && !a->stats) return fail(SP_EINVAL, "stats is NULL");
    }
    return SP_OK;
}

// Workgroups of a row: few rows are cut so that about `want` workgroups run, in pieces of at least `piece` bytes; rows of less than `whole` are not.
int splits_of(const sp_distill_args *a, i64 want, i64 whole, i64 piece) {
    const i64 bytes = a->n_cols * (a->dtype == SP_DT_F32 ? 4 : 2);
    if (a->n_rows <= 0 || bytes < whole) return 1;
    const i64 s = ceil_div(want, a->n_rows), most = bytes / piece;
    return (int)(s > most ? most : s);
}
// A row in pieces needs a second launch for the loss: 1 row of 200 KB whole / in pieces 9 / 13 us, 256 rows 13 / 18; 64 rows of 400 KB 18 / 13,
// 256 rows 29 / 25; 1 row of 1.2 MB 22 / 12.  (With pieces for 1024 workgroups 512 rows of 200 .. 1200 KB take 4 .. 8 % longer.)
int scan_splits(const sp_distill_args *a) { return splits_of(a, SCAN_WGS, 384 << 10, 128 << 10); }
// The gradient: every piece reads the row's list again, 2048 workgroups are worth that only where the scores come from memory.  (2048 / 1024:
// 1024 x 84 432 float32 with the loss 231 / 242 us, 512 x 200 000 259 / 265, 256 x 100 000 80 / 75, 512 x 100 000 bf16 83 / 77.  Pieces of 4 KB: 64 x
// 40 000 float32 31 us, of 32 KB 23.5, of 64 KB 24.4.)
int grad_splits(const sp_distill_args *a) {
    const bool cached = a->n_rows * a->n_cols * (a->dtype == SP_DT_F32 ? 4 : 2) <= CACHE_BYTES;
    return splits_of(a, cached ? GRAD_WGS / 2 : GRAD_WGS, 64 << 10, 32 << 10);
}
i64 chunk_of(const sp_distill_args *a, int splits) { return ceil_div(ceil_div(a->n_cols, splits), 64) * 64; }

// The one-call kernel keeps `nt * 16` vectors of 16 bytes in registers and more in a share of the LDS of a CU that `wgs` workgroups have.
constexpr i64 LDS_BYTES = 163840;
i64 lds_room(const sp_distill_args *a, int nt, int wgs) {
    const i64 r = (LDS_BYTES / wgs - ListLds::grad_bytes(a->k, nt) - 512) / 16;
    return r < 0 ? 0 : r;
}
// It is taken from as many rows on as fill the card, a workgroup each, and for fewer rows that a CU can keep: one launch instead of three.  (One
// kernel / scan, join and gradient: 1 row of 40 000 bf16 12.0 / 16.1 us, of 100 000 17.7 / 16.0, of 100 000 float32 14.2 / 16.1; 64 rows 12.1 / 23.4,
// 22.6 / 29.2, 19.6 / 31.2.  Rows of 300 000 bf16, which are not kept: 1 36 / 16, 64 42 / 37, 128 49 / 53; 256 of 100 000 bf16 28 / 44.)
constexpr i64 FUSED_ROWS = 256;
bool one_kernel(const sp_distill_args *a) {
    return a->n_rows >= FUSED_ROWS || a->n_cols / (a->dtype == SP_DT_F32 ? 4 : 8) <= 16 * 1024 + lds_room(a, 1024, 1);
}

// the workspace: row statistics between the two halves of a call that is not one kernel, and the partial ones of rows in several pieces
size_t distill_stats_bytes(const sp_distill_args *a) { return one_kernel(a) ? 0 : ((size_t)a->n_rows * 8 + 255) & ~(size_t)255; }
i64 distill_ws_bytes(const sp_distill_args *a, bool grad) {
    if (grad && one_kernel(a)) return 0;
    const int splits = scan_splits(a);
    return (grad ? (i64)distill_stats_bytes(a) : 0) + (splits > 1 ? a->n_rows * splits * 8 : 0);
}
int check_workspace(const void *ws, i64 have, i64 need) {
    if (need > 0 && (!ws || have < need)) return fail(SP_EWORKSPACE, "workspace too small: need %lld bytes, got %lld", need, ws ? have : 0ll);
    return SP_OK;
}

DistillParams distill_params(const sp_distill_args *a, bool both = false) {
    DistillParams p{};
    p.student = a->student; p.grad = a->grad;
    p.n_rows = a->n_rows; p.n_cols = a->n_cols; p.ld_student = a->ld_student; p.ld_grad = a->ld_grad;
    p.k = a->k; p.cols64 = a->cols64; p.values_dtype = a->values_dtype;
    p.tau = a->temperature; p.inv_tau = 1.f / a->temperature; p.c = (float)(1.4426950408889634074 / (double)a->temperature);
    p.cols = a->cols; p.values = a->values; p.counts = a->counts; p.teacher_lse = a->teacher_lse;
    p.loss = a->loss; p.stats = a->stats; p.grad_loss = a->grad_loss;
    p.part = (float *)((unsigned char *)a->workspace + (both ? distill_stats_bytes(a) : 0));
    return p;
}

// a kernel's limit of dynamic LDS is raised where a launch needs more than every kernel may have
int allow_lds(const void *kernel, size_t bytes) {
    if (bytes > 48 * 1024) HIP_TRY(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return SP_OK;
}

int launch_scan(const sp_distill_args *a, DistillParams p, hipStream_t stream) {
    p.splits = scan_splits(a);
    p.chunk = chunk_of(a, p.splits);
    const size_t lists = (size_t)ListLds::loss_bytes(a->k);
    return with_type(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        TRY(allow_lds((const void *)sp_distill_scan_kernel<T, DI_NT>, lists));
        TRY(allow_lds((const void *)sp_distill_join_kernel<T>, lists));
        hipLaunchKernelGGL((sp_distill_scan_kernel<T, DI_NT>), dim3((unsigned)(a->n_rows * p.splits)), dim3(DI_NT), lists, stream, p);
        if (p.splits > 1) hipLaunchKernelGGL((sp_distill_join_kernel<T>), dim3((unsigned)a->n_rows), dim3(64), lists, stream, p);
        HIP_TRY(hipGetLastError());
        return (int)SP_OK;
    });
}
int launch_grad(const sp_distill_args *a, DistillParams p, hipStream_t stream) {
    p.splits = grad_splits(a);
    p.chunk = chunk_of(a, p.splits);
    return with_type(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        const size_t lists = (size_t)ListLds::grad_bytes(a->k, DI_NT);
        TRY(allow_lds((const void *)sp_distill_grad_kernel<T, DI_NT>, lists));
        hipLaunchKernelGGL((sp_distill_grad_kernel<T, DI_NT>), dim3((unsigned)(a->n_rows * p.splits)), dim3(DI_NT), lists, stream, p);
        HIP_TRY(hipGetLastError());
        return (int)SP_OK;
    });
}

}  // namespace

extern "C" {

int sp_embed_rows(const sp_embed_args *a) {
    sp_set_error(0, "");
    TRY(check_embed(a));
    if (a->out_dtype != a->dtype) return fail(SP_EINVAL, "out_dtype must be the table's dtype");
    if (a->n_rows == 0 || a->dim == 0) return SP_OK;
    if (!a->out || (a->n_vocab > 0 && !a->src)) return fail(SP_EINVAL, "NULL table or out");
    if (a->n_rows > 1 && a->ld_out < a->dim) return fail(SP_EINVAL, "rows of out overlap");
    TRY(check_embed_launch(a));
    OnDevice dev;
    TRY(dev.enter(a->device));
    return run_embed(a);
}

int64_t sp_embed_rows_grad_workspace_bytes(const sp_embed_args *a) {
    TRY(check_embed(a));
    return (int64_t)grad_layout(a).total;
}

int sp_embed_rows_grad(const sp_embed_args *a) {
    sp_set_error(0, "");
    TRY(check_embed(a));
    if (a->out_dtype != a->dtype && a->out_dtype != SP_DT_F32) return fail(SP_EINVAL, "out_dtype must be dtype or SP_DT_F32");
    if (a->n_vocab == 0 || a->dim == 0) return SP_OK;
    if (!a->out || (a->n_rows > 0 && !a->src)) return fail(SP_EINVAL, "NULL gradient or out");
    if (a->n_vocab > 1 && a->ld_out < a->dim) return fail(SP_EINVAL, "rows of out overlap");
    TRY(check_grad_launch(a));
    TRY(check_workspace(a->workspace, a->workspace_bytes, a->nnz > 0 ? (i64)grad_layout(a).total : 0));
    OnDevice dev;
    TRY(dev.enter(a->device));
    return with_type(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        return a->out_dtype == a->dtype ? run_embed_grad_as<T, T>(a) : run_embed_grad_as<T, float>(a);
    });
}

int sp_adjust_scores(const sp_adjust_args *a) {
    sp_set_error(0, "");
    if (!a || a->struct_size != sizeof(sp_adjust_args)) return fail(SP_EINVAL, "sp_adjust_args size mismatch");
    if (a->flags) return fail(SP_EINVAL, "flags must be 0");
    if (bad_dtype(a->dtype) || (a->bias && bad_dtype(a->bias_dtype))) return fail(SP_EINVAL, "bad dtype");
    if (a->n_rows < 0 || a->n_rows > I32_MAX || a->n_cols < 0 || a->n_cols > COLS_MAX) return fail(SP_EINVAL, "bad shape");
    TRY(check_pattern(a->history, "history"));
    TRY(check_pattern(a->filter, "filter"));
    TRY(check_pattern(a->target, "target"));
    if (a->n_rows == 0 || a->n_cols == 0) return SP_OK;
    if (!a->scores || !a->out) return fail(SP_EINVAL, "NULL scores or out");
    if (a->n_rows > 1 && a->ld_out < a->n_cols) return fail(SP_EINVAL, "rows of out overlap");
    // a history without any penalty changes nothing
    const bool counts = a->history.indptr && (a->repetition || a->presence || a->frequency || a->repetition_all != 1.f || a->presence_all != 0.f || a->frequency_all != 0.f);
    if (counts && !a->repetition && !(a->repetition_all > 0.f)) return fail(SP_EINVAL, "repetition_all must be positive");
    OnDevice dev;
    TRY(dev.enter(a->device));
    AdjustParams p{};
    p.scores = a->scores; p.out = a->out; p.n_rows = a->n_rows; p.n_cols = a->n_cols; p.ld_scores = a->ld_scores; p.ld_out = a->ld_out;
    p.targets = a->targets; p.targets64 = a->targets64; p.bias_dtype = a->bias_dtype;
    p.history = pattern_of(a->history); p.filter = pattern_of(a->filter); p.target = pattern_of(a->target);
    p.repetition = a->repetition; p.presence = a->presence; p.frequency = a->frequency;
    p.repetition_all = a->repetition_all; p.presence_all = a->presence_all; p.frequency_all = a->frequency_all;
    p.bias = a->bias; p.ld_bias = a->ld_bias; p.allowed = a->allowed; p.ld_allowed = a->ld_allowed;
    return with_type(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        return launch_adjust<T>(p, counts, (hipStream_t)a->stream);
    });
}

int64_t sp_distill_workspace_bytes(const sp_distill_args *a) {
    if (!a || a->struct_size != sizeof(sp_distill_args)) return fail(SP_EINVAL, "sp_distill_args size mismatch");
    if (a->n_rows < 0 || a->n_rows > I32_MAX || a->n_cols < 0 || a->n_cols > COLS_MAX) return fail(SP_EINVAL, "bad shape");
    return (int64_t)distill_ws_bytes(a, a->grad != nullptr);
}

int sp_distill_loss(const sp_distill_args *a) {
    sp_set_error(0, "");
    TRY(check_distill(a, DISTILL_LOSS));
    if (a->n_rows == 0) return SP_OK;
    TRY(check_workspace(a->workspace, a->workspace_bytes, distill_ws_bytes(a, false)));
    OnDevice dev;
    TRY(dev.enter(a->device));
    return launch_scan(a, distill_params(a), (hipStream_t)a->stream);
}

int sp_distill_grad(const sp_distill_args *a) {
    sp_set_error(0, "");
    TRY(check_distill(a, DISTILL_GRAD));
    if (a->n_rows == 0 || a->n_cols == 0) return SP_OK;
    if (a->n_rows > 1 && a->ld_grad < a->n_cols) return fail(SP_EINVAL, "rows of grad overlap");
    OnDevice dev;
    TRY(dev.enter(a->device));
    return launch_grad(a, distill_params(a), (hipStream_t)a->stream);
}

int sp_distill_loss_grad(const sp_distill_args *a) {
    sp_set_error(0, "");
    TRY(check_distill(a, DISTILL_LOSS | DISTILL_GRAD));
    if (a->n_rows == 0) return SP_OK;
    if (a->n_rows > 1 && a->ld_grad < a->n_cols) return fail(SP_EINVAL, "rows of grad overlap");
    TRY(check_workspace(a->workspace, a->workspace_bytes, distill_ws_bytes(a, true)));
    OnDevice dev;
    TRY(dev.enter(a->device));
    hipStream_t stream = (hipStream_t)a->stream;
    DistillParams p = distill_params(a, true);
    if (!one_kernel(a)) {
        p.stats = (float *)a->workspace;
        TRY(launch_scan(a, p, stream));
        return launch_grad(a, p, stream);
    }
    return with_type(a->dtype, [&](auto tag) {
        using T = decltype(tag);
        // The row in registers and LDS, by the smallest kind of workgroup that holds all of it: 8 of 256 threads on a CU, 4 or 2 of 512, one
        // of 1024; the last one takes longer rows as well, and reads the rest twice.
        const i64 vecs = a->n_cols / VecOf<T>::N;
        auto room = [&](int nt, int wgs) { return lds_room(a, nt, wgs); };
        auto launch = [&](auto kernel, int nt, int rv, int wgs) {
            const i64 more = vecs - (i64)nt * rv;
            p.stage = (int)(more < 0 ? 0 : more < room(nt, wgs) ? more : room(nt, wgs));
            const size_t lds = (size_t)(ListLds::grad_bytes(a->k, nt) + (i64)p.stage * 16);
            TRY(allow_lds((const void *)kernel, lds));
            hipLaunchKernelGGL(kernel, dim3((unsigned)a->n_rows), dim3((unsigned)nt), lds, stream, p);
            HIP_TRY(hipGetLastError());
            return (int)SP_OK;
        };
        if (vecs <= 4 * 256 + room(256, 8)) return launch(sp_distill_loss_grad_kernel<T, 256, 4>, 256, 4, 8);
        if (vecs <= 4 * 512 + room(512, 4)) return launch(sp_distill_loss_grad_kernel<T, 512, 4>, 512, 4, 4);
        if (vecs <= 16 * 512 + room(512, 2)) return launch(sp_distill_loss_grad_kernel<T, 512, 16>, 512, 16, 2);
        return launch(sp_distill_loss_grad_kernel<T, 1024, 16>, 1024, 16, 1);
    });
}

}  // extern "C"
