/*
 * sp_dense.h — C ABI of the operators on DENSE tensors that libsimilaripy_hip.so offers next to the sparse kernel
 * (include/sp_knn.h): what stands on either side of the top-k lists when a model with an embedding table learns from
 * them or is served with the same selectors.
 *
 *   sp_embed_rows        rows of a CSR (histories: ids and weights) times an embedding table; a plain lookup is the CSR
 *                        whose rows hold one entry each
 *   sp_embed_rows_grad   the gradient of the table: the CSR's transpose times the gradient of the rows, by sorted ids
 *   sp_adjust_scores     penalties for repeated ids, biases and masks on rows of dense scores: the selectors
 *                        (filter_cols, target_cols) and targets of sp_knn_f32_i32, for scores a dense model produced
 *   sp_distill_loss      divergence of a student's dense scores from a teacher's top-k lists, in the layout that
 *                        sp_knn_f32_i32 writes them (cols, values, out_counts)
 *   sp_distill_grad      its gradient, from the row statistics that sp_distill_loss left
 *   sp_distill_loss_grad both in one call
 *
 * Every pointer is device memory on `device`; every call is asynchronous on `stream`, allocates nothing, leaves the
 * calling thread's current device as it was and may be captured into a graph.  `flags` is 0 (reserved).
 * Same conventions as sp_knn.h: plain pointers and sizes, 0 or a negative SP_E* code, sp_last_error().
 * A launch has fewer than 2^32 threads.  A call that would need more is refused with SP_EINVAL, before anything is launched,
 * and has to be cut by the caller.  Threads, with `slabs` = a row's KB rounded up:
 *   lookup          n_rows * slabs * lanes, the 8, 16, 32 or 64 lanes that cover a row (64: from 513 bytes on) by 16 bytes each
 *   bags            n_rows * slabs * 64, n_rows rounded up to a multiple of 4, whatever the width
 *   gradient        256 * slabs for every min(ceil(n_vocab / 512), 2048) ids with up to 1024 entries; for every chunk of the sorted
 *                   entries, of which there are at most 262144 / lanes, with more
 *   adjustment      n_rows * 256 * segments, a segment for every 16384 columns (few rows are cut further, up to 2048 segments)
 *   distillation    (n_rows + 2048) * 512
 * Sums, row statistics and list probabilities are formed in 32 bits or more whatever the type of the tensors.
 */
#ifndef SP_DENSE_H_
#define SP_DENSE_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types of the dense tensors */
#define SP_DT_F32   0
#define SP_DT_BF16  1
#define SP_DT_F16   2

#define SP_DISTILL_KMAX 4096      /* longest list of a row */

typedef struct sp_embed_args {
    uint32_t struct_size;      /* = sizeof(sp_embed_args); checked */
    uint32_t flags;
    int32_t  device;
    int32_t  dtype;            /* SP_DT_*: the table (sp_embed_rows), the gradient of the rows (sp_embed_rows_grad) */
    int32_t  out_dtype;        /* sp_embed_rows: = dtype; sp_embed_rows_grad: dtype or SP_DT_F32 */
    int32_t  index64;          /* 1: indices and indptr are int64, 0: int32 */
    int32_t  accumulate;       /* sp_embed_rows_grad: 1 adds to `out` (rows without entries are not touched), 0 writes all of it */
    float    scale;
    int64_t  n_rows;           /* rows of the CSR */
    int64_t  n_vocab;          /* rows of the table, < 2^31 - 1 */
    int64_t  dim;
    int64_t  nnz;              /* entries of `indices`, < 2^31 */
    int64_t  ld_src;            /* elements between rows of `src` */
    int64_t  ld_out;           /* ... and of `out` */
    const void  *src;          /* sp_embed_rows: table [n_vocab, dim]; sp_embed_rows_grad: gradient of the rows [n_rows, dim] */
    const void  *indices;      /* [nnz]; an id outside [0, n_vocab) contributes nothing */
    const void  *indptr;       /* [n_rows + 1], or NULL: row i holds entry i alone (nnz = n_rows) */
    const float *data;         /* [nnz] weights, or NULL: ones */
    void        *out;          /* sp_embed_rows: [n_rows, dim]; sp_embed_rows_grad: [n_vocab, dim] */
    void        *stream;
    void        *workspace;    /* sp_embed_rows_grad: >= sp_embed_rows_grad_workspace_bytes() */
    int64_t      workspace_bytes;
} sp_embed_args;

/* out[i, :] = scale * sum over the entries j of row i of data[j] * src[indices[j], :], in 32 bits, rounded once.  The order of the additions
 * depends on the sizes and the row alone (groups of lanes take a row's entries in turn, their sums are added as a tree): equal calls give
 * equal bits. */
int sp_embed_rows(const sp_embed_args *args);

/* out[v, :] = scale * sum over the entries j with indices[j] = v of data[j] * src[row of j, :] (+ out[v, :] with accumulate).
 * The entries are sorted by id, stably, and added in ascending j within a chunk of the sorted entries; the sums of an id that has entries in
 * several chunks are joined in their order.  No atomics: equal calls give equal bits. */
int sp_embed_rows_grad(const sp_embed_args *args);
int64_t sp_embed_rows_grad_workspace_bytes(const sp_embed_args *args);

/* a CSR pattern: per-row lists of column ids, in any order, repeats allowed; ids outside [0, n_cols) are passed over */
typedef struct sp_csr_pattern {
    const void *indptr;        /* [n_rows + 1]; NULL: the pattern is not given */
    const void *indices;       /* [nnz] */
    int64_t     n_rows;
    int64_t     nnz;
    int32_t     index64;       /* 1: both arrays are int64, 0: int32 */
    int32_t     _pad0;
} sp_csr_pattern;

typedef struct sp_adjust_args {
    uint32_t struct_size;      /* = sizeof(sp_adjust_args); checked */
    uint32_t flags;
    int32_t  device;
    int32_t  dtype;            /* SP_DT_* of scores and out */
    int64_t  n_rows;
    int64_t  n_cols;           /* < 2^31 - 65536 */
    int64_t  ld_scores;        /* elements between rows */
    int64_t  ld_out;
    const void *scores;        /* [n_rows, n_cols] */
    void       *out;           /* [n_rows, n_cols]; may be `scores` itself (with the same ld) */
    const void *targets;       /* [n_rows] row ids into the three patterns (absolute, as in sp_knn_f32_i32), or NULL: 0 .. n_rows-1;
                                  an id outside a pattern's rows stands for an empty row */
    int32_t  targets64;
    int32_t  bias_dtype;       /* SP_DT_* */
    sp_csr_pattern history;    /* ids whose scores are penalised; the count of a column is how often its row lists it */
    sp_csr_pattern filter;     /* listed columns become -inf */
    sp_csr_pattern target;     /* columns that are NOT listed become -inf */
    const float *repetition;   /* [n_rows] or NULL: all rows repetition_all (> 0 where a history is given) */
    const float *presence;     /* [n_rows] or NULL: presence_all */
    const float *frequency;    /* [n_rows] or NULL: frequency_all */
    float    repetition_all, presence_all, frequency_all;
    int32_t  _pad0;
    const void *bias;          /* [n_cols] (ld_bias 0) or [n_rows, n_cols], or NULL */
    int64_t  ld_bias;
    const uint32_t *allowed;   /* [words] (ld_allowed 0) or [n_rows, words], words = ceil(n_cols / 32); bit c%32 of word c/32 clear: column c becomes -inf; or NULL */
    int64_t  ld_allowed;       /* words between rows */
    void    *stream;
} sp_adjust_args;

/* y = s;  listed c > 0 times in the history: y = (y > 0 ? y / repetition : y * repetition) - presence - frequency * c;
 * y += bias;  y = -inf where a mask says so (also for NaN).  One rounding, at the end. */
int sp_adjust_scores(const sp_adjust_args *args);

typedef struct sp_distill_args {
    uint32_t struct_size;      /* = sizeof(sp_distill_args); checked */
    uint32_t flags;
    int32_t  device;
    int32_t  dtype;            /* SP_DT_* of student and grad */
    int64_t  n_rows;
    int64_t  n_cols;           /* < 2^31 - 65536 */
    int64_t  ld_student;
    int64_t  ld_grad;
    int32_t  k;                /* slots of a list, 0 .. SP_DISTILL_KMAX */
    int32_t  cols64;           /* 1: cols is int64, 0: int32 */
    int32_t  values_dtype;     /* SP_DT_* */
    float    temperature;      /* > 0 */
    const void  *student;      /* [n_rows, n_cols] */
    const void  *cols;         /* [n_rows, k]; entries outside [0, n_cols) are not in the list; a column listed twice counts twice */
    const void  *values;       /* [n_rows, k] the teacher's scores */
    const int32_t *counts;     /* [n_rows] valid slots of each list, or NULL: all k */
    const float *teacher_lse;  /* [n_rows] log-sum-exp of ALL the teacher's scores / temperature, or NULL: p is normalised over the list */
    float   *loss;             /* [n_rows] */
    float   *stats;            /* [n_rows, 2] m = max of student, sum of exp((student - m) / temperature); OUT of sp_distill_loss, IN of sp_distill_grad */
    const float *grad_loss;    /* [n_rows] gradient of the loss of each row, or NULL: ones */
    void    *grad;             /* [n_rows, n_cols]; may be `student` itself (with the same ld) */
    void    *stream;
    void    *workspace;        /* >= sp_distill_workspace_bytes() */
    int64_t  workspace_bytes;
} sp_distill_args;

/* p_j = softmax of values / temperature over the list (or exp(values / temperature - teacher_lse)), q = softmax of student / temperature:
 *   loss = temperature^2 * sum_j p_j (log p_j - log q[cols_j])                  (0 for an empty list; p_j = 0 contributes 0)
 *   grad[v] = grad_loss * temperature * (q[v] * sum_j p_j - sum over cols_j = v of p_j) */
int sp_distill_loss(const sp_distill_args *args);        /* writes loss and stats (either may be NULL) */
int sp_distill_grad(const sp_distill_args *args);        /* reads stats, writes grad */
int sp_distill_loss_grad(const sp_distill_args *args);   /* writes loss (may be NULL) and grad */
int64_t sp_distill_workspace_bytes(const sp_distill_args *args);      /* of sp_distill_loss, or, where `grad` is set, of sp_distill_loss_grad */

#ifdef __cplusplus
}
#endif
#endif /* SP_DENSE_H_ */
