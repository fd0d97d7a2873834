/*
 * Operators of a decoder layer that holds activations, weights and the
 * key/value cache as int8 with scales, for programs that decode token by
 * token on one MI355X.
 *
 * None of these has a counterpart in the reference runtime, whose packages
 * have fixed shapes and no cache: a decoder's rows, lengths and pages change
 * from call to call.  So they are calls of their own beside spkv2_run:
 *
 *  - every pointer is DEVICE memory of the caller's (spkv2_device_malloc, any
 *    HIP allocation), except the argument struct itself, which is read before
 *    the call returns;
 *  - a call enqueues its kernels on `stream` (a hipStream_t of the current
 *    device; NULL is the default stream) and returns without waiting; it
 *    allocates nothing, keeps nothing for a later call and can be captured
 *    into a HIP graph;
 *  - 0: enqueued (also where there is nothing to do); -1: a bad argument;
 *    SPKV2_E_UNSUPPORTED: a size or type that no kernel covers; SPKV2_E_HIP:
 *    the launch failed.  spkv2_mi355x_last_error says which; nothing has been
 *    enqueued then;
 *  - strides count elements, and the last axis of every tensor is contiguous;
 *    rows of any alignment are taken (16-byte aligned ones are faster);
 *  - outputs may not overlap inputs, or each other, except where said.
 *
 * Quantisation is symmetric: a vector of the last axis becomes codes
 * q = rint(127 v / max|v|) in [-127, 127], ties to the even code, and one
 * float scale max|v| / 127.  The codes are those of exact arithmetic, whatever
 * the order of a kernel's sums.  A vector of zeros has scale 0; a vector that
 * holds a NaN or an infinity has scale NaN and codes 0, so that what is
 * computed from it is NaN.
 */
#ifndef SPKV2_DECODER_H
#define SPKV2_DECODER_H

#include <stddef.h>
#include <stdint.h>
#include "spkv2_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of these operators' tensors: SPKV2_DTYPE_FP32, SPKV2_DTYPE_FP16 and
 * this one, which packages do not hold. */
#define SPKV2_DTYPE_BF16 4

/* ---- rows: norm, quantisation ------------------------------------------- */

/* h = x + residual (rounded to the rows' type, as it is stored), then
 * q, scale = quantised h weight / sqrt(mean(h^2) + eps), row by row. */
typedef struct {
    const void *x;        /* [rows, cols] */
    const void *residual; /* [rows, cols], or NULL: h = x */
    const void *weight;   /* [cols], or NULL: ones */
    void *residual_out;   /* [rows, cols]: h; may be x's or residual's own memory (with its stride); NULL: not stored */
    int8_t *q;            /* [rows, cols] */
    float *scale;         /* [rows] */
    int64_t rows, cols;
    int64_t x_stride, residual_stride, residual_out_stride, q_stride; /* elements between rows */
    int32_t dtype;        /* of x, residual and residual_out */
    int32_t weight_dtype; /* dtype, or SPKV2_DTYPE_FP32 */
    int32_t norm;         /* 0: quantise h weight itself, without the norm */
    float eps;            /* at least 0 */
} Spkv2RmsNormI8;
int spkv2_mi355x_rmsnorm_i8(const Spkv2RmsNormI8 *args, void *stream);

/* out = scale q, row by row */
typedef struct {
    const int8_t *q;    /* [rows, cols] */
    const float *scale; /* [rows] */
    void *out;          /* [rows, cols] */
    int64_t rows, cols;
    int64_t q_stride, out_stride;
    int32_t dtype; /* of out */
    int32_t reserved;
} Spkv2DequantizeI8;
int spkv2_mi355x_dequantize_i8(const Spkv2DequantizeI8 *args, void *stream);

/* ---- product ------------------------------------------------------------- */

/* out[m, n] = a_scale[m] b_scale[n] sum_k a[m, k] b[n, k] + bias[n]: sums
 * that are exact up to k = 2^17, of -128 too (larger k is refused, and m above
 * 2^21 or n above 2^26), scaled in fp32 and rounded once to out's type: the same
 * bits whatever the strides and the sizes beside a row and a channel. */
typedef struct {
    const int8_t *a;      /* [m, k]: one row for each token */
    const int8_t *b;      /* [n, k]: one row for each output channel */
    const float *a_scale; /* [m] */
    const float *b_scale; /* [n] */
    const float *bias;    /* [n], or NULL */
    void *out;            /* [m, n] */
    int64_t m, n, k;
    int64_t a_stride, b_stride, out_stride;
    int32_t dtype; /* of out */
    int32_t reserved;
} Spkv2MatmulI8;
int spkv2_mi355x_matmul_i8(const Spkv2MatmulI8 *args, void *stream);
/* name of the kernel that the call takes at these sizes, strides and type
 * ("matmul_tiles<128x128>", ...; its pointers are not looked at; empty: none),
 * for reports and tests */
int spkv2_mi355x_matmul_i8_kernel_name(const Spkv2MatmulI8 *args, char *buf, size_t buf_size);

/* ---- key/value cache ----------------------------------------------------- */

/* A paged cache: pages of page_size tokens, in each of them the heads' codes
 * one after the other, so that a head's page is contiguous.  Token `i` of a
 * sequence is row i % page_size of page table[i / page_size]. */
typedef struct {
    int8_t *k, *v;           /* [pages, kv_heads, page_size, head_dim], 16-byte aligned */
    float *k_scale, *v_scale; /* [pages, kv_heads, page_size], 16-byte aligned */
    int64_t pages;           /* at least 1 */
    int32_t kv_heads;
    int32_t page_size; /* a multiple of 16 */
    int32_t head_dim;  /* a multiple of 16, at most 256 */
    int32_t reserved;
} Spkv2KvCacheI8;

/* Quantises each token's keys and values, head by head, into its slot
 * page * page_size + row.  A token whose slot is negative, or past the cache,
 * is not written.  Two tokens of one call may not have the same slot. */
typedef struct {
    const void *k, *v;    /* [tokens, kv_heads, head_dim], heads contiguous */
    const int64_t *slots; /* [tokens] */
    int64_t tokens;
    int64_t k_stride, v_stride; /* elements between tokens */
    int32_t dtype;              /* of k and v */
    int32_t reserved;
} Spkv2KvWrite;
int spkv2_mi355x_kv_write_i8(const Spkv2KvCacheI8 *cache, const Spkv2KvWrite *args, void *stream);

/* Reads tokens first[s] .. first[s] + offsets[s + 1] - offsets[s] of each
 * sequence s back, scaled, into rows offsets[s] .. of k and v.  Tokens past a
 * table's end, or on a page that the cache does not have, are zeros. */
typedef struct {
    const int32_t *table;   /* [sequences, table_width] */
    const int32_t *first;   /* [sequences], or NULL: zeros */
    const int32_t *offsets; /* [sequences + 1], from 0, not decreasing */
    void *k, *v;            /* [tokens, kv_heads, head_dim], heads contiguous; one of them may be NULL */
    int64_t tokens;         /* rows of k and v: those from offsets[sequences] on are not written */
    int64_t k_stride, v_stride;
    int32_t sequences;
    int32_t table_width; /* pages of a table's row */
    int32_t dtype;       /* of k and v */
    int32_t reserved;
} Spkv2KvRead;
int spkv2_mi355x_kv_read_i8(const Spkv2KvCacheI8 *cache, const Spkv2KvRead *args, void *stream);

/* ---- attention ------------------------------------------------------------ */

/* out = softmax(scale q k^T) v of each sequence's queries and its first
 * lengths[s] cached tokens.  Query head h reads kv head h / (heads / kv_heads).
 * Query i of n is token lengths[s] - n + i of its sequence: causal, it reads
 * the tokens up to itself, and the last `window` of them where window > 0.
 * Not causal (an encoder's states), every query reads all tokens.  A query
 * whose mask leaves nothing (no tokens yet; a position before the first) gets
 * zeros.  Tokens past a table's end, or on a page that the cache does not
 * have, are as masked.
 * The cached codes are read as 16-bit floats, exactly; queries are held with
 * 11 bits (22 for fp32 rows), and to within 2^-39 of their row's largest
 * element; softmax weights times their tokens' value scales with as many, and
 * to within 2^-28 of the largest of those that the row reads; sums and softmax
 * statistics are fp32.  Value scales are meant to lie between 2^-96 and 2^96,
 * where smaller ones lose bits, key scales below 2^64.  A token whose key or
 * value scale is not finite makes the rows that read it NaN, and no other; what
 * a row does not read changes no bit of it.
 *
 * max_queries and max_length bound the sequences' counts of queries and
 * lengths; what a sequence has beyond them is not computed (queries) or not
 * read (tokens).  They set the launch's size and the workspace's: rows of
 * partial sums where one sequence's tokens are split over several workgroups.
 * spkv2_mi355x_attention_i8_workspace gives its size in bytes (0: none is
 * needed).  The workspace need not be cleared and holds nothing after the
 * call's kernels have run; calls on one stream can share it. */
typedef struct {
    const void *q;          /* [queries, heads, head_dim], heads contiguous */
    void *out;              /* [queries, heads, head_dim], heads contiguous */
    const int32_t *table;   /* [sequences, table_width] */
    const int32_t *lengths; /* [sequences] */
    const int32_t *offsets; /* [sequences + 1]: rows of q, from 0, not decreasing */
    void *workspace;        /* 16-byte aligned */
    size_t workspace_size;
    int64_t queries; /* rows of q and out */
    int64_t q_stride, out_stride;
    int64_t max_queries, max_length;
    int32_t sequences;
    int32_t table_width;
    int32_t heads; /* a multiple of the cache's kv_heads */
    int32_t dtype; /* of q and out */
    int32_t causal;
    int32_t window; /* 0: no window; causal only */
    float scale;
    int32_t reserved;
} Spkv2AttentionI8;
int spkv2_mi355x_attention_i8(const Spkv2KvCacheI8 *cache, const Spkv2AttentionI8 *args, void *stream);
/* bytes of workspace that the call needs (its pointers and workspace are not looked at); -1 codes as above */
int spkv2_mi355x_attention_i8_workspace(const Spkv2KvCacheI8 *cache, const Spkv2AttentionI8 *args, size_t *size);
/* name of the kernel that the call takes ("attend_rows<waves=4,splits=3>", ...), likewise, for reports and tests */
int spkv2_mi355x_attention_i8_kernel_name(const Spkv2KvCacheI8 *cache, const Spkv2AttentionI8 *args, char *buf, size_t buf_size);

#ifdef __cplusplus
}
#endif

#endif /* SPKV2_DECODER_H */
