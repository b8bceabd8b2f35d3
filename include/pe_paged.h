/*
 * pe_paged.h — C ABI of the paged key/value cache in libpe_attn.so (gfx950): attention over pages,
 * rotary positions, the write of new tokens into pages and copies of pages.
 *
 * Conventions are pe_attn.h's: plain pointers and sizes, status codes (pe_attn_strerror) and no
 * exceptions, launches on the caller's stream on the current device, no allocation, no
 * synchronisation, no device-to-host read, so every entry point can be captured into a HIP graph.
 *
 * A cache holds k and v in pages of page_size tokens each. Page x, slot t and kv head h of k is the row
 *   k_pages + x * k_stride_page + t * k_stride_token + h * k_stride_head   (head_dim elements)
 * and key j of sequence s is slot j % page_size of page page_table[s * table_stride + j / page_size].
 * An entry outside [0, n_pages) (-1 by convention) maps no page: attention treats its keys as masked,
 * pe_paged_append_fwd drops their rows.
 *
 * The call's new tokens are packed: sequence s has rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1
 * (cu_seqlens does not descend), and
 * they are the last of its seqlens_k[s] keys: row r of Lq sits at key position seqlens_k[s] - Lq + r.
 */
#ifndef PE_PAGED_H
#define PE_PAGED_H

#include "pe_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PE_PAGED_PAGE_MULTIPLE 16    /* page_size is a multiple of this */
#define PE_PAGED_MAX_KEYS (1 << 29) /* largest max_seqlen_k and window, else PE_ATTN_EUNSUPPORTED */

/* Attention of the new tokens (their k and v already in the pages):
 *     allowed(i, j) = j < seqlens_k && (window_left < 0 || i - j <= window_left)
 *                  && (window_right < 0 || j - i <= window_right) && (!causal || j <= i)
 *                  && key j's page is mapped                      (i, j key positions)
 *     out[i] = sum_j softmax_j(scale * q_i . k_j over allowed j) * v_j
 * with pe_attn.h's arithmetic. A row that reaches no key is zero. k and v of keys a row may not
 * reach do not enter it, whatever they hold (infinities and NaN included), nor what pages hold past
 * a sequence's keys. A sequence with more rows than max_seqlen, or more keys than max_seqlen_k or
 * than its table's max_pages pages hold, or a negative count, is skipped: its rows are not written,
 * like those at or beyond cu_seqlens[n_seq]. */
typedef struct pe_paged_args {
    uint32_t struct_size; /* sizeof(pe_paged_args) */
    int32_t dtype;        /* PE_ATTN_DTYPE_BF16 */
    const void *q;        /* [total_tokens, n_heads_q, head_dim] */
    const void *k_pages;  /* [n_pages, page_size, n_heads_kv, head_dim] by the strides */
    const void *v_pages;
    void *o;                   /* [total_tokens, n_heads_q, head_dim] (written); overlaps no input */
    const int32_t *page_table; /* device [n_seq, max_pages] */
    const int32_t *cu_seqlens; /* device [n_seq + 1] */
    const int32_t *seqlens_k;  /* device [n_seq] */
    /* strides in elements; the head_dim stride is 1. Base pointers 16-byte aligned, strides of q, k, v
       and o non-negative multiples of 8. */
    int64_t q_stride_token, q_stride_head;
    int64_t k_stride_page, k_stride_token, k_stride_head;
    int64_t v_stride_page, v_stride_token, v_stride_head;
    int64_t o_stride_token, o_stride_head;
    int64_t table_stride; /* of a sequence, in int32 entries */
    int32_t n_seq;
    int32_t total_tokens;
    int32_t max_seqlen;   /* host bound on the new tokens of a sequence */
    int32_t max_seqlen_k; /* host bound on its keys */
    int32_t n_heads_q;
    int32_t n_heads_kv; /* divides n_heads_q */
    int32_t head_dim;   /* 64, 128 or 256 */
    int32_t n_pages;
    int32_t page_size; /* a multiple of PE_PAGED_PAGE_MULTIPLE */
    int32_t max_pages; /* entries of a sequence in page_table */
    float softmax_scale;
    int32_t window_left;  /* -1: unbounded */
    int32_t window_right; /* -1: unbounded */
    int32_t causal;       /* 0 or 1; causal is window_right = 0 */
} pe_paged_args;

/* Bytes of device workspace pe_paged_attn_fwd needs (host-only, from the sizes): the partial rows of a
   call whose keys are split over workgroups, else 0. At most 256 MiB. */
int pe_paged_workspace_size(const pe_paged_args *args, size_t *bytes);

/* The workspace is 16-byte aligned, holds nothing between calls, and may be shared by calls that are
   ordered on one stream. */
int pe_paged_attn_fwd(const pe_paged_args *args, void *workspace, size_t workspace_bytes, hipStream_t stream);

/* Rotary positions: pair i < half of a head of token t is elements (i, i + half), or (2 i, 2 i + 1)
 * when interleaved, of its first 2 * half elements, turned by positions[t] * inv_freq[i] (or by its
 * opposite: the gradient) and scaled:
 *     a' = scale * (a cos - b sin),  b' = scale * (b cos + a sin)
 * in fp32 (the angle's reduction in fp64), rounded once; the head's other elements are copied. out
 * may be x itself when x is contiguous, and overlaps no input otherwise. */
#define PE_ROTARY_BF16 1
#define PE_ROTARY_FP16 2
#define PE_ROTARY_FP32 3
#define PE_ROTARY_MAX_PAIRS 256
typedef struct pe_rotary_args {
    uint32_t struct_size; /* sizeof(pe_rotary_args) */
    int32_t dtype;        /* PE_ROTARY_* */
    const void *x;        /* [n_tokens, n_heads, head_dim] by the strides (elements; head_dim's is 1) */
    void *out;            /* [n_tokens, n_heads, head_dim], contiguous (written) */
    const void *positions; /* device [n_tokens], int64 or (positions_32) int32 */
    const float *inv_freq; /* device [half] */
    int64_t x_stride_token, x_stride_head;
    int64_t n_tokens;
    int32_t n_heads;
    int32_t head_dim;
    int32_t half; /* 1 .. PE_ROTARY_MAX_PAIRS, 2 * half <= head_dim */
    int32_t positions_32;
    int32_t interleaved; /* 0 or 1 */
    int32_t inverse;     /* 1: the opposite angle */
    float scale;
} pe_rotary_args;

int pe_rotary_fwd(const pe_rotary_args *args, hipStream_t stream);

/* New tokens into the pages: row r of sequence s goes to the slot of its key position. k is rotated as
 * pe_rotary_fwd does (bf16) by that position, v is copied; with q, its rows are rotated likewise into
 * q_out. half 0 rotates nothing. Rows whose position is negative, beyond the table, or in no mapped
 * page are dropped; rows at or beyond cu_seqlens[n_seq] are left alone. Two tokens of one call may not
 * share a slot. */
typedef struct pe_append_args {
    uint32_t struct_size; /* sizeof(pe_append_args) */
    int32_t dtype;        /* PE_ATTN_DTYPE_BF16 */
    const void *q;        /* optional [total_tokens, n_heads_q, head_dim]; NULL for none */
    void *q_out;          /* contiguous, with q (written); overlaps no input */
    const void *k;        /* [total_tokens, n_heads_kv, head_dim] */
    const void *v;
    void *k_pages; /* written */
    void *v_pages;
    const int32_t *page_table;
    const int32_t *cu_seqlens;
    const int32_t *seqlens_k;
    const float *inv_freq; /* device [half] */
    int64_t q_stride_token, q_stride_head;
    int64_t k_stride_token, k_stride_head;
    int64_t v_stride_token, v_stride_head;
    int64_t kp_stride_page, kp_stride_token, kp_stride_head; /* of k_pages */
    int64_t vp_stride_page, vp_stride_token, vp_stride_head; /* of v_pages */
    int64_t table_stride;
    int32_t n_seq;
    int32_t total_tokens;
    int32_t n_heads_q; /* 0 without q */
    int32_t n_heads_kv;
    int32_t head_dim; /* a multiple of 8 */
    int32_t n_pages;
    int32_t page_size;
    int32_t max_pages;
    int32_t half;
    int32_t interleaved;
    float rope_scale;
} pe_append_args;

int pe_paged_append_fwd(const pe_append_args *args, hipStream_t stream);

/* Copies page src[i] to page dst[i], i < n_pairs, in each of n_bases caches: a page is page_bytes bytes
 * (a multiple of 16, as are page_stride and the bases) at base + page * page_stride. bases, src and dst
 * are host arrays, read before the call returns. Pages lie in [0, n_pages); a page is the target of at
 * most one pair and then no pair's source (else PE_ATTN_EINVAL and nothing is copied). */
int pe_copy_pages(void *const *bases, int32_t n_bases, int64_t page_stride, int64_t page_bytes, int32_t n_pages,
                  const int32_t *src, const int32_t *dst, int32_t n_pairs, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* PE_PAGED_H */
