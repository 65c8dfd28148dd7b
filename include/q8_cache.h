/*
 * C-ABI of the operators between a decoder block's products, in
 * libsgemm_shim.so (gfx950): positions, a paged cache of 8-bit keys and values,
 * and attention over it.
 *
 *   q8_rotary        heads turned by their tokens' positions, on one or several
 *                    axes; and turned back (the gradient)
 *   q8_cache_write   new tokens' keys and values to 8 bits, into their pages
 *   q8_cache_read    and back
 *   q8_attention     attention of each sequence's new tokens over its cache: one
 *                    token each (decoding), chunks, whole prompts
 *
 * Conventions, handle, types and 8-bit rows are those of q8_shim.h.  Besides:
 *   - A token is a row; its heads follow one another in it, `dim` values each.
 *     Rows lie `ld` values apart, so queries, keys and values may be columns of
 *     one product's rows.
 *   - An 8-bit row is one head of one token, with its own scale.
 *   - What lies in device memory (positions, starts, lengths, table) is read when
 *     the work runs, not when it is enqueued: a captured call serves other values
 *     of the same sizes.  No value there makes a kernel read or write outside
 *     the tensors that the call names.
 * No counterpart in the reference, which multiplies FP32 matrices only.
 */
#ifndef Q8_CACHE_H
#define Q8_CACHE_H

#include "q8_shim.h"

#ifdef __cplusplus
extern "C" {
#endif

#define Q8_MAX_DIM 256u     /* values of a head */
#define Q8_MAX_AXES 8u

/* How positions turn a head's values: the first 2 pairs of them in pairs, the
 * rest not at all. */
typedef struct q8_rotation {
    uint32_t dim;           /* 1 .. Q8_MAX_DIM */
    uint32_t pairs;         /* 2 pairs <= dim */
    uint32_t axes;          /* 1 .. Q8_MAX_AXES: time; time, height, width; ... */
    uint32_t neighbours;    /* 0: pair j is values j and pairs + j;  1: 2j and 2j + 1 */
    uint8_t axis[128];      /* of each pair, below axes */
} q8_rotation;

/* Keys and values of one layer in pages of `page_tokens` tokens.  The row of a
 * page's slot and head is
 *     k + ((page * heads + head) * page_tokens + slot) * row_bytes
 * with row_bytes = dim rounded up to 16 (what lies past dim is 0 once written),
 * its scale k_scale[(page * heads + head) * page_tokens + slot]; v likewise.
 * k and v are aligned to 16 bytes. */
typedef struct q8_cache {
    int8_t* k;
    int8_t* v;
    float* k_scale;
    float* v_scale;
    uint32_t pages;
    uint32_t page_tokens;
    uint32_t heads;
    uint32_t dim;           /* 1 .. Q8_MAX_DIM */
} q8_cache;

/* Sequences and their new tokens (chunks).  Sequence b's chunk is rows
 * starts[b] .. starts[b + 1] of the tokens; lengths[b] counts its tokens in all,
 * the chunk's, which are the last ones, among them; and its token at position p
 * lies in page table[b * table_ld + p / page_tokens], slot p % page_tokens.
 * A page below 0 or not below `pages` stands for one that is not there, and so
 * does every position from width * page_tokens on.  Starts ascend; what of
 * them lies outside 0 .. tokens is cut off. */
typedef struct q8_batch {
    const int32_t* starts;      /* seqs + 1, on the device */
    const int32_t* lengths;     /* seqs */
    const int32_t* table;       /* seqs rows of `width` pages */
    uint32_t seqs;
    uint32_t tokens;            /* rows that the tensors have */
    uint32_t width;
    uint32_t table_ld;
    uint32_t longest;           /* tokens of the longest chunk, as far as known; 0: not known.  It chooses
                                 * between kernels; another value gives the same results to rounding. */
} q8_batch;

/* y = x with the heads turned: with a = positions[axis_j * ldp + i] freq_j for
 * pair j of token i,
 *     (y1, y2) = (x1 cos a - x2 sin a, x2 cos a + x1 sin a),
 * or with -a where `inverse` is not 0, which takes the gradient of y to that of x.
 * a is exact to 2^-52 of a turn for |a| below 2^40, sine and cosine are FP32 values; the
 * other values are copied.  freq has `pairs` values.  y may be x (same pointer
 * and ld). */
int q8_rotary(q8_handle* h, int dtype, const q8_rotation* form, const void* x, uint32_t ldx, const int32_t* positions,
              uint32_t ldp, const float* freq, void* y, uint32_t ldy, uint32_t tokens, uint32_t heads, int inverse);

/* Keys and values of the chunks' tokens (rows of cache->heads heads) into their
 * pages, as q8_quantize would round each head.  A token whose page is not
 * there, or whose position is below 0, is left out.  If two tokens have one place,
 * what it holds afterwards is not defined. */
int q8_cache_write(q8_handle* h, int dtype, const q8_cache* cache, const q8_batch* batch, const void* k, uint32_t ldk,
                   const void* v, uint32_t ldv);

/* The chunks' tokens read back, as q8_dequantize does; where a page is not there,
 * zeros.  (Starts that count whole sequences read all of them.)  Rows of no chunk
 * are left as they are. */
int q8_cache_read(q8_handle* h, int dtype, const q8_cache* cache, const q8_batch* batch, void* k, uint32_t ldk, void* v,
                  uint32_t ldv);

/* Row i of `out`, head a: the chunk's token at position p = lengths[b] - n + i of
 * a chunk of n tokens attends to the keys of head a / (heads / cache->heads) at positions
 * 0 .. p below lengths[b], with `window` > 0 only to the last `window` of them,
 * and to no page that is not there:
 *     t_j = scale sum_d q_d k_jd,  out = sum_j exp(t_j) v_j / sum_j exp(t_j)
 *     lse = log sum_j exp(t_j)           (FP32, tokens x heads; may be NULL)
 * with scale in -2^100 .. 2^100.
 * A row that attends to nothing is 0, its lse -infinity; one of a NaN scale that it sees is NaN.
 * Rows of no chunk are left as they are.  The scores are FP32 values of any size; one below -2^100 counts
 * as not there.  Sums are in FP32; exp(t_j) sv_j, sv_j the scale of v_j, is rounded to 11 bits before its product with
 * the 8-bit values, or to 2^-31 of the row's largest exp(t_i) max(|sv_i|, 2^-100); in Q8_F32 not at all.  An exp(t_j)
 * below 2^-132 of that largest product counts as 0.  Scales may be 0. */
int q8_attention(q8_handle* h, int dtype, const q8_cache* cache, const q8_batch* batch, uint32_t heads, const void* q,
                 uint32_t ldq, float scale, uint32_t window, void* out, uint32_t ldo, float* lse);

/* The workspace that q8_attention takes with these sizes (the pointers in cache
 * and batch are not looked at); q8_cache_write, q8_cache_read and q8_rotary take none. */
int q8_attention_workspace(int dtype, const q8_cache* cache, const q8_batch* batch, uint32_t heads, size_t* bytes);

#ifdef __cplusplus
}
#endif

#endif /* Q8_CACHE_H */
