/*
 * manta_cache.h -- the operators of a model that reads what was retrieved (a
 * reranker over a shared question, a model that answers from passages):
 * rotary positions, and a key/value cache of pages held in 8 bits, with its
 * attention and the bookkeeping of its pages.
 *
 * Conventions are manta_rocm.h's: int status and malloc'd message, "_dev"
 * pointers are device addresses, calls are asynchronous on the runtime's
 * stream.  None of the calls below allocates device memory, so all but
 * create / bind may be recorded into a HIP graph.  What only the device can
 * see (an index in a device array) is checked by the kernels: such an entry
 * is skipped, nothing out of range is read or written, and the next
 * synchronizing call (manta_rocm_synchronize / manta_rocm_download) reports
 * it.  A call takes at most 2^25 tokens and 2^21 sequences, attention 2^28
 * rows (tokens * heads).  The reference has no counterpart: its row-wise `rope` kernel
 * (compiler/compiler.go:746-802) rotates f32 rows at positions 0, 1, 2, ...
 */
#ifndef MANTA_CACHE_H
#define MANTA_CACHE_H

#include "manta_rocm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations. */
enum {
    MANTA_ROCM_F32 = 32,
    MANTA_ROCM_F16 = 16,
    MANTA_ROCM_BF16 = 17,
};

/* One activation tensor [tokens, heads, head_dim] and where its result goes.
 * Strides are in elements; head_dim is contiguous, and rows that are written
 * may not run into each other.  out_dev may be x_dev with
 * the same strides; otherwise the two must not overlap. */
typedef struct MantaRocmHeads {
    const void* x_dev;
    void* out_dev;
    int64_t heads;
    int64_t x_token, x_head;
    int64_t out_token, out_head;
} MantaRocmHeads;

/* ---- rotary positions --------------------------------------------------- */

typedef struct MantaRocmRotary MantaRocmRotary;

/* Which columns of the first `rot` make pair p: HALF p and p + rot/2,
 * INTERLEAVED 2p and 2p + 1. */
enum {
    MANTA_ROCM_ROTARY_HALF = 0,
    MANTA_ROCM_ROTARY_INTERLEAVED = 1,
};

/* How frequencies are stretched for contexts longer than a model was trained
 * on (f_p = base^(-2p/rot) radians a token):
 *   NONE    f_p
 *   LINEAR  f_p / factor
 *   BASE    base * factor^(rot/(rot-2)) in place of base (rot > 2)
 *   BLEND   f_p * ((1 - g) / factor + g), g = (turns - low) / (high - low)
 *           cut to [0, 1], turns = original * f_p / (2 pi): pairs that turned
 *           `high` times or more over the trained length stay, those below
 *           `low` are stretched, the rest lie between */
enum {
    MANTA_ROCM_ROTARY_NONE = 0,
    MANTA_ROCM_ROTARY_LINEAR = 1,
    MANTA_ROCM_ROTARY_BASE = 2,
    MANTA_ROCM_ROTARY_BLEND = 3,
};

/* The frequencies of rot/2 pairs, on the host. */
int manta_rocm_rotary_freqs(int64_t rot, double base, int scaling, double factor, double low, double high,
                            double original, double* out, char** err);

/* Bind frequencies (rot/2 of them, radians a token, any finite values).
 * magnitude multiplies the rotated columns (1 for none). */
int manta_rocm_rotary_bind(MantaRocm* rt, const double* freqs, int64_t rot, int layout, double magnitude,
                           MantaRocmRotary** out, char** err);
void manta_rocm_rotary_unbind(MantaRocmRotary* rot);

/* Rotate the first rot columns of each head by the token's angles
 * (positions_dev int32 [tokens]) and copy the others, for up to 4 tensors in
 * one launch (a model's q and k):
 *   y1 = m (x1 cos a - x2 sin a),  y2 = m (x2 cos a + x1 sin a),
 *   a = position * freq,
 * in f32 from angles reduced in f64, rounded once.  inverse != 0 negates the
 * angle: the gradient of x from the gradient of y. */
int manta_rocm_rotary(MantaRocm* rt, const MantaRocmRotary* rot, int dtype, const int32_t* positions_dev,
                      int64_t tokens, int64_t head_dim, const MantaRocmHeads* parts, int64_t nparts, int inverse,
                      char** err);

/* ---- the cache ---------------------------------------------------------- */

typedef struct MantaRocmCache MantaRocmCache;

typedef struct MantaRocmCacheShape {
    int64_t layers;       /* a page holds page_tokens tokens of every layer */
    int64_t pages;
    int64_t page_tokens;  /* 16, 32, 64 or 128 */
    int64_t kv_heads;
    int64_t head_dim;     /* 1 to 256 */
    int64_t seqs;         /* sequence slots */
    int64_t table_pages;  /* pages a sequence may name */
} MantaRocmCacheShape;

/* The cache's device memory, for saving, restoring and inspection:
 *   k_codes int8 [layers][pages][kv_heads][page_tokens][pitch]
 *   v_codes int8 [layers][pages][kv_heads][pitch][page_tokens]
 *   k_max, v_max f32 [layers][pages][kv_heads]: a code stands for
 *     code * max / 127
 *   book int32: refs [pages] (tables naming a page; 0 = free), lengths
 *     [seqs], tables [seqs][table_pages] (-1 past a sequence's pages)
 * pitch is head_dim rounded up to 32; padding codes are 0. */
typedef struct MantaRocmCacheBuffers {
    int8_t* k_codes_dev;
    int8_t* v_codes_dev;
    float* k_max_dev;
    float* v_max_dev;
    int32_t* book_dev;
    int64_t pitch;
    int64_t code_bytes;  /* of k_codes, and of v_codes */
    int64_t max_count;   /* of k_max, and of v_max */
    int64_t book_count;
} MantaRocmCacheBuffers;

/* An empty cache: every page free, every sequence of length 0.  Beside the
 * buffers it holds 96 MiB for attention's partial results. */
int manta_rocm_cache_create(MantaRocm* rt, const MantaRocmCacheShape* shape, MantaRocmCache** out, char** err);
/* Frees the handle and, unless the runtime went first, its device memory. */
void manta_rocm_cache_destroy(MantaRocmCache* cache);
int manta_rocm_cache_shape(const MantaRocmCache* cache, MantaRocmCacheShape* out);
int manta_rocm_cache_buffers(const MantaRocmCache* cache, MantaRocmCacheBuffers* out);

/* -- pages.  The sequence lists are int32 device arrays of n distinct slots.
 * fork and release skip an entry that is wrong and do the others; extend does
 * all of its entries or, where one is wrong or pages are too few, none. */

/* Grow sequences by counts_dev[i] >= 0 tokens: each takes the lowest free
 * pages, in the order of the list; one whose last page is partly filled and
 * shared when the call begins first gets a copy of it (every layer).  The
 * new tokens' contents are undefined until they are appended.  A refused call
 * leaves its sequences as they are until it is reported: appends skip them and
 * extends that name one are refused too, so that the steps that were already
 * on their way (or in a graph) cost nothing that the cache holds. */
int manta_rocm_cache_extend(MantaRocm* rt, MantaRocmCache* cache, const int32_t* seqs_dev, const int32_t* counts_dev,
                            int64_t n, char** err);
/* children_dev[i] (empty, and no parent of this call) takes the first
 * tokens_dev[i] tokens of parents_dev[i] (all when tokens_dev is NULL),
 * sharing its pages. */
int manta_rocm_cache_fork(MantaRocm* rt, MantaRocmCache* cache, const int32_t* parents_dev,
                          const int32_t* children_dev, const int32_t* tokens_dev, int64_t n, char** err);
/* Cut sequences to their first keep_dev[i] tokens (0 when keep_dev is NULL),
 * giving up the pages past them. */
int manta_rocm_cache_release(MantaRocm* rt, MantaRocmCache* cache, const int32_t* seqs_dev, const int32_t* keep_dev,
                             int64_t n, char** err);
/* Move the live pages that lie past the live count into the free ones below
 * it (both in ascending order) and rewrite every table; *live_dev, when
 * given, receives the live count: pages at or past it hold nothing. */
int manta_rocm_cache_compact(MantaRocm* rt, MantaRocmCache* cache, int32_t* live_dev, char** err);
/* Copy pages src_dev[i] to dst_dev[i], every layer; no page of dst_dev occurs
 * twice or in src_dev.  The book is not changed. */
int manta_rocm_cache_copy_pages(MantaRocm* rt, MantaRocmCache* cache, const int32_t* src_dev, const int32_t* dst_dev,
                                int64_t n, char** err);

/* -- contents.  A ragged batch: sequence seqs_dev[i] (i when seqs_dev is
 * NULL) owns rows offsets_dev[i] .. offsets_dev[i+1] (int32 [n+1], ascending,
 * within [0, tokens]) of the activation tensors, and they are its last
 * tokens: with c rows and length l, row j is at position l - c + j.  Rows of
 * negative position are skipped.  Offsets that descend leave rows to nobody or
 * to several sequences (still nothing out of range is read or written);
 * attention may skip such a batch as a whole and report it. */

/* Quantise k and v [tokens, kv_heads, head_dim] of one layer into the pages
 * (extended before; the sequences are distinct, and a page that another table
 * names too is skipped and reported).  Per page and head, max is the largest
 * magnitude of the tokens appended to it since its first, and code =
 * round_half_even(x * 127 / max), in f32; +-127 where x * 127 is past the
 * largest number (magnitudes above 2.67e36).  Tokens that the page held before
 * keep their codes; when the new tokens raise max, they become
 * round_half_even(code * old / max), at any magnitude.  A max below 2^-126
 * counts as 0 (all codes 0); a new value that is not finite makes max NaN, and
 * with it every result that attends to the page's head.
 * A max only rises until the page's first token is appended again: after
 * release, or fork to a part of a page, it may be that of a token that is gone,
 * and what is appended then is coded by it.  (A NaN stays likewise: the tokens
 * left have lost their codes to it.) */
int manta_rocm_cache_append(MantaRocm* rt, MantaRocmCache* cache, int64_t layer, int dtype, const void* k_dev,
                            int64_t k_token, int64_t k_head, const void* v_dev, int64_t v_token, int64_t v_head,
                            const int32_t* offsets_dev, const int32_t* seqs_dev, int64_t n, int64_t tokens,
                            char** err);
/* The cache's values code * max / 127 as rows (f32, rounded once to dtype). */
int manta_rocm_cache_read(MantaRocm* rt, const MantaRocmCache* cache, int64_t layer, int dtype, void* k_dev,
                          int64_t k_token, int64_t k_head, void* v_dev, int64_t v_token, int64_t v_head,
                          const int32_t* offsets_dev, const int32_t* seqs_dev, int64_t n, int64_t tokens, char** err);

/* softmax(scale q k^T) v over the cached tokens of each row's sequence.  q:
 * q->x_dev [tokens, heads, head_dim], heads a multiple of kv_heads (query
 * head j reads kv head j / (heads / kv_heads)), f16 or bf16; q->out_dev the
 * same shape and type.  causal: a row at position p sees tokens 0..p, with
 * window > 0 only p - window + 1 .. p; otherwise (window must be 0) all.  A
 * row that sees nothing gets zeros.  lse_dev, when given, f32
 * [tokens, heads]: log of the sum of exp(scale q k), -inf for such a row.
 * Scores and sums are f32; the operand of the second product, weight times the
 * page's v_max against the largest of those that the row sees, is rounded to
 * f16 (2^-11, and to zero below 2^-32 of that largest one).
 * longest: about the longest sequence of the batch (it sets how the work is
 * split, not the result's meaning). */
int manta_rocm_cache_attention(MantaRocm* rt, const MantaRocmCache* cache, int64_t layer, int dtype,
                               const MantaRocmHeads* q, float* lse_dev, const int32_t* offsets_dev,
                               const int32_t* seqs_dev, int64_t n, int64_t tokens, double scale, int causal,
                               int64_t window, int64_t longest, char** err);

/* Device-to-device copy on the runtime's stream (a snapshot of a book, a page
 * pool set aside); the ranges must not overlap. */
int manta_rocm_copy(MantaRocm* rt, void* dst_dev, const void* src_dev, size_t bytes, char** err);

#ifdef __cplusplus
}
#endif
#endif
