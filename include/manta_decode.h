/*
 * manta_decode.h -- the operators of a model that writes an answer from what
 * was retrieved, beside those of manta_cache.h: products in 8 bits with a
 * scale for each token and each output column, norms of queries and keys with
 * their rotation in one pass, and beams: the choice of the next ones and the
 * cache's sequences following it.
 *
 * Conventions are manta_cache.h's: int status and malloc'd message, "_dev"
 * pointers are device addresses, calls are asynchronous on the runtime's
 * stream, none but bind / create allocates device memory (so all others may
 * be recorded into a HIP graph), and what only the device can see is checked
 * by the kernels and reported by the next synchronizing call.  The reference
 * has no counterpart: it widens q8 weights to f32 (runtime/backend/
 * tensor.go:49-71) and has no decoder.
 */
#ifndef MANTA_DECODE_H
#define MANTA_DECODE_H

#include "manta_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- products in 8 bits ------------------------------------------------- */

typedef struct MantaRocmWeight MantaRocmWeight;

/* What becomes of a product of two halves (bind):
 *   NONE  x W
 *   SILU  silu(x G) * (x U), silu(a) = a / (1 + exp(-a))
 *   GELU  gelu(x G) * (x U), the tanh form of the encoder's gelu step */
enum {
    MANTA_ROCM_GATE_NONE = 0,
    MANTA_ROCM_GATE_SILU = 1,
    MANTA_ROCM_GATE_GELU = 2,
};

/* Bind a weight: host codes int8 [width, columns] and a scale f32 per column,
 * the form of the encoder's matrices.  columns is n, or 2 n when gated: n
 * columns of G, then n of U.  width is 1 to 131072 (int32 sums stay exact). */
int manta_rocm_weight_bind(MantaRocm* rt, const int8_t* codes, const float* scales, int64_t width, int64_t n, int gate,
                           MantaRocmWeight** out, char** err);
void manta_rocm_weight_unbind(MantaRocmWeight* w);

/* Bytes of the codes of `rows` quantised rows: rows rounded up to 16 times
 * width rounded up to 128.  They lie in blocks of 16 rows and 64 columns, as
 * the matrix cores take them: the code of (r, c) is byte
 *   ((r / 16) * (pitch / 64) + c / 64) * 1024 + (c % 64) / 16 * 256 + r % 16 * 16 + c % 16.
 * The first starts on 16 bytes.  -1 where rows or width is out of range. */
int64_t manta_rocm_quantized_bytes(int64_t rows, int64_t width);

/* Quantise rows x [rows, width] (row r at x + r * x_row elements; f32, f16 or
 * bf16) to 8 bits with a scale a row:
 *   z = x, or x * norm[c] rounded to f32 with norm_dev (f32 [width]);
 *   code = round_half_even(z * 127 / max|z|) in f32 (also where z * 127 is past
 *   its range), scale = max|z| / 127,
 *   times 1 / sqrt(mean(x^2) + eps) with norm_dev: the RMS norm's factor
 *   cancels in the codes.
 * A row whose max|z| is below 2^-126 has codes and scale 0, one with a z that
 * is not finite codes 0 and scale NaN.  Padding columns are 0, padding rows
 * undefined.  eps is at least 2^-126 (not looked at without norm_dev). */
int manta_rocm_quantize_rows(MantaRocm* rt, int dtype, const void* x_dev, int64_t x_row, int64_t rows, int64_t width,
                             const float* norm_dev, double eps, int8_t* codes_dev, float* scales_dev, char** err);

/* Quantised rows times a bound weight: with y = code sums (exact, int32) *
 * (row scale * column scale) in f32,
 *   out[r, c] = y + add[r, c], or act(y of G) * y of U when gated,
 * rounded once to dtype.  add_dev (not with a gated weight) may be NULL or
 * out_dev with the same stride; otherwise out_dev overlaps no other operand.
 * Strides are in elements and at least n. */
int manta_rocm_matmul_q8(MantaRocm* rt, const MantaRocmWeight* w, const int8_t* codes_dev, const float* scales_dev,
                         int64_t rows, int dtype, const void* add_dev, int64_t add_row, void* out_dev, int64_t out_row,
                         char** err);

/* ---- norms of queries and keys with their rotation ---------------------- */

/* manta_rocm_rotary of tensors whose heads are RMS normed first, in the same
 * pass: y = rotate(x / sqrt(mean(x^2) + eps) * norm), the mean over a head's
 * head_dim columns, in f32 (the sum of squares in f64), rounded once.
 * norms_dev[i], f32 [head_dim] in device memory, belongs to parts[i]; NULL:
 * that tensor is rotated only.  eps is at least 2^-126.  As the formula has it,
 * a NaN makes its whole head NaN, an infinity its own pair (or column), and the
 * head's other columns 0. */
int manta_rocm_rotary_normed(MantaRocm* rt, const MantaRocmRotary* rot, int dtype, const int32_t* positions_dev,
                             int64_t tokens, int64_t head_dim, const MantaRocmHeads* parts,
                             const float* const* norms_dev, int64_t nparts, double eps, char** err);

/* ---- beams -------------------------------------------------------------- */

typedef struct MantaRocmBeams MantaRocmBeams;

/* The scratch memory of beam_select for up to `groups` groups of `beams`
 * beams (1 to 64) and `best` results a group (1 to 64).  Calls that may
 * overlap, on streams or in graphs, take a handle each. */
int manta_rocm_beams_create(MantaRocm* rt, int64_t groups, int64_t beams, int64_t best, MantaRocmBeams** out,
                            char** err);
void manta_rocm_beams_destroy(MantaRocmBeams* b);

/* The best continuations of every group's beams: of the totals
 *   scores[g, b] + logits[g, b, t] - log(sum over u of exp(logits[g, b, u]))
 * the `best` largest, in descending order, equal ones by the lower beam, those
 * of one beam by the larger logit, then the lower token (so that within a beam
 * the order is that of its logits): the beam to out_parents, t to out_tokens,
 * the total to out_scores, each [groups, best].  logits_dev: f32, f16 or bf16
 * [groups * beams, vocab], rows logits_row elements apart; scores_dev f32
 * [groups, beams].  Totals are formed and compared in f64 and rounded once.
 * out_scores_dev may be scores_dev where best is beams.
 * ended_dev, when given: int32 [groups, beams]; a beam whose entry is not 0
 * has one continuation, end_token, of total scores[g, b], and its logits are
 * not read.  out_ended_dev, when given: int32 [groups, best], 1 where the
 * continuation is end_token, else 0: the next call's ended_dev (which it may
 * be, where best is beams).
 * A total that is -inf or NaN is no continuation (a masked token; a beam of
 * score -inf; every one of a beam with a NaN or +inf among its logits); where
 * a group has too few, the rest is parent -1, token -1, -inf. */
int manta_rocm_beam_select(MantaRocm* rt, MantaRocmBeams* b, int dtype, const void* logits_dev, int64_t logits_row,
                           int64_t groups, int64_t beams, int64_t vocab, const float* scores_dev,
                           const int32_t* ended_dev, int64_t end_token, int64_t best, int32_t* out_parents_dev,
                           int32_t* out_tokens_dev, float* out_scores_dev, int32_t* out_ended_dev, char** err);

/* What the next step reads: out[i] = tokens[i], or `instead` where that is
 * negative (no continuation).  out_dev may be tokens_dev; n is at most 2^25. */
int manta_rocm_beam_inputs(MantaRocm* rt, const int32_t* tokens_dev, int64_t n, int64_t instead, int32_t* out_dev,
                           char** err);

/* Beams that go on from others: seqs_dev (int32 [n], distinct slots) holds
 * n / group groups, and its entry i takes over what entry parents_dev[i] (0
 * to group - 1) of its own group held when the call began, sharing its pages;
 * -1 empties it.  Pages that no sequence names any more are free.  All
 * entries or, where one is wrong, none: as a refused extend, which see, and
 * so is a call that names a sequence of one.  n is at most 4096, group at
 * most 1024.  (extend then copies a last page that several go on from.) */
int manta_rocm_cache_reorder(MantaRocm* rt, MantaRocmCache* cache, const int32_t* seqs_dev, const int32_t* parents_dev,
                             int64_t n, int64_t group, char** err);

#ifdef __cplusplus
}
#endif
#endif
