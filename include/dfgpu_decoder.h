/*
 * dfgpu_decoder -- C ABI of the operators that stand around the attention of a decoder's step: norms of query and key heads with
 * their rotary positions, products of 8-bit integers with a scale for each token and channel, and beam search over a paged cache.
 * Part of libdfgpu.so; types, status codes, dfgpu_last_error() and the shape of every launcher are those of dfgpu.h (device pointers
 * in port order, caller-owned scratch that needs no clearing, no allocation and no synchronisation inside a launcher, launches capture
 * into CUDA graphs). They are calls beside the graph and the calls of dfgpu_cache.h.
 *
 * Ids and flags in device memory (parents, finished) are never trusted with an address. Unless a port says so, an output must not overlap
 * an input or another output.
 */
#ifndef DFGPU_DECODER_H
#define DFGPU_DECODER_H

#include "dfgpu.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bumped whenever a params struct, a pointer list or an enumeration of this header changes (dfgpu_abi_version() is dfgpu.h's). */
int dfgpu_decoder_abi_version(void);

/* INT8: two's-complement bytes. A storage type of the calls below only; its number continues dfgpu.h's. */
enum { DFGPU_I8 = 12 };

/* ---- norms of heads, with their positions -------------------------------------------------
   Row x of D channels (a token's head): r = 1 / sqrt(mean(x^2) + epsilon), n(i) = x(i) r (gain(i) + gain_offset), and with positions
   the pairs of n turn as in dfgpu_rope (dfgpu_cache.h: frequencies, interleaved, scale; channels R..D-1 stay n). Sums, products and r are
   f32 (a row whose squares pass f32's range gives zeros), angles are reduced in 64 bits; one rounding to Y's type.
   tensors: {X, Y, gain or null, positions or null, frequencies or null, X2 or null, Y2 or null, gain2 or null}. X, Y [B, H, S, D]
   FLOAT, HALF or BFLOAT16, the same type (any strides; D contiguous, at most 1024); X2, Y2 [B, H2, S, D], a second pair in the same launch
   (keys beside queries), rank 0: absent. gain, gain2 FLOAT, HALF or BFLOAT16 [1, 1 or H, 1, D], D contiguous, rank 0: a factor of one (no offset). positions
   INT32 or INT64 [B or 1, 1, S, 1] and frequencies FLOAT [1, 1, 1, R/2], R <= D; both rank 0: no position is applied. Y may be X itself (same
   pointer, same strides), Y2 X2. */
enum { DFGPU_HEAD_NORM_AUTO = 0, DFGPU_HEAD_NORM_VECTOR = 1, DFGPU_HEAD_NORM_SCALAR = 2 };
typedef struct dfgpu_head_norm_params {
    dfgpu_tensor x, y, x2, y2;
    dfgpu_tensor gain, gain2;
    dfgpu_tensor positions, frequencies;
    int32_t interleaved;
    float scale; /* of the turned channels: 1, or the magnitude of the frequencies' scaling */
    float epsilon, gain_offset;
    int32_t kernel, reserved;
} dfgpu_head_norm_params;
int dfgpu_query_head_norm(const dfgpu_head_norm_params*, dfgpu_plan_info*);
int dfgpu_head_norm(const dfgpu_head_norm_params*, void* const* tensors, void* scratch, void* stream);

/* The gradients: with u the channels of dY turned back (times scale), v = u (gain + gain_offset) and m = mean(v x),
   dX = r v - x r^3 m and dgain(i) = sum over the rows that share it of u(i) x(i) r. Partial sums of dgain are f32 over at most 1280 rows each (a head's
   16 tokens with gains of every head) and meet in 64 bits, always in the same order.
   A row whose squares pass f32's range has r = 0: its dX and its terms of dgain are zeros (NaN where the sum of v x passes it too).
   tensors: {X, dY, dX, gain or null, dgain or null, positions or null, frequencies or null, X2, dY2, dX2, gain2, dgain2 (null where absent)}.
   dX has X's extents and type and may be X or dY itself (same pointer, same strides); dX2 likewise. dgain has gain's extents, FLOAT, HALF or
   BFLOAT16, rank 0: not wanted; where gain is absent it may still be wanted, [1, 1 or H, 1, D]. Scratch holds the partial sums: none where no dgain is
   wanted, which saves the second launch too. */
typedef struct dfgpu_head_norm_grad_params {
    dfgpu_tensor x, dy, dx, x2, dy2, dx2;
    dfgpu_tensor gain, dgain, gain2, dgain2;
    dfgpu_tensor positions, frequencies;
    int32_t interleaved;
    float scale;
    float epsilon, gain_offset;
    int32_t kernel, reserved;
} dfgpu_head_norm_grad_params;
int dfgpu_query_head_norm_grad(const dfgpu_head_norm_grad_params*, dfgpu_plan_info*);
int dfgpu_head_norm_grad(const dfgpu_head_norm_grad_params*, void* const* tensors, void* scratch, void* stream);

/* ---- 8-bit integers with a scale for each token -------------------------------------------
   Row by row: scale = max |x| / 127, y = x / scale to the nearest whole number, ties to even, within [-127, 127]; both quotients are f32's,
   rounded once, so codes are the same wherever they are computed. A row of zeros (or below 2^-143) has scale 0 and codes 0; one with an infinity has an
   infinite scale and codes 0, one with a NaN a NaN scale and codes 0: its products are NaN.
   tensors: {X, Y, scale}. X FLOAT, HALF or BFLOAT16 [..., M, K], rank 2 to 4, K contiguous; Y INT8 of the same extents, K contiguous; scale
   FLOAT [..., M, 1]. Weights [N, K] are quantised channel by channel in the same way. DFGPU_TOKEN_QUANTIZE_VECTOR: rows of whole 16-byte vectors on their
   boundaries; DFGPU_TOKEN_QUANTIZE_SCALAR: any rows. */
enum { DFGPU_TOKEN_QUANTIZE_AUTO = 0, DFGPU_TOKEN_QUANTIZE_VECTOR = 1, DFGPU_TOKEN_QUANTIZE_SCALAR = 2 };
typedef struct dfgpu_token_quantize_params {
    dfgpu_tensor x, y, scale;
    int32_t kernel, reserved;
} dfgpu_token_quantize_params;
int dfgpu_query_token_quantize(const dfgpu_token_quantize_params*, dfgpu_plan_info*);
int dfgpu_token_quantize(const dfgpu_token_quantize_params*, void* const* tensors, void* scratch, void* stream);

/* C(m, n) = sum_k A(m, k) B(k, n) * a_scale(m) * b_scale(n) + bias(n): the sum in 32-bit integers (exact: K is at most 131071), then an f32 of
   it, the two products and the sum with the bias in f32, in this order, and one rounding to C's type.
   tensors: {A, B, C, a_scale, b_scale, bias or null}. A INT8 [..., M, K], B INT8 [..., K, N], C FLOAT, HALF or BFLOAT16 [..., M, N], equal rank
   2 to 8; batch axes of A and B are C's or 1. a_scale FLOAT [..., M or 1, 1], b_scale FLOAT [..., 1, N or 1], bias FLOAT, HALF or BFLOAT16
   [..., 1, N], of the same rank, their batch axes 1 or (a_scale) A's. DFGPU_MATMUL_INT8_UMMA: tcgen05 (kind::i8); A with K contiguous, B with K or N
   contiguous, their rows on 16-byte boundaries (any extents), C and the bias with N contiguous, batch axes that fold into M. DFGPU_MATMUL_INT8_FEW: at
   most 16 rows of A, A and B with K contiguous on 16-byte boundaries, batch axes that fold into M, any C and bias: for a decoder's step, bound by B. AUTO takes the quicker of the two
   where it can; everything else goes to the CUDA cores, which take any layout at 20 to 75 times the time: rows or columns off the 16-byte boundaries, an A whose K
   is not contiguous, a B for each batch entry, and batches whose rows do not lie evenly (a padded buffer: call once an entry instead). The result does not depend on the kernel. */
enum { DFGPU_MATMUL_INT8_AUTO = 0, DFGPU_MATMUL_INT8_CORES = 1, DFGPU_MATMUL_INT8_UMMA = 2, DFGPU_MATMUL_INT8_FEW = 3 };
typedef struct dfgpu_matmul_int8_params {
    dfgpu_tensor a, b, c;
    dfgpu_tensor a_scale, b_scale, bias;
    int32_t kernel, reserved;
} dfgpu_matmul_int8_params;
int dfgpu_query_matmul_int8(const dfgpu_matmul_int8_params*, dfgpu_plan_info*);
int dfgpu_matmul_int8(const dfgpu_matmul_int8_params*, void* const* tensors, void* scratch, void* stream);

/* ---- beam search -------------------------------------------------------------------------------
   A batch entry has W beams (at most 32). Beam w that is not finished continues with each of the V tokens t, at score(w) + logits(w, t) - ln sum exp logits(w, .); one that
   is finished with the token `pad` alone, at score(w). The W continuations of the greatest worth are kept, in falling order; equals go to the lower
   beam, then the lower token. Worth is the score; with lengths, score / n^length_penalty, where n = max(1, lengths(w) + 1), for a finished beam max(1, lengths(w));
   length_penalty is within -28 and 28.
   Sums of exponentials are f32 over at most 64 terms of a thread and meet in 64 bits, where scores are added and compared. A beam whose score is not
   finite, or whose logits have no finite sum of exponentials (a NaN, +inf, all -inf), continues at -inf: with its tokens 0, 1, ...,
   which are kept only where fewer than W others are finite; the same holds for logits of -inf.
   tensors: {logits, scores, finished or null, lengths or null, scores_out, tokens, parents, finished_out or null, lengths_out or null, forks or null}.
   logits FLOAT, HALF or BFLOAT16 [B, W, V], V contiguous, below 2^26; scores, scores_out FLOAT, the others INT32 [B, W] (any
   strides): tokens and the beams (0..W-1) they continue, whether a beam is finished (not 0; afterwards 1 also where its token is `end`; no token is where
   `end` is negative), and tokens so far (lengths_out: n of the beam). scores_out, finished_out and lengths_out may be scores,
   finished and lengths themselves. forks INT32 [B * W, 2], packed: (source_base + b W + parent, target_base + b W + w), the list that dfgpu_cache_pages FORK takes to
   continue the sequences from source_base on as those from target_base on. Scratch: 16-byte aligned. */
typedef struct dfgpu_beam_select_params {
    dfgpu_tensor logits, scores, finished, lengths;
    dfgpu_tensor scores_out, tokens, parents, finished_out, lengths_out, forks; /* rank 0: absent */
    float length_penalty; /* read only with lengths */
    int32_t end, pad;
    int32_t source_base, target_base;
    int32_t reserved;
} dfgpu_beam_select_params;
int dfgpu_query_beam_select(const dfgpu_beam_select_params*, dfgpu_plan_info*);
int dfgpu_beam_select(const dfgpu_beam_select_params*, void* const* tensors, void* scratch, void* stream);

/* States of beams follow: target(l, b, w, :) = source(l, b, parents(b, w), :), byte by byte, for up to 8 states in one launch. A parent outside
   [0, W) leaves its rows as they are. tensors: {parents, source 0, target 0, source 1, target 1, ...}. parents INT32 [B, W]; source and target [layers, B, W, n] of any
   type of whole bytes, the same, n contiguous (any other strides); a target must not overlap a source, its own or another. Quickest where all rows start on 8-byte
   boundaries and are whole multiples of 8 bytes; half as quick by 2 bytes, a quarter by single ones. */
#define DFGPU_BEAM_MAX_STATES 8
typedef struct dfgpu_beam_reorder_params {
    dfgpu_tensor parents;
    dfgpu_tensor source[DFGPU_BEAM_MAX_STATES], target[DFGPU_BEAM_MAX_STATES];
    int32_t count, reserved;
} dfgpu_beam_reorder_params;
int dfgpu_query_beam_reorder(const dfgpu_beam_reorder_params*, dfgpu_plan_info*);
int dfgpu_beam_reorder(const dfgpu_beam_reorder_params*, void* const* tensors, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif
#endif
