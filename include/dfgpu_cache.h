/*
 * dfgpu_cache -- C ABI of the operators around a paged key/value cache in 8 bits: rotary positions, writing new tokens into the
 * cache, attention over it, and the bookkeeping of its pages. Part of libdfgpu.so; types, status codes, dfgpu_last_error()
 * and the shape of every launcher are those of dfgpu.h (device pointers in port order, caller-owned scratch, no allocation and
 * no synchronisation inside a launcher, launches capture into CUDA graphs). They are calls beside the graph:
 * the importer refuses graphs with the reference's own rotary nodes (ROPE, ROPE_BWD; lib/Compiler/SequenceGraph.cpp) and its PAGED_CACHE_LOAD
 * as before. Writing to a paged cache, holding it in 8 bits and moving its pages have no counterpart there.
 *
 * The cache. K and V are containers [pages, Hk, T, D] of FP8_E4M3 codes, T tokens a page, as the SDPA node's paged containers
 * are, and each has a tensor of FP8_E8M0 scales [pages, Hk, T / t, 1]: one power of two for every t consecutive tokens of a page
 * and head (t divides T). A value is decode(code) * 2^(scale - 127). A sequence's tokens lie in the pages that its row of an INT32
 * page table [B, 1, P, 1] names, T to a page in order.
 *
 * Sequence lengths, page tables and page ids are read on the device and are never trusted with an address: a page id outside
 * [0, pages) or a position past P * T reads as zeros and is not written.
 */
#ifndef DFGPU_CACHE_H
#define DFGPU_CACHE_H

#include "dfgpu.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bumped whenever a params struct, a pointer list or an enumeration of this header changes (dfgpu_abi_version() is dfgpu.h's). */
int dfgpu_cache_abi_version(void);

/* ---- rotary positions -----------------------------------------------------------------
   With angle a(s, i) = position(s) * frequency(i), i < R/2, the pair (x1, x2) of channels (i, i + R/2), or with `interleaved`
   (2i, 2i + 1), becomes scale * (x1 cos a - x2 sin a, x2 cos a + x1 sin a); channels R..D-1 are copied. `inverse` turns by -a:
   with the same scale that is the transposed map, the gradient of X from that of Y. The angle is reduced to one turn in
   64 bits, so far positions keep f32 accuracy; products and sums are f32, rounded once to Y's type.
   tensors: {X, Y, positions, frequencies, X2 or null, Y2 or null}. X, Y [B, H, S, D] FLOAT, HALF or BFLOAT16, the same type
   (any strides; D contiguous); X2, Y2 [B, H2, S, D], a second pair of tensors turned in the same launch (keys beside queries),
   rank 0: absent. Y may be X itself (same pointer, same strides) and must not overlap it, X2 or Y2 otherwise. positions INT32 or INT64
   [B or 1, 1, S, 1]; frequencies FLOAT [1, 1, 1, R/2], R = 2 * that extent <= D. The largest D is 1024. */
enum { DFGPU_ROPE_AUTO = 0, DFGPU_ROPE_VECTOR = 1, DFGPU_ROPE_SCALAR = 2 };
typedef struct dfgpu_rope_params {
    dfgpu_tensor x, y, x2, y2;
    dfgpu_tensor positions, frequencies;
    int32_t interleaved, inverse;
    float scale; /* 1, or the magnitude that the scaling below reports */
    int32_t kernel;
} dfgpu_rope_params;
int dfgpu_query_rope(const dfgpu_rope_params*, dfgpu_plan_info*);
int dfgpu_rope(const dfgpu_rope_params*, void* const* tensors, void* scratch, void* stream);

/* Fills HOST memory frequencies[rotary / 2] with base^(-2i / rotary), scaled for contexts `factor` times as long as the
   `original` one, in 64 bits and rounded once; *magnitude receives the factor for dfgpu_rope_params.scale (may be null).
     NONE    as they are; magnitude 1
     LINEAR  all divided by factor (position interpolation)
     BASE    ("NTK-aware") the base becomes base * factor^(rotary / (rotary - 2)): the last pair's frequency is divided by factor, the first's kept
     RAMP    ("NTK by parts", YaRN) a pair that makes more than `high` turns over the original length is kept, one that makes fewer than `low` is divided
             by factor, and between the pair numbers at which that is so (rounded outwards, within [0, R - 1], a step of 0.001 where they
             meet: that method's conventions, which its users' frequencies follow) a linear ramp blends the two; magnitude 0.1 ln(factor) + 1
     BANDS   the same borders with a blend linear in the number of turns (bands of wavelengths); magnitude 1 */
enum { DFGPU_ROPE_SCALING_NONE = 0, DFGPU_ROPE_SCALING_LINEAR = 1, DFGPU_ROPE_SCALING_BASE = 2, DFGPU_ROPE_SCALING_RAMP = 3, DFGPU_ROPE_SCALING_BANDS = 4 };
typedef struct dfgpu_rope_scaling {
    int32_t kind;
    int32_t rotary;   /* R, even */
    double base;      /* 10000 */
    double factor;    /* >= 1; not read by NONE */
    double original;  /* RAMP, BANDS: the context length before */
    double low, high; /* RAMP, BANDS: turns, 0 < low < high */
} dfgpu_rope_scaling;
int dfgpu_rope_frequencies(const dfgpu_rope_scaling*, float* frequencies, float* magnitude);

/* ---- new tokens into the cache -----------------------------------------------------------
   Token j < added(b) of sequence b goes to position lengths(b) + j. Where the new tokens of one call meet a scale block
   (t tokens of a page and head), its scale becomes the larger of 2^ceil(log2(amax / 448)) over them (BLOCK_SCALE_QUANTIZE's rule;
   a block of zeros takes 2^-127, which bounds nothing, a NaN 0xff) and, where the block holds tokens of this sequence already,
   their scale; if that grew, the codes they hold are encoded again in the new one. Codes are x / scale as BLOCK_SCALE_QUANTIZE
   encodes them. A block whose first token is written forgets what it held before. Nothing else in the containers changes.
   tensors: {K, V, K container, V container, K scale, V scale, page table of K, page table of V, lengths, added or null,
   lengths_out or null}. K, V [B, Hk, S, D] FLOAT, HALF or BFLOAT16 (any strides, D contiguous); page tables INT32 [B,1,P,1]
   (both may be the same); lengths, added, lengths_out INT32 [B,1,1,1]: tokens before the call (a negative one counts as 0), new
   tokens (absent: S; clamped to [0, S]), and their sum (clamped to P * T of the K table), which may be `lengths` itself, but not `added`. Positions past a table's P * T are not
   written. A page that two sequences share must not be written: fork first. */
enum { DFGPU_CACHE_APPEND_AUTO = 0, DFGPU_CACHE_APPEND_VECTOR = 1, DFGPU_CACHE_APPEND_SCALAR = 2 };
typedef struct dfgpu_cache_append_params {
    dfgpu_tensor k, v;
    dfgpu_tensor k_cache, v_cache, k_scale, v_scale;
    dfgpu_tensor page_table_k, page_table_v;
    dfgpu_tensor lengths, added, lengths_out; /* added, lengths_out: rank 0 where absent */
    int32_t kernel, reserved;
} dfgpu_cache_append_params;
int dfgpu_query_cache_append(const dfgpu_cache_append_params*, dfgpu_plan_info*);
int dfgpu_cache_append(const dfgpu_cache_append_params*, void* const* tensors, void* scratch, void* stream);

/* ---- attention over the cache ---------------------------------------------------------------
   O = softmax(attn_scale * Q K^T) V over the keys that SDPA's masks leave: kv < min(SEQ_LEN_KV, s_kv) and, counted from
   shift = bottom_right ? SEQ_LEN_KV - SEQ_LEN_Q : 0, kv <= q + shift + right_bound (with has_right_bound) and
   kv > q + shift - left_bound (with has_left_bound). Query rows from SEQ_LEN_Q on, and rows without keys, give O = 0 and
   Stats = -inf. A key whose page id is out of range reads as zeros, as in SDPA. Products take the codes as they are
   (exact in f16), scales and everything else are f32; the probabilities that weight V are rounded to f16 (2^-11 of each, 2^-36 of
   the row's largest where that is more), and Q is taken to within 2^-39 of its row's largest magnitude. A code or scale of a masked key, NaN or not, has no effect. Values under a V scale more than 2^80 below
   that of an earlier key of the sequence count as zeros.
   tensors: {Q, K container, V container, O, Stats or null, K scale, V scale, SEQ_LEN_Q or null, SEQ_LEN_KV, Page_table_K,
   Page_table_V}. Q, O [B, Hq, Sq, D] HALF or BFLOAT16, the same type (O may be FLOAT); D contiguous, 64, 128 or 256; Hq a
   multiple of Hk. O must not overlap Q or any other input. Containers with D contiguous, their other strides positive multiples of 16 and 16-byte aligned; T and t multiples of 16. Stats FLOAT
   [B, Hq, Sq, 1]: max + ln(sum). SEQ_LEN_Q absent: all Sq rows. s_kv bounds the keys of every sequence (at most P * T). */
enum { DFGPU_CACHE_SDPA_AUTO = 0, DFGPU_CACHE_SDPA_STREAM = 1, DFGPU_CACHE_SDPA_UMMA = 2 };
typedef struct dfgpu_cache_sdpa_params {
    dfgpu_tensor q, k, v, o, stats;
    dfgpu_tensor k_scale, v_scale;
    dfgpu_tensor seq_q, seq_kv;
    dfgpu_tensor page_table_k, page_table_v;
    float attn_scale;
    int32_t has_left_bound, has_right_bound, bottom_right;
    int64_t left_bound, right_bound;
    int64_t s_kv;
    int32_t kernel, reserved;
} dfgpu_cache_sdpa_params;
int dfgpu_query_cache_sdpa(const dfgpu_cache_sdpa_params*, dfgpu_plan_info*);
int dfgpu_cache_sdpa(const dfgpu_cache_sdpa_params*, void* const* tensors, void* scratch, void* stream);

/* ---- pages -------------------------------------------------------------------------------------
   A page is free where its reference count is 0 (or less; one that is taken has a count of 1). Every operation reads {page table, lengths, refs} and writes whole tables of
   what they are afterwards to {table_out, lengths_out, refs_out}, each of which may be its input itself. A sequence of n tokens uses its
   first ceil(n / block) slots (lengths are clamped to [0, P * block]); ids outside [0, pages) there count for nothing. Free pages are taken
   lowest id first. Results do not depend on timing.
     RESERVE  list [B, 1]: tokens that each sequence is going to add (negative: 0). Sequences get the pages that they lack for that,
              in order; one whose tokens pass P * block, or whose pages and those of all before it that fit their rows are more
              than the free ones, is refused and keeps its row. Lengths stay. The table has fewer than 2^31 slots.
     FORK     list [n, 2]: (source, target) sequences. The target, which must be empty and named by no earlier entry of the kind,
              gets the source's length and shares its full pages (counts grow by one); a last page that is partly filled is copied
              into a free one. Refused: ids out of range, source == target, a target with tokens, and entries for whose copies, and those of all
              entries before them that are not refused for another reason, the free pages do not suffice. The rest of the target's row becomes -1.
     FREE     list [n, 1]: sequences (one named twice counts once; ids out of range are refused). Their pages' counts fall by one,
              not below 0; their rows become -1 and their lengths 0.
     COMPACT  no list. With L pages in use, those with ids >= L move to the free ids < L, in order: contents, counts and the
              used slots of all tables follow.
     COPY     list [n, 2]: (source, target) pages. Refused: ids out of range, source == target, and entries whose source is another entry's
              target (one of ids in range that differ, refused or not). Of the entries that name a target, ids out of range and equal ones apart, only the last
              counts: it is copied, or where it is refused for its source, nothing is; the others are neither copied nor refused. Table, lengths and counts stay.
   Entries of a list whose first id is negative are skipped without being refused (FORK, FREE, COPY), so a list may be longer than what it says.
   report INT32 [4] (or null): free pages afterwards; pages taken, given back or moved (COPY: copied); page copies; entries refused.
   tensors: {page table, lengths, refs, list or null, table_out, lengths_out, refs_out, report or null, pool 0, ...}. page table
   INT32 [B,1,P,1], lengths INT32 [B,1,1,1], refs INT32 [pages], list INT32, all packed; at most 8 pools [layers, pages, n] of any type of whole bytes, n contiguous:
   what lies under a page's id (codes, scales; K and V), copied byte by byte for every layer. COPY reads no table, lengths
   and counts and may be given null for these and their outputs. One launch of a single thread-block cluster, and one more that copies where pools are given (FORK, COMPACT, COPY). */
enum { DFGPU_CACHE_PAGES_RESERVE = 0, DFGPU_CACHE_PAGES_FORK = 1, DFGPU_CACHE_PAGES_FREE = 2, DFGPU_CACHE_PAGES_COMPACT = 3, DFGPU_CACHE_PAGES_COPY = 4 };
#define DFGPU_CACHE_MAX_POOLS 8
typedef struct dfgpu_cache_pages_params {
    int32_t op, pool_count;
    int64_t block; /* tokens per page */
    dfgpu_tensor page_table, lengths, refs, list;
    dfgpu_tensor pools[DFGPU_CACHE_MAX_POOLS];
} dfgpu_cache_pages_params;
int dfgpu_query_cache_pages(const dfgpu_cache_pages_params*, dfgpu_plan_info*);
int dfgpu_cache_pages(const dfgpu_cache_pages_params*, void* const* tensors, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif
#endif
