/*
 * turbovec_hip.h -- C ABI of the MI355X (gfx950) search path for turbovec.
 *
 * The library replaces ONE crate-internal function of the reference,
 *     search::search(...)                       turbovec/src/search.rs:3206-3221
 * whose only caller is
 *     TurboQuantIndex::try_search_with_mask     turbovec/src/lib.rs:1462-1477
 * plus the small amount of index state that function reads (codes, per-vector
 * scales, rotation tables, centroids, TQ+ calibration), kept resident in HBM.
 *
 * Conventions: every entry point returns a tv_status; nothing throws or aborts
 * across the boundary; all buffers are caller-owned host memory unless the name
 * ends in _dev; sizes are element counts.  Functions that mutate an index
 * (upload / append / swap_remove / set_*) need external exclusion, exactly as
 * the reference's `&mut self` methods do; tv_search* may be called from many
 * threads at once: the GPU serves one launch at a time, so calls that arrive
 * while the index is busy wait, and whoever gets the index next serves every
 * waiting tv_search (or tv_search_dev) call with the same k and the same mask
 * pointer together with its own, as one batch; each caller receives exactly the
 * rows a call of its own would have returned.  A process
 * that has used the library must not fork() and keep using it in the child.
 *
 * Device buffers (_dev entry points, device pointers): the library runs on a
 * stream of its own per index, not on the caller's.  Every device buffer handed
 * in must be complete -- the work that writes it finished, e.g. the producing
 * stream synchronised -- before the call, and must stay untouched until the call
 * returns; outputs are complete when the call returns (it synchronises its
 * stream before returning).
 */
#ifndef TURBOVEC_HIP_H
#define TURBOVEC_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct tv_index tv_index;

/* Status codes.  1..5 are the reference's SearchError variants
 * (turbovec/src/error.rs:234-276). */
typedef enum {
    TV_OK = 0,
    TV_ERR_QUERY_BUFFER_NOT_MULTIPLE_OF_DIM = 1, /* lib.rs:1363-1369 */
    TV_ERR_INVALID_QUERY_VALUE = 2,              /* lib.rs:1374-1380, encode.rs:76-83 */
    TV_ERR_MASK_LENGTH_MISMATCH = 3,             /* lib.rs:1427-1434 */
    TV_ERR_ALLOWLIST_EMPTY = 4,                  /* id_map.rs:672 */
    TV_ERR_UNKNOWN_ID = 5,                       /* id_map.rs:677 */
    TV_ERR_BAD_ARGUMENT = 6,                     /* ConstructError / FromPartsError class */
    TV_ERR_HIP = 7,                              /* a HIP runtime call failed */
    TV_ERR_NO_DEVICE = 8,                        /* no gfx950 device visible */
    TV_ERR_INDEX_OUT_OF_RANGE = 9,
    TV_ERR_BAD_IMAGE = 10        /* snapshot bytes refused; tv_last_error says why */
} tv_status;

/* Which integer score definition the scan uses (the reference picks one at run
 * time from CPU features, turbovec/src/pack.rs:1189-1219, search.rs:2975-2980). */
typedef enum {
    TV_SCORE_AUTO = 0,      /* what an AVX-512 VNNI / dotprod host runs: P at 4-bit, L_U32 at 2/3-bit */
    TV_SCORE_L_SCALAR = 1,  /* u8 LUT terms added one by one in f32, bias first   search.rs:3113-3128 (the
                               definition; what FORCE_SCALAR_FALLBACK selects, search.rs:313-316) */
    TV_SCORE_L_CLASSIC = 2, /* u8 LUT sums, fma flush per 256 byte-groups   search.rs:516-582 */
    TV_SCORE_L_U32 = 3,     /* u8 LUT sums, (acc*scale+bias)*vec_scale      search.rs:1174-1177 */
    TV_SCORE_P = 4          /* int8 permute-dot, fma(acc,scale,bias)*vs     search.rs:1519-1524 (4-bit only) */
} tv_score_mode;

const char *tv_status_string(int status);
/* Text of the last HIP failure on the calling thread ("" if none). */
const char *tv_last_error(void);

/* ---- index life cycle -------------------------------------------------- */

/* Replaces the lazily built caches of TurboQuantIndex (lib.rs:1404-1415): the
 * rotation tables (rotation.rs:141-187) and Lloyd-Max centroids
 * (codebook.rs:50) are derived inside and uploaded.  dim: positive multiple of
 * 8, <= 16384; bits in {2,3,4} (lib.rs:629-668).  device: HIP ordinal.
 * Device blocks of 1 MiB and more that an index gives up -- it grew, or was
 * destroyed -- are kept for the indexes of that device, up to 2 GiB, while any
 * index lives there: handed on to a request they exceed by a quarter at most,
 * given back to the device when an allocation of this library fails and when
 * the device's last index is destroyed.  When that is not enough, a failing
 * allocation also takes what the device's indexes keep of filtered searches'
 * allowed rows (tv_debug_workspace_bytes), and room that no search is using of
 * the next kind.  Batches of 65 queries and more over large indexes of 2- or
 * 3-bit codes need room for the rows that they look at twice: up to 1 GiB a
 * search, 2 GiB in all, lent to one search of the device at a time and kept for
 * the next until the device's last index is destroyed; a search that finds none
 * runs without, up to three times as long.  Other allocators of the process do
 * not see any of this.  Calls on host arrays pass through pinned host memory that the
 * device's indexes share too: allocated on first use, up to 256 MiB, freed with
 * the last index. */
int tv_index_create(int dim, int bits, int device, tv_index **out);
int tv_index_destroy(tv_index *ix);

/* Hand over the caller's own tables instead of the derived ones: signs and
 * perms are round 0 then round 1 (2*dim each, rotation.rs:110-115), centroids
 * 2^bits values.  Any pointer may be NULL to keep the current table. */
int tv_index_set_tables(tv_index *ix, const float *signs, const uint32_t *perms, const float *centroids);
/* TQ+ pair (lib.rs:329-330), dim values each; both NULL = uncalibrated. */
int tv_index_set_calibration(tv_index *ix, const float *shift, const float *scale);
int tv_index_set_score_mode(tv_index *ix, int mode);

/* Read back the tables in use (for cross-checking against the caller's). */
int tv_index_get_tables(const tv_index *ix, float *signs, uint32_t *perms, float *centroids, float *boundaries);

/* Replace the contents with n_vectors rows given in the sequential-blocked
 * layout the reference persists (pack.rs:336-361: byte of (block b, group g,
 * lane l) at (b*G+g)*32+l, ceil(n/32)*G*32 bytes) and their per-vector scales
 * (lib.rs:312).  Replaces BlockedCache (lib.rs:253-256). */
int tv_index_upload_seq(tv_index *ix, const uint8_t *seq_codes, size_t n_vectors, const float *scales);
/* Same, from device memory (both pointers are device pointers). */
int tv_index_upload_seq_dev(tv_index *ix, const uint8_t *d_seq_codes, size_t n_vectors, const float *d_scales);
/* Append n_new rows; rows[i*G + g] is row i's code byte of group g (the
 * per-vector form extract_codes_flat yields, pack.rs:306).  Replaces
 * append_lanes (pack.rs:211-233). */
int tv_index_append_rows(tv_index *ix, const uint8_t *rows, const float *scales, size_t n_new);
/* Encode n_new raw float rows (n_new*dim values) on the device and append them:
 * normalise, rotate, quantise against the codebook (and the TQ+ pair when one is
 * set), derive the per-vector scale, pack, append.  Codes and scales are
 * bit-identical to the CPU encoder's.  Replaces the encode half of
 * TurboQuantIndex::add (lib.rs:738-966 -> encode.rs:1418-1476, :560-664,
 * :900-932).  Values must be finite with |x| < 1e16 (encode.rs:76-83):
 * TV_ERR_INVALID_QUERY_VALUE otherwise, and nothing is added: tv_index_len counts
 * the rows once all of them have passed.  The index's buffers may have grown all
 * the same (tv_index_device_ptrs). */
int tv_index_add(tv_index *ix, const float *vectors, size_t n_new);
/* Fit the TQ+ per-coordinate pair from n >= 2 sample rows and commit it
 * (TurboQuantIndex::calibrate, lib.rs:2599; fit encode.rs:737-857): the sample is
 * normalised and rotated on the device, the order statistics are taken on the
 * host.  Only on an empty index: re-encoding stored rows under a new pair
 * (lib.rs:2599-2835) is not built.  The fitted pair equals the reference's bit
 * for bit. */
int tv_index_calibrate(tv_index *ix, const float *sample, size_t n);
/* The committed pair: *n_calib is 0 (uncalibrated) or dim; shift/scale may be NULL. */
int tv_index_get_calibration(const tv_index *ix, float *shift, float *scale, size_t *n_calib);
/* Same, rows already in device memory, at any address a float may have (not validated: the caller checked them). */
int tv_index_add_dev(tv_index *ix, const float *d_vectors, size_t n_new);
/* lib.rs:2864-3028: move the last vector into slot idx, zero the vacated lane. */
int tv_index_swap_remove(tv_index *ix, size_t idx);
/* Copy the index back in the sequential-blocked layout (codes_blocked_seq,
 * lib.rs:2088); seq_out holds ceil(n/32)*G*32 bytes, scales_out n floats. */
int tv_index_download_seq(const tv_index *ix, uint8_t *seq_out, float *scales_out);
size_t tv_index_len(const tv_index *ix);
int tv_index_dim(const tv_index *ix);
int tv_index_bits(const tv_index *ix);

/* ---- search ------------------------------------------------------------- */

/* Caller-side validation the reference performs before the seam
 * (lib.rs:1363-1380): len must be a multiple of dim, every value must satisfy
 * |x| < 1e16.  On TV_ERR_INVALID_QUERY_VALUE *bad_index is the flat offset. */
int tv_validate_queries(const float *queries, size_t len, int dim, size_t *bad_index);
/* lib.rs:1435-1456: one byte per slot (non-zero = allowed) to u64 words, LSB =
 * lowest slot; returns the number of allowed slots in *n_allowed. */
int tv_pack_mask(const uint8_t *mask_bytes, size_t n, uint64_t *words_out, size_t *n_allowed);

/* search::search (search.rs:3206).  queries: nq*dim floats.  mask_words: NULL
 * or ceil(n/64) words.  Writes nq*k_eff scores and slot indices, rows sorted
 * (score desc, slot asc), k_eff = min(k, n, popcount(mask)) returned in
 * *out_k_eff; out buffers must hold nq*min(k,n) entries.  k_eff == 0 or
 * nq == 0 writes nothing. */
int tv_search(tv_index *ix, const float *queries, size_t nq, size_t k,
              const uint64_t *mask_words, size_t n_mask_words,
              float *out_scores, int64_t *out_indices, size_t *out_k_eff);

/* tv_validate_queries and tv_search in one: the values checked are the snapshot of them that is searched
 * (turbovec-python/src/lib.rs:617-629 copies the array first for that).  On TV_ERR_INVALID_QUERY_VALUE
 * *bad_index is the flat offset and nothing is searched. */
int tv_search_checked(tv_index *ix, const float *queries, size_t nq, size_t k,
                      const uint64_t *mask_words, size_t n_mask_words,
                      float *out_scores, int64_t *out_indices, size_t *out_k_eff, size_t *bad_index);

/* Same, with queries, mask words and outputs already in device memory and the
 * mask's popcount supplied by the caller (the reference's caller counts it
 * while packing, lib.rs:1446).  Returns after the work is enqueued and
 * completed on the index's stream. */
int tv_search_dev(tv_index *ix, const float *d_queries, size_t nq, size_t k,
                  const uint64_t *d_mask_words, size_t n_allowed,
                  float *d_out_scores, int64_t *d_out_indices, size_t *out_k_eff);

/* tv_search_dev for callers that cannot allocate device memory (tight serving loops, harnesses
 * that forbid hipMalloc, code that must not disturb a caching allocator).  No counterpart in the
 * reference.  Like tv_search_dev it runs on the index's own stream and synchronises that stream
 * before it returns (it reads the overflow flags of its passes on the host), so it cannot be
 * recorded into a HIP graph under capture.
 * Same arguments, results and status codes as tv_search_dev, but everything the search carves
 * -- rotated queries, tables, candidate segments, the exact path's lists -- comes out of a
 * fixed array in the library's device image (tv_noalloc_scratch_bytes() bytes, 64 MiB, held by
 * every GPU the library runs on until the process ends), and the call makes no hipMalloc,
 * hipFree, event or stream creation.  A search whose worst case does not fit (at 1536
 * dimensions, 4-bit: more than about 400 queries per call; k > 32 on an index of millions of
 * rows, whose exact fallback ranks dense score rows) is refused with TV_ERR_BAD_ARGUMENT and
 * tv_last_error() names the bytes needed; nothing is written then.  All calls on one GPU share
 * the array: within a process they are serialised by the library; the array keeps the previous
 * call's bytes and every search overwrites what it reads.  Scan timings (tv_last_scan_ms) are
 * not taken on this path. */
int tv_search_dev_noalloc(tv_index *ix, const float *d_queries, size_t nq, size_t k,
                          const uint64_t *d_mask_words, size_t n_allowed,
                          float *d_out_scores, int64_t *d_out_indices, size_t *out_k_eff);
size_t tv_noalloc_scratch_bytes(void);

/* ---- operators beside the search ------------------------------------------
 *
 * Rows in 8 and 4 bits, their products, re-scoring of what a search returned,
 * a norm that ends in such rows, drawing a slot from scores, and log probabilities
 * of slots with their gradient.  No counterpart in the reference.  They hold no
 * state and take no index: every pointer but `stream` is a device pointer of
 * `device`, and the call puts its kernels on `stream` (a hipStream_t of that
 * device; NULL: its default stream) and returns without waiting.  Inputs must
 * be complete in that stream's order and stay untouched until the kernels have
 * run.  Nothing is allocated: a call may be recorded into a graph, which holds
 * the buffers and the workspace it was recorded with.  Calls that may run at
 * the same time need workspaces of their own; a workspace needs no clearing and
 * holds nothing from one call to the next.  Any thread may call; the caller's
 * current device stays what it was.  Strides count elements from one row to the
 * next, elements of a row lie next to each other.  Results overlap no input.
 * Arguments are checked before anything is launched (TV_ERR_BAD_ARGUMENT,
 * tv_last_error() says which); what lies in device memory is not.  Calls of
 * no rows do nothing. */

/* Types of values, and of the scales of 8-bit rows. */
typedef enum { TV_F32 = 0, TV_F16 = 1, TV_BF16 = 2 } tv_value_type;
typedef enum {
    TV_SCALE_E8M0 = 0, /* a byte e: 2^(e - 127); 255 is NaN */
    TV_SCALE_F32 = 1   /* a float */
} tv_scale_type;

/* 8-bit rows hold e4m3 codes (1 sign, 4 exponent and 3 mantissa bits, no infinity, largest value 448) of
 * dim coordinates, 1 to 16384, and a scale for every block of 128 coordinates (the last may be shorter) of
 * `group` rows: 1, or 128 (the last tile may hold fewer).  A coordinate is code * scale.  Scale of row r and
 * coordinate c: scales[(r / group) * scale_stride + c / 128]. */

/* Makes 8-bit rows of values.  With `amax` the largest finite magnitude of a block, its scale is
 * max(amax / 448, 2^-126) as a float, or the smallest power of two 2^e, e >= -126, with amax <= 448 * 2^e;
 * codes are x / scale rounded to the nearest, ties to even.  Infinities and NaN become NaN codes and leave
 * their block's scale to the others. */
int tv_fp8_quantize_dev(int device, void *stream, const void *d_x, int x_type, size_t x_stride, size_t rows, size_t dim,
                        int scale_type, int group, uint8_t *d_codes, size_t code_stride, void *d_scales, size_t scale_stride);
/* out[i][j] = the inner product of row i of a (m rows, a scale of each row) with row j of b (n rows, scales of
 * `group` rows): sums of products of codes within a block times both scales, blocks added in 32 bits, rounded
 * once to out_type.  For 16-bit results the products are added in groups of eight neighbouring coordinates, each
 * cut off towards zero at 2^-13 of the group's largest (whose factors count as the powers of two at or below them):
 * on random rows 1.4e-5 of the usual result, so that results close to 0 are off by more of themselves.  32-bit
 * results lose what 32-bit sums do.  Float scales multiply a block's sum in 32 bits, a's first: as long as a's lie
 * between 2^-108 and 2^103, nothing is lost to numbers that 32 bits do not hold, but for the result itself.  With e8m0
 * scales and 32-bit results a coordinate, code * scale, counts as bfloat16 holds it: infinite from 2^128 on, in
 * multiples of 2^-133.  Rows that start at multiples of 16 bytes (codes and stride) are read fastest.  A result of
 * more tiles than one launch has (2^24 of 64 x 64) fails before anything is written. */
int tv_fp8_matmul_dev(int device, void *stream, const uint8_t *d_a, size_t a_stride, const void *d_a_scales, size_t a_scale_stride, size_t m,
                      const uint8_t *d_b, size_t b_stride, const void *d_b_scales, size_t b_scale_stride, size_t n, int group,
                      size_t dim, int scale_type, void *d_out, int out_type, size_t out_stride);
/* Scores the m slots of each query (m <= 16384) against their 8-bit rows and writes the k <= m best, sorted
 * (score desc, slot asc), as the search does: nq * k scores and slots.  Products and sums are taken in 64 bits,
 * a score is rounded once.  A slot below 0 or not below n counts as absent, the same slot twice as two
 * candidates; a query with fewer than k present ends in scores of -infinity at slot -1.  NaN scores come last.
 * A scale that is NaN or infinite makes its rows' scores NaN or infinite. */
int tv_fp8_rescore_dev(int device, void *stream, const void *d_queries, int q_type, size_t q_stride, size_t nq,
                       const uint8_t *d_rows, size_t row_stride, const void *d_scales, size_t scale_stride, size_t n, int group, size_t dim, int scale_type,
                       const int64_t *d_slots, size_t slot_stride, size_t m, size_t k, float *d_out_scores, int64_t *d_out_slots,
                       void *d_workspace, size_t workspace_bytes);
size_t tv_fp8_rescore_workspace(size_t nq, size_t m, size_t dim);
/* Draws one slot from each row of n scores.  Allowed are the slots whose mask bit is set (d_mask_words NULL: all;
 * 64 slots a word, as tv_pack_mask makes them; mask_stride 0: one mask for all rows) and whose score is neither NaN nor
 * -infinity.  With slots ranked by score, ties to the lower slot, and w = exp((score - best) / temperature):
 * top_k > 0 keeps the first top_k; of those, top_p < 1 keeps a slot while the ones before it hold less than
 * top_p of their mass; of those, min_p > 0 keeps w >= min(min_p, 1); the best one always stays.  Drawn is the first
 * slot, in order of slots, at which the running sum of the kept w exceeds u times their sum, 0 <= u < 1.  A temperature
 * that is not above 0 draws the best.  out_probs: w over the sum of the kept ones.  A row that allows nothing: slot -1,
 * probability 0.  Weights are taken in 64 bits and held in whole multiples of 2^-(63 - ceil(log2 n)), rounded down; sums of them are exact,
 * so that a draw never depends on the order of additions.  A slot of less weight than that is never drawn, and a row loses less than n times that in all: 2e-5
 * of the best slot's weight at ten million slots, 0.15 % at 10^8, half of it at 2^31 - 1.  d_u holds a value a row; each of the four parameters does
 * too, or is NULL: temperature 1, no limit. */
int tv_sample_dev(int device, void *stream, const void *d_scores, int score_type, size_t score_stride, size_t rows, size_t n,
                  const uint64_t *d_mask_words, size_t mask_stride, const float *d_u, const float *d_temperature, const int32_t *d_top_k,
                  const float *d_top_p, const float *d_min_p, int64_t *d_out_slots, float *d_out_probs, void *d_workspace, size_t workspace_bytes);
size_t tv_sample_workspace(size_t rows, size_t n);

/* 4-bit rows hold e2m1 codes (1 sign, 2 exponent bits, 1 of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6; the sign is the highest
 * bit) of dim coordinates, 1 to 16384, two a byte, coordinate 2i in the low half of byte i, and an e8m0 scale for every
 * block of 32 coordinates (the last may be shorter) of a row.  A coordinate is code * scale.  The high half of the last byte of an
 * odd dim is written as 0 and not looked at.  Strides of codes and scales count bytes. */

/* Makes 4-bit rows of values.  With `amax` the largest magnitude of a block, its scale is the smallest power of two 2^e,
 * e >= -126, with amax < 7 * 2^e (so that the largest value is off by half a step at most, as all others are; a conversion that takes
 * 2^(floor(log2 amax) - 2), as is usual for the format, has half that scale where amax is 1.75 times a power of two or more, and cuts what is above 6 of it: rows made so are
 * rows here too, of other bytes); codes are x / scale
 * rounded to the nearest, ties to even, at most 6.  There is no code for them: an infinity or a NaN makes its block's scale NaN (255). */
int tv_fp4_quantize_dev(int device, void *stream, const void *d_x, int x_type, size_t x_stride, size_t rows, size_t dim,
                        uint8_t *d_codes, size_t code_stride, uint8_t *d_scales, size_t scale_stride);
/* The coordinates that 4-bit rows stand for: code * scale rounded once to out_type (32 bits hold it as long as it is below 2^128, bfloat16 too). */
int tv_fp4_values_dev(int device, void *stream, const uint8_t *d_codes, size_t code_stride, const uint8_t *d_scales, size_t scale_stride,
                      size_t rows, size_t dim, void *d_out, int out_type, size_t out_stride);
/* out[i][j] = the inner product of row i of a (m rows) with row j of b (n rows): products of codes within a block times both scales, added in
 * 32 bits and rounded once to out_type.  A block's sum is exact; a sum of blocks loses what 32-bit sums do, and is infinite where it, or
 * a block's part of it, passes 2^128.  Rows that start at multiples of 16 bytes (codes and stride) are read fastest.  A result of more tiles than one
 * launch has (2^24 of 64 x 64; 2^26 of 16 x 16 where rows are below 16 bytes, or 8 MB and more apart) fails before anything is written. */
int tv_fp4_matmul_dev(int device, void *stream, const uint8_t *d_a, size_t a_stride, const uint8_t *d_a_scales, size_t a_scale_stride, size_t m,
                      const uint8_t *d_b, size_t b_stride, const uint8_t *d_b_scales, size_t b_scale_stride, size_t n,
                      size_t dim, void *d_out, int out_type, size_t out_stride);

/* Kinds of rows that a norm ends in. */
typedef enum { TV_ROWS_FP8 = 0, TV_ROWS_FP4 = 1 } tv_row_kind;

/* h = x + residual (d_residual NULL: x), y = h / sqrt(mean of h^2 over the row + eps) * weight (d_weight NULL: 1), taken in 32 bits
 * and made into rows of 8 bits, as tv_fp8_quantize_dev with a group of 1, or of 4 (scale_type TV_SCALE_E8M0), as tv_fp4_quantize_dev.  The norm is of h before
 * it is rounded; d_sum, unless NULL, receives h rounded to x_type.  x, residual and sum have x_type; the sum may take the place of
 * x or of the residual (same address and stride) and overlaps neither in any other way.  eps: finite, not below 0.  A row of zeros with eps 0 has
 * no norm, nor has one with a NaN or an infinity: its values are NaN.  (Squares are taken in 32 bits, up to 16 of them added there and
 * those sums in 64: an |h| from 2^64 on counts as infinite, one from 2^62 on may; of a row that is below 2^-63 throughout the squares lose bits, below 2^-75 all of them, and eps is what
 * remains.)  A power of two as a scale is the one that h in 32 bits
 * and all that follows in 64 would have, but for a few in 10^8 blocks. */
int tv_rms_norm_dev(int device, void *stream, const void *d_x, int x_type, size_t x_stride, const void *d_residual, size_t residual_stride,
                    void *d_sum, size_t sum_stride, const void *d_weight, int weight_type, float eps, size_t rows, size_t dim,
                    int row_kind, int scale_type, uint8_t *d_codes, size_t code_stride, void *d_scales, size_t scale_stride);

/* Log probabilities under a softmax of rows of n scores, divided by a temperature a row (NULL: 1; one below 2^-126 or NaN is the limit
 * towards 0, the best slots share the mass; an infinite one gives all slots that have a probability the same).  A score that is 2^128 or more below the row's largest
 * has probability 0 at every temperature.  Slots whose mask bit is not set (d_mask_words NULL: all are; mask_stride 0: one mask for all rows) and slots of score
 * -infinity have probability 0, whatever else stands there.  For each row: out_log_probs, of the `given` slots in d_slots (-infinity for a slot of
 * probability 0 or outside 0 .. n - 1; the same slot may stand there twice); out_entropy, -sum p log p; the `top` slots of the highest scores,
 * ties to the lower slot, with their log probabilities (slot -1, -infinity where fewer have a probability; a NaN is not among them).  given and top are at
 * most 128; either may be 0.  A row with nothing allowed has entropy 0; one where an allowed score is NaN or +infinity has NaN for
 * the entropy and every log probability that is not -infinity.  d_out_stats, unless NULL, receives four floats a row for the gradient.  All sums are taken in 32 bits: a thread
 * adds up to 32 scores for themselves and those sums, no more than n / 4096 and a dozen (n / 8192 of two-byte scores), one after the other. */
int tv_log_probs_dev(int device, void *stream, const void *d_scores, int score_type, size_t score_stride, size_t rows, size_t n,
                     const uint64_t *d_mask_words, size_t mask_stride, const float *d_temperature, const int64_t *d_slots, size_t slot_stride, size_t given,
                     size_t top, float *d_out_log_probs, float *d_out_entropy, int64_t *d_out_top_slots, float *d_out_top_log_probs, float *d_out_stats,
                     void *d_workspace, size_t workspace_bytes);
size_t tv_log_probs_workspace(size_t rows, size_t n, size_t top);
/* The gradient of the scores, in their type, from those of the log probabilities and of the entropy (either may be NULL), with the call's own inputs and the stats
 * that it left: (sum over given of g [slot] - G p - g_entropy p (log p + entropy)) / temperature, G the sum of g over given slots that have a
 * probability; a slot of probability 0 has gradient 0, and so has a row at the limit.  The same given slot twice adds up. */
int tv_log_probs_grad_dev(int device, void *stream, const void *d_scores, int score_type, size_t score_stride, size_t rows, size_t n,
                          const uint64_t *d_mask_words, size_t mask_stride, const float *d_temperature, const int64_t *d_slots, size_t slot_stride, size_t given,
                          const float *d_stats, const float *d_grad_log_probs, const float *d_grad_entropy, void *d_grad_scores, size_t grad_stride);

/* ---- host-only derivations (no GPU touched) ------------------------------- */

/* The tables tv_index_create derives: Rotation::new (rotation.rs:141-187;
 * signs/perms 2*dim each, round 0 first) and codebook::codebook (codebook.rs:50). */
int tv_host_rotation_tables(int dim, float *signs, uint32_t *perms, int *block, float *inv_sqrt_block);
int tv_host_codebook(int bits, int dim, float *boundaries, float *centroids);

/* ---- snapshot images (turbovec/src/io_v7.rs) ------------------------------- */

/* The byte form TurboQuantIndex::to_bytes (lib.rs:2167) / IdMapIndex::to_bytes
 * (id_map.rs:971) and `write` produce: an unclaimed generation-0 TV7 image
 * (io_v7.rs:902-925 write_image: superblock :516-542, header slot :549-599,
 * units :602-629, CRC-32C :128-141).  kind 0 = slot-addressed index, 1 = id map.
 * format 7 is that image; format 6 is the flat TVPI / TVIM container of the
 * release before (convert.rs:14-31, :453-512), which the reference's committed
 * sha256 digests of to_bytes() still hash.  These four touch no GPU. */
size_t tv_host_snapshot_len(int format, int dim, int bits, int kind, size_t n_calib, size_t n);
/* seq: sequential-blocked codes of n rows (what tv_index_download_seq returns);
 * shift/scale: n_calib floats each (n_calib is 0 or dim); ids: n values, kind 1 only.
 * out must hold tv_host_snapshot_len(...) bytes. */
int tv_host_snapshot_compose(int format, int dim, int bits, int kind, const float *boundaries, const float *centroids,
                             size_t n_calib, const float *shift, const float *scale,
                             const uint8_t *seq, size_t n, const float *scales, const uint64_t *ids,
                             uint8_t *out);
/* Validate an image of either format (magic, revision, checksums, geometry, that a TV7
 * image is a snapshot and not a synced container with pending operations) and report its shape. */
int tv_host_snapshot_info(const uint8_t *bytes, size_t len, int *format, int *kind, int *dim, int *bits,
                          size_t *n_calib, size_t *n);
/* Unpack a validated image; any output pointer may be NULL.  seq: ceil(n/32)*G*32 bytes. */
int tv_host_snapshot_extract(const uint8_t *bytes, size_t len, float *boundaries, float *centroids,
                             float *shift, float *scale, uint8_t *seq, float *scales, uint64_t *ids);
/* Snapshot of a device-resident index.  ids == NULL writes kind 0, otherwise kind 1 with
 * ids[slot] (id_map.rs slot_to_id).  out == NULL only reports *len. */
int tv_index_to_bytes(const tv_index *ix, const uint64_t *ids, int format, uint8_t *out, size_t cap, size_t *len);
/* Build a device-resident index from an image (replaces from_v7_image, lib.rs:2196);
 * ids_out (may be NULL) receives n ids for a kind-1 image. */
int tv_index_from_bytes(const uint8_t *bytes, size_t len, int device, tv_index **out, uint64_t *ids_out);

/* ---- test / measurement hooks -------------------------------------------- */

/* Integer accumulators and final float scores of every (query, slot) pair,
 * nq*n each (either may be NULL): what the parity tests compare bit-for-bit. */
int tv_debug_scan(tv_index *ix, const float *queries, size_t nq, int32_t *acc_out, float *scores_out);
/* Query preparation only: rotated (and TQ+-calibrated) rows nq*dim, and per
 * query scale and bias of the active score mode (any may be NULL). */
int tv_debug_prepare(tv_index *ix, const float *queries, size_t nq,
                     float *q_rot_out, float *scale_out, float *bias_out);
/* Duration in milliseconds of the full scans of the most recent tv_search* call
 * on this index (of its first chunk of queries, or the first one of each 8192)
 * and how many launches they were.  Where another launch of the call comes
 * before the full scan, the duration is the span between two readings of the
 * device clock -- as that launch ends, and as the selection behind the scan
 * starts -- and the gaps between the launches count; a scan from open floors
 * and the exact path are measured with HIP events around the first 32 launches. */
int tv_last_scan_ms(const tv_index *ix, float *ms, int *launches);
/* Queries one full-scan launch of the last search served (a full launch of a large batch). */
int tv_debug_queries_per_launch(const tv_index *ix, int *queries);
/* Path selection for tests (results must be identical either way): bit 0 makes
 * every search take the full-range list / dense-select path instead of
 * sample-then-filter; bit 1 keeps large batches on the one-tile-per-launch scan
 * instead of the batched ones; bit 2 keeps them off the all-queries-per-pass
 * kernel only; bit 3 keeps u8-LUT batches on the scan that holds whole tables in
 * LDS (at most 8 queries per pass) instead of the larger ones; bit 4 samples
 * small indexes (bits 1 and 2 do too), and those of up to 16384 blocks by the
 * levels of rows that tests lay data out against; bit 6 has filtered searches
 * gather the allowed rows first whatever their number; bit 7 has u8-LUT batches
 * take the int8 scan in front of the tables (65 queries and more over a large
 * index of 2- or 3-bit codes otherwise) wherever it has an instance for the row
 * length and there are four blocks of rows to sample; without bit 6 any other bit, bit 5
 * of no other meaning too, has them read the mask as they scan. */
int tv_debug_set_path(tv_index *ix, int force_full_lists);
/* The sampling ladder a search for the k best of nq queries (its first chunk of up to 1024) runs
 * on this index as it stands, unfiltered: block strides of the successive scans, strides[0 ..
 * *count), the last one 1 (the full scan); level i reads blocks 0, strides[i], 2*strides[i], ...,
 * and in the repeated pass of queries whose candidates overflowed it starts at block
 * repeat_offsets[i].  At most cap entries are written (either array may be NULL); *count = 0 means
 * the search does not sample (large k, an index so small that every block is scored and its best
 * row kept, or the exact path is forced).  For tests and the bench,
 * which lay rows out against the ladder. */
int tv_debug_sampling_plan(const tv_index *ix, size_t nq, size_t k, uint32_t *strides, uint32_t *repeat_offsets,
                           size_t cap, size_t *count);
/* A sampling level whose candidates do not fit (its floor came from a level that happened to read
 * poor rows) runs a second time, on the device, from the floor taken from what did fit.  track = 1
 * makes searches report such levels (a few hundred bytes more in the flag copy), 0 stops that,
 * negative leaves it as it is; *count (may be NULL) = levels repeated so far while tracking. */
int tv_debug_level_repeats(tv_index *ix, int track, size_t *count);
/* Bytes of the index's cached search workspace -- with what its filtered searches keep of their
 * allowed rows, up to 1.25 GiB and four bytes a row, which is given back when an allocation of this
 * library fails on that device -- and of its host-call staging allocation (either pointer may be
 * NULL).  They grow otherwise, and tv_search_dev_noalloc touches neither.  What the device's indexes
 * share (tv_index_create) is not in them. */
int tv_debug_workspace_bytes(const tv_index *ix, size_t *workspace, size_t *staging);
/* How many filtered searches so far ran on their allowed rows alone, and how many of
 * those read them in place, without a copy. */
int tv_debug_gathered_searches(const tv_index *ix, size_t *count, size_t *in_place);
/* How many queries so far did not finish in the single sampled pass because their
 * candidate buffer overflowed (they are scanned once more, all together, from a raised
 * floor), and how many of those went on to the exact list / select path. */
int tv_debug_overflow_redos(const tv_index *ix, size_t *count);
int tv_debug_exact_redos(const tv_index *ix, size_t *count);
/* How many tv_search / tv_search_dev calls so far were served by another caller's launch: calls
 * that arrive while the index is busy are merged, by the next caller to get it, with every
 * waiting call of the same k and mask into one batch. */
int tv_debug_merged_calls(const tv_index *ix, size_t *count);
/* Bandwidth probe on the index's stream: reps launches of a pure read-sum over
 * d_src (d_dst NULL) or of a plain copy d_src -> d_dst, bytes each; mean
 * milliseconds per launch.  Calibrates the achievable HBM rate and gives the
 * hardware counters a kernel of known traffic. */
int tv_debug_stream_probe(tv_index *ix, const void *d_src, void *d_dst, size_t bytes, int reps, float *ms_per_rep);
/* Matrix-unit probe on the index's stream: reps launches of the batched scan's
 * MFMA loop alone (int8 32x32x32, A operands in registers, B operands read from
 * LDS, pseudo-random bytes, no HBM traffic), iters x 48 MFMAs per wavefront;
 * mean milliseconds per launch and the int8 operations (2 per multiply-add) of
 * one launch.  Calibrates the rate the matrix unit sustains on this chip under
 * its power management, as the read probe does for HBM.  No counterpart in the
 * reference (its roofline probe is the read one, examples/stream_bw.rs:30-66). */
int tv_debug_mfma_probe(tv_index *ix, int iters, int reps, float *ms_per_rep, double *ops_per_rep);
/* Device pointers of the resident index (native layout) for tools. */
int tv_index_device_ptrs(const tv_index *ix, void **d_codes, void **d_scales, size_t *code_bytes);

#ifdef __cplusplus
}
#endif
#endif
