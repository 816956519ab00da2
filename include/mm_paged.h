/*
 * mm_paged.h -- C ABI of the paged-cache decode and beam-search operators on DEVICE pointers. A
 * paged cache is a pool of pages (an mm_latent_cache whose rows are pages and whose positions are
 * a page's entries) and a page table: position t of table row r is entry t % page of page
 * table[r][t / page]. The reference keeps one contiguous fp32 cache per request (CpuDecoder,
 * src/infer/inference.cpp:47-174) and decodes greedily or by sampling (inference.cpp:345-426);
 * these are the forms a server of many long requests and a beam search need.
 *
 * Conventions are those of mm_latent.h: enqueued on `stream` of the current device, nothing is
 * allocated, no wait (mm_paged_status alone waits), 0 or 1 + ErrorCode, messages by
 * mm_latent_last_error. What only the device holds (tables, lengths, positions, parents) is clamped
 * or skipped, so no access leaves a buffer. Results do not depend on scheduling: equal inputs give
 * equal bits.
 */
#ifndef MM_PAGED_H
#define MM_PAGED_H

#include "mm_latent.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct mm_paged_cache {
    mm_latent_cache pool;      /* rows = pages, positions = entries of a page */
    const int32_t* table;      /* [table_rows][table_columns], columns adjacent */
    int64_t table_stride;
    int32_t table_rows, table_columns;
} mm_paged_cache;

/* Waits for `stream` and reports whether a kernel of mm_paged_attention on the current device gave
 * up on a wait since the last report (a defect or a fault of the machine, never the input): 0, or
 * MM_GPU_ERROR (the results it concerns are NaN). */
int mm_paged_status(void* stream);

/* Stores n new positions. values [n][kv + rope_dim] of `dtype` (row stride in elements) are a
 * projection's results: kv latent values, then a rotary key before its rotation. Token i goes to
 * position positions[i] of table row rows[i] (rows NULL: row i); a token whose position is negative or
 * past the table, whose row is outside it, or whose page is outside the pool is skipped. With
 *   c = latent * norm / sqrt(mean(latent^2) + eps)    (norm fp32 [kv]; NULL: c = latent)
 *   (a, b) -> (a cos t - b sin t, a sin t + b cos t),  t = position * theta^(-2 j / rope_dim)
 * on the adjacent pairs j of the key (angles in fp64, src/model/ops.cpp:88-108), a 16-bit pool gets
 * c and the key rounded once; an MM_E4M3 one scale = max(max |c| / 448, 2^-100), codes e4m3(c / scale)
 * and the key in its rope_kind. (Without norm the codes are exactly those; with it c and the quotient are off by some units
 * in the last place of fp32, by how many depends on the strides, which may show in the code of a quotient that is as near to
 * the middle of two.) Two tokens of one call for one position leave a mix of both. */
int mm_paged_append(const mm_paged_cache* cache, const void* values, int64_t values_stride, int dtype,
                    const int32_t* rows, const int32_t* positions, int64_t n, double theta,
                    const float* norm, float eps, void* stream);

/* Absorbed latent attention of one query token per row over its pages. Row b sees the positions
 * j < lengths[b] of table row b with j < sinks or j >= lengths[b] - window (window 0: all of them),
 * except those of pages outside the pool (entries of pages that were given back may hold -1):
 *   s = scale * q . K_j,  out = sum_j softmax(s)_j K_j[0, kv),  lse = ln sum_j e^s
 * A query that sees no position gets out = 0, lse = -infinity. What unseen positions hold (NaN
 * included) never reaches a result; a NaN or an infinity in a seen one reaches its row's alone, as the
 * formula has it (a score of -infinity is a weight of zero). e4m3 scales above 2^100 may make results infinite.
 * Lengths are clamped to [0, max_length], max_length <= table_columns * page: a host-side
 * bound that sizes the launch.
 * q: MM_F16 / MM_BF16 [rows][heads][kv + rope_dim], last dimension adjacent; 16-bit pools have its
 * type, e4m3 ones its rope_kind. out [rows][heads][kv] of dtype and lse [rows][heads] fp32 (may be
 * NULL) are contiguous. The tensor-core form (128 + 16 and 512 + 32 wide, pages of a multiple of 16
 * positions) needs pool rows of 16-byte multiples at 16-byte addresses, q at an 8-byte one with
 * strides of multiples of 4 and out at an 8-byte one; other calls take a slower form. */
typedef struct mm_paged_attention_desc {
    const void* q;
    int64_t q_row_stride, q_head_stride;
    const int32_t* lengths;
    int32_t dtype, rows, heads, max_length, window, sinks;
    float scale;
    int32_t reserved;
    void* out;
    float* lse;
} mm_paged_attention_desc;

/* Bytes of workspace the call needs (0 possible), or -(1 + ErrorCode). */
int64_t mm_paged_attention_workspace(const mm_paged_attention_desc* desc, const mm_paged_cache* cache);
int mm_paged_attention(const mm_paged_attention_desc* desc, const mm_paged_cache* cache, void* workspace,
                       size_t workspace_bytes, void* stream);

/* Self-test of what follows a wait that ran out: mm_paged_attention in which the loads of every other CTA end after `steps`
 * steps of a run of tiles, so that its other warps wait for what does not come (a second or two). The rows that it has
 * tiles of are NaN, the others as ever, and mm_paged_status reports MM_GPU_ERROR once. Refused for calls of the slower form, which has no
 * waits. */
int mm_paged_selftest_wait_timeout(const mm_paged_attention_desc* desc, const mm_paged_cache* cache, void* workspace,
                                   size_t workspace_bytes, int steps, void* stream);

/* Beam search's selection. For batch entry b, candidate (k, v) has the score
 *   scores[b][k] + logits[b][k][v] - ln sum_u exp(logits[b][k][u]),
 * a finished beam (finished[b][k] != 0) the one candidate (k, eos) with scores[b][k]. The `count`
 * best go to out_scores / out_parents / out_tokens [batch][count] in descending order, ties to the
 * lowest k * vocab + v. Candidates without a finite fp32 score (dead beams of score -infinity, banned
 * tokens, a beam whose scores hold a NaN or +infinity) are never taken; entries that are left over
 * are (-infinity, min(entry, beams - 1), -1). Scores are compared in fp64.
 * logits of `dtype` with strides in elements, tokens adjacent; scores and finished (bytes, may be
 * NULL) [batch][beams] contiguous. beams, count <= 32, vocab <= 2^20, eos < vocab. */
int64_t mm_beam_select_workspace(int batch, int beams, int vocab, int count);
int mm_beam_select(const void* logits, int64_t batch_stride, int64_t beam_stride, int dtype, const float* scores,
                   const uint8_t* finished, int eos, int batch, int beams, int vocab, int count, float* out_scores,
                   int32_t* out_parents, int32_t* out_tokens, void* workspace, size_t workspace_bytes, void* stream);

/* Rows take over their parents' caches. Every row owns its last, partly filled page, the pages of the table
 * entries behind it that it may grow into, and a spare page. Row i with parent p = parents[i] and n =
 * lengths[p] gets table entries [0, n / page) of p (full pages are shared). When p != i, and n % page > 0 or n !=
 * lengths[i], its spare page becomes its entry n / page, with p's n % page positions copied into it in every
 * layer, and its own page at entry lengths[i] / page is its new spare (-1 where its lengths fill the table, which
 * leaves it without). Other entries stay, but for those of a row that takes over one shorter by a page or more
 * (of pages that it would write, and others read): what stands between n / page and lengths[i] / page becomes -1 where
 * another row has that page; so does, in the call after which the row begins a page (n % page = 0) or lays one aside
 * unwritten, an entry that another row has or that is the row's spare page. Such a row needs a page of its own where its
 * entry is -1 before it stores there, and between two calls it stores no further than to the end of its last page.
 * (Other tables that hold a page are not looked at.) out_lengths[i] = n. A parent outside [0, rows) is the row itself;
 * lengths are clamped to the table.
 * `cache` describes layer 0 (pages, page entries) and its table; layer l is layer_strides[0..2] * l
 * elements further in latent, rope and scale. out_table [rows][columns] contiguous, out_spare and
 * out_lengths [rows] are other memory than their inputs. Pages in use and spare pages are distinct. */
int mm_beam_reorder(const mm_paged_cache* cache, int layers, const int64_t layer_strides[3], const int32_t* spare,
                    const int32_t* lengths, const int32_t* parents, int32_t* out_table, int32_t* out_spare,
                    int32_t* out_lengths, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MM_PAGED_H */
