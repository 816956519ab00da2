/*
 * mm_latent.h -- C ABI of the shared-prompt decode operators on DEVICE pointers: an 8-bit
 * compressed (MLA) cache, attention of a batch whose rows share stored prompts, and the
 * verification of drafted tokens. The reference keeps one fp32 cache per request
 * (CpuDecoder, src/infer/inference.cpp:47-174) and decodes one token at a time
 * (inference.cpp:469-579); these are the forms a batched server or a group rollout needs.
 *
 * Conventions:
 *   - every call validates what the host can see, enqueues its kernels on `stream` (a
 *     cudaStream_t of the current device; NULL = the legacy default stream) and returns
 *     without waiting (mm_latent_status alone waits). Nothing is allocated and no context is involved; scratch is the
 *     caller's `workspace` and may be reused by the next call on the same stream;
 *   - returns 0 or 1 + ErrorCode as include/mm_cuda.h; mm_latent_last_error() gives the
 *     calling thread's last message. No C++ exception leaves an entry;
 *   - what only the device holds (lengths, group bounds, slots, draft tokens) is not checked
 *     on the host; kernels clamp or skip out-of-range values, so no access leaves a buffer;
 *   - results do not depend on scheduling (no floating-point atomics): equal inputs give equal
 *     bits (a slot written twice by one call excepted);
 *   - memory past a length may hold anything, NaN included: it never reaches a result;
 *   - the attention kernel's waits are bounded. One that runs out (a defect or a fault of the
 *     machine, never the input) makes the results it concerns NaN, and mm_latent_status says so.
 */
#ifndef MM_LATENT_H
#define MM_LATENT_H

#include <stddef.h>
#include <stdint.h>

#include "mm_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { MM_F32 = 0, MM_F16 = 1, MM_BF16 = 2, MM_E4M3 = 3 };

/* A latent cache of `rows` x `positions` entries, each kv latent values and rope_dim rotated
 * key values; strides in elements of the array they belong to, positions of `scale` adjacent.
 *   kind MM_F16 / MM_BF16: latent holds [kv | rope_dim] values per position, rope and scale
 *     are unused (the layout of the context's own cache);
 *   kind MM_E4M3: latent holds kv e4m3 bytes, rope rope_dim 16-bit values (rope_kind), scale
 *     one fp32 factor per position: value = code * scale. One factor per position (not per
 *     block) because the rows are RMS-normalised and it then factors out of both products of
 *     attention. The rope key stays 16-bit: its magnitude is not normalised with the latent. */
typedef struct mm_latent_cache {
    void* latent;
    void* rope;
    float* scale;
    int64_t row_stride, pos_stride;
    int64_t rope_row_stride, rope_pos_stride;
    int64_t scale_row_stride;
    int32_t rows, positions, kv, rope_dim;
    int32_t kind, rope_kind;
} mm_latent_cache;

/* Copies the calling thread's last message (NUL-terminated, truncated to cap); returns its
 * length. */
size_t mm_latent_last_error(char* buf, size_t cap);

/* Waits for `stream` and reports whether a kernel of this library on the current device gave up on
 * a wait since the last report: 0, or MM_GPU_ERROR (results of a call in between are then NaN). */
int mm_latent_status(void* stream);

/* Quantises n new positions into an MM_E4M3 cache. latent [n][kv] and rope [n][rope_dim] of
 * `dtype` (row strides in elements); position i goes to slots[i] = row * positions + position;
 * slots outside [0, rows * positions) are skipped. The others are distinct: a position given twice
 * in one call may end with the codes, scale and rope key of different inputs (nothing else changes).
 *   scale = max(max_c |x_c| / 448, 2^-100), code = e4m3(x / scale) round to nearest even,
 * both in IEEE fp32. A NaN reads back as NaN; an infinity makes its position read back NaN. */
int mm_latent_cache_write(const mm_latent_cache* cache, const void* latent, int64_t latent_stride,
                          const void* rope, int64_t rope_stride, int dtype, const int64_t* slots,
                          int64_t n, void* stream);

/* Reads n positions of an MM_E4M3 cache back: out [n][kv + rope_dim] of out_dtype (row stride
 * out_stride); slots as above, rows of skipped slots are zeros. */
int mm_latent_cache_read(const mm_latent_cache* cache, const int64_t* slots, int64_t n, void* out,
                         int64_t out_stride, int out_dtype, void* stream);

/* Absorbed latent attention of `tokens` query tokens per row over a shared prefix and the
 * row's own suffix. Rows [group_start[g], group_start[g + 1]) (non-decreasing, device int32
 * [groups + 1]) are group g and attend over prefix row g, positions [0, prefix_len[g]); a row
 * outside every group has no prefix. Row b's suffix is suffix row b: its last `tokens`
 * positions are the query tokens' own, so token t sees positions
 * [0, suffix_len[b] - (tokens - 1 - t)). With K the concatenation of both,
 *   s = scale * q . K_j,  out = sum_j softmax(s)_j K_j[0, kv),  lse = ln sum_j e^s
 * and a query that sees no position gets out = 0, lse = -infinity.
 * A latent NaN or infinity, or a scale that is one, makes the results of the queries that see its
 * position not finite, and no other's.
 * Lengths are clamped to [0, max_prefix] and [0, max_suffix]; max_* are host-side bounds
 * (<= the caches' positions) that size the launch, as is max_group (rows of the largest group;
 * larger groups leave their further rows without the prefix).
 * q: dtype MM_F16 / MM_BF16 with element strides, last dimension contiguous; 16-bit caches
 * have the same dtype, e4m3 caches the same rope_kind. out [rows][tokens][heads][kv] of dtype
 * and lse [rows][tokens][heads] fp32 (may be NULL) are contiguous. prefix may be NULL (with
 * groups = 0), and so may suffix. Pointers are aligned to their elements; the tensor-core form
 * (128 + 16 and 512 + 32 wide) also needs q and cache rows of 16-byte multiples at 16-byte
 * addresses and out at an 8-byte one, other calls take a slower form of the same results. */
typedef struct mm_shared_prefix_desc {
    const void* q;
    int64_t q_row_stride, q_token_stride, q_head_stride;
    int32_t dtype, rows, tokens, heads;
    const int32_t* group_start;
    const int32_t* prefix_len;
    const int32_t* suffix_len;
    int32_t groups, max_group, max_prefix, max_suffix;
    float scale;
    int32_t reserved;
    void* out;
    float* lse;
} mm_shared_prefix_desc;

/* Bytes of workspace the call needs (0 possible), or -(1 + ErrorCode). */
int64_t mm_shared_prefix_attention_workspace(const mm_shared_prefix_desc* desc,
                                             const mm_latent_cache* prefix,
                                             const mm_latent_cache* suffix);
int mm_shared_prefix_attention(const mm_shared_prefix_desc* desc, const mm_latent_cache* prefix,
                               const mm_latent_cache* suffix, void* workspace,
                               size_t workspace_bytes, void* stream);

/* Verification of drafted tokens (speculative sampling) from given random numbers. For row b,
 * with p = target_probs [rows][drafts + 1][vocab], q = draft_probs [rows][drafts][vocab] (NULL:
 * deterministic drafts, q = 1 at the drafted token) of `dtype`, contiguous rows of vocab:
 *   draft i < draft_len[b] is accepted while u_accept[b][i] * q_i(x_i) < p_i(x_i) in fp32 (a
 *   token outside the vocabulary is rejected); with j the first rejected position (or
 *   draft_len[b]) the row emits its j accepted tokens and one more: the first y with
 *   sum_{x <= y} w_x > floor(k W / 2^24), W = sum_x w_x, k = floor(2^24 u_sample[b]) clamped to
 *   [0, 2^24), w_x = floor(2^38 clamp(r_x, 0, 1)), r = max(p_j - q_j, 0) after a rejection (p_j
 *   where that is all zeros) and p_j when every draft was accepted.
 * The sums are exact integers, so the token does not depend on their order. out_tokens
 * [rows][drafts + 1] int32: accepted tokens, the sampled one, then -1; accepted [rows] = j. A
 * row whose weights are all zero emits -1 as its sampled token. vocab <= 262,144. */
int mm_verify_drafts(const void* target_probs, const void* draft_probs, int dtype,
                     const int32_t* draft_tokens, const int32_t* draft_len, const float* u_accept,
                     const float* u_sample, int rows, int drafts, int vocab, int32_t* out_tokens,
                     int32_t* accepted, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MM_LATENT_H */
