/*
 * cbq_serve.h -- batched serving over a paged key/value cache
 * (libcbq_hip.so, csrc/cbq_paged_append.hip and csrc/cbq_prefix_attn*.hip), and
 * the verification of drafted tokens (csrc/cbq_verify.hip).
 *
 * These entry points have no counterpart in the reference's C/HIP libraries:
 * its models run HF's attention over one dense cache per sequence.  They let
 * a batch of sequences share one pool of key/value pages and one prefix (a
 * system prompt, a document) whose pages are stored, and in attention read,
 * once for all of them.
 *
 * Conventions as cbq_hip.h: device pointers, asynchronous on `stream`, no
 * allocation, no synchronisation, no host copy of device data (so every call
 * can be captured in a HIP graph), return 0 / 1 (HIP error) / 2 (invalid
 * argument, nothing launched).
 *
 * What only the device knows (positions, slots, lengths, page tables) is
 * checked there, so that no value of it reads or writes out of range:
 *   - a length counts as 0 below 0 and as the row's capacity above it;
 *   - a table entry outside [0, n_pages) hides the keys of its page from every
 *     query (-1 is the value to write where no page is taken);
 *   - a slot outside the pool stores nothing.
 */
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CBQ_F32 0
#define CBQ_BF16 1
#define CBQ_F16 2

/* A pool of pages.  Element d of row r (0 <= r < page) of kv head h of page p
 * is base[p * stride[0] + h * stride[1] + r * stride[2] + d]; strides are in
 * elements and d is contiguous, so both [pages, heads, rows, hd] and [pages,
 * rows, heads, hd] layouts, and keys and values in one tensor, are described.
 * 1 <= page <= 65536; n_pages * page < 2^31.  The attention also needs page and
 * row strides of 0 or more whose largest offset is below 2^32 times the largest
 * power of two (4096 at most) that divides all of them in bytes: any pool up to
 * 512 GiB if they are whole 128 bytes. */
typedef struct cbq_paged_kv {
    void *k, *v;
    int64_t k_stride[3], v_stride[3];
    int64_t n_pages;
    int32_t page, n_kv, hd;
    int32_t dtype;                          /* CBQ_F32, CBQ_BF16 or CBQ_F16 */
} cbq_paged_kv;

/* New tokens into the cache.  For each token t < N, with p = positions[t]:
 *   q_out[t, i]    = rope_p(rmsnorm(q[t, i]) * q_weight)       i < n_q
 *   k page of slot = rope_p(rmsnorm(k[t, j]) * k_weight)        j < n_kv
 *   v page of slot = v[t, j]
 * slots[t] = page_id * page + row.  rmsnorm(x) = x * rsqrt(mean(x^2) + eps),
 * left out (with its weight) when norm is 0; weights [hd] may be NULL (ones).
 * rope_p turns the pairs (x[d], x[d + rot/2]), d < rot/2, by the angle whose
 * cosine and sine are cos_table[p, d] and sin_table[p, d] (tables [n_pos,
 * rot] of float; their second halves repeat the first and are not read); the
 * elements from rot on pass.  All of it in fp32, rounded once, to the cache's
 * type, which is x's type, or any type when x is fp32.  q_out [N, n_q, hd] is
 * contiguous, of the cache's type, and may not alias q, k or v.
 * q, k, v: element [t, h, d] at t * stride[0] + h * stride[1] + d.
 * A token whose position is outside [0, n_pos) stores nothing, and its query
 * is turned by row 0; two tokens with one slot leave pieces of either's row.
 * hd even, 2..256; rot even, 2..hd; N * (n_q + 2 n_kv) < 2^31. */
int cbq_paged_append(const void *q, const void *k, const void *v, int x_dtype,
                     const int64_t *q_stride, const int64_t *k_stride, const int64_t *v_stride,
                     const float *cos_table, const float *sin_table, int64_t n_pos, int rot,
                     const int64_t *positions, const int64_t *slots, int norm,
                     const float *q_weight, const float *k_weight, float eps, void *q_out,
                     const cbq_paged_kv *cache, int64_t N, int n_q, hipStream_t stream);

/* One query token for each of `batch` sequences: sequence b sees the shared
 * prefix (`prefix` keys, in the pages prefix_table names in order) and its own
 * lengths[b] keys (pages tables[b * table_stride + i], i < width), and
 *   out[b, i] = softmax(q[b, i] . k_j * scale) . v_j     over the keys it sees,
 * query head i reading kv head i / (n_q / n_kv); a sequence that sees no key
 * gets zeros.  The prefix is read once for all sequences, or by each where
 * keys are so few that this takes less time.  q [batch, n_q, hd] with strides
 * {token, head} in elements, 16-byte aligned as the pages are; out contiguous,
 * of q's type, which is the cache's.  Scores, maxima, sums and the weighted
 * values are fp32; for 16-bit types the weights exp(s - max) are rounded to
 * that type for the matrix cores.  hd in {64, 128, 256}; n_q % n_kv == 0;
 * n_q < 2^20, batch < 2^30, batch * n_q < 2^31; prefix + width * page <=
 * 2^31 - 65536.
 * workspace: cbq_prefix_attn_decode_workspace bytes (which may be 0), 16-byte
 * aligned, overwritten by every call. */
size_t cbq_prefix_attn_decode_workspace(const cbq_paged_kv *cache, int64_t prefix, int width,
                                        int batch, int n_q);
int cbq_prefix_attn_decode(const void *q, const int64_t *q_stride, const cbq_paged_kv *cache,
                           const int32_t *prefix_table, int64_t prefix, const int32_t *tables,
                           int64_t table_stride, int width, const int32_t *lengths, int batch,
                           int n_q, float scale, void *out, void *workspace,
                           size_t workspace_bytes, hipStream_t stream);

/* A run of new tokens for each sequence: run b is tokens q_start[b] ..
 * q_start[b + 1] - 1 of q [N, n_q, hd] (q_start [batch + 1], ascending from 0
 * to N; tokens before the first run and after the last get zeros).  Its own
 * keys, lengths[b] of them, end with the run's: the token that is i-th from
 * the run's end sees the prefix and the own keys up to the i-th from the end.
 * Otherwise as cbq_prefix_attn_decode; N * n_q < 2^31 and N / 16 * n_q +
 * min(batch, N) * n_kv < 2^31. */
size_t cbq_prefix_attn_prompt_workspace(const cbq_paged_kv *cache, int64_t prefix, int width,
                                        int batch, int64_t N, int n_q);
int cbq_prefix_attn_prompt(const void *q, const int64_t *q_stride, const int32_t *q_start,
                           const cbq_paged_kv *cache, const int32_t *prefix_table, int64_t prefix,
                           const int32_t *tables, int64_t table_stride, int width,
                           const int32_t *lengths, int batch, int64_t N, int n_q, float scale,
                           void *out, void *workspace, size_t workspace_bytes,
                           hipStream_t stream);

/* Drafted tokens against the target's probabilities.  Sequence b has n = n_drafts[b]
 * drafts (as a length, inside 0..drafts; all of them when n_drafts is NULL) d_i, drawn
 * from q_i = draft_probs[b, i], the target's p_i = probs[b, i] (i <= n; p_n is the
 * row behind them all) and random numbers u_i = uniforms[b, i] of [0, 1).  Drafts are
 * kept while
 *   u_i q_i(d_i) < p_i(d_i),
 * and behind the a that are kept one token is drawn by u = uniforms[b, drafts] from
 *   w = max(p_a - q_a, 0) if a < n, or from w = p_n:
 * the first token whose sum w(0) + .. + w(token) exceeds u times the sum of all (the
 * last one of w > 0 where rounding leaves none).  So the tokens are distributed as the
 * target's.  Without draft_probs (NULL) a draft is taken as certain: q_i is 1 at d_i
 * and 0 elsewhere.  Products, differences and sums are in 64 bits.
 *   tokens[b] = d_0 .. d_(a-1), the drawn one, then -1;  counts[b] = a + 1.
 * What is NaN or below 0 in w counts as 0; where all of w is 0, p_a is taken in its
 * place, and where that is too, the token is -1.  A draft outside [0, vocab) has the
 * probability 0; its q is 1 without draft_probs, else 0.
 * probs, draft_probs: dtype CBQ_F32, CBQ_BF16 or CBQ_F16, element [b, i, v] at b *
 * stride[0] + i * stride[1] + v.  drafts [batch, drafts], uniforms [batch, drafts + 1],
 * tokens [batch, drafts + 1] and counts [batch] are contiguous.  1 <= vocab < 2^31,
 * 0 <= drafts = n_max < 2^20, 0 <= batch < 2^24, batch * drafts < 2^30.
 * workspace: cbq_verify_drafts_workspace bytes, 16-byte aligned, overwritten. */
size_t cbq_verify_drafts_workspace(int batch, int64_t vocab);
int cbq_verify_drafts(const void *probs, const int64_t *p_stride, const int64_t *drafts,
                      const void *draft_probs, const int64_t *q_stride, int dtype,
                      const int32_t *n_drafts, const float *uniforms, int batch, int n_max,
                      int64_t vocab, int64_t *tokens, int32_t *counts, void *workspace,
                      size_t workspace_bytes, hipStream_t stream);

#ifdef __cplusplus
}
#endif
