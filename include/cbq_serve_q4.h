/*
 * cbq_serve_q4.h -- batched serving over a paged key/value cache of 4 bits
 * (libcbq_hip.so, csrc/cbq_q4_append.hip and csrc/cbq_q4_attn*.hip).
 *
 * As cbq_serve.h, whose conventions and device-side checks hold here too, with
 * keys and values quantised as they are written and read in that form: 4.5 bits
 * a value.  No counterpart in the reference, which compresses weights only.
 *
 * The format.  A row of hd values (one token, one kv head) is hd / 64 groups of
 * 64 neighbouring values.  A group has two bf16 numbers, scale s and mid m, and
 * 64 codes c of 0..15; it stands for the values
 *     m + s * (c - 7.5).
 * Written from x, in 64 bits with bf16's nearest (by way of fp32) where it says so:
 *     m = bf16((max x + min x) / 2)
 *     s = bf16(max(max x - m, m - min x) / 7.5)
 *     c = min(max(floor((x - m) / s) + 8, 0), 15), 8 where s is 0
 * so a value comes back within 0.52 s.  A group that holds a NaN or an infinity,
 * or whose m or s is none of bf16's finite numbers, is stored with m = NaN and
 * reads as NaN.  A row's codes lie in the order in which the attention's matrix
 * products take them, four of each group side by side: value 64 g + e has the low
 * (e even) or high four bits of byte (e / 4) * (hd / 32) + 2 g + e % 4 / 2.  A group's
 * pair is {s, m}.
 */
#pragma once

#include "cbq_serve.h"

#ifdef __cplusplus
extern "C" {
#endif

#define CBQ_Q4_GROUP 64

/* A pool of pages.  Row r of kv head h of page p has its hd / 2 bytes of codes at
 * k_codes + p * code_stride[0] + h * code_stride[1] + r * code_stride[2], and its hd
 * / 64 pairs at k_scales (16-bit numbers) + p * scale_stride[0] + h *
 * scale_stride[1] + r * scale_stride[2]; the values lie as the keys do.  Codes
 * are 16-byte aligned, strides too; scales 4-byte aligned, strides even; strides 0
 * or more.  hd 64, 128 or 256; 1 <= page <= 65536; n_pages * page < 2^31; offsets
 * of codes below 64 GiB, of scales below 16 GiB. */
typedef struct cbq_paged_q4 {
    void *k_codes, *v_codes, *k_scales, *v_scales;
    int64_t code_stride[3], scale_stride[3];
    int64_t n_pages;
    int32_t page, n_kv, hd;
} cbq_paged_q4;

/* As cbq_paged_append, into a pool of 4 bits: keys and values are quantised (keys
 * normed and turned in 64 bits first, so that a value next to a border between two
 * codes falls to the same side whatever the order of the sums), and q_out is of
 * x's type.  q_out may not alias q, k or v.  rot even, 2..hd; two tokens with one
 * slot leave pieces of either's row. */
int cbq_paged_append_q4(const void *q, const void *k, const void *v, int x_dtype,
                        const int64_t *q_stride, const int64_t *k_stride, const int64_t *v_stride,
                        const float *cos_table, const float *sin_table, int64_t n_pos, int rot,
                        const int64_t *positions, const int64_t *slots, int norm,
                        const float *q_weight, const float *k_weight, float eps, void *q_out,
                        const cbq_paged_q4 *cache, int64_t N, int n_q, hipStream_t stream);

/* The rows slots[t] = page_id * page + row, t < N, as values of type dtype: k_out
 * and v_out [N, n_kv, hd], contiguous and 16-byte aligned: in fp32, then to the type.
 * A slot outside the pool gives zeros.  N * n_kv * hd < 2^39. */
int cbq_paged_read_q4(const cbq_paged_q4 *cache, const int64_t *slots, int64_t N, int dtype,
                      void *k_out, void *v_out, hipStream_t stream);

/* The newest tokens of each of `batch` sequences, `tokens` each (one, or one and the
 * drafts behind it): sequence b's lengths[b] own keys end with theirs, so its token t
 * sees the prefix (`prefix` keys, in the pages prefix_table names in order) and the
 * own keys up to the (tokens - 1 - t)-th from the end, and
 *   out[b * tokens + t, i] = softmax(q[b * tokens + t, i] . k_j * scale) . v_j
 * over the keys it sees, query head i reading kv head i / (n_q / n_kv); a token that
 * sees no key gets zeros.  The prefix's keys are read for many sequences at a time (a
 * short prefix's by each sequence, where that is less work).  q [batch * tokens, n_q, hd]
 * of type dtype, strides {token, head} in elements, 16-byte aligned; out contiguous, of q's
 * type.  Keys and values count as the values they stand for; scores, maxima, sums and the
 * weighted values are fp32.  A weight times a value's scale is rounded to an fp16 number
 * (of fp32 queries to two: 22 bits, down to 2^-15 of the largest scale, below that 2^-37 of
 * it); a long prefix that more than 16 query rows a kv head share is, for bf16 queries,
 * made into fp16 numbers, and its weights are.  A query that is not finite gives
 * NaN where it sees a key; keys whose scale passes 2^96 may, whatever the query.
 * n_q % n_kv == 0; n_q < 2^20, batch < 2^30, batch * tokens * n_q <= 2^31 - 65536;
 * prefix + width * page <= 2^31 - 65536, fewer than 2^30 entries of a table.
 * workspace: cbq_prefix_attn_decode_q4_workspace bytes (which may be 0), 16-byte
 * aligned, overwritten by every call. */
size_t cbq_prefix_attn_decode_q4_workspace(const cbq_paged_q4 *cache, int64_t prefix, int width,
                                           int batch, int tokens, int n_q, int dtype);
int cbq_prefix_attn_decode_q4(const void *q, const int64_t *q_stride, int dtype,
                              const cbq_paged_q4 *cache, const int32_t *prefix_table,
                              int64_t prefix, const int32_t *tables, int64_t table_stride,
                              int width, const int32_t *lengths, int batch, int tokens, int n_q,
                              float scale, void *out, void *workspace, size_t workspace_bytes,
                              hipStream_t stream);

#ifdef __cplusplus
}
#endif
