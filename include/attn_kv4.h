/* attn_kv4.h -- a paged key cache held in 4 bits on B200 (sm_100a): the producer that writes it, the
 * attention that reads it, and its tokens back as bf16. The counterpart of attn_qkv_rope_paged_stream
 * and attn_flash_paged_stream (attn_qkv_rope.h, attn_flash.h) at 17/64 of their cache bytes; the
 * reference keeps K and V in bf16 (flash.c:727-729).
 *
 * The cache. A key (or value) of one token and kv head is a vector of D bf16 values, cut into groups of
 * ATTN_KV4_GROUP consecutive elements. A group is stored as
 *   s    one E4M3 byte (as OCP FP8 defines it): a / 7 rounded to nearest even, a the group's largest
 *        magnitude (at most 448)
 *   q_i  one nibble each, q_i + 8 with q_i = x_i / s rounded to nearest even, within [-8, 7]
 * and stands for q_i * s, which bf16 holds exactly. A group whose s is zero stands for zeros; a NaN is
 * stored as 0 and an infinity as the group's largest code: the cache holds finite values. The pools, all
 * device memory, uint8:
 *   K_codes, V_codes    [num_pages][Hkv][page_size][D / 2]    byte i: element 2i in the low nibble,
 *                                                             2i + 1 in the high one
 *   K_scales, V_scales  [num_pages][Hkv][page_size][D / 32]
 * Position p of sequence b lives in page block_table[b * max_pages + p / page_size], row p % page_size.
 *
 * D is 64 or 128; page_size 8, 16, 32, 64 or a multiple of 128; pools, Q, K, V, O and qkv 16-byte
 * aligned; all tensors contiguous, on the current device. Calls are asynchronous on `stream` and return
 * ATTN_OK or an ATTN_ERR_* code; scratch, threads and status as in attn_flash.h (any block sized by
 * attn_flash_scratch_bytes for this D). Captured calls that may run at the same time need a scratch
 * block each.
 */
#ifndef ATTN_KV4_B200_H
#define ATTN_KV4_B200_H

#include "attn_flash_mod.h"
#include "attn_qkv_rope.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ATTN_KV4_GROUP 32 /* elements that share a scale */

/* attn_qkv_rope_paged_stream into the 4-bit cache: split qkv [B*S][(Hq + 2*Hkv) * D], norm and rotate
 * the q and k heads, write Q [B*Hq][S][D] in bf16, and the keys and values, first rounded to bf16 as
 * that call writes them, in 4 bits. The norm of the k heads is summed in double precision, so that the
 * codes do not depend on an order of summation. Two tokens of one call must not name the same slot. A
 * token outside the table, the cache or the pool is skipped whole and reported by attn_flash_status. */
int attn_qkv_rope_kv4_stream(const uint16_t *qkv, const int *positions, const float *cos_sin, int max_pos,
                             const uint16_t *q_norm_w, const uint16_t *k_norm_w, float eps, int B, int S, int Hq,
                             int Hkv, int D, int rot, int style, uint16_t *Q, uint8_t *K_codes, uint8_t *K_scales,
                             uint8_t *V_codes, uint8_t *V_scales, const int *block_table, int page_size,
                             int num_pages, int max_pages, void *scratch, void *stream);

/* The tokens at positions [B*S] (token t = b*S + s of sequence b) as bf16: K and V [B*Hkv][S][D], the
 * layout attn_flash and attn_flash_mod_stream read. A token outside the table or the pool leaves its rows
 * as they were and is reported by attn_flash_status. */
int attn_kv4_unpack_stream(const uint8_t *K_codes, const uint8_t *K_scales, const uint8_t *V_codes,
                           const uint8_t *V_scales, const int *block_table, const int *positions, uint16_t *K,
                           uint16_t *V, int B, int S, int Hkv, int D, int page_size, int num_pages, int max_pages,
                           void *scratch, void *stream);

/* Attention over the cache for single tokens or a few new positions: Q [B*Hq][Sq][D] bf16, O the same
 * in fp32 or bf16 (out_dtype as attn_flash_stream_out); sequence b has seq_lens[b] keys (clamped to
 * [0, max_pages * page_size]; none: zero rows), its queries are its last Sq positions. mod (may be NULL)
 * as in attn_flash_mod_paged_stream: cap, bias, key ranges and causality over the sequence's keys. Rows
 * of a page past the sequence's end, and keys that no row of a unit sees (here up to 16 rows of a kv head), are not
 * read as numbers. Of its block table the entries of the pages from the first key that any of its queries sees to
 * the last are read (with more than 16 positions those of all its keys). A page
 * id outside the pool there is reported by attn_flash_status; that sequence's rows are then undefined. At least
 * a million kv heads over all sequences are taken (their bookkeeping lies in scratch). Weights
 * are rounded to fp16 once (11 bits down to 2^-26 of a row's largest, steps of 2^-36 of it below) and
 * dequantised elements are exact in fp16; scores, maxima, sums and accumulators are fp32. */
int attn_flash_kv4_stream(const uint16_t *Q, const uint8_t *K_codes, const uint8_t *K_scales,
                          const uint8_t *V_codes, const uint8_t *V_scales, const int *block_table,
                          const int *seq_lens, void *O, int out_dtype, int B, int Hq, int Hkv, int Sq, int D,
                          const attn_mod *mod, int page_size, int num_pages, int max_pages, void *scratch,
                          void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ATTN_KV4_B200_H */
