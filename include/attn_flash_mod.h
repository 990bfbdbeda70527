/* attn_flash_mod.h -- attention with modified scores on B200 (sm_100a): capped scores, a bias by
 * distance, and per-row key ranges (packed documents, visible prefixes, windows, padded batches).
 * Extends attn_flash (attn_flash.h), whose reference masks by causality alone (flash.c:799-800,
 * 535-543). For a query at position pos_i = Sk - Sq + i (bottom-right, as attn_flash's causal rule)
 * and key j:
 *   s   = q_i . k_j / sqrt(D)
 *   s'  = softcap * tanh(s / softcap)              when softcap > 0
 *   s'' = s' - slope[h] * |pos_i - j|              when slopes is given
 *   key j is seen when key_begin[b][i] <= j < key_end[b][i] (each bound only when given; values
 *   outside [0, Sk] act as the nearest of its ends) and, when causal, j <= pos_i
 *   o_i = sum_j softmax(s'')_j v_j over the seen keys; a row that sees none is zero.
 * A key that no row of a unit sees (a unit: up to 256 consecutive packed rows of one kv head) is not
 * read as a number: what such a slot holds (NaN, infinities) reaches no output. A key that some row of
 * the unit sees is multiplied by a zero weight for the unit's other rows, so an infinity or NaN in its
 * value reaches those too, as it does in a masked matrix product.
 *
 * Layouts are attn_flash's with batch folded into heads: Q [B*Hq][Sq][D], K and V [B*Hkv][Sk][D] bf16
 * bits, O [B*Hq][Sq][D] fp32 or bf16 bits. Tensors are contiguous and live on the current device.
 * P is rounded to bf16 for the second product (as flash.c rounds it); scores, maxima, sums and
 * accumulators are fp32. With a cap of up to 52, slopes of zero or more and more than 16 query rows of a kv
 * head, weights are taken against a fixed score instead of a row's maximum, so they may reach 2^50, and a
 * row's largest may be as low as 2^-100: values above 2^60 may then overflow, and values below 2^-20 lose bits in
 * rows whose every score is near -softcap. Asynchronous on `stream`; the same threads, scratch and status contract as
 * attn_flash_stream. Calls can be captured into CUDA graphs; graphs that may run at the same time
 * need a scratch block each.
 */
#ifndef ATTN_FLASH_MOD_B200_H
#define ATTN_FLASH_MOD_B200_H

#include "attn_flash.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The bounds of a score cap (0 means none). */
#define ATTN_SOFTCAP_MIN 1e-3f
#define ATTN_SOFTCAP_MAX 1e6f

/* How scores are modified. The struct is read during the call; its arrays are device memory that the
 * work on the stream reads. No cap, slopes or ranges: plain attention. Over contiguous K/V that is then
 * attn_flash_stream_out, bit for bit, whose masked keys all have zero weights: an infinity or NaN in the value of
 * a key past the causal limit may reach the rows of its unit there. */
typedef struct attn_mod {
    float softcap;        /* 0, or within [ATTN_SOFTCAP_MIN, ATTN_SOFTCAP_MAX] */
    int causal;           /* nonzero: key j is seen only when j <= pos_i */
    const float *slopes;  /* fp32 [Hq], or NULL: no bias */
    const int *key_begin; /* int32 [B][Sq], or NULL: from key 0 */
    const int *key_end;   /* int32 [B][Sq], or NULL: to the last key */
} attn_mod;

/* Attention over contiguous K/V. out_dtype as attn_flash_stream_out. mod may be NULL (none). D in
 * [1, 256]; D a multiple of 8 up to 128 with 16-byte aligned tensors runs on the tensor cores, any
 * other call on the general path. Returns ATTN_OK or an ATTN_ERR_* code. */
int attn_flash_mod_stream(const uint16_t *Q, const uint16_t *K, const uint16_t *V, void *O, int out_dtype, int B,
                          int Hq, int Hkv, int Sq, int Sk, int D, const attn_mod *mod, void *scratch, void *stream);

/* Attention over a paged K/V cache: attn_flash_paged_stream's pools, tables and limits (D a multiple
 * of 8 up to 128), with modified scores and a choice of output type. A sequence's key axis is its
 * seq_lens entry, so pos_i = seq_lens[b] - Sq + i. Rows of a page at or past the sequence's end are
 * not read as numbers. Of a sequence's block table the entries of the pages from the first key that any of its
 * queries sees to the last are read, both ends rounded outwards to 128 keys; before and behind it may hold
 * anything. An entry read that names no page of the pool is reported by attn_flash_status. */
int attn_flash_mod_paged_stream(const uint16_t *Q, const uint16_t *K_pages, const uint16_t *V_pages,
                                const int *block_table, const int *seq_lens, void *O, int out_dtype, int B, int Hq,
                                int Hkv, int Sq, int D, const attn_mod *mod, int page_size, int num_pages,
                                int max_pages, void *scratch, void *stream);

/* Key ranges of S tokens that hold n_docs documents one after another: document d is tokens
 * [cu_docs[d], cu_docs[d + 1]) (int32 [n_docs + 1], rising; device memory). Writes key_begin and
 * key_end (int32 [S], device): token i of a document sees
 *   causal:     the document up to itself, and the document's first prefix[d] tokens (prefix: int32
 *               [n_docs], or NULL: none)
 *   otherwise:  the whole document
 * and, when window > 0, no key before i - window + 1 (not together with prefix). Tokens outside every
 * document see nothing. Pass the arrays to attn_flash_mod_stream with causal = 0, B = 1 and
 * Sq = Sk = S. */
int attn_mask_ranges_stream(const int *cu_docs, const int *prefix, int n_docs, int S, int causal, int window,
                            int *key_begin, int *key_end, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* ATTN_FLASH_MOD_B200_H */
