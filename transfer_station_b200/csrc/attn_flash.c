/* attn_flash.c -- the C host layer of the B200 attention path.
 *
 * Mirrors the driver half of flash.c's attn_flash (flash.c:727-772: bk check, group,
 * scale, scratch carve) and its two sizing entry points, then hands a validated problem to
 * the CUDA launchers. No allocation happens here: the only device memory touched besides
 * the caller's tensors is the caller-owned scratch block.
 */
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "attn_flash.h"
#include "attn_flash_diag.h"
#include "attn_flash_mod.h"
#include "attn_kv4.h"
#include "fa_launch.h"

/* flash.c:641-647: a bk the caller did not also size scratch with must fail loudly, never
 * mis-stride a tile. Same bounds, same message shape, same abort(). */
static void attn_bk_check(int bk, const char *who) {
    if (bk < ATTN_BK_MIN || bk > ATTN_BK_MAX || (bk & (bk - 1)) != 0) {
        fprintf(stderr, "%s: bk=%d is invalid -- bk must be a POWER OF TWO in [%d, %d]\n", who, bk, ATTN_BK_MIN,
                ATTN_BK_MAX);
        abort();
    }
}

/* Scratch carve: status word, then partial m, l, acc sized for ATTN_PARTIAL_ROWS rows at
 * this head_dim. One function measures and carves, as flash.c:658-672 insists. */
typedef struct ts_scratch {
    int *status;
    float *m, *l, *acc;
} ts_scratch;

static size_t ts_scratch_layout(void *base, int D, ts_scratch *s) {
    const size_t a = ATTN_SCRATCH_ALIGN;
    const size_t d = D < 1 ? 1u : (size_t)D;
    const size_t rows = ATTN_PARTIAL_ROWS;
    size_t off = 0;
    char *b = (char *)base;
    if (s) s->status = base ? (int *)(b + off) : NULL;
    off += TS_SCRATCH_CTRL_BYTES;
    off = (off + a - 1) & ~(a - 1);
    if (s) s->m = base ? (float *)(b + off) : NULL;
    off += rows * sizeof(float);
    off = (off + a - 1) & ~(a - 1);
    if (s) s->l = base ? (float *)(b + off) : NULL;
    off += rows * sizeof(float);
    off = (off + a - 1) & ~(a - 1);
    if (s) s->acc = base ? (float *)(b + off) : NULL;
    off += rows * d * sizeof(float);
    return (off + a - 1) & ~(a - 1);
}

size_t attn_flash_scratch_bytes(int D, int bk) {
    attn_bk_check(bk, "attn_flash_scratch_bytes");
    return ts_scratch_layout(NULL, D, NULL);
}

/* README.md:359-436 of the reference: working_set(D, bk) = 6*bk*(D+BQ) + 6*BQ*D + 4*D +
 * 12*BQ, pick the largest power-of-two bk with 2*working_set <= l2_bytes; never below
 * ATTN_BK_MIN (even if nothing fits), never above ATTN_BK_MAX; D < 1 clamped to 1; D
 * widened to size_t before any arithmetic (the reference's own overflow fix). The GPU's
 * query block is BQ = 128. The result is then capped at the kernel's key tile. */
int attn_flash_pick_bk(int D, size_t l2_bytes) {
    const size_t BQ = 128;
    const size_t d = D < 1 ? 1u : (size_t)D;
    const size_t per_bk = 6u * (d + BQ);
    const size_t fixed = 6u * BQ * d + 4u * d + 12u * BQ;
    const size_t half = l2_bytes / 2u; /* 2*ws <= l2  <=>  ws <= floor(l2/2) */
    int best = ATTN_BK_MIN;
    for (int bk = ATTN_BK_MIN; bk <= ATTN_BK_MAX; bk *= 2) {
        const size_t ws = per_bk * (size_t)bk + fixed;
        if (ws > half) break;
        best = bk;
    }
    return best < ATTN_GPU_KEY_TILE ? best : ATTN_GPU_KEY_TILE;
}

const char *attn_flash_strerror(int status) {
    switch (status) {
    case ATTN_OK: return "ok";
    case ATTN_ERR_ARGS: return "invalid arguments (shape, null pointer, Hq % Hkv, or D outside [1, 256])";
    case ATTN_ERR_ALIGN: return "misaligned pointer";
    case ATTN_ERR_CUDA: return "CUDA runtime/driver error";
    case ATTN_ERR_DEVICE: return "device-side failure reported in the scratch status word (bounded wait ran out)";
    case ATTN_ERR_NOT_SM100: return "current device is not a compute-capability 10.x (B200) GPU";
    default: return "unknown status";
    }
}

/* Work plan. First the split-KV plan for problems with few CTAs (decode): pick nsplit
 * minimising the modelled makespan
 *   T(s) = ceil(ctas*s / SMs) * (blocks/s + 1)
 * (the +1 is the per-CTA prologue/epilogue, in key-block units), subject to the partial
 * rows fitting the scratch and every split keeping >= 2 key blocks. Otherwise, on the
 * tensor-core path without causal masking, the tail wave: when the last wave of CTAs would
 * run at most half full, its L units are split into floor(SMs / L) key pieces, so the last
 * wave takes a fraction of a full CTA's time; their partials are merged afterwards. */
static void ts_plan_core(fa_problem *p, int tc, int sms, int ctas) {
    const long long rows = (long long)p->Hq * p->Sq;
    const int nblk = (p->Sk + ATTN_GPU_KEY_TILE - 1) / ATTN_GPU_KEY_TILE;
    if (sms < 1) sms = 1;
    p->n_direct = 0;
    p->row_base = 0;
    const long long room = p->part_cap > 0 ? p->part_cap : ATTN_PARTIAL_ROWS;
    long long cap = rows > 0 ? room / rows : 0;
    int smax = nblk / 2;
    if (smax > cap) smax = (int)cap;
    if (smax > 256) smax = 256;
    int best = 1;
    double best_t = 1e300;
    for (int s = 1; s <= (smax > 1 ? smax : 1); ++s) {
        const int bps = (nblk + s - 1) / s;
        const int seff = (nblk + bps - 1) / bps;
        if (seff != s) continue; /* same plan as a smaller s */
        const long long tot = (long long)ctas * s;
        const double t = (double)((tot + sms - 1) / sms) * ((double)bps + 1.0);
        if (t < best_t * 0.999) {
            best_t = t;
            best = s;
        }
    }
    int bps = (nblk + best - 1) / best;
    p->nsplit = best;
    p->keys_per_split = bps * ATTN_GPU_KEY_TILE;
    if (best > 1 || !tc || p->causal || ctas <= sms) return;
    const int L = ctas % sms;
    if (L == 0 || 2 * L > sms) return;
    const int ur = ts_tc_unit_rows(p); /* query rows per unit */
    const int tiles = ctas / p->Hkv;
    const int u0 = ctas - L;
    const long long rows_per_kv = (long long)(p->Hq / p->Hkv) * p->Sq;
    const long long row_base = (long long)(u0 / tiles) * rows_per_kv + (long long)(u0 % tiles) * ur;
    int s = sms / L;
    if (s > nblk / 2) s = nblk / 2;
    while (s >= 2 && (rows - row_base) * s > room) --s;
    if (s < 2) return;
    bps = (nblk + s - 1) / s;
    p->nsplit = (nblk + bps - 1) / bps;
    p->keys_per_split = bps * ATTN_GPU_KEY_TILE;
    p->n_direct = u0;
    p->row_base = (int)row_base;
}

static void ts_plan(fa_problem *p) {
    const int tc = ts_tc_supported(p);
    const long long rows = (long long)p->Hq * p->Sq;
    if (p->order) return; /* whole units (ts_fill's plan), sorted by their lengths */
    ts_plan_core(p, tc, ts_num_sms(), tc ? ts_tc_ctas_per_split(p) : (int)((rows + 7) / 8));
}

static int ts_validate(const void *Q, const void *K, const void *V, int Hq, int Hkv, int Sq, int Sk, int D,
                       const void *scratch) {
    if (!Q || !K || !V || !scratch) return ATTN_ERR_ARGS;
    if (Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || Sq < 1 || Sk < 1 || D < 1 || D > ATTN_D_MAX) return ATTN_ERR_ARGS;
    if ((long long)Hq * Sq > 0x7fffffffLL || (long long)Hkv * Sk > 0x7fffffffLL) return ATTN_ERR_ARGS;
    if (((uintptr_t)scratch) & 15u) return ATTN_ERR_ALIGN;
    if (ts_cc_major() != 10) return ATTN_ERR_NOT_SM100;
    return ATTN_OK;
}

static void ts_fill(fa_problem *p, const uint16_t *Q, const uint16_t *K, const uint16_t *V, int Hq, int Hkv,
                    int Sq, int Sk, int D, int causal, int v_prepacked) {
    memset(p, 0, sizeof *p);
    p->Q = Q;
    p->K = K;
    p->V = V;
    p->Hq = Hq;
    p->Hkv = Hkv;
    p->Sq = Sq;
    p->Sk = Sk;
    p->Sk_total = Sk;
    p->k_begin = 0;
    p->D = D;
    p->causal = causal ? 1 : 0;
    p->v_prepacked = v_prepacked ? 1 : 0;
    p->scale_log2 = (1.0f / sqrtf((float)D)) * 1.4426950408889634f;
    p->nsplit = 1;
    p->keys_per_split = ((Sk + ATTN_GPU_KEY_TILE - 1) / ATTN_GPU_KEY_TILE) * ATTN_GPU_KEY_TILE;
}

int attn_diag_plan(int Hq, int Hkv, int Sq, int Sk, int D, int causal, int sms, int out[5]) {
    if (!out || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || Sq < 1 || Sk < 1 || D < 1 || D > ATTN_D_MAX || sms < 1)
        return ATTN_ERR_ARGS;
    if ((long long)Hq * Sq > 0x7fffffffLL || (long long)Hkv * Sk > 0x7fffffffLL) return ATTN_ERR_ARGS;
    fa_problem p;
    ts_fill(&p, NULL, NULL, NULL, Hq, Hkv, Sq, Sk, D, causal, 0);
    const int ctas = ts_tc_ctas_per_split(&p);
    ts_plan_core(&p, 1, sms, ctas);
    out[0] = p.nsplit;
    out[1] = p.keys_per_split;
    out[2] = p.n_direct;
    out[3] = p.row_base;
    out[4] = ctas;
    return ATTN_OK;
}

static int ts_run(fa_problem *p, void *scratch, void *stream) {
    ts_scratch s;
    ts_scratch_layout(scratch, p->D, &s);
    p->status = s.status;
    ts_plan(p);
    if (p->nsplit > 1) {
        p->part_m = s.m;
        p->part_l = s.l;
        p->part_acc = s.acc;
    } else if (p->write_partials) {
        p->part_m = p->out_m;
        p->part_l = p->out_l;
        p->part_acc = p->out_acc;
    }
    /* the tensor-core kernel clears the status word itself (no memset between two launches,
     * so consecutive calls can overlap under programmatic dependent launch); the general path
     * needs the memset */
    if (ts_tc_supported(p)) {
        p->status_gen = ts_next_status_gen();
    } else {
        int rc = ts_clear_status(s.status, stream);
        if (rc != ATTN_OK) return rc;
    }
    return ts_launch_attention(p, stream);
}

int attn_flash_stream(const uint16_t *Q, const uint16_t *K, const uint16_t *V, float *O, int Hq, int Hkv, int Sq,
                      int Sk, int D, int causal, int bk, void *scratch, int v_prepacked, void *stream) {
    attn_bk_check(bk, "attn_flash");
    if (!O) return ATTN_ERR_ARGS;
    int rc = ts_validate(Q, K, V, Hq, Hkv, Sq, Sk, D, scratch);
    if (rc != ATTN_OK) return rc;
    fa_problem p;
    ts_fill(&p, Q, K, V, Hq, Hkv, Sq, Sk, D, causal, v_prepacked);
    p.O = O;
    return ts_run(&p, scratch, stream);
}

int attn_flash_stream_out(const uint16_t *Q, const uint16_t *K, const uint16_t *V, void *O, int out_dtype, int Hq,
                          int Hkv, int Sq, int Sk, int D, int causal, int bk, void *scratch, int v_prepacked,
                          void *stream) {
    attn_bk_check(bk, "attn_flash");
    if (!O || (out_dtype != ATTN_OUT_F32 && out_dtype != ATTN_OUT_BF16)) return ATTN_ERR_ARGS;
    int rc = ts_validate(Q, K, V, Hq, Hkv, Sq, Sk, D, scratch);
    if (rc != ATTN_OK) return rc;
    fa_problem p;
    ts_fill(&p, Q, K, V, Hq, Hkv, Sq, Sk, D, causal, v_prepacked);
    p.O = (float *)O;
    p.o_bf16 = out_dtype == ATTN_OUT_BF16;
    return ts_run(&p, scratch, stream);
}

static int ts_page_size_ok(int ps) {
    if (ps == 8 || ps == 16 || ps == 32 || ps == 64) return 1;
    return ps > 0 && ps % ATTN_GPU_KEY_TILE == 0;
}

/* The argument checks of a paged call. */
static int ts_paged_check(const void *Q, const void *K_pages, const void *V_pages, const int *block_table,
                          const int *seq_lens, const void *O, int B, int Hq, int Hkv, int Sq, int D, int page_size,
                          int num_pages, int max_pages, const void *scratch) {
    if (!Q || !K_pages || !V_pages || !block_table || !seq_lens || !O || !scratch) return ATTN_ERR_ARGS;
    if (B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || Sq < 1 || num_pages < 1 || max_pages < 1)
        return ATTN_ERR_ARGS;
    if (D < 8 || D > 128 || D % 8 != 0 || !ts_page_size_ok(page_size)) return ATTN_ERR_ARGS;
    if ((long long)B * Hq * Sq > 0x7fffffffLL || (long long)max_pages * page_size > 0x7fffffffLL ||
        (long long)B * max_pages > 0x7fffffffLL)
        return ATTN_ERR_ARGS;
    if (((uintptr_t)Q | (uintptr_t)K_pages | (uintptr_t)V_pages | (uintptr_t)O | (uintptr_t)scratch) & 15u)
        return ATTN_ERR_ALIGN;
    if (ts_cc_major() != 10) return ATTN_ERR_NOT_SM100;
    return ATTN_OK;
}

int attn_flash_paged_stream(const uint16_t *Q, const uint16_t *K_pages, const uint16_t *V_pages,
                            const int *block_table, const int *seq_lens, float *O, int B, int Hq, int Hkv, int Sq,
                            int D, int causal, int page_size, int num_pages, int max_pages, void *scratch,
                            void *stream) {
    const int rc = ts_paged_check(Q, K_pages, V_pages, block_table, seq_lens, O, B, Hq, Hkv, Sq, D, page_size, num_pages,
                                  max_pages, scratch);
    if (rc != ATTN_OK) return rc;
    fa_problem p;
    ts_fill(&p, Q, K_pages, V_pages, B * Hq, B * Hkv, Sq, max_pages * page_size, D, causal, 0);
    p.O = O;
    p.paged = 1;
    p.block_table = block_table;
    p.seq_lens = seq_lens;
    p.page_size = page_size;
    p.max_pages = max_pages;
    p.num_pages = num_pages;
    p.hkv_local = Hkv;
    if (!ts_tc_supported(&p)) return ATTN_ERR_ARGS;
    return ts_run(&p, scratch, stream);
}

/* Checks a call's modifiers and sets the problem's (Hkv kv heads per sequence). A plain call keeps
 * mod 0 and takes the plain kernels. */
static int ts_set_mod(fa_problem *p, const attn_mod *mod, int Hkv) {
    p->hkv_local = Hkv;
    if (!mod) return ATTN_OK;
    p->causal = mod->causal ? 1 : 0;
    const float cap = mod->softcap;
    if (!(cap == 0.0f || (cap >= ATTN_SOFTCAP_MIN && cap <= ATTN_SOFTCAP_MAX))) return ATTN_ERR_ARGS;
    if ((((uintptr_t)mod->slopes) | ((uintptr_t)mod->key_begin) | ((uintptr_t)mod->key_end)) & 3u) return ATTN_ERR_ALIGN;
    p->key_begin = mod->key_begin;
    p->key_end = mod->key_end;
    p->slopes = mod->slopes;
    if (cap > 0.0f) {
        p->cap_in = 1.0f / (cap * sqrtf((float)p->D));
        p->cap_out = cap * 1.4426950408889634f;
    }
    if (cap > 0.0f || mod->slopes)
        p->mod = cap > 0.0f ? (mod->slopes ? 4 : 2) : 3;
    else if (mod->key_begin || mod->key_end)
        p->mod = 1;
    return ATTN_OK;
}

/* Query positions a unit's ranges are read from by the kernel itself; longer calls get their bounds
 * from a kernel of their own first (about 2 us, against 256 dependent reads per unit and role). */
#define TS_MOD_INLINE_ROWS 8

/* Runs a problem with modified scores. The bounds of the units' ranges and the units' order sit at the end
 * of the scratch block's partial accumulators, which the plan then uses less of. */
static int ts_run_mod(fa_problem *p, void *scratch, void *stream) {
    if (ts_few_rows(p)) {
        ts_scratch s;
        ts_scratch_layout(scratch, p->D, &s);
        p->status = s.status;
        p->part_m = s.m;
        p->part_l = s.l;
        p->part_acc = s.acc;
        return ts_launch_few_rows(p, stream);
    }
    if (p->mod && ts_tc_supported(p)) {
        const int ranges = p->key_begin || p->key_end, per_kv = ts_tc_ctas_per_split(p) / p->Hkv;
        const long long units = (long long)per_kv * p->Hkv, tiles = units / p->hkv_local;
        /* units of different lengths that the kernel's own order would not put longest first */
        const int misfit = p->causal && p->Hq != p->Hkv && p->Sq % ts_tc_unit_rows(p) != 0;
        const int order = units > ts_num_sms() && (ranges || p->paged || misfit);
        const size_t row_bytes = (size_t)p->D * sizeof(float);
        const size_t bytes = (size_t)tiles * 8 * sizeof(int) + (order ? (size_t)units * sizeof(int) : 0);
        const size_t taken = (bytes + row_bytes - 1) / row_bytes + 1;
        /* no room: the kernel reads the ranges itself */
        if ((order || (ranges && p->Sq > TS_MOD_INLINE_ROWS)) && taken <= ATTN_PARTIAL_ROWS / 2) {
            ts_scratch s;
            ts_scratch_layout(scratch, p->D, &s);
            p->part_cap = ATTN_PARTIAL_ROWS - (int)taken;
            /* 16-byte aligned, within the rows taken (one more than they fill) */
            p->bounds = (int *)(((uintptr_t)(s.acc + (size_t)p->part_cap * (size_t)p->D) + 15u) & ~(uintptr_t)15u);
            if (order) p->order = p->bounds + 8 * tiles;
        }
    }
    return ts_run(p, scratch, stream);
}

int attn_flash_mod_stream(const uint16_t *Q, const uint16_t *K, const uint16_t *V, void *O, int out_dtype, int B,
                          int Hq, int Hkv, int Sq, int Sk, int D, const attn_mod *mod, void *scratch, void *stream) {
    if (!O || (out_dtype != ATTN_OUT_F32 && out_dtype != ATTN_OUT_BF16) || B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0)
        return ATTN_ERR_ARGS;
    if ((long long)B * Hq > 0x7fffffffLL) return ATTN_ERR_ARGS;
    fa_problem p;
    ts_fill(&p, Q, K, V, B * Hq, B * Hkv, Sq, Sk, D < 1 ? 1 : D, 0, 0);
    int rc = ts_set_mod(&p, mod, Hkv);
    if (rc == ATTN_ERR_ARGS) return rc;
    const int valid = ts_validate(Q, K, V, B * Hq, B * Hkv, Sq, Sk, D, scratch);
    if (valid == ATTN_ERR_ARGS) return valid;
    if (rc != ATTN_OK) return rc;
    if (valid != ATTN_OK) return valid;
    p.O = (float *)O;
    p.o_bf16 = out_dtype == ATTN_OUT_BF16;
    return ts_run_mod(&p, scratch, stream);
}

int attn_flash_mod_paged_stream(const uint16_t *Q, const uint16_t *K_pages, const uint16_t *V_pages,
                                const int *block_table, const int *seq_lens, void *O, int out_dtype, int B, int Hq,
                                int Hkv, int Sq, int D, const attn_mod *mod, int page_size, int num_pages,
                                int max_pages, void *scratch, void *stream) {
    if (out_dtype != ATTN_OUT_F32 && out_dtype != ATTN_OUT_BF16) return ATTN_ERR_ARGS;
    int rc = ts_paged_check(Q, K_pages, V_pages, block_table, seq_lens, O, B, Hq, Hkv, Sq, D, page_size, num_pages,
                            max_pages, scratch);
    if (rc == ATTN_ERR_ARGS) return rc;
    fa_problem p;
    ts_fill(&p, Q, K_pages, V_pages, B * Hq, B * Hkv, Sq, max_pages * page_size, D, 0, 0);
    const int mrc = ts_set_mod(&p, mod, Hkv);
    if (mrc != ATTN_OK) return mrc;
    /* (the plain kernels multiply what lies behind a sequence's end by zero: a NaN there would reach its rows) */
    if (!p.mod) p.mod = 1;
    if (rc != ATTN_OK) return rc;
    p.O = (float *)O;
    p.o_bf16 = out_dtype == ATTN_OUT_BF16;
    p.paged = 1;
    p.block_table = block_table;
    p.seq_lens = seq_lens;
    p.page_size = page_size;
    p.max_pages = max_pages;
    p.num_pages = num_pages;
    if (!ts_tc_supported(&p)) return ATTN_ERR_ARGS;
    return ts_run_mod(&p, scratch, stream);
}

int attn_flash_kv4_stream(const uint16_t *Q, const uint8_t *K_codes, const uint8_t *K_scales, const uint8_t *V_codes,
                          const uint8_t *V_scales, const int *block_table, const int *seq_lens, void *O, int out_dtype,
                          int B, int Hq, int Hkv, int Sq, int D, const attn_mod *mod, int page_size, int num_pages,
                          int max_pages, void *scratch, void *stream) {
    if (!K_scales || !V_scales || (out_dtype != ATTN_OUT_F32 && out_dtype != ATTN_OUT_BF16)) return ATTN_ERR_ARGS;
    if (D != 64 && D != 128) return ATTN_ERR_ARGS;
    int rc = ts_paged_check(Q, K_codes, V_codes, block_table, seq_lens, O, B, Hq, Hkv, Sq, D, page_size, num_pages,
                            max_pages, scratch);
    if (rc == ATTN_ERR_ARGS) return rc;
    /* (the kernel looks a few tiles past the last key: its key indexes stay within 32 bits) */
    if ((long long)page_size * max_pages > 0x7fffffffLL - 65536 || (long long)B * Hkv > 0x7fffffffLL) return ATTN_ERR_ARGS;
    fa_problem f;
    ts_fill(&f, Q, NULL, NULL, B * Hq, B * Hkv, Sq, max_pages * page_size, D, 0, 0);
    const int mrc = ts_set_mod(&f, mod, Hkv);
    if (mrc != ATTN_OK) return mrc;
    if ((((uintptr_t)K_scales) | ((uintptr_t)V_scales)) & 15u) return ATTN_ERR_ALIGN;
    if (rc != ATTN_OK) return rc;
    ts_scratch s;
    ts_scratch_layout(scratch, D, &s);
    ts_kv4_problem P;
    memset(&P, 0, sizeof P);
    P.Q = Q;
    P.k_codes = K_codes;
    P.k_scales = K_scales;
    P.v_codes = V_codes;
    P.v_scales = V_scales;
    P.block_table = block_table;
    P.seq_lens = seq_lens;
    P.O = O;
    P.o_bf16 = out_dtype == ATTN_OUT_BF16;
    P.B = B;
    P.Hq = Hq;
    P.Hkv = Hkv;
    P.Sq = Sq;
    P.D = D;
    P.causal = f.causal;
    P.page_size = page_size;
    P.num_pages = num_pages;
    P.max_pages = max_pages;
    P.scale_log2 = f.scale_log2;
    P.cap_in = f.cap_in;
    P.cap_out = f.cap_out;
    P.slopes = f.slopes;
    P.key_begin = f.key_begin;
    P.key_end = f.key_end;
    P.status = s.status;
    P.part_m = s.m;
    P.part_l = s.l;
    P.part_acc = s.acc;
    P.part_rows = ATTN_PARTIAL_ROWS;
    return ts_launch_kv4(&P, stream);
}

int attn_mask_ranges_stream(const int *cu_docs, const int *prefix, int n_docs, int S, int causal, int window,
                            int *key_begin, int *key_end, void *stream) {
    if (!cu_docs || !key_begin || !key_end || n_docs < 1 || S < 1 || window < 0 || (window > 0 && prefix))
        return ATTN_ERR_ARGS;
    if ((((uintptr_t)cu_docs) | ((uintptr_t)prefix) | ((uintptr_t)key_begin) | ((uintptr_t)key_end)) & 3u)
        return ATTN_ERR_ALIGN;
    if (ts_cc_major() != 10) return ATTN_ERR_NOT_SM100;
    return ts_launch_mask_ranges(cu_docs, prefix, n_docs, S, causal ? 1 : 0, window, key_begin, key_end, stream);
}

int attn_flash_partial_stream(const uint16_t *Q, const uint16_t *K, const uint16_t *V, float *m, float *l,
                              float *acc, int Hq, int Hkv, int Sq, int Sk_local, int Sk_total, int k_begin, int D,
                              int causal, int bk, void *scratch, int v_prepacked, void *stream) {
    attn_bk_check(bk, "attn_flash_partial");
    if (!m || !l || !acc || k_begin < 0 || Sk_total < (long long)k_begin + Sk_local) return ATTN_ERR_ARGS;
    int rc = ts_validate(Q, K, V, Hq, Hkv, Sq, Sk_local, D, scratch);
    if (rc != ATTN_OK) return rc;
    fa_problem p;
    ts_fill(&p, Q, K, V, Hq, Hkv, Sq, Sk_local, D, causal, v_prepacked);
    p.Sk_total = Sk_total;
    p.k_begin = k_begin;
    p.write_partials = 1;
    p.out_m = m;
    p.out_l = l;
    p.out_acc = acc;
    return ts_run(&p, scratch, stream);
}

int attn_flash_decode_peers_stream(const uint16_t *Q, const uint16_t *K, const uint16_t *V, float *O, int Hq,
                                   int Hkv, int Sq, int Sk_local, int Sk_total, int k_begin, int D, int causal, int bk,
                                   void *scratch, void *const *blocks, int world, int rank, unsigned int epoch,
                                   void *stream) {
    attn_bk_check(bk, "attn_flash_decode_peers");
    if (!O || !blocks || world < 1 || world > ATTN_PEERS_MAX || rank < 0 || rank >= world || epoch == 0 ||
        Sk_local < 0 || k_begin < 0 || Sk_total < 1 || (long long)k_begin + Sk_local > Sk_total)
        return ATTN_ERR_ARGS;
    for (int r = 0; r < world; ++r)
        if (!blocks[r]) return ATTN_ERR_ARGS;
        else if (((uintptr_t)blocks[r]) & 255u) return ATTN_ERR_ALIGN;
    /* validated as the whole key axis when this shard is empty (K and V are not read then) */
    int rc = ts_validate(Q, Sk_local > 0 ? K : Q, Sk_local > 0 ? V : Q, Hq, Hkv, Sq, Sk_local > 0 ? Sk_local : 1, D,
                         scratch);
    if (rc != ATTN_OK) return rc;
    if ((long long)Hq * Sq > ATTN_PARTIAL_ROWS) return ATTN_ERR_ARGS;
    ts_scratch s;
    ts_scratch_layout(scratch, D, &s);
    int nparts = 0;
    if (Sk_local > 0) {
        fa_problem p;
        ts_fill(&p, Q, K, V, Hq, Hkv, Sq, Sk_local, D, causal, 0);
        p.Sk_total = Sk_total;
        p.k_begin = k_begin;
        p.status = s.status;
        /* the tensor-core kernel clears the status word itself (no memset between this step's
         * kernels and the previous step's, which keeps their launches overlapping) */
        if (ts_tc_supported(&p)) {
            p.status_gen = ts_next_status_gen();
        } else {
            rc = ts_clear_status(s.status, stream);
            if (rc != ATTN_OK) return rc;
        }
        ts_plan(&p);
        if (p.n_direct > 0) { /* a prefill tail split: run every unit whole instead */
            p.nsplit = 1;
            p.n_direct = 0;
            p.row_base = 0;
            p.keys_per_split = ((Sk_local + ATTN_GPU_KEY_TILE - 1) / ATTN_GPU_KEY_TILE) * ATTN_GPU_KEY_TILE;
        }
        /* every piece lands in the scratch partial arrays as [piece][row] */
        p.write_partials = 1;
        p.part_m = p.out_m = s.m;
        p.part_l = p.out_l = s.l;
        p.part_acc = p.out_acc = s.acc;
        rc = ts_launch_attention_pieces(&p, stream);
        if (rc != ATTN_OK) return rc;
        nparts = p.nsplit;
    } else {
        rc = ts_clear_status(s.status, stream);
        if (rc != ATTN_OK) return rc;
    }
    return ts_launch_peer_merge(s.m, s.l, s.acc, nparts, Hq * Sq, D, O, blocks, world, rank, epoch, s.status, stream);
}

int attn_flash_combine_stream(const float *m, const float *l, const float *acc, int nparts, int rows, int D,
                              float *O, void *stream) {
    if (!m || !l || !acc || !O || nparts < 1 || rows < 0 || D < 1 || D > ATTN_D_MAX) return ATTN_ERR_ARGS;
    if (ts_cc_major() != 10) return ATTN_ERR_NOT_SM100;
    return ts_launch_combine(m, l, acc, nparts, rows, D, O, NULL, NULL, 0, stream);
}

size_t attn_flash_packed_floats(int rows, int D) {
    if (rows < 0 || D < 1) return 0;
    return ((2 * (size_t)rows + 3) & ~(size_t)3) + (size_t)rows * D;
}

int attn_flash_combine_packed_stream(const float *parts, int nparts, int rows, int D, float *O, void *stream) {
    if (!parts || !O || nparts < 1 || rows < 0 || D < 1 || D > ATTN_D_MAX) return ATTN_ERR_ARGS;
    if (ts_cc_major() != 10) return ATTN_ERR_NOT_SM100;
    const size_t ml = (2 * (size_t)rows + 3) & ~(size_t)3;
    const size_t stride = attn_flash_packed_floats(rows, D);
    return ts_launch_combine_strided(parts, parts + rows, parts + ml, nparts, rows, D, stride, stride, O, NULL, NULL,
                                     0, stream);
}

int attn_flash_status(void *scratch, void *stream, int *device_code) {
    if (!scratch) return ATTN_ERR_ARGS;
    ts_scratch s;
    ts_scratch_layout(scratch, 1, &s);
    int v = 0;
    int rc = ts_read_status(s.status, stream, &v);
    if (device_code) *device_code = v;
    if (rc != ATTN_OK) return rc;
    return v ? ATTN_ERR_DEVICE : ATTN_OK;
}

void attn_flash(const uint16_t *Q, const uint16_t *K, const uint16_t *V, float *O, int Hq, int Hkv, int Sq, int Sk,
                int D, int causal, int bk, void *scratch, int v_prepacked, struct attn_times *tm) {
    int rc = attn_flash_stream(Q, K, V, O, Hq, Hkv, Sq, Sk, D, causal, bk, scratch, v_prepacked, NULL);
    int code = 0;
    if (rc == ATTN_OK) rc = attn_flash_status(scratch, NULL, &code);
    /* flash.c:822-849 adds each phase's seconds into *tm (its harness zeroes it once and
     * divides by the call count). The four phases run fused in one kernel here, so there is
     * nothing to add: *tm is left as the caller's running totals stand. */
    (void)tm;
    if (rc != ATTN_OK) {
        fprintf(stderr, "attn_flash: %s (device code %d)\n", attn_flash_strerror(rc), code);
        abort();
    }
}
