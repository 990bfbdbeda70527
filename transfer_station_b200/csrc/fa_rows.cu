// fa_rows.cu -- attention with modified scores (attn_flash_mod.h) for up to 16 query rows of each kv head:
// single tokens, a few new positions.
//
// What bounds it: the bytes of K and V, read once. The kernel for prompts gives such a call 128-row tiles of
// which 4 or 16 rows exist, and caps, biases and masks all 128: with a cap, 16 sequences of 8,192 keys took
// 124 us there, 3 times the time of their bytes. Here keys are the M side of mma.m16n8k16 and the query rows
// the N side, so no row is padding beyond the next 8: an SM sub-partition needs 16 MMAs (8 cycles each) and
// about 200 other instructions for 16 keys, while their 8 KB take it 1,400 cycles to arrive.
//
// One producer warp streams 64-key tiles by TMA (128-byte swizzle, the layout ldmatrix reads without bank
// conflicts) into a 96 KB ring; four consumer warps take 16 keys of each, with a running maximum and an
// accumulator of their own, merged in shared memory at a unit's end. Two such CTAs share an SM, so that one
// streams while the other is between units (one CTA with twice the ring: 64 sequences of 300 keys, 16 rows, 39 us, not
// 33). The work split is rows_plan.cuh's.
//
// Measured, 16 sequences of 8,192 keys, 4 rows, D = 128, cap: 51.8 us of 42.3 for the bytes (ragged lengths); all of full
// length 85 us, 6.3 TB/s; over pages of 8 keys 96, 16 90, 32 and more 88; 16 rows 94.
#include <cuda_bf16.h>

#include <atomic>
#include <type_traits>

#include "attn_flash_mod.h"
#include "rows_plan.cuh"
#include "score_cap.cuh"

namespace ts {

namespace {

constexpr int kTile = 64;   // keys per stage
constexpr int kWarps = 4;   // consumer warps, 16 keys of a tile each
constexpr int kThreads = 32 * (kWarps + 1);
constexpr float kMost = 7.f;  // a reference moves when a score exceeds it by this (log2 units)

struct FewParams : RowsParams {
    float cap_in, cap_out, tanh_k[5];
};

// DP: head elements in shared memory (64 or 128; those past D are zeros). NT: blocks of 8 query rows.
template <int DP, int NT>
struct FewConfig {
    static constexpr int HALF = kTile * 128;           // 64 elements of a tile's keys
    static constexpr int TILE_BYTES = HALF * (DP / 64);
    static constexpr int STAGE = 2 * TILE_BYTES;       // K, V
    static constexpr int NS = 98304 / STAGE;
    static constexpr int ROWS = 8 * NT;
    static constexpr int ROUNDS = NT * DP / 64;        // of the merge, to fit two CTAs on an SM
    static constexpr int COLS = DP / ROUNDS;
    static constexpr int MERGE = kWarps * ROWS * (COLS + 4) * 4;
    static constexpr int OFF_MERGE = NS * STAGE;
    static constexpr int OFF_ML = OFF_MERGE + MERGE;   // m, l [kWarps][ROWS]
    static constexpr int OFF_BAR = OFF_ML + 2 * kWarps * ROWS * 4;
    static constexpr int SMEM = OFF_BAR + 2 * NS * 8 + 1024;  // + alignment of the swizzled tiles
    static_assert(2 * (SMEM + 2048) <= 228 * 1024, "");
};

__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int DP, int NT>
__global__ void __launch_bounds__(kThreads, 2)
    few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const FewParams p) {
    using C = FewConfig<DP, NT>;
    constexpr int KT = DP / 16;  // 16-element steps of the first product, tiles of the output
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ int abort_flag_s;
    volatile int *abort_flag = &abort_flag_s;
    const uint32_t base = smem_u32(smem), bars = base + C::OFF_BAR;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (C::NS + s); };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        abort_flag_s = 0;
        for (int s = 0; s < C::NS; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kWarps);
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
    }
    pdl_wait();
    pdl_trigger();
    const Share sh = find_share<kTile>(p, blockIdx.x, gridDim.x);  // (its barriers also publish the set-up)
    if (sh.t0 >= sh.t1) return;

    const int units = p.Hkv * p.row_blocks;
    long long left = sh.t1 - sh.t0;
    int b = sh.b, u = sh.u, tile = sh.tile;

    if (warp == kWarps) {
        // ================= producer: the CTA's tiles, in order, into the ring
        const int P = p.block_table ? p.page_size : kTile;
        const int rows = P < kTile ? P : kTile;      // keys per copy
        const int per_tile = kTile / rows;           // copies per operand half and tile
        int st = 0;                                  // next stage, and the round of the ring it is in
        uint32_t round = 0;
        bool ok = true;
        while (left > 0 && ok) {
            const Span sp = seq_span<kTile>(p, b);
            const int len = sp.len, nt = sp.nt;
            const int kvh = u / p.row_blocks;
            const int *table = p.block_table ? p.block_table + (size_t)b * p.max_pages : nullptr;
            const int end = (int)((long long)nt < tile + left ? (long long)nt : tile + left);
            // page ids of the next 32 chunks (a chunk: `rows` keys), one a lane
            int win = -1, id = -1;
            for (int i = tile; i < end && ok; ++i) {
                const int c0 = (sp.t0 + i) * per_tile;
                if (table && (win < 0 || c0 + per_tile > win + 32)) {
                    win = c0;
                    const long long key = (long long)(c0 + lane) * rows;
                    const int page = (int)(key / P);
                    id = -1;
                    if (key < sp.hi && key + rows > sp.lo) {  // (what else the table holds is not read)
                        id = ld_plan(table + page);
                        if (id < 0 || id >= p.num_pages) {
                            report_pending(p, kDevErrBadPage);
                            id = -1;
                        }
                    }
                }
                if (round > 0) ok = ring_wait(empty(st), (round - 1) & 1u, abort_flag, p, kDevErrTimeoutKV);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int page_id = __shfl_sync(0xffffffffu, id, (c0 - win + lane) & 31);
                // a contiguous tile that begins past the keys (a sequence without any) is not loaded
                const int my_id = table ? page_id : ((long long)c0 * rows < len ? 0 : -1);
                const bool mine = lane < per_tile && my_id >= 0;
                const int n = __popc(__ballot_sync(0xffffffffu, mine));
                const uint32_t bytes = (uint32_t)rows * 128u;
                if (lane == 0) mbar_expect_tx(full(st), (uint32_t)n * bytes * (2u * (DP / 64)));
                __syncwarp();
                if (mine) {
                    const int row0 = table ? (int)(((long long)(c0 + lane) * rows) % P) : c0 * rows;
                    const int plane = table ? my_id * p.Hkv + kvh : b * p.Hkv + kvh;
                    const uint32_t dst = base + st * C::STAGE + lane * bytes, bar = full(st);
#pragma unroll
                    for (int h = 0; h < DP / 64; ++h) {
                        tma_load_3d(dst + h * C::HALF, &tmK, bar, 64 * h, row0, plane);
                        tma_load_3d(dst + C::TILE_BYTES + h * C::HALF, &tmV, bar, 64 * h, row0, plane);
                    }
                }
                __syncwarp();
                if (++st == C::NS) {
                    st = 0;
                    ++round;
                }
            }
            left -= end - tile;
            tile = 0;
            if (++u == units) {
                u = 0;
                ++b;
            }
        }
        // copies in flight land before the CTA exits: the last issue of each stage
        for (int j = 0; j < C::NS; ++j) {
            volatile int never = 0;
            if (j < st)
                ring_wait(full(j), round & 1u, &never, p, kDevErrTimeoutDrain);
            else if (round > 0)
                ring_wait(full(j), (round - 1) & 1u, &never, p, kDevErrTimeoutDrain);
        }
        return;
    }

    // ================= consumers
    const int g = lane >> 2, t = lane & 3;
    float *merge = reinterpret_cast<float *>(smem + C::OFF_MERGE);
    float *ml = reinterpret_cast<float *>(smem + C::OFF_ML);
    const int rows_all = p.group * p.Sq, D = p.D;
    const bool has_cap = p.cap_out > 0.f, has_bias = p.slopes != nullptr;
    const float fac1 = has_cap ? p.cap_in : p.scale_log2, fac[2] = {fac1, fac1};
    // ldmatrix: matrix m = lane / 8 is keys 8 (m % 2) .. of chunk m / 2 for K (an A operand), keys 8 (m / 2) ..
    // of chunk m % 2 for V (transposed to one); a chunk: 16 bytes, swizzled by the key's low bits.
    const int r8 = lane & 7, m8 = lane >> 3;
    const uint32_t k_row = (16 * warp + r8 + 8 * (m8 & 1)) * 128, v_row = (16 * warp + r8 + 8 * (m8 >> 1)) * 128;
    const int k_chunk = m8 >> 1, v_chunk = m8 & 1;
    int st = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (left > 0) {
        const Span span = seq_span<kTile>(p, b);
        const int len = span.len, nt = span.nt;
        const int kvh = u / p.row_blocks, rb = u - kvh * p.row_blocks;
        const int begin = tile, end = (int)((long long)nt < tile + left ? (long long)nt : tile + left);
        const int row0 = rb * C::ROWS;
        const size_t qrow0 = ((size_t)b * p.Hkv + kvh) * rows_all + row0;  // row of Q and O

        // ---- Q as B operand: lane (g, t) holds elements 2t, 2t + 1 and 2t + 8, 2t + 9 of each 16 of row g
        uint32_t qf[NT][KT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const bool have = row0 + 8 * n + g < rows_all;
            const uint16_t *src = p.Q + (qrow0 + 8 * n + g) * D + 2 * t;
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    qf[n][i][h] = have && 16 * i + 8 * h < D ? *reinterpret_cast<const uint32_t *>(src + 16 * i + 8 * h) : 0u;
        }
        // ---- this lane's query columns: keys seen, position, bias
        int lo[NT][2], hi[NT][2], pos[NT][2];
        float slope2[NT][2], near[NT][2];
        int all_lo = 0, all_hi = len;  // every row sees [all_lo, all_hi)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int row = min(row0 + 8 * n + 2 * t + c, rows_all - 1), i = row % p.Sq;
                pos[n][c] = len - p.Sq + i;
                lo[n][c] = 0;
                hi[n][c] = p.causal ? min(len, pos[n][c] + 1) : len;
                const size_t at = (size_t)b * p.Sq + i;
                if (p.key_begin) lo[n][c] = min(max(0, ld_plan(p.key_begin + at)), len);
                if (p.key_end) hi[n][c] = min(hi[n][c], ld_plan(p.key_end + at));
                hi[n][c] = max(hi[n][c], 0);
                near[n][c] = (float)max(0, max(lo[n][c] - pos[n][c], pos[n][c] - (hi[n][c] - 1)));
                slope2[n][c] = has_bias ? ld_plan(p.slopes + kvh * p.group + row / p.Sq) * 1.4426950408889634f : 0.f;
                all_lo = max(all_lo, lo[n][c]);
                all_hi = min(all_hi, hi[n][c]);
            }
        all_lo = __reduce_max_sync(0xffffffffu, all_lo);
        all_hi = __reduce_min_sync(0xffffffffu, all_hi);

        float ref[NT][2], most[NT][2], l[NT][2], acc[NT][KT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            ref[n][0] = ref[n][1] = 0.f;
            most[n][0] = most[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < KT; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[n][i][c] = 0.f;
        }

        for (int i = begin; i < end; ++i) {
            if (!__all_sync(0xffffffffu, ok && mbar_try_wait(full(st), phase))) {
                if (ok) ok = ring_wait(full(st), phase, abort_flag, p, kDevErrTimeoutKV);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
            const uint32_t kt = base + st * C::STAGE, vt = kt + C::TILE_BYTES;
            const int key0 = (span.t0 + i) * kTile + 16 * warp;  // this warp's keys
            if (key0 < span.hi && key0 + 16 > span.lo) {
                // ---- S^T = K Q^T, in two chains
                float s[NT][4], s1[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = s1[n][e] = 0.f;
#pragma unroll
                for (int k = 0; k < KT; k += 2) {
                    uint32_t a[4], a1[4];
                    const uint32_t half = kt + (k >> 2) * C::HALF + k_row;
                    ldmatrix4(a, half + (((2 * (k & 3) + k_chunk) ^ r8) << 4));
                    ldmatrix4(a1, half + (((2 * (k & 3) + 2 + k_chunk) ^ r8) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_bf16(s[n], a, qf[n][k][0], qf[n][k][1]);
                        mma_bf16(s1[n], a1, qf[n][k + 1][0], qf[n][k + 1][1]);
                    }
                }
                // ---- scores less their column's reference, log2 units: element e is key g + 8 (e / 2), query
                // column e % 2
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] += s1[n][e];
                if (has_cap) {
                    float far = 0.f;
#pragma unroll
                    for (int n = 0; n < NT; ++n) cap_argument(s[n], fac, far);
                    if (__any_sync(0xffffffffu, far > kTanhMaxSq)) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) cap_any(s[n], p.tanh_k, p.cap_out, ref[n]);
                    } else {
#pragma unroll
                        for (int n = 0; n < NT; ++n) cap_near(s[n], p.tanh_k, ref[n]);
                    }
                } else {
#pragma unroll
                    for (int n = 0; n < NT; ++n) scale_less(s[n], fac, ref[n]);
                }
                if (has_bias) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float at[2] = {(float)(key0 - pos[n][0] + g), (float)(key0 - pos[n][1] + g)};
                        less_bias(s[n], 0.f, at, near[n], slope2[n]);
                    }
                }
                const bool whole = key0 >= all_lo && key0 + 16 <= all_hi;
                uint32_t v_keep[2] = {0xffffffffu, 0xffffffffu};  // keys 2t, 2t + 1 and 2t + 8, 2t + 9
                if (!whole) {
                    bool seen[2] = {false, false};
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = key0 + g + 8 * (e >> 1);
                            const bool in = key >= lo[n][e & 1] && key < hi[n][e & 1];
                            seen[e >> 1] |= in;
                            if (!in) s[n][e] = -INFINITY;
                        }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // what no row sees is no number
                        const uint32_t lanes = __ballot_sync(0xffffffffu, seen[h]) >> (8 * t);
                        v_keep[h] = ((lanes & 0x0fu) ? 0x0000ffffu : 0u) | ((lanes & 0xf0u) ? 0xffff0000u : 0u);
                    }
                }
                bool above = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) above |= fmaxf(s[n][c], s[n][c + 2]) > most[n][c];
                // A column's reference is its maximum when it was set and moves only when a score exceeds it by
                // kMost: bf16 weights are as exact at 2^7 as at 1. (Until a column has seen a key, most is -inf
                // and the reference 0.)
                if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float mx = fmaxf(s[n][c], s[n][c + 2]);
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            const bool first = most[n][c] == -INFINITY;
                            if (mx == -INFINITY) continue;  // (uniform over the column's lanes)
                            const float by = first ? mx : fmaxf(0.f, mx);
                            const float alpha = first ? 0.f : ex2(-by);
                            ref[n][c] += by;
                            most[n][c] = kMost;
                            l[n][c] *= alpha;
                            s[n][c] -= by;
                            s[n][c + 2] -= by;
#pragma unroll
                            for (int q = 0; q < KT; ++q) {
                                acc[n][q][c] *= alpha;
                                acc[n][q][c + 2] *= alpha;
                            }
                        }
                }
                // ---- weights, their transpose as the B operand of O^T += V^T P^T
                uint32_t pf[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e] = ex2(s[n][e]);
                        l[n][e & 1] += w[e];
                    }
                    pf[n][0] = transpose8x8(pack_bf16x2(w[0], w[1]));
                    pf[n][1] = transpose8x8(pack_bf16x2(w[2], w[3]));
                }
                // (`whole` is uniform: the masked copy of the loop serves a row's first and last tile)
                auto second = [&](auto masked) {
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        uint32_t a[4];
                        ldmatrix4_trans(a, vt + (k >> 2) * C::HALF + v_row + (((2 * (k & 3) + v_chunk) ^ r8) << 4));
                        if (decltype(masked)::value) a[0] &= v_keep[0], a[1] &= v_keep[0], a[2] &= v_keep[1], a[3] &= v_keep[1];
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma_bf16(acc[n][k], a, pf[n][0], pf[n][1]);
                    }
                };
                if (whole)
                    second(std::false_type{});
                else
                    second(std::true_type{});
            }
            fence_proxy_async_smem();  // this stage's reads before the copies that refill it
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(st));
            if (++st == C::NS) {
                st = 0;
                phase ^= 1u;
            }
        }

        // ---- merge the four warps: rows [ROWS] x DP
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
                l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
                l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
                if (g == 0) {
                    ml[warp * C::ROWS + 8 * n + 2 * t + c] = most[n][c] == -INFINITY ? -INFINITY : ref[n][c];
                    ml[(kWarps + warp) * C::ROWS + 8 * n + 2 * t + c] = l[n][c];
                }
            }
        const bool cut = begin > 0 || end < nt;
        const size_t slot = ((size_t)2 * blockIdx.x + (begin > 0 ? 0 : 1)) * C::ROWS;
        if (threadIdx.x == 0 && begin == 0) {
            int2 d = make_int2(blockIdx.x, blockIdx.x);
            if (cut) {  // the unit's last tile: this CTA's share ends inside the unit
                const long long at = sh.t1 - left + nt - 1;
                d.y = owner(at, sh.total, sh.ctas);
            }
            p.desc[(size_t)b * units + u] = d;
        }
        constexpr int V4 = C::COLS / 4;
#pragma unroll
        for (int round = 0; round < C::ROUNDS; ++round) {
            const int col0 = round * C::COLS;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float *dst = merge + (warp * C::ROWS + 8 * n + 2 * t + c) * (C::COLS + 4) + g;
#pragma unroll
                    for (int k = 0; k < C::COLS / 16; ++k) {
                        dst[16 * k] = acc[n][round * (C::COLS / 16) + k][c];
                        dst[16 * k + 8] = acc[n][round * (C::COLS / 16) + k][c + 2];
                    }
                }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
            for (int x = threadIdx.x; x < C::ROWS * V4; x += 32 * kWarps) {
                const int r = x / V4, c4 = x - r * V4, col = col0 + 4 * c4;
                float mw[kWarps], M = -INFINITY, L = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    mw[w] = ml[w * C::ROWS + r];
                    M = fmaxf(M, mw[w]);
                }
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float f = mw[w] == -INFINITY ? 0.f : ex2(mw[w] - M);
                    const float4 v = *reinterpret_cast<const float4 *>(merge + (w * C::ROWS + r) * (C::COLS + 4) + 4 * c4);
                    L = fmaf(f, ml[(kWarps + w) * C::ROWS + r], L);
                    o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
                }
                if (cut) {
                    if (col == 0) {
                        p.part_m[slot + r] = M;
                        p.part_l[slot + r] = L;
                    }
                    *reinterpret_cast<float4 *>(p.part_acc + (slot + r) * DP + col) = o;
                } else if (row0 + r < rows_all && col < D) {
                    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
                    const size_t at = (qrow0 + r) * D + col;
                    if (p.o_bf16)
                        *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p.O) + at) =
                            make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
                    else
                        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.O) + at) =
                            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                }
            }
            asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");  // the merge area is free again
        }
        left -= end - begin;
        tile = 0;
        if (++u == units) {
            u = 0;
            ++b;
        }
    }
}

// K or V as {D, keys of a plane, planes}, boxes of 64 elements and a copy's keys.
bool make_map(CUtensorMap *m, const uint16_t *data, const fa_problem *P) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t keys = (cuuint64_t)(P->paged ? P->page_size : P->Sk), D = (cuuint64_t)P->D;
    cuuint64_t dims[3] = {D, keys, P->paged ? (cuuint64_t)P->num_pages * P->hkv_local : (cuuint64_t)P->Hkv};
    cuuint64_t strides[2] = {2 * D, 2 * D * keys};
    cuuint32_t box[3] = {64, (cuuint32_t)(P->paged && keys < kTile ? keys : kTile), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t *>(data), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int NT>
int run(const fa_problem *P, cudaStream_t st) {
    static std::atomic<int> cache[64];
    const int fit = resident(few_kernel<DP, NT>, kThreads, FewConfig<DP, NT>::SMEM, cache);
    FewParams p;
    p.Q = P->Q;
    p.O = P->O;
    p.o_bf16 = P->o_bf16;
    p.B = P->Hkv / P->hkv_local, p.Hkv = P->hkv_local, p.Sq = P->Sq, p.D = P->D;
    p.group = P->Hq / P->Hkv;
    p.causal = P->causal;
    p.block_table = P->paged ? P->block_table : nullptr;
    p.seq_lens = P->paged ? P->seq_lens : nullptr;
    p.page_size = P->page_size, p.num_pages = P->num_pages, p.max_pages = P->max_pages;
    p.Sk = P->Sk;
    p.scale_log2 = P->scale_log2;
    p.slopes = P->slopes;
    p.key_begin = P->key_begin, p.key_end = P->key_end;
    p.status = P->status;
    p.unit = 1.f;
    p.part_m = P->part_m, p.part_l = P->part_l, p.part_acc = P->part_acc;
    p.cap_in = P->cap_in, p.cap_out = P->cap_out;
    for (int i = 0; i < 5; ++i) p.tanh_k[i] = P->cap_out * kTanhC[i];
    int ctas = 0;
    const int planned = plan_rows<kTile, DP, 8 * NT>(p, fit, ATTN_PARTIAL_ROWS, ctas);
    if (planned != ATTN_OK) return planned;
    CUtensorMap tmK, tmV;
    if (!make_map(&tmK, P->K, P) || !make_map(&tmV, P->V, P)) return ATTN_ERR_CUDA;
    const int rc = launch(few_kernel<DP, NT>, dim3((unsigned)ctas), dim3(kThreads), FewConfig<DP, NT>::SMEM, st, tmK, tmV, p);
    if (rc != ATTN_OK) return rc;
    return launch_combine<DP, 8 * NT>(p, st);
}

}  // namespace

}  // namespace ts

extern "C" int ts_few_rows(const fa_problem *P) {
    // More than 16 rows would read the cache twice, from L2: 16 sequences of 8,192 keys, capped, took here and
    // in the kernel for prompts 117 and 164 us at 16 rows, 195 and 166 at 24 (one of 32,768: 47 and 55, 64 and 57). Since
    // then 94 here at 16 rows, and there 155 and 49 at 24, 163 at 64.
    // (As many units as descriptors find room behind the partials; key indexes look a few tiles past the end.)
    return P->mod && (long long)(P->Hq / P->Hkv) * P->Sq <= 16 && P->Hkv <= 65536 && P->Sk <= 0x7fffffff - 65536 &&
           ts_tc_supported(P);
}

extern "C" int ts_launch_few_rows(const fa_problem *P, void *stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool one = P->Hq / P->Hkv * P->Sq <= 8;
    if (P->D <= 64) return one ? ts::run<64, 1>(P, st) : ts::run<64, 2>(P, st);
    return one ? ts::run<128, 1>(P, st) : ts::run<128, 2>(P, st);
}
