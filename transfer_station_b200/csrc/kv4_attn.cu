// kv4_attn.cu -- attention over the 4-bit paged key cache (attn_kv4.h), for single tokens and a few new
// positions per sequence.
//
// What bounds it: the cache bytes, D/2 + D/32 per key and per value, read once (68 B at D = 128 against
// 256 in bf16). At the measured copy rate an SM receives about 24 bytes, 46 elements, per clock, and every
// element has to reach the tensor cores as a number. What an SM sub-partition was measured to take: an
// m16n8k16 fp16 MMA 8.2 cycles, a logic or fp16 instruction 2, and they overlap little (an MMA and four
// LOPs: 13). So:
//   * A nibble n under a mask is already a number: the fp16 subnormal n * 2^-24 (n * 2^-20 for the high
//     nibble of a byte), two to an operand register by one LOP. MMAs take subnormals exactly, though the sum
//     is then aligned as if they were normal and loses up to ten bits (24 of them remain, measured).
//   * First product: the keys enter like that; the high nibbles' factor 16 is in Q's fragment. The offset 8
//     and the scales stay off the elements: one accumulator per 32-element group gets -8 * 2^-24 *
//     sum(Q over the group) added and is multiplied by the key's scale once. (e4m3 operands, whose
//     nibbles need no more than a mask either and pair with Q split in two, ran at half this speed.)
//   * Second product: one LOP3 and one HFMA2 turn a pair of nibbles into the values themselves, (n - 8) * s, exact.
//     The weights stay as they are for every group. (The scale in the weight instead took 127 us where this takes
//     133, but rounded twice, the second time below fp16's normal numbers: behind a key that holds most of the
//     weight, or at small scales, the other keys' products lost their bits or were zero.)
//   * ldmatrix gives each lane one 32-bit word of one group per key (K), and, transposed, two keys' same
//     four elements in the halves of a register (V): the operand layouts without a permute. The code tiles
//     come by TMA with the 64-byte (D = 64: 32-byte) swizzle, so the eight rows of a matrix lie in
//     different banks.
// Keys are the M side of mma.m16n8k16 and the query rows of a kv head the N side: up to 8 rows cost one
// MMA per 16 keys x 16 elements, with no padding rows. tcgen05 would need the operand tile written back to
// shared memory (2 bytes an element: 92 of the 128 bytes a clock) and 128 rows of queries. fp16 rather than
// bf16: the weights keep 11 bits, and Q, 8 bits wide, is exact after a power-of-two scale per row.
//
// Work split: rows_plan.cuh. One producer warp per CTA streams tiles into a ring of shared-memory stages (codes by
// TMA, scales by 16-byte copies); four consumer warps take 32 keys of each tile, each with its own
// running maximum and accumulator, merged in shared memory at a unit's end.
//
// Measured (D = 128, 32 / 8 heads): 64 sequences of 8,192 keys 133 us, 4 of 131,072 (64 / 8 heads) 130 us, each 571 MB
// of cache, 4.3 TB/s, with the SM at 1.965 GHz; the time follows that clock, and a call repeated for long is held to
// 1.8 to 1.9 GHz by the power limit: 137 to 144. With a cap of 50 143 us, a bias 150, both 159; a window of half the
// keys 77. Streaming the same tiles without arithmetic takes 96 us. 9 to 16 rows of a kv head in one
// column pair (64 sequences of 8,192 keys, 16 rows): 243 us, D = 64 138; two passes of 8 took 246 and 169.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "attn_kv4.h"
#include "fa_launch.h"
#include "rows_plan.cuh"
#include "score_cap.cuh"

namespace ts {

namespace {

constexpr int kTile = 128;       // keys per stage
constexpr int kWarps = 4;        // consumer warps, 32 keys of a tile each
constexpr int kSlabs = 2;        // 16-key MMA rows of a warp and tile
constexpr int kThreads = 32 * (kWarps + 1);

constexpr float kHead = 12.f, kMost = 15.f;  // see the weights
// With small pages the copy engine is bound by the number of copies, and a page's 64 bytes of scales take as
// long as its codes: up to this page size the producer's lanes fetch them. 64 sequences of 4,096 keys (32 / 8 heads,
// D = 128), by the engine and by the lanes: pages of 8 149 and 122 us, 16 93 and 83, 32 76 and 75, 64 70 and 71. (With the
// values at their scale 107 to 111, 86, 79, and 75 by the engine at 64.)
constexpr int kSmallPage = 32;

struct Kv4Params : RowsParams {
    const uint8_t *kc, *ks, *vc, *vs;
    float cap_in, cap_out, tanh_k[5];
};

// 16 bytes from global to shared memory, asynchronously; and one arrival at a barrier once this thread's copies so
// far have landed.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

template <int D, int NT>
struct Kv4Config {
    static constexpr int CODES = kTile * D / 2, SCALES = kTile * D / ATTN_KV4_GROUP;
    static constexpr int STAGE = 2 * (CODES + SCALES);
    static constexpr int NS = D == 128 ? 3 : 6;
    static constexpr int V_CODES = CODES, K_SCALES = 2 * CODES, V_SCALES = 2 * CODES + SCALES;  // in a stage
    static constexpr int ROWS = 8 * NT;
    static constexpr int MERGE = kWarps * ROWS * (D + 4) * 4;  // one warp's accumulator rows, padded
    static constexpr int OFF_MERGE = NS * STAGE;
    static constexpr int OFF_ML = OFF_MERGE + MERGE;           // m, l [kWarps][ROWS]
    static constexpr int OFF_BAR = OFF_ML + 2 * kWarps * ROWS * 4;
    static constexpr int SMEM = OFF_BAR + 2 * NS * 8 + 1024;  // + alignment of the swizzled tiles
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(  // (not volatile: a pure function of its operands, free to be scheduled)
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma16816_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2 *>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t *>(&v); }

// Two E4M3 bytes (the low half word) -> fp16.
__device__ __forceinline__ __half2 scales2(uint32_t bytes) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)bytes, __NV_E4M3);
    return __half2(r);
}

constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;   // fp16: n * 2^-24, n * 2^-20
constexpr float kKeyUnit = 1.f / 16777216.f, kUnit = 1.f / 8.f;  // 2^-24 and 2^-3: what 1 stands for as a key, a value

// A pair of nibbles (of two keys) -> the values (n - 8) * s over 8, exact: under an exponent of their own the nibbles
// are 128 + n / 8 and 8 + n / 8, and (128 + n / 8) * s - 129 s is rounded once, to a number of 8 bits. s has 4
// bits, so 129 s has 11 at most and 9 s has 8; with the largest scale, 448, all stay below 65504. (The constants as
// bits: the conversion functions are not folded.)
constexpr uint32_t k128 = 0x58005800u, k8 = 0x48004800u, kMinus129 = 0xd808d808u, kMinus9 = 0xc880c880u;
struct ValueScales {  // s, -129 s, -9 s of two keys
    __half2 s, low, high;
    __device__ __forceinline__ explicit ValueScales(__half2 v)
        : s(v), low(__hmul2(v, as_half2(kMinus129))), high(__hmul2(v, as_half2(kMinus9))) {}
};
// (x & mask) | exponent as one LOP3: written out, the compiler emits two with an immediate each
__device__ __forceinline__ __half2 under(uint32_t x, uint32_t mask, uint32_t exponent) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(mask), "r"(exponent));
    return as_half2(r);
}
__device__ __forceinline__ uint32_t value_low(uint32_t x, const ValueScales &v) {
    return as_u32(__hfma2(under(x, kLow, k128), v.s, v.low));
}
__device__ __forceinline__ uint32_t value_high(uint32_t x, const ValueScales &v) {
    return as_u32(__hfma2(under(x, kHigh, k8), v.s, v.high));
}

// A slab's 16 rows of codes: lane (g, t) gets word t of every group of rows g and g + 8, or transposed the
// 16-bit column g of every group of rows 2t, 2t + 1 and 2t + 8, 2t + 9. `off`: the lane's swizzled row.
template <int D, bool TRANS>
__device__ __forceinline__ void load_rows(uint32_t slab, uint32_t off, uint32_t (&r0)[D / 32], uint32_t (&r1)[D / 32]) {
    auto load = [](uint32_t (&r)[4], uint32_t addr) {
        if constexpr (TRANS)
            ldmatrix4_trans(r, addr);
        else
            ldmatrix4(r, addr);
    };
    if constexpr (D == 128) {
        load(r0, slab + off);
        load(r1, slab + off + 8 * 64);
    } else {
        uint32_t r[4];
        load(r, slab + off);
        r0[0] = r[0], r0[1] = r[1], r1[0] = r[2], r1[1] = r[3];
    }
}

// MOD: the call has a cap, a bias or key ranges.
template <int D, int NT, bool MOD>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2)
    kv4_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Kv4Params p) {
    using C = Kv4Config<D, NT>;
    constexpr int MT = D / 16;             // 16-element tiles of the output
    constexpr int GROUPS = D / ATTN_KV4_GROUP;
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
            mbar_init(full(s), 1 + (p.page_size <= kSmallPage ? 32 : 0));  // (each producer lane's scales)
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
        const int P = p.page_size;
        const int rows = P < kTile ? P : kTile;      // keys per copy
        const int per_tile = kTile / rows;           // copies per pool and tile
        int st = 0;                                  // next stage, and the round of the ring it is in
        uint32_t round = 0;
        bool ok = true;
        auto produce = [&](auto small_pages) {
            constexpr bool small = decltype(small_pages)::value;
            while (left > 0 && ok) {
                const Span sp = seq_span<kTile>(p, b);
                const int nt = sp.nt;
                const int kvh = u / p.row_blocks;
                const int *table = p.block_table + (size_t)b * p.max_pages;
                const int end = (int)((long long)nt < tile + left ? (long long)nt : tile + left);
                // chunk ids (a chunk: `rows` keys) of the next 32 chunks, one a lane
                int win = -1, id = -1;
                for (int i = tile; i < end && ok; ++i) {
                    const int c0 = (sp.t0 + i) * per_tile;
                    if (win < 0 || c0 + per_tile > win + 32) {
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
                    const int my_id = __shfl_sync(0xffffffffu, id, (c0 - win + lane) & 31);
                    const bool mine = lane < per_tile && my_id >= 0;
                    const int n = __popc(__ballot_sync(0xffffffffu, mine));
                    const uint32_t code_bytes = (uint32_t)(rows * (D / 2)), scale_bytes = (uint32_t)(rows * GROUPS);
                    const uint32_t dst = base + st * C::STAGE, bar = full(st);
                    if (lane == 0) mbar_expect_tx(bar, (uint32_t)n * 2u * (code_bytes + (small ? 0u : scale_bytes)));
                    __syncwarp();
                    if (mine) {
                        const int row0 = (int)(((long long)(c0 + lane) * rows) % P);
                        const int plane = my_id * p.Hkv + kvh;
                        const size_t at = ((size_t)plane * P + row0) * GROUPS;  // in the scale pools
                        tma_load_3d(dst + lane * code_bytes, &tmK, bar, 0, row0, plane);
                        if (!small) bulk_load(dst + C::K_SCALES + lane * scale_bytes, p.ks + at, scale_bytes, bar);
                        tma_load_3d(dst + C::V_CODES + lane * code_bytes, &tmV, bar, 0, row0, plane);
                        if (!small) bulk_load(dst + C::V_SCALES + lane * scale_bytes, p.vs + at, scale_bytes, bar);
                    }
                    if constexpr (small) {  // the scales in pieces of 16 bytes
                        constexpr int KEYS = 16 / GROUPS, PIECES = kTile / KEYS;  // keys of a piece, pieces of a pool and tile
                        const int key = (lane & (PIECES - 1)) * KEYS;
                        const int sid = __shfl_sync(0xffffffffu, id, (c0 - win + key / rows) & 31);
                        if (sid >= 0) {
                            const int row = (int)(((long long)c0 * rows + key) % P);
                            const size_t at = ((size_t)(sid * p.Hkv + kvh) * P + row) * GROUPS;
                            if (PIECES == 32 || lane < PIECES) copy16(dst + C::K_SCALES + key * GROUPS, p.ks + at);
                            if (PIECES == 32 || lane >= PIECES) copy16(dst + C::V_SCALES + key * GROUPS, p.vs + at);
                        }
                        copy_arrive(bar);
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
        };
        if (P <= kSmallPage)
            produce(std::true_type{});
        else
            produce(std::false_type{});
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
    const int rows_all = p.group * p.Sq;
    const bool has_cap = MOD && p.cap_out > 0.f, has_bias = MOD && p.slopes != nullptr;
    // This lane's row and 16-byte chunk for ldmatrix, swizzled. D = 128: matrix m is chunk m of rows 0..7 (a
    // second load takes rows 8..15); D = 64: chunk m % 2 of rows 8 (m / 2) ..
    uint32_t rows_off;
    if constexpr (D == 128) {
        const int r = lane & 7, m = lane >> 3;
        rows_off = r * 64 + ((m ^ ((r >> 1) & 3)) << 4);
    } else {
        const int r = (lane & 7) + 8 * (lane >> 4), m = (lane >> 3) & 1;
        rows_off = r * 32 + ((m ^ ((r >> 2) & 1)) << 4);
    }
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

        // ---- Q fragments: lane (g, t) holds, of query row g, elements 8t..8t+7 of every group, scaled by a
        // power of two per row
        uint32_t qf[NT][GROUPS][4];
        float start[NT][GROUPS][2];  // -8 * 2^-24 * sum of Q over a group, for this lane's two query columns
        float fac[NT][2];            // accumulator -> scaled score, for the same
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const bool have = row0 + 8 * n + g < rows_all;
            const uint16_t *src = p.Q + (qrow0 + 8 * n + g) * D + 8 * t;
            uint32_t raw[GROUPS][4];
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < GROUPS; ++w) {
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (have) v = *reinterpret_cast<const uint4 *>(src + ATTN_KV4_GROUP * w);
                raw[w][0] = v.x, raw[w][1] = v.y, raw[w][2] = v.z, raw[w][3] = v.w;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    a = fmax3(a, fabsf(__uint_as_float(raw[w][i] << 16)), fabsf(__uint_as_float(raw[w][i] & 0xffff0000u)));
            }
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 1));
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, 2));
            // 2^(4-e) puts the row's largest magnitude into [16, 32) (a zero or non-finite row stays)
            const int e = (int)(__float_as_uint(a) >> 23) - 127;
            const bool plain = a == 0.f || e >= 128 || e <= -120;
            const float down = plain ? 1.f : __uint_as_float((uint32_t)(131 - e) << 23);
            const float up = plain ? 1.f : __uint_as_float((uint32_t)(123 + e) << 23);
#pragma unroll
            for (int w = 0; w < GROUPS; ++w) {
                // a word's nibbles pair up as elements (0,4) (1,5) (2,6) (3,7); the odd pairs are high nibbles
                auto element = [&](int i) {
                    const uint32_t v = raw[w][i >> 1];
                    return __uint_as_float((i & 1) ? (v & 0xffff0000u) : (v << 16)) * down;
                };
                float sum = 0.f;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const float part = (h & 1) ? 0.0625f : 1.f;
                    const __half2 q = __floats2half2_rn(element(h) * part, element(h + 4) * part);
                    qf[n][w][h] = as_u32(q);
                    const float2 f = __half22float2(q);
                    sum += (f.x + f.y) / part;
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= -8.f * kKeyUnit;
                start[n][w][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                start[n][w][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            }
            // Held below 2^100, so that rows past 2^83 stay finite: an accumulator is a multiple of 2^-57 below 2, and scores
            // that differ at all then lie 2^43 apart.
            const float unit = (has_cap ? p.cap_in : p.scale_log2) / kKeyUnit;
            fac[n][0] = fminf(__shfl_sync(0xffffffffu, up, 8 * t) * unit, 0x1p100f);
            fac[n][1] = fminf(__shfl_sync(0xffffffffu, up, 8 * t + 4) * unit, 0x1p100f);
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

        float ref[NT][2], most[NT][2], l[NT][2], acc[NT][MT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            ref[n][0] = ref[n][1] = 0.f;
            most[n][0] = most[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[n][i][c] = 0.f;
        }

        for (int i = begin; i < end; ++i) {
            if (!__all_sync(0xffffffffu, ok && mbar_try_wait(full(st), phase))) {
                if (ok) ok = ring_wait(full(st), phase, abort_flag, p, kDevErrTimeoutKV);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
            const uint8_t *stage = smem + st * C::STAGE;
            const uint32_t stage_at = base + st * C::STAGE;
            const int key0 = (span.t0 + i) * kTile + 16 * kSlabs * warp;  // this warp's keys
            if (key0 < span.hi && key0 + 16 * kSlabs > span.lo) {
                // ---- S^T = K Q^T
                float s[kSlabs][NT][4];
#pragma unroll
                for (int b = 0; b < kSlabs; ++b) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.f;
                    const int r0 = 16 * (kSlabs * warp + b);  // the slab's first row in the stage
                    uint32_t k0[GROUPS], k1[GROUPS];          // this lane's word of every group, keys g and g + 8
                    load_rows<D, false>(stage_at + r0 * (D / 2), rows_off, k0, k1);
                    const uint8_t *sp = stage + C::K_SCALES + (r0 + g) * GROUPS;
                    float2 f0[GROUPS / 2], f1[GROUPS / 2];    // their scales
                    if constexpr (GROUPS == 4) {
                        const uint32_t w0 = *reinterpret_cast<const uint32_t *>(sp);
                        const uint32_t w1 = *reinterpret_cast<const uint32_t *>(sp + 8 * GROUPS);
                        f0[0] = __half22float2(scales2(w0 & 0xffffu)), f0[1] = __half22float2(scales2(w0 >> 16));
                        f1[0] = __half22float2(scales2(w1 & 0xffffu)), f1[1] = __half22float2(scales2(w1 >> 16));
                    } else {
                        f0[0] = __half22float2(scales2(*reinterpret_cast<const uint16_t *>(sp)));
                        f1[0] = __half22float2(scales2(*reinterpret_cast<const uint16_t *>(sp + 8 * GROUPS)));
                    }
                    float d[GROUPS][NT][4];
#pragma unroll
                    for (int w = 0; w < GROUPS; ++w) {
                        const uint32_t xs = k0[w] >> 8, ys = k1[w] >> 8;
                        const uint32_t a0[4] = {k0[w] & kLow, k1[w] & kLow, k0[w] & kHigh, k1[w] & kHigh};
                        const uint32_t a1[4] = {xs & kLow, ys & kLow, xs & kHigh, ys & kHigh};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16816_zero(d[w][n], a0, qf[n][w][0], qf[n][w][1]);
                            mma16816(d[w][n], a1, qf[n][w][2], qf[n][w][3]);
                        }
                    }
#pragma unroll
                    for (int w = 0; w < GROUPS; ++w) {
                        const float c0 = (w & 1) ? f0[w >> 1].y : f0[w >> 1].x, c1 = (w & 1) ? f1[w >> 1].y : f1[w >> 1].x;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            s[b][n][0] = fmaf(d[w][n][0] + start[n][w][0], c0, s[b][n][0]);
                            s[b][n][1] = fmaf(d[w][n][1] + start[n][w][1], c0, s[b][n][1]);
                            s[b][n][2] = fmaf(d[w][n][2] + start[n][w][0], c1, s[b][n][2]);
                            s[b][n][3] = fmaf(d[w][n][3] + start[n][w][1], c1, s[b][n][3]);
                        }
                    }
                }
                // ---- scores less their column's reference, log2 units: element e is key g + 8 (e / 2) of its
                // slab, query column e % 2
                const bool whole = key0 >= all_lo && key0 + 16 * kSlabs <= all_hi;
                if (has_cap) {
                    float far = 0.f;
#pragma unroll
                    for (int b = 0; b < kSlabs; ++b)
#pragma unroll
                        for (int n = 0; n < NT; ++n) cap_argument(s[b][n], fac[n], far);
                    if (__any_sync(0xffffffffu, far > kTanhMaxSq)) {
#pragma unroll
                        for (int b = 0; b < kSlabs; ++b)
#pragma unroll
                            for (int n = 0; n < NT; ++n) cap_any(s[b][n], p.tanh_k, p.cap_out, ref[n]);
                    } else {
#pragma unroll
                        for (int b = 0; b < kSlabs; ++b)
#pragma unroll
                            for (int n = 0; n < NT; ++n) cap_near(s[b][n], p.tanh_k, ref[n]);
                    }
                } else {
#pragma unroll
                    for (int b = 0; b < kSlabs; ++b)
#pragma unroll
                        for (int n = 0; n < NT; ++n) scale_less(s[b][n], fac[n], ref[n]);
                }
                if (has_bias) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float at[2] = {(float)(key0 - pos[n][0] + g), (float)(key0 - pos[n][1] + g)};
#pragma unroll
                        for (int b = 0; b < kSlabs; ++b) less_bias(s[b][n], 16.f * b, at, near[n], slope2[n]);
                    }
                }
                uint32_t seen[kSlabs];  // bits 0 to 3: some row sees key 2t, 2t + 1, 2t + 8, 2t + 9 of the slab
                if (!whole) {
#pragma unroll
                    for (int b = 0; b < kSlabs; ++b) {
                        bool any[2] = {false, false};
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int key = key0 + 16 * b + g + 8 * (e >> 1);
                                const bool in = key >= lo[n][e & 1] && key < hi[n][e & 1];
                                any[e >> 1] |= in;
                                if (!in) s[b][n][e] = -INFINITY;
                            }
                        seen[b] = 0;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t lanes = __ballot_sync(0xffffffffu, any[h]) >> (8 * t);
                            seen[b] |= ((lanes & 0x0fu) ? 1u << (2 * h) : 0u) | ((lanes & 0xf0u) ? 2u << (2 * h) : 0u);
                        }
                    }
                }
                bool above = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = fmaxf(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
                        for (int b = 1; b < kSlabs; ++b) mx = fmax3(mx, s[b][n][c], s[b][n][c + 2]);
                        above |= mx > most[n][c];
                    }
                // A column's reference is its maximum less kHead when it was set, and moves only when a score
                // exceeds it by kMost: weights reach from 2^kHead at the maximum up to 2^kMost, the upper end of fp16,
                // and keep its 11 bits down to 2^-26 of the largest. (Until a column has seen a key, most is -inf and
                // the reference 0.)
                if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float mx = fmaxf(s[0][n][c], s[0][n][c + 2]);
#pragma unroll
                            for (int b = 1; b < kSlabs; ++b) mx = fmax3(mx, s[b][n][c], s[b][n][c + 2]);
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            const bool first = most[n][c] == -INFINITY;
                            if (mx == -INFINITY) continue;  // (uniform over the column's lanes)
                            const float by = first ? mx - kHead : fmaxf(0.f, mx - kHead);
                            const float alpha = first ? 0.f : ex2(-by);
                            ref[n][c] += by;
                            most[n][c] = kMost;
                            l[n][c] *= alpha;
#pragma unroll
                            for (int b = 0; b < kSlabs; ++b) {
                                s[b][n][c] -= by;
                                s[b][n][c + 2] -= by;
                            }
#pragma unroll
                            for (int q = 0; q < MT; ++q) {
                                acc[n][q][c] *= alpha;
                                acc[n][q][c + 2] *= alpha;
                            }
                        }
                }
#pragma unroll
                for (int b = 0; b < kSlabs; ++b) {
                    // ---- weights, and their transpose as the B operand of O^T += V^T P^T
                    uint32_t pf[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w[e] = ex2(s[b][n][e]);
                            l[n][e & 1] += w[e];
                        }
                        pf[n][0] = transpose8x8(as_u32(__floats2half2_rn(w[0], w[1])));
                        pf[n][1] = transpose8x8(as_u32(__floats2half2_rn(w[2], w[3])));
                    }
                    // ---- V^T: lane (g, t) holds elements 4g..4g+3 of every group for keys 2t, 2t+1 and 2t+8, 2t+9
                    const int r0 = 16 * (kSlabs * warp + b);
                    uint32_t v0[GROUPS], v1[GROUPS];
                    load_rows<D, true>(stage_at + C::V_CODES + r0 * (D / 2), rows_off, v0, v1);
                    // the keys' scales, pairs of keys side by side: sc[half][..] bytes (A0 B0 A1 B1) (A2 B2 A3 B3)
                    const uint8_t *sp = stage + C::V_SCALES + (r0 + 2 * t) * GROUPS;
                    uint32_t sc[2][GROUPS / 2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if constexpr (GROUPS == 4) {
                            uint2 w = *reinterpret_cast<const uint2 *>(sp + 8 * j * GROUPS);
                            sc[j][0] = __byte_perm(w.x, w.y, 0x5140);
                            sc[j][1] = __byte_perm(w.x, w.y, 0x7362);
                        } else {
                            sc[j][0] = __byte_perm(*reinterpret_cast<const uint32_t *>(sp + 8 * j * GROUPS), 0u, 0x3120);
                        }
                    }
                    if (!whole) {
                        // what an unseen slot holds may be any byte, a NaN scale among them: it becomes zero
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (!((seen[b] >> j) & 1u))
#pragma unroll
                                for (int w = 0; w < GROUPS / 2; ++w) sc[j >> 1][w] &= (j & 1) ? 0x00ff00ffu : 0xff00ff00u;
                        }
                    }
#pragma unroll
                    for (int w = 0; w < GROUPS; ++w) {
                        const uint32_t x = v0[w], y = v1[w], xs = x >> 8, ys = y >> 8;
                        const ValueScales s0(scales2((w & 1) ? sc[0][w >> 1] >> 16 : sc[0][w >> 1] & 0xffffu));
                        const ValueScales s1(scales2((w & 1) ? sc[1][w >> 1] >> 16 : sc[1][w >> 1] & 0xffffu));
                        const uint32_t a0[4] = {value_low(x, s0), value_high(x, s0), value_low(y, s1), value_high(y, s1)};
                        const uint32_t a1[4] = {value_low(xs, s0), value_high(xs, s0), value_low(ys, s1), value_high(ys, s1)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16816(acc[n][2 * w], a0, pf[n][0], pf[n][1]);
                            mma16816(acc[n][2 * w + 1], a1, pf[n][0], pf[n][1]);
                        }
                    }
                }
            }
            fence_proxy_async_smem();  // this stage's reads before the copies that refill it
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(st));
            if (++st == C::NS) {
                st = 0;
                phase ^= 1u;
            }
        }

        // ---- merge the four warps: rows [ROWS] x D
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
                // elements 4g..4g+3 of every group
                float *dst = merge + (warp * C::ROWS + 8 * n + 2 * t + c) * (D + 4) + 4 * g;
#pragma unroll
                for (int w = 0; w < GROUPS; ++w)
                    *reinterpret_cast<float4 *>(dst + ATTN_KV4_GROUP * w) =
                        make_float4(acc[n][2 * w][c], acc[n][2 * w][c + 2], acc[n][2 * w + 1][c],
                                    acc[n][2 * w + 1][c + 2]);
            }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
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
        constexpr int V4 = D / 4;
        for (int x = threadIdx.x; x < C::ROWS * V4; x += 32 * kWarps) {
            const int r = x / V4, c4 = x - r * V4;
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
                const float4 v = *reinterpret_cast<const float4 *>(merge + (w * C::ROWS + r) * (D + 4) + 4 * c4);
                L = fmaf(f, ml[(kWarps + w) * C::ROWS + r], L);
                o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
            }
            if (cut) {
                if (c4 == 0) {
                    p.part_m[slot + r] = M;
                    p.part_l[slot + r] = L;
                }
                *reinterpret_cast<float4 *>(p.part_acc + (slot + r) * D + 4 * c4) = o;
            } else if (row0 + r < rows_all) {
                const float inv = L > 0.f ? 1.f / (kUnit * L) : (L == 0.f ? 0.f : L);
                const size_t at = (qrow0 + r) * D + 4 * c4;
                if (p.o_bf16)
                    *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p.O) + at) =
                        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
                else
                    *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.O) + at) =
                        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");  // the merge area is free again
        left -= end - begin;
        tile = 0;
        if (++u == units) {
            u = 0;
            ++b;
        }
    }
}

// A code pool as {D/2 bytes, rows of a page, page x kv head}, boxes of one page's rows up to a tile.
bool make_code_map(CUtensorMap *m, const uint8_t *codes, const ts_kv4_problem *P, int D) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t row = (cuuint64_t)D / 2, ps = (cuuint64_t)P->page_size;
    cuuint64_t dims[3] = {row, ps, (cuuint64_t)P->num_pages * P->Hkv};
    cuuint64_t strides[2] = {row, row * ps};
    cuuint32_t box[3] = {(cuuint32_t)row, (cuuint32_t)(ps < kTile ? ps : kTile), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(codes), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, D == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int NT, bool MOD>
int run(const ts_kv4_problem *P, cudaStream_t st) {
    static std::atomic<int> cache[64];
    const int fit = resident(kv4_kernel<D, NT, MOD>, kThreads, Kv4Config<D, NT>::SMEM, cache);
    if (fit < 0) return ATTN_ERR_CUDA;
    Kv4Params p;
    p.Q = P->Q;
    p.O = P->O;
    p.o_bf16 = P->o_bf16;
    p.B = P->B, p.Hkv = P->Hkv, p.Sq = P->Sq, p.D = D;
    p.group = P->Hq / P->Hkv;
    p.causal = P->causal;
    p.block_table = P->block_table;
    p.seq_lens = P->seq_lens;
    p.page_size = P->page_size, p.num_pages = P->num_pages, p.max_pages = P->max_pages;
    p.Sk = P->max_pages * P->page_size;
    p.scale_log2 = P->scale_log2;
    p.slopes = P->slopes;
    p.key_begin = P->key_begin, p.key_end = P->key_end;
    p.status = P->status;
    p.unit = kUnit;
    p.part_m = P->part_m, p.part_l = P->part_l, p.part_acc = P->part_acc;
    p.kc = P->k_codes, p.ks = P->k_scales, p.vc = P->v_codes, p.vs = P->v_scales;
    p.cap_in = P->cap_in, p.cap_out = P->cap_out;
    for (int i = 0; i < 5; ++i) p.tanh_k[i] = P->cap_out * kTanhC[i];
    int ctas = 0;
    const int planned = plan_rows<kTile, D, 8 * NT>(p, fit, P->part_rows, ctas);
    if (planned != ATTN_OK) return planned;
    CUtensorMap tmK, tmV;
    if (!make_code_map(&tmK, P->k_codes, P, D) || !make_code_map(&tmV, P->v_codes, P, D)) return ATTN_ERR_CUDA;
    const int rc = launch(kv4_kernel<D, NT, MOD>, dim3((unsigned)ctas), dim3(kThreads), Kv4Config<D, NT>::SMEM, st, tmK, tmV, p);
    if (rc != ATTN_OK) return rc;
    return launch_combine<D, 8 * NT>(p, st);
}

}  // namespace

}  // namespace ts

extern "C" int ts_launch_kv4(const ts_kv4_problem *P, void *stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long rows = (long long)(P->Hq / P->Hkv) * P->Sq;
    // up to 8 query rows of a kv head: one column tile; more: two, so that a cache row serves 16
    const bool mod = P->cap_out > 0.f || P->slopes || P->key_begin || P->key_end;
    if (P->D == 64) {
        if (mod) return rows <= 8 ? ts::run<64, 1, true>(P, st) : ts::run<64, 2, true>(P, st);
        return rows <= 8 ? ts::run<64, 1, false>(P, st) : ts::run<64, 2, false>(P, st);
    }
    if (mod) return rows <= 8 ? ts::run<128, 1, true>(P, st) : ts::run<128, 2, true>(P, st);
    return rows <= 8 ? ts::run<128, 1, false>(P, st) : ts::run<128, 2, false>(P, st);
}
