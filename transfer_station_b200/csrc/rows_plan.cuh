// rows_plan.cuh -- what the attention kernels for a few query rows of each kv head share (single tokens, a few
// new positions): the division of all sequences' keys among the CTAs, bounded waits and error reports,
// the merge of cut units, and the launch.
//
// Tiles of TILE keys of all (sequence, kv head, row block) units form one list; CTA c of G takes the c-th G-th
// of it, whatever the lengths are, so a ragged batch stays balanced without the host knowing a length. A unit
// cut between CTAs leaves (m, l, acc) partials, merged by rows_combine.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "attn_flash.h"
#include "fa_launch.h"
#include "sm100_ptx.cuh"

extern "C" void ts_count_launch(void);

namespace ts {

namespace {

struct RowsParams {
    const uint16_t *Q;
    void *O;
    int o_bf16;
    int B, Hkv, Sq, D, group, row_blocks, causal;  // Hkv: of one sequence
    const int *block_table, *seq_lens;             // paged; NULL: [B * Hkv][Sk][D]
    int page_size, num_pages, max_pages;
    int Sk;                                        // keys of a sequence, at most
    float scale_log2;                              // log2(e) / sqrt(D)
    const float *slopes;
    const int *key_begin, *key_end;
    int *status;                                   // [0]: result; [2], [3]: reports of the running call and its generation
    unsigned gen;
    float unit;                                    // what a value of 1 stands for in the accumulators
    float *part_m, *part_l, *part_acc;  // [2 * CTAs][rows]([D]): slot 2c of CTA c for a unit begun before it, 2c + 1 after
    int2 *desc;                         // [units]: first and last CTA of a unit (equal: nothing to merge)
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Four 8x8 matrices of 16-bit elements; lane l gives the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// A sequence: its keys, the span [lo, hi) outside which no query of it sees one, and the tiles of that
// span (at least one, so that a sequence without keys gets its zero rows). The span is read from the key
// ranges for up to kSpanRows query positions; longer calls walk the whole sequence.
constexpr int kSpanRows = 16;
struct Span {
    int len, lo, hi, t0, nt;
};
template <int TILE>
__device__ __forceinline__ Span seq_span(const RowsParams &p, int b) {
    Span s;
    const int n = p.seq_lens ? ld_plan(p.seq_lens + b) : p.Sk;
    s.len = n < 0 ? 0 : (n < p.Sk ? n : p.Sk);
    s.lo = 0;
    s.hi = s.len;
    if ((p.key_begin || p.key_end) && p.Sq <= kSpanRows) {
        int lo = s.len, hi = 0;
        for (int i = 0; i < p.Sq; ++i) {
            const size_t at = (size_t)b * p.Sq + i;
            const int x0 = p.key_begin ? max(ld_plan(p.key_begin + at), 0) : 0;
            int x1 = p.key_end ? min(ld_plan(p.key_end + at), s.len) : s.len;
            if (p.causal) x1 = min(x1, s.len - p.Sq + i + 1);
            if (x0 >= x1) continue;  // (sees none)
            lo = min(lo, x0);
            hi = max(hi, x1);
        }
        s.lo = lo;
        s.hi = hi;
    }
    s.t0 = s.lo / TILE;
    s.nt = s.hi > s.lo ? (s.hi + TILE - 1) / TILE - s.t0 : 1;
    return s;
}

// Where a CTA's share of the tile list begins, and what the list is.
struct Share {
    long long total, t0, t1;  // all tiles; this CTA's
    int ctas;                 // CTAs that have a share
    int b;                    // first sequence
    int u;                    // first unit within it
    int tile;                 // first tile of that unit's span
};

// All threads of the CTA. Units are ordered by sequence, then kv head, then row block.
template <int TILE>
__device__ __forceinline__ Share find_share(const RowsParams &p, int cta, int grid) {
    __shared__ long long warp_sum[32];
    __shared__ long long found_rem;
    __shared__ int found_b;
    const int n = blockDim.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = n >> 5;
    const int units = p.Hkv * p.row_blocks;
    const int chunk = (p.B + n - 1) / n;
    const int b0 = min(p.B, tid * chunk), b1 = min(p.B, b0 + chunk);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += (long long)seq_span<TILE>(p, b).nt * units;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    if (tid == 0) found_b = p.B;
    __syncthreads();
    long long before = 0, total = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) before += warp_sum[w];
        total += warp_sum[w];
    }
    Share s;
    s.total = total;
    s.ctas = (int)(total < grid ? total : grid);
    s.t0 = cta < s.ctas ? cta * total / s.ctas : total;
    s.t1 = cta < s.ctas ? (cta + 1) * total / s.ctas : total;
    long long at = before + incl - mine;
    if (s.t0 >= at && s.t0 < at + mine) {
        int b = b0;
        for (; b < b1; ++b) {
            const long long here = (long long)seq_span<TILE>(p, b).nt * units;
            if (s.t0 < at + here) break;
            at += here;
        }
        found_b = b;
        found_rem = s.t0 - at;
    }
    __syncthreads();
    s.b = found_b;
    s.u = s.tile = 0;
    if (s.t0 < s.t1) {
        const int nt = seq_span<TILE>(p, s.b).nt;
        s.u = (int)(found_rem / nt);
        s.tile = (int)(found_rem - (long long)s.u * nt);
    }
    return s;
}

// The CTA that has tile x of the list.
__device__ __forceinline__ int owner(long long x, long long total, int ctas) {
    int c = (int)(x * ctas / total);
    while (c + 1 < ctas && (c + 1) * total / ctas <= x) ++c;
    return c;
}

// Reports gather in a pair (generation, codes) that rows_combine moves to the status word: a report can
// neither meet the clearing of an earlier call's nor be lost by a replayed graph's.
__device__ __forceinline__ void report_pending(const RowsParams &p, int code) {
    unsigned long long *at = reinterpret_cast<unsigned long long *>(p.status + 2);
    unsigned long long old = *reinterpret_cast<volatile unsigned long long *>(at);
    while (true) {
        const unsigned long long now = (unsigned)(old >> 32) == p.gen ? old | (unsigned)code
                                                                      : ((unsigned long long)p.gen << 32) | (unsigned)code;
        const unsigned long long seen = atomicCAS(at, old, now);
        if (seen == old) return;
        old = seen;
    }
}

// Bounded wait on a barrier of this CTA.
__device__ __forceinline__ bool ring_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, const RowsParams &p,
                                          int code) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
            *abort_flag = 1;
            report_pending(p, code);
            return false;
        }
    }
}

// Merges a cut unit's partials (accumulators D wide, outputs p.D): block (unit, row), its warps take pieces in turn. Block 0 also moves the
// call's reports to the status word.
template <int D, int ROWS>
__global__ void __launch_bounds__(128) rows_combine(const RowsParams p) {
    constexpr int PER = D / 32;
    __shared__ float sm[4], sl[4], sacc[4][D];
    pdl_wait();
    pdl_trigger();
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
        unsigned long long *at = reinterpret_cast<unsigned long long *>(p.status + 2);
        const unsigned long long v = *reinterpret_cast<volatile unsigned long long *>(at);
        p.status[0] = (unsigned)(v >> 32) == p.gen ? (int)(unsigned)v : 0;
        *at = 0;
    }
    const int r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int units = p.Hkv * p.row_blocks;
    const int2 d = make_int2(ld_plan(&p.desc[blockIdx.x].x), ld_plan(&p.desc[blockIdx.x].y));
    if (d.x == d.y) return;
    const int b = blockIdx.x / units, u = blockIdx.x - b * units;
    const int kvh = u / p.row_blocks, rb = u - kvh * p.row_blocks;
    const int row = rb * ROWS + r, rows_all = p.group * p.Sq;
    if (row >= rows_all) return;
    auto slot = [&](int c) { return ((size_t)2 * c + (c == d.x ? 1 : 0)) * ROWS + r; };
    float m = -INFINITY, l = 0.f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    for (int c = d.x + warp; c <= d.y; c += 4) {
        const size_t at = slot(c);
        const float mc = p.part_m[at], lc = p.part_l[at];
        float v[PER];
        if constexpr (PER == 4) {
            *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(p.part_acc + at * D + PER * lane);
        } else {
            *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(p.part_acc + at * D + PER * lane);
        }
        const float to = fmaxf(m, mc);
        const float f0 = m == -INFINITY ? 0.f : ex2(m - to), f1 = mc == -INFINITY ? 0.f : ex2(mc - to);
        l = l * f0 + lc * f1;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = acc[i] * f0 + v[i] * f1;
        m = to;
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) sacc[warp][PER * lane + i] = acc[i];
    __syncthreads();
    const int col = threadIdx.x;
    if (col >= p.D) return;
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float L = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = sm[w] == -INFINITY ? 0.f : ex2(sm[w] - M);
        L = fmaf(f, sl[w], L);
        o = fmaf(f, sacc[w][col], o);
    }
    const float inv = L > 0.f ? 1.f / (p.unit * L) : (L == 0.f ? 0.f : L);
    const size_t at = (((size_t)b * p.Hkv + kvh) * rows_all + row) * p.D + col;
    if (p.o_bf16)
        reinterpret_cast<uint16_t *>(p.O)[at] = (uint16_t)pack_bf16x2(o * inv, 0.f);
    else
        reinterpret_cast<float *>(p.O)[at] = o * inv;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn fn = []() -> EncodeTiledFn {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<EncodeTiledFn>(ptr);
        return nullptr;
    }();
    return fn;
}

template <typename... KArgs, typename... Args>
int launch(void (*kern)(KArgs...), dim3 grid, dim3 block, int smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...) != cudaSuccess) return ATTN_ERR_CUDA;
    ts_count_launch();
    return ATTN_OK;
}

// CTAs of a kernel that fit on an SM (cached per device in the kernel's own array, with the shared-memory opt-in done).
template <typename... KArgs>
int resident(void (*kern)(KArgs...), int threads, int smem, std::atomic<int> (&cache)[64]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -1;
    const bool cached = dev >= 0 && dev < 64;
    if (cached) {
        const int r = cache[dev].load(std::memory_order_acquire);
        if (r > 0) return r;
    }
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -1;
    int r = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&r, kern, threads, smem) != cudaSuccess || r < 1) r = 1;
    if (cached) cache[dev].store(r, std::memory_order_release);
    return r;
}

// Row blocks of ROWS query rows, CTAs, and the scratch: the partials take the rows of the first 2 * ctas slots,
// the units' descriptors lie behind their accumulators. `fit`: CTAs resident on an SM.
template <int TILE, int D, int ROWS>
int plan_rows(RowsParams &p, int fit, int part_rows, int &ctas) {
    if (fit < 0) return ATTN_ERR_CUDA;
    p.row_blocks = (p.group * p.Sq + ROWS - 1) / ROWS;
    // (spread over 32 bits, an odd factor: what a fresh scratch block happens to hold, small numbers mostly, must not
    // pass for this call's reports)
    p.gen = ts_next_status_gen() * 2654435761u;
    const long long units = (long long)p.B * p.Hkv * p.row_blocks, tiles = ((long long)p.Sk + TILE - 1) / TILE;
    long long n = (long long)ts_num_sms() * fit;
    if (n > part_rows / (2 * ROWS)) n = part_rows / (2 * ROWS);
    if (tiles * units < n) n = tiles * units;
    const long long room = ((long long)part_rows * p.D - 2 * units) / (2 * ROWS * D);  // (accumulator rows are p.D wide)
    if (n > room) n = room;
    if (n < 1) return ATTN_ERR_ARGS;
    const size_t acc = (size_t)2 * n * ROWS * D;
    p.desc = reinterpret_cast<int2 *>(p.part_acc + acc);
    ctas = (int)n;
    return ATTN_OK;
}

template <int D, int ROWS>
int launch_combine(const RowsParams &p, cudaStream_t st) {
    const int rows = p.group * p.Sq < ROWS ? p.group * p.Sq : ROWS;
    return launch(rows_combine<D, ROWS>, dim3((unsigned)((long long)p.B * p.Hkv * p.row_blocks), rows), dim3(128), 0, st, p);
}

}  // namespace

}  // namespace ts
