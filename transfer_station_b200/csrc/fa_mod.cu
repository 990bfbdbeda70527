// fa_mod.cu -- what stands around the attention kernel with modified scores: the key ranges of packed
// documents, the bounds of a unit's ranges, the units' order by length, and the choice of the kernel form.
// Small kernels bound by latency: 1.8 us (ranges of 6,007 tokens), 2 us each (bounds, order).
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_flash_mod.h"
#include "fa_launch.h"
#include "sm100_ptx.cuh"

extern "C" void ts_count_launch(void);
extern "C" int ts_launch_tc_mod1(const fa_problem *P, void *stream);
extern "C" int ts_launch_tc_mod2(const fa_problem *P, void *stream);
extern "C" int ts_launch_tc_mod3(const fa_problem *P, void *stream);
extern "C" int ts_launch_tc_mod4(const fa_problem *P, void *stream);

namespace ts {

constexpr int kBlock = ATTN_GPU_KEY_TILE;  // keys of the attention kernel's block
constexpr int kBins = 2048;
constexpr int kMostRows = 256;             // of a unit

// One warp per (sequence, row tile of a kv head): the least begin and greatest end over the tile's
// query positions that see a key ({0, 0} when none does), the greatest begin and least end of all. Rows of a
// tile are packed (query head, position), so positions repeat; a tile of at least Sq rows covers all of them.
// A tile across the border of two query heads holds the last positions and the first: between what the two
// parts see may lie a hole, {begin, end} of the second int4, whose third member is the tile's key blocks and
// whose fourth says that some row sees each key from the least begin to the greatest end: within a part
// the rows that see keys follow one another, and each one's range touches the next one's.
struct BoundsTask {
    const int *key_begin, *key_end, *seq_lens;
    int4 *out;
    int n, tiles, unit_rows, rows_per_kv, Sq, Smax, causal;
};

__device__ __forceinline__ void tile_bounds(const BoundsTask &p, int w, int lane) {
    const int b = w / p.tiles, row0 = (w - b * p.tiles) * p.unit_rows, Sq = p.Sq;
    const int rows = min(min(p.unit_rows, p.rows_per_kv - row0), Sq), i0 = row0 % Sq;
    const int Sk = p.seq_lens ? max(0, min(ld_plan(p.seq_lens + b), p.Smax)) : p.Smax;
    const size_t at = (size_t)b * Sq;
    constexpr int kTurns = kMostRows / 32;  // all loads in flight at once
    int b0[kTurns], b1[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
        const int e = 32 * k + lane, i = i0 + e >= Sq ? i0 + e - Sq : i0 + e;
        b0[k] = 0;
        b1[k] = Sk;
        if (e < rows) {
            if (p.key_begin) b0[k] = ld_plan(p.key_begin + at + i);
            if (p.key_end) b1[k] = ld_plan(p.key_end + at + i);
        }
    }
    int lo[2] = {0x7fffffff, 0x7fffffff}, hi[2] = {0, 0}, lo1 = 0, hi1 = Sk;  // [1]: past the border
    int runs[2] = {0, 0}, apart = 0;  // runs of rows that see keys, neighbours that do not touch
    int last0 = 0, last1 = 0;         // the keys of the row before this turn's
#pragma unroll
    for (int k = 0; k < kTurns; ++k) {
        const int e = 32 * k + lane, past = i0 + e >= Sq, i = past ? i0 + e - Sq : i0 + e;
        const int x0 = max(b0[k], 0);
        int x1 = min(b1[k], Sk);
        if (p.causal) x1 = min(x1, Sk - Sq + i + 1);
        int c0 = __shfl_up_sync(0xffffffffu, x0, 1), c1 = __shfl_up_sync(0xffffffffu, x1, 1);  // the row before
        if (lane == 0) c0 = last0, c1 = last1;
        if (i == 0) c1 = c0;  // (none in this part)
        last0 = __shfl_sync(0xffffffffu, x0, 31);
        last1 = __shfl_sync(0xffffffffu, x1, 31);
        if (e >= rows) continue;
        if (x0 < x1) {
            lo[past] = min(lo[past], x0);
            hi[past] = max(hi[past], x1);
            if (c0 >= c1)
                ++runs[past];
            else
                apart |= max(x0, c0) > min(x1, c1);
        }
        lo1 = max(lo1, x0);
        hi1 = min(hi1, x1);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        lo[h] = __reduce_min_sync(0xffffffffu, lo[h]);
        hi[h] = __reduce_max_sync(0xffffffffu, hi[h]);
        runs[h] = __reduce_add_sync(0xffffffffu, runs[h]);
    }
    apart = __any_sync(0xffffffffu, apart);
    lo1 = __reduce_max_sync(0xffffffffu, lo1);
    hi1 = __reduce_min_sync(0xffffffffu, hi1);
    const int a = min(lo[0], lo[1]), z = max(hi[0], hi[1]);
    if (z <= a) {
        if (lane == 0) p.out[2 * w] = p.out[2 * w + 1] = make_int4(0, 0, 0, 0);
        return;
    }
    int h0 = 0, h1 = 0;
    if (hi[0] > 0 && hi[1] > 0) {
        const int first = lo[1] < lo[0];  // the part whose keys come first
        if (hi[first] < lo[1 - first]) h0 = hi[first], h1 = lo[1 - first];
    }
    // blocks from the first key's on, less whole ones of the hole (as the attention kernel walks them)
    const int base = a / kBlock * kBlock, skip = h1 > h0 ? (h1 - base) / kBlock - (h0 - base + kBlock - 1) / kBlock : 0;
    const int blocks = (z - base + kBlock - 1) / kBlock - max(skip, 0);
    if (lane == 0) {
        p.out[2 * w] = make_int4(a, z, lo1, hi1);
        p.out[2 * w + 1] = make_int4(h0, h1, blocks, runs[0] <= 1 && runs[1] <= 1 && !apart && h1 <= h0);
    }
}

__global__ void __launch_bounds__(256) mod_bounds_kernel(const BoundsTask p) {
    pdl_wait();
    pdl_trigger();
    const int w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (w < p.n) tile_bounds(p, w, threadIdx.x & 31);
}

// The units, longest first: a counting sort of the tiles by their key blocks (in steps of 2^shift blocks),
// every tile standing for its sequence's kv heads. Up to kRanked tiles are ranked by comparing all of them, which
// leaves equal ones in their own order (a launch's time then repeats, too); among more, equal ones come as
// they happen to. No result depends on the order.
constexpr int kRanked = 1024;
__global__ void __launch_bounds__(1024) mod_order_kernel(const int4 *bounds, int *order, int n, int tiles, int hkv, int shift) {
    __shared__ int count[kBins], warp_sum[32];
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto place = [&](int w, int at) {
        const int b = w / tiles, tile = w - b * tiles;
        for (int h = 0; h < hkv; ++h) order[at + h] = (b * hkv + h) * tiles + tile;
    };
    if (n <= kRanked) {
        const int mine = tid < n ? ld_plan(bounds + 2 * tid + 1).z : 0;
        if (tid < n) count[tid] = mine;
        __syncthreads();
        int rank = 0;
        for (int w = 0; w < n; ++w) rank += count[w] > mine || (count[w] == mine && w < tid);
        if (tid < n) place(tid, rank * hkv);
        return;
    }
    for (int i = tid; i < kBins; i += 1024) count[i] = 0;
    __syncthreads();
    // bin 0: the longest
    auto bin = [&](int w) { return kBins - 1 - min(ld_plan(bounds + 2 * w + 1).z >> shift, kBins - 1); };
    for (int w = tid; w < n; w += 1024) atomicAdd(&count[bin(w)], hkv);
    __syncthreads();
    // exclusive sums: two bins a thread
    static_assert(kBins == 2048, "");
    const int c0 = count[2 * tid], c1 = count[2 * tid + 1];
    int incl = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int before = incl - c0 - c1;
    for (int i = 0; i < warp; ++i) before += warp_sum[i];
    count[2 * tid] = before;
    count[2 * tid + 1] = before + c0;
    __syncthreads();
    for (int w = tid; w < n; w += 1024) place(w, atomicAdd(&count[bin(w)], hkv));
}

// Token i of document [s, e) sees keys [s, i] and the document's first prefix tokens (causal), or the
// whole document; with a window only its last `window` keys. The document is found by bisection.
__global__ void __launch_bounds__(256) mask_ranges_kernel(const int *cu, const int *prefix,
                                                          int n_docs, int S, int causal, int window,
                                                          int *key_begin, int *key_end) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= S) return;
    int begin = 0, end = 0;
    if (i >= ld_plan(cu) && i < ld_plan(cu + n_docs)) {
        int a = 0, b = n_docs;  // cu[a] <= i < cu[b]
        while (b - a > 1) {
            const int m = (a + b) >> 1;
            if (ld_plan(cu + m) <= i)
                a = m;
            else
                b = m;
        }
        const int s = ld_plan(cu + a), e = min(ld_plan(cu + a + 1), S);
        begin = s;
        end = e;
        if (causal) {
            end = i + 1;
            if (prefix) end = max(end, (int)min((long long)e, (long long)s + ld_plan(prefix + a)));
        }
        if (window > 0) begin = max(begin, i - window + 1);
    }
    key_begin[i] = begin;
    key_end[i] = end;
}

template <typename... KArgs, typename... Args>
static int launch(void (*kern)(KArgs...), unsigned grid, unsigned block, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
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

}  // namespace ts

extern "C" int ts_launch_mod_bounds(const fa_problem *P, void *stream) {
    const int tiles = ts_tc_ctas_per_split(P) / P->Hkv, n = P->Hkv / P->hkv_local * tiles;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const ts::BoundsTask task = {P->key_begin, P->key_end, P->paged ? P->seq_lens : nullptr,
                                 reinterpret_cast<int4 *>(P->bounds), n, tiles, ts_tc_unit_rows(P),
                                 P->Hq / P->Hkv * P->Sq, P->Sq, P->Sk, P->causal};
    const int rc = ts::launch(ts::mod_bounds_kernel, (unsigned)((n + 7) / 8), 256, st, task);
    if (rc != ATTN_OK || !P->order) return rc;
    int shift = 0;
    while (((P->Sk - 1) / ts::kBlock + 1) >> shift >= ts::kBins) ++shift;
    return ts::launch(ts::mod_order_kernel, 1u, 1024, st, task.out, P->order, n, tiles, P->hkv_local, shift);
}

extern "C" int ts_launch_mask_ranges(const int *cu_docs, const int *prefix, int n_docs, int S, int causal, int window,
                                     int *key_begin, int *key_end, void *stream) {
    return ts::launch(ts::mask_ranges_kernel, (unsigned)(((long long)S + 255) / 256), 256, static_cast<cudaStream_t>(stream), cu_docs,
                      prefix, n_docs, S, causal, window, key_begin, key_end);
}

extern "C" int ts_launch_tc_mod(const fa_problem *P, void *stream) {
    switch (P->mod) {
    case 1: return ts_launch_tc_mod1(P, stream);
    case 2: return ts_launch_tc_mod2(P, stream);
    case 3: return ts_launch_tc_mod3(P, stream);
    case 4: return ts_launch_tc_mod4(P, stream);
    default: return ATTN_ERR_ARGS;
    }
}
