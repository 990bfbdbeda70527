// fa_mod.cu -- what stands around the attention kernel with modified scores: the key ranges of packed
// documents, the bounds of a unit's ranges, and the choice of the kernel form.
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

// One warp per (sequence, row tile of a kv head): the least begin and greatest end over the tile's
// query positions that see a key ({0, 0} when none does), the greatest begin and least end of all. Rows of a tile are packed (query head,
// position), so positions repeat; a tile of at least Sq rows covers all of them.
__global__ void __launch_bounds__(256) mod_bounds_kernel(const int *__restrict__ key_begin,
                                                         const int *__restrict__ key_end, int4 *__restrict__ out,
                                                         int n, int tiles, int unit_rows, int rows_per_kv, int Sq, int Sk) {
    pdl_wait();
    pdl_trigger();
    const int w = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (w >= n) return;
    const int b = w / tiles, row0 = (w - b * tiles) * unit_rows;
    const int rows = min(min(unit_rows, rows_per_kv - row0), Sq);
    const size_t at = (size_t)b * Sq;
    int lo = 0x7fffffff, hi = 0, lo1 = 0, hi1 = Sk;
    for (int e = lane; e < rows; e += 32) {
        const int i = (row0 + e) % Sq;
        const int b0 = key_begin ? key_begin[at + i] : 0, b1 = key_end ? key_end[at + i] : Sk;
        if (b0 < b1) {
            lo = min(lo, b0);
            hi = max(hi, b1);
        }
        lo1 = max(lo1, b0);
        hi1 = min(hi1, b1);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    lo1 = __reduce_max_sync(0xffffffffu, lo1);
    hi1 = __reduce_min_sync(0xffffffffu, hi1);
    if (lane == 0) out[w] = hi > lo ? make_int4(lo, hi, lo1, hi1) : make_int4(0, 0, 0, 0);
}

// Token i of document [s, e) sees keys [s, i] and the document's first prefix tokens (causal), or the
// whole document; with a window only its last `window` keys. The document is found by bisection.
__global__ void __launch_bounds__(256) mask_ranges_kernel(const int *__restrict__ cu, const int *__restrict__ prefix,
                                                          int n_docs, int S, int causal, int window,
                                                          int *__restrict__ key_begin, int *__restrict__ key_end) {
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= S) return;
    int begin = 0, end = 0;
    if (i >= cu[0] && i < cu[n_docs]) {
        int a = 0, b = n_docs;  // cu[a] <= i < cu[b]
        while (b - a > 1) {
            const int m = (a + b) >> 1;
            if (cu[m] <= i)
                a = m;
            else
                b = m;
        }
        const int s = cu[a], e = min(cu[a + 1], S);
        begin = s;
        end = e;
        if (causal) {
            end = i + 1;
            if (prefix) end = max(end, (int)min((long long)e, (long long)s + prefix[a]));
        }
        if (window > 0) begin = max(begin, i - window + 1);
    }
    key_begin[i] = begin;
    key_end[i] = end;
}

template <typename... KArgs, typename... Args>
static int launch(void (*kern)(KArgs...), unsigned grid, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(256);
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
    return ts::launch(ts::mod_bounds_kernel, (unsigned)((n + 7) / 8), static_cast<cudaStream_t>(stream), P->key_begin,
                      P->key_end, reinterpret_cast<int4 *>(P->bounds), n, tiles, ts_tc_unit_rows(P),
                      P->Hq / P->Hkv * P->Sq, P->Sq, P->Sk);
}

extern "C" int ts_launch_mask_ranges(const int *cu_docs, const int *prefix, int n_docs, int S, int causal, int window,
                                     int *key_begin, int *key_end, void *stream) {
    return ts::launch(ts::mask_ranges_kernel, (unsigned)(((long long)S + 255) / 256), static_cast<cudaStream_t>(stream), cu_docs,
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
