// fa_mod_inst.cuh -- the instances of one MOD of the tensor-core attention kernel: head widths 64 and
// 128, one or two query tiles per unit, contiguous or paged K/V.
#pragma once
#include "fa_fwd_kernel.cuh"

namespace ts {

template <int MOD>
static int launch_tc_mod(const fa_problem *P, void *stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int nqt = nqt_for(P);
    const int tiles = ts_tc_ctas_per_split(P) / P->Hkv;
    if (P->D <= 64) {
        if (nqt == 2) return launch_tc<64, 2, false, false, MOD>(P, st, tiles);
        return launch_tc<64, 1, false, false, MOD>(P, st, tiles);
    }
    if (nqt == 2) return launch_tc<128, 2, false, false, MOD>(P, st, tiles);
    return launch_tc<128, 1, false, false, MOD>(P, st, tiles);
}

}  // namespace ts
