// fa_fwd_sm100.cu -- the plain forms of the tensor-core attention kernel (fa_fwd_kernel.cuh): which
// calls it takes and the launcher behind ts_launch_attention.
#include "fa_fwd_kernel.cuh"

extern "C" int ts_tc_supported(const fa_problem *P) {
    if (P->D % 8 != 0 || P->D > 128 || P->D < 8) return 0;
    if (P->v_prepacked && P->Sk % 8 != 0) return 0;
    if (((uintptr_t)P->Q | (uintptr_t)P->K | (uintptr_t)P->V) & 15u) return 0;
    const float *out = P->O ? P->O : P->part_acc;
    if (((uintptr_t)out) & 15u) return 0;
    if (ts::encode_fn() == nullptr) return 0;
    return 1;
}

extern "C" int ts_tc_unit_rows(const fa_problem *P) { return ts::kBM * ts::nqt_for(P); }

extern "C" int ts_tc_ctas_per_split(const fa_problem *P) {
    const long long rows = (long long)(P->Hq / P->Hkv) * P->Sq;
    const int nqt = ts::nqt_for(P);
    const long long tiles = (rows + ts::kBM * nqt - 1) / (ts::kBM * nqt);
    return (int)(tiles * P->Hkv);
}

// attn_diag_wait_timeout's launch: the NOQ build at head_dim 128, one 128-row tile per unit.
extern "C" int ts_launch_tc_noq(const fa_problem *P, void *stream) {
    using namespace ts;
    if (P->D != 128 || (long long)(P->Hq / P->Hkv) * P->Sq > kBM || P->paged || P->v_prepacked) return ATTN_ERR_ARGS;
    if (encode_fn() == nullptr) return ATTN_ERR_CUDA;
    return launch_tc<128, 1, false, true>(P, static_cast<cudaStream_t>(stream), 1);
}

extern "C" int ts_launch_tc(const fa_problem *P, void *stream) {
    using namespace ts;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long rows = (long long)(P->Hq / P->Hkv) * P->Sq;
    const int nqt = nqt_for(P);
    const int tiles = (int)((rows + kBM * nqt - 1) / (kBM * nqt));
    const int dp = P->D <= 64 ? 64 : 128;
    const bool vt = P->v_prepacked != 0;
#define TS_LAUNCH(DPV, NQTV)                                                                      \
    do {                                                                                          \
        return vt ? launch_tc<DPV, NQTV, true>(P, st, tiles) : launch_tc<DPV, NQTV, false>(P, st, tiles); \
    } while (0)
    if (dp == 64) {
        if (nqt == 2) TS_LAUNCH(64, 2);
        TS_LAUNCH(64, 1);
    }
    if (nqt == 2) TS_LAUNCH(128, 2);
    TS_LAUNCH(128, 1);
#undef TS_LAUNCH
}
