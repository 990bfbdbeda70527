// fa_mod_cap.cu -- the tensor-core attention kernel with capped scores (and key ranges).
#include "fa_mod_inst.cuh"

extern "C" int ts_launch_tc_mod2(const fa_problem *P, void *stream) { return ts::launch_tc_mod<2>(P, stream); }
