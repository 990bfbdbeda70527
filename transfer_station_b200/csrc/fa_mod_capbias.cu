// fa_mod_capbias.cu -- the tensor-core attention kernel with capped scores and a distance bias (and key ranges).
#include "fa_mod_inst.cuh"

extern "C" int ts_launch_tc_mod4(const fa_problem *P, void *stream) { return ts::launch_tc_mod<4>(P, stream); }
