// fa_mod_bias.cu -- the tensor-core attention kernel with a distance bias (and key ranges).
#include "fa_mod_inst.cuh"

extern "C" int ts_launch_tc_mod3(const fa_problem *P, void *stream) { return ts::launch_tc_mod<3>(P, stream); }
