// fa_mod_range.cu -- the tensor-core attention kernel with key ranges.
#include "fa_mod_inst.cuh"

extern "C" int ts_launch_tc_mod1(const fa_problem *P, void *stream) { return ts::launch_tc_mod<1>(P, stream); }
