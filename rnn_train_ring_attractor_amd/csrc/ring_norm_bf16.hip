// The kernels of norm, gate and scaled residual for bf16 rows.
#include "ring_norm.hpp"

hipError_t ring_launch_norm_bf16(const RingNormArgs& p, bool wide, bool back, hipStream_t st) { return ring_norm::launch<__bf16>(p, wide, back, st); }
