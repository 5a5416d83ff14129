// The kernels of norm, gate and scaled residual for fp32 rows.
#include "ring_norm.hpp"

hipError_t ring_launch_norm_f32(const RingNormArgs& p, bool wide, bool back, hipStream_t st) { return ring_norm::launch<float>(p, wide, back, st); }
