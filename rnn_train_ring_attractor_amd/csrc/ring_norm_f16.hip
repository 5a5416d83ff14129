// The kernels of norm, gate and scaled residual for fp16 rows.
#include "ring_norm.hpp"

hipError_t ring_launch_norm_f16(const RingNormArgs& p, bool wide, bool back, hipStream_t st) { return ring_norm::launch<_Float16>(p, wide, back, st); }
