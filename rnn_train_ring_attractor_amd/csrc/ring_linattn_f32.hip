// The chunk kernels of linear attention for fp32 rows.
#include "ring_linattn.hpp"

hipError_t ring_launch_linattn_f32(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  return ring_lin::launch<float>(a, rev, state_only, st);
}

hipError_t ring_launch_linattn_pair_f32(const RingLinArgs& a, hipStream_t st) { return ring_lin::launch_pair<float>(a, st); }
