// The chunk kernels of linear attention for fp16 rows.
#include "ring_linattn.hpp"

hipError_t ring_launch_linattn_f16(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  return ring_lin::launch<_Float16>(a, rev, state_only, st);
}

hipError_t ring_launch_linattn_pair_f16(const RingLinArgs& a, hipStream_t st) { return ring_lin::launch_pair<_Float16>(a, st); }
