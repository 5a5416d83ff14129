// The chunk kernels of linear attention for bf16 rows.
#include "ring_linattn.hpp"

hipError_t ring_launch_linattn_bf16(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  return ring_lin::launch<__bf16>(a, rev, state_only, st);
}

hipError_t ring_launch_linattn_pair_bf16(const RingLinArgs& a, hipStream_t st) { return ring_lin::launch_pair<__bf16>(a, st); }
