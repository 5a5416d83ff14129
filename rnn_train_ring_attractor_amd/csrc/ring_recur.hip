// Sums over parts, for the gradients of parameters: every workgroup that finds a part writes it out, and the parts are added in their order, so that
// a result is the same from run to run.
#include "ring_recur.hpp"

// Bound by latency: 4 to 5 us for parts of 5 to 64 rows, of up to 20000 columns.
template <int W> __global__ __launch_bounds__(256) void ring_sum_parts_kernel(RingSumArgs p) {
  __shared__ float sums[256];
  ring_recur::sum_parts<W>(p, blockIdx.x, sums);
}

hipError_t ring_launch_sum_parts(const RingSumArgs& p, hipStream_t st) {
  const dim3 grid(ring_recur::sum_blocks(p));
  if (ring_recur::sum_ways(p) > 1) hipLaunchKernelGGL(ring_sum_parts_kernel<ring_recur::kWays>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(ring_sum_parts_kernel<1>, grid, dim3(256), 0, st, p);
  return hipGetLastError();
}
