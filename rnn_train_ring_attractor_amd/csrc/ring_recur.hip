// Sums over parts, for the gradients of parameters: every workgroup that finds a part writes it out, and the parts are added in their order, so that
// a result is the same from run to run.
#include "ring_recur.hpp"

// A workgroup takes 256 / W columns; W threads share a column's parts and are added in their order.  Bound by latency: 4 to 5 us for parts of 5 to 64 rows, of up to
// 20000 columns.
template <int W>
__global__ __launch_bounds__(256) void ring_sum_parts_kernel(RingSumArgs p) {
  constexpr int COLS = 256 / W;
  __shared__ float sums[256];
  const size_t i = (size_t)blockIdx.x * COLS + threadIdx.x % COLS;
  const int w = threadIdx.x / COLS, each = (p.parts + W - 1) / W, end = min(p.parts, (w + 1) * each);
  float sum = 0.f;
  if (i < p.n)
#pragma unroll 8
    for (int k = w * each; k < end; ++k) sum += p.part[(size_t)k * p.n + i];
  if constexpr (W > 1) {
    sums[threadIdx.x] = sum;
    __syncthreads();
    if (w > 0) return;
    for (int k = 1; k < W; ++k) sum += sums[k * COLS + threadIdx.x];
  }
  if (i >= p.n) return;
  const size_t column = i / p.per;
  const int k = (int)(i - column * p.per), more = k - (p.per - p.rest);
  if (k < p.N) {
    if (p.out) p.out[column * p.N + k] = sum;
  } else if (more >= 0 && p.more[more]) {
    p.more[more][column] = sum;
  }
}

hipError_t ring_launch_sum_parts(const RingSumArgs& p, hipStream_t st) {
  if (p.parts >= 16) hipLaunchKernelGGL(ring_sum_parts_kernel<8>, dim3((unsigned)((p.n + 31) / 32)), dim3(256), 0, st, p);
  else hipLaunchKernelGGL(ring_sum_parts_kernel<1>, dim3((unsigned)((p.n + 255) / 256)), dim3(256), 0, st, p);
  return hipGetLastError();
}
