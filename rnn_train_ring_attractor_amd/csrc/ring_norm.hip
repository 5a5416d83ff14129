// Norm, gate and scaled residual: how the rows are read, the launches, the sums over the workgroups' parts.
#include "ring_norm.hpp"

using namespace ring_norm;

// dw, dscale, dnext [C] from the workgroups' parts, in their order.  512 parts of 2048 columns: 6 us, bound by latency.
__global__ __launch_bounds__(256) void ring_norm_sum_kernel(RingNormArgs p) {
  constexpr int W = 16, COLS = 256 / W;
  __shared__ float sums[256];
  const int k = blockIdx.y, c = blockIdx.x * COLS + threadIdx.x % COLS, w = threadIdx.x / COLS, each = (p.parts + W - 1) / W;
  float* out = k == 0 ? p.dw : (k == 1 ? p.dscale : p.dnext);
  if (!out) return;
  float sum = 0.f;
  if (c < p.C)
#pragma unroll 4
    for (int m = w * each; m < min(p.parts, (w + 1) * each); ++m) sum += p.part[((size_t)m * 3 + k) * p.C + c];
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (w > 0 || c >= p.C) return;
  for (int m = 1; m < W; ++m) sum += sums[m * COLS + threadIdx.x];
  out[c] = sum;
}

// 16 bytes at a time where rows, groups and addresses are whole numbers of that
static bool is_wide(const RingNormArgs& p, int V) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.gate) | reinterpret_cast<uintptr_t>(p.residual) |
                        reinterpret_cast<uintptr_t>(p.dy) | reinterpret_cast<uintptr_t>(p.dn) | reinterpret_cast<uintptr_t>(p.w) |
                        reinterpret_cast<uintptr_t>(p.scale) | reinterpret_cast<uintptr_t>(p.next);
  return p.group % V == 0 && (all & 15) == 0 && (p.xs | p.gs | p.rs | p.dys | p.dns) % V == 0;
}

static hipError_t launch_type(RingNormArgs p, int type, bool back, hipStream_t st) {
  const int V = type == RINGATTR_F32 ? 4 : 8;
  const bool wide = is_wide(p, V);
  p.each = 1.f / (float)p.group;
  p.each_row = 1.f / (float)p.C;
  if (back) p.parts = parts_of(plan_of(p.C, p.group, wide ? V : 1), p.rows);
  hipError_t e = type == RINGATTR_F32 ? ring_launch_norm_f32(p, wide, back, st) : (type == RINGATTR_BF16 ? ring_launch_norm_bf16(p, wide, back, st) : ring_launch_norm_f16(p, wide, back, st));
  if (e != hipSuccess || !back || !p.part) return e;
  hipLaunchKernelGGL(ring_norm_sum_kernel, dim3((unsigned)((p.C + 15) / 16), 3), dim3(256), 0, st, p);
  return hipGetLastError();
}

size_t ring_norm_bwd_bytes(int type, long rows, int C, int group, bool params) {
  if (!params) return 0;
  const int V = type == RINGATTR_F32 ? 4 : 8, a = group % V == 0 ? parts_of(plan_of(C, group, V), rows) : 0, b = parts_of(plan_of(C, group, 1), rows);
  return (size_t)(a > b ? a : b) * 3 * C * sizeof(float);
}

hipError_t ring_norm_fwd(const RingNormArgs& p, int type, hipStream_t st) { return launch_type(p, type, false, st); }
hipError_t ring_norm_bwd(RingNormArgs p, int type, hipStream_t st) { return launch_type(p, type, true, st); }
