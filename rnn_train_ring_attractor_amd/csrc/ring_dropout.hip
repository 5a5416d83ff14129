// Dropout whose mask is never stored: whether element i is kept is a function of (seed, offset, i), so the backward finds it again.
//
//   y_i = residual_i + (word_i >= p 2^32 ? x_i / (1 - p) : 0)
//
// word_i is word i % 4 of block i / 4 of Philox with four words and seven rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011; seven rounds are the fewest that pass the tests there): counter (block, offset), key seed.
// Bound by memory: 67 million bf16 values, forward with the residual and backward, 671 MB in 120 us, 5.6 TB/s (a large copy: 5.2 to
// 5.4).  Seven rounds for four values hide behind the loads; a stored mask would be written and read besides.
// What is dropped is left out, not multiplied by zero: an infinity there does not become NaN.
#include "ring_common.hpp"
#include "ring_kernels.hpp"
#include "ringattr.h"

namespace {

struct Words { unsigned w[4]; };

__device__ __forceinline__ Words philox(unsigned long long block, unsigned long long offset, unsigned long long seed) {
  unsigned x0 = (unsigned)block, x1 = (unsigned)(block >> 32), x2 = (unsigned)offset, x3 = (unsigned)(offset >> 32);
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const unsigned long long a = (unsigned long long)x0 * 0xD2511F53u, b = (unsigned long long)x2 * 0xCD9E8D57u;
    x0 = (unsigned)(b >> 32) ^ x1 ^ k0;
    x1 = (unsigned)b;
    x2 = (unsigned)(a >> 32) ^ x3 ^ k1;
    x3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{x0, x1, x2, x3}};
}

}  // namespace

// A thread takes W values at a time, whole blocks of four words, from WIDE memory accesses or one by one.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void ring_dropout_kernel(RingDropoutArgs p) {
  constexpr int W = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(W)));
  const T *x = (const T*)p.x, *res = (const T*)p.residual;
  T* y = (T*)p.y;
  const unsigned long long offset = p.offset + (p.offset_ptr ? (unsigned long long)*p.offset_ptr : 0ull);
  const size_t units = (p.n + W - 1) / W;
  for (size_t u = (size_t)blockIdx.x * 256 + threadIdx.x; u < units; u += (size_t)gridDim.x * 256) {
    const size_t i0 = u * W;
    const int here = p.n - i0 < W ? (int)(p.n - i0) : W;
    vec v, a;
    if (WIDE && here == W) {
      v = *(const vec*)(x + i0);
      if (res) a = *(const vec*)(res + i0);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        v[e] = e < here ? x[i0 + e] : (T)0.f;
        a[e] = res && e < here ? res[i0 + e] : (T)0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < W / 4; ++q) {
      const Words w = philox(u * (W / 4) + q, offset, p.seed);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f = w.w[e] >= p.threshold ? (float)v[4 * q + e] * p.scale : 0.f;
        if (res) f = (float)a[4 * q + e] + f;
        v[4 * q + e] = (T)f;
      }
    }
    if (WIDE && here == W) {
      *(vec*)(y + i0) = v;
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e)
        if (e < here) y[i0 + e] = v[e];
    }
  }
}

template <typename T> static hipError_t launch(const RingDropoutArgs& p, hipStream_t st) {
  constexpr size_t W = 16 / sizeof(T);
  const size_t blocks = ((p.n + W - 1) / W + 255) / 256;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384)), block(256);
  const bool wide = ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.residual) | reinterpret_cast<uintptr_t>(p.y)) & 15) == 0;
  if (wide) hipLaunchKernelGGL((ring_dropout_kernel<T, true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((ring_dropout_kernel<T, false>), grid, block, 0, st, p);
  return hipGetLastError();
}

hipError_t ring_launch_dropout(const RingDropoutArgs& p, int type, hipStream_t st) {
  if (type == RINGATTR_F32) return launch<float>(p, st);
  if (type == RINGATTR_BF16) return launch<__bf16>(p, st);
  return launch<_Float16>(p, st);
}
