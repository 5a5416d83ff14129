// What the kernels of the recurrent layer's operators (short convolution, selective scan, norm and gate) share: functions in fp32 and
// rows of values read and written some at a time.
#pragma once
#include "ring_common.hpp"
#include "ring_kernels.hpp"

namespace ring_recur {

constexpr float kLog2e = 1.44269504088896341f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.693147180559945309f;

// Functions for rows of fp32 (FINE) and of 16 bits.  FINE: a power's argument as a sum of two numbers, the second to first order, otherwise one
// (off by |x| 2^-24 then, which is less than the rounding of a 16-bit argument by far).

// e^x, FINE: for |x| <= 87
template <bool FINE> __device__ __forceinline__ float exp_of(float x) {
  const float high = x * kLog2e, e = __builtin_amdgcn_exp2f(high);
  if constexpr (!FINE) return e;
  const float low = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -high));
  return fmaf(e, low * kLn2, e);
}

// x log2(e), rounded once
__device__ __forceinline__ float times_log2e(float x) { return fmaf(x, kLog2e, x * kLog2eLow); }

// 1 / (1 + e^-x)  (FINE, of NaN: a number; its users multiply by x as well, or look at it themselves)
template <bool FINE> __device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + exp_of<FINE>(FINE ? __builtin_amdgcn_fmed3f(-x, -87.f, 87.f) : -x));
}
template <bool FINE> __device__ __forceinline__ float silu(float x) { return x * sigmoid<FINE>(x); }
// the derivative of x sigmoid(x), s = sigmoid(x)
__device__ __forceinline__ float silu_slope(float x, float s) { return s * fmaf(x, 1.f - s, 1.f); }

// ln(1 + e^x) = max(x, 0) + ln(1 + e), e = e^-|x|, and its derivative.  What 1 + e loses of e is added to the logarithm of the sum, whose slope there is one
// to first order (together within 3.5 2^-24 of ln(1 + e), measured from e = 2^-24 to 1).
template <bool FINE> __device__ __forceinline__ float softplus(float x, float& slope) {
  const float e = exp_of<FINE>(FINE ? __builtin_amdgcn_fmed3f(-fabsf(x), -87.f, 0.f) : -fabsf(x)), w = 1.f + e;
  const float y = fmaf(__builtin_amdgcn_logf(w), kLn2, e - (w - 1.f)) + __builtin_amdgcn_fmed3f(x, 0.f, INFINITY), r = __builtin_amdgcn_rcpf(w);
  slope = x > 0.f ? r : e * r;
  return FINE ? (x == x ? y : x) : y;        // (NaN: otherwise through e)
}
template <bool FINE> __device__ __forceinline__ float softplus(float x) {
  float slope;
  return softplus<FINE>(x, slope);
}

// `rows` rows of `st` values as a buffer: what is read behind them is zero, what is written there is left out.  (Their places within it are 32-bit numbers that
// stay the same from chunk to chunk, the buffer's own address is scalar: no vector instruction for either.)
template <typename T> __device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const T* p, long st, int rows) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), 0, (int)(rows * st * (long)sizeof(T)), 0x00027000);
}
constexpr int kOutside = 0x7ffffff0;   // a place behind every buffer

// E values, neighbours in memory.  WIDE: the address is a whole number of min(16, E sizeof(T)) bytes; otherwise one by one, `here` of them.
template <typename T, int E> struct Row {
  typedef T vec __attribute__((ext_vector_type(E)));
  T v[E];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = (T)0.f;
  }
  __device__ __forceinline__ void load(const T* p, bool wide, int here) {
    constexpr int W = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
    typedef T part __attribute__((ext_vector_type(W)));
    if (wide) {
      if (here >= E) {
#pragma unroll
        for (int i = 0; i < E / W; ++i) {
          const part w = *reinterpret_cast<const part*>(p + i * W);
#pragma unroll
          for (int e = 0; e < W; ++e) v[i * W + e] = w[e];
        }
      } else {
        zero();
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = e < here ? p[e] : (T)0.f;
    }
  }
  // One by one without conditions: `here` of them (at least one) and copies of the last
  __device__ __forceinline__ void read(const T* p, int here) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = p[min(e, here - 1)];
  }
  // From and to a buffer, at a number of bytes
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t b, int at) {
    constexpr int BYTES = E * sizeof(T);
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const auto x = __builtin_amdgcn_raw_buffer_load_b128(b, at + 16 * i, 0, 0);
        __builtin_memcpy(v + i * (16 / sizeof(T)), &x, 16);
      }
    } else if constexpr (BYTES == 8) {
      const auto x = __builtin_amdgcn_raw_buffer_load_b64(b, at, 0, 0);
      __builtin_memcpy(v, &x, 8);
    } else if constexpr (BYTES == 4) {
      const auto x = __builtin_amdgcn_raw_buffer_load_b32(b, at, 0, 0);
      __builtin_memcpy(v, &x, 4);
    } else {
      const auto x = __builtin_amdgcn_raw_buffer_load_b16(b, at, 0, 0);
      __builtin_memcpy(v, &x, 2);
    }
  }
  __device__ __forceinline__ void give(__amdgpu_buffer_rsrc_t b, int at) const {
    constexpr int BYTES = E * sizeof(T);
    typedef unsigned four __attribute__((ext_vector_type(4)));
    typedef unsigned two __attribute__((ext_vector_type(2)));
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        four x;
        __builtin_memcpy(&x, v + i * (16 / sizeof(T)), 16);
        __builtin_amdgcn_raw_buffer_store_b128(x, b, at + 16 * i, 0, 0);
      }
    } else if constexpr (BYTES == 8) {
      two x;
      __builtin_memcpy(&x, v, 8);
      __builtin_amdgcn_raw_buffer_store_b64(x, b, at, 0, 0);
    } else if constexpr (BYTES == 4) {
      unsigned x;
      __builtin_memcpy(&x, v, 4);
      __builtin_amdgcn_raw_buffer_store_b32(x, b, at, 0, 0);
    } else {
      unsigned short x;
      __builtin_memcpy(&x, v, 2);
      __builtin_amdgcn_raw_buffer_store_b16(x, b, at, 0, 0);
    }
  }
  __device__ __forceinline__ void store(T* p, bool wide, int here) const {
    constexpr int W = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
    typedef T part __attribute__((ext_vector_type(W)));
    if (wide) {
      if (here >= E) {
#pragma unroll
        for (int i = 0; i < E / W; ++i) {
          part w;
#pragma unroll
          for (int e = 0; e < W; ++e) w[e] = v[i * W + e];
          *reinterpret_cast<part*>(p + i * W) = w;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < here) p[e] = v[e];
    }
  }
};

// Sums across lanes.  Of a and b, the wave's halves (its odd and even rows of 16) added: a's sum in the lower half (even rows), b's in the other.
__device__ __forceinline__ float fold32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// the lane's value plus that of the lane CTRL names within a row of 16
template <int CTRL> __device__ __forceinline__ float plus_dpp(float x) {
  return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}
constexpr int kRor8 = 0x128, kUp4 = 0x104, kDown4 = 0x114, kXor1 = 0xB1, kXor2 = 0x4E;      // (up 4: the lane four further on)

// Sums over parts in their order (RingSumArgs): a workgroup of 256 takes 256 / W columns; W threads share a column's parts and are added in their order
constexpr int kWays = 8;
inline int sum_ways(const RingSumArgs& p) { return p.parts >= 16 ? kWays : 1; }
inline unsigned sum_blocks(const RingSumArgs& p) { return (unsigned)((p.n * sum_ways(p) + 255) / 256); }
template <int W> __device__ __forceinline__ void sum_parts(const RingSumArgs& p, unsigned block, float* sums) {
  constexpr int COLS = 256 / W;
  const size_t i = (size_t)block * COLS + threadIdx.x % COLS;
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

__device__ __forceinline__ int length_of(const int* lengths, int b, int T) { return lengths ? min(max(lengths[b], 0), T) : T; }

}  // namespace ring_recur
