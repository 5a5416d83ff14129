// Rotary positions: pair m of a head's values, (a, b), is turned by the angle position * frequency[m],
//
//   (a, b) -> scale (a cos - b sin, b cos + a sin),
//
// pairs being halves apart (m, m + rot / 2) or neighbours (2m, 2m + 1); what lies behind the first `rot` values of a head is copied.
// Backwards the same with the opposite angle.  A position is a count of tokens or an angle of its own (a heading; the pairs then turn
// with its harmonics).
//
// Bound by memory: everything is read once and written once: 8 x 4096 tokens, 16 + 4 heads of 128, bf16: 336 MB in 69 us, 4.9 TB/s (a
// large copy: 5.2).  A workgroup takes a few tokens through all heads of both tensors, so a
// token's angles are found once: the number of turns as a product in 64 bits, whose whole part is taken off before it is rounded (at
// position 2^20 a product in 32 bits is off by 0.06 rad), then one sine and cosine in 32.
#include "ring_common.hpp"
#include "ring_kernels.hpp"
#include "ringattr.h"

namespace {

constexpr int kAngles = 1024;      // (cos, sin) that a workgroup keeps
// Bytes that a call reads and writes from which on it leaves nothing in the last cache (256 MB) that a reader behind it would find
constexpr size_t kPastCache = 320000000;

__device__ __forceinline__ double position_of(const RingRotaryArgs& p, long at) {
  if (p.position_type == RINGATTR_POS_F32) return (double)((const float*)p.positions)[at];
  if (p.position_type == RINGATTR_POS_I32) return (double)((const int*)p.positions)[at];
  return (double)((const long long*)p.positions)[at];
}

}  // namespace

// V values at a time, neighbours in memory (V = 1: any strides and widths).  PAST: results are stored past the caches, where the call
// passes them anyway and its inputs would be pushed out (kPastCache), in rows of whole lines (16 + 4 heads of 128, bf16, halves, us with
// and without: 336 MB with inputs just written 55, 68, inputs from memory 68.4, 69.6, and a call that reads the results 135, 142; smaller,
// 252 MB: that 106, 97; rows of 128 bytes, 302 MB: 64.4, 63.1 and 130, 125).  Dropout gains nothing by it (403 and 268 MB there and back:
// 124, 120).
template <typename T, int V, bool HALF, bool PAST>
__global__ __launch_bounds__(256) void ring_rotary_kernel(RingRotaryArgs p) {
  constexpr int P = HALF ? V : (V + 1) / 2;                    // pairs of a unit
  typedef T vec __attribute__((ext_vector_type(V)));
  auto store = [](T* at, vec x) {
    if constexpr (PAST) __builtin_nontemporal_store(x, (vec*)at);
    else *(vec*)at = x;
  };
  __shared__ f32x2 trig[kAngles];
  const int tid = threadIdx.x, r = p.rot / 2, D = p.D;
  const long first = ((long)blockIdx.z * gridDim.x + blockIdx.x) * p.tokens, all = (long)p.B * p.T;
  if (first >= all) return;
  const int here = (int)(all - first < p.tokens ? all - first : p.tokens);
  for (int i = tid; i < here * r; i += 256) {
    const int tok = i / r, m = i - tok * r;
    const long b = (first + tok) / p.T, t = (first + tok) - b * p.T;
    const double pos = position_of(p, b * p.pos_b + t * p.pos_t), f = p.frequencies[m] * 0.15915494309189535;      // turns
    const double turns = rint(pos * f);
    const float x = 2.f * (float)fma(pos, f, -turns);
    float s, c;
    sincospif(x, &s, &c);
    trig[i] = f32x2{p.scale * c, p.inverse ? -p.scale * s : p.scale * s};
  }
  __syncthreads();
  // a row's units: P pairs each, then V values to copy
  const int turned = r / P, units = turned + (D - p.rot) / V;
  const int heads = p.heads[0] + p.heads[1], h0 = blockIdx.y * p.heads_per, h1 = min(heads, h0 + p.heads_per), nh = h1 - h0;
  for (int i = tid; i < here * nh * units; i += 256) {
    const int row = i / units, u = i - row * units, tok = row / nh;
    int h = h0 + row - tok * nh;
    const int which = h >= p.heads[0];
    if (which) h -= p.heads[0];
    const long b = (first + tok) / p.T, t = (first + tok) - b * p.T;
    const RingLinTensor& in = p.in[which];
    const T* x = (const T*)in.p + b * in.sb + t * in.st + h * in.sh;
    T* y = (T*)p.out[which] + ((first + tok) * p.heads[which] + h) * D;
    const f32x2* cs = trig + tok * r + u * P;
    if (u >= turned) {
      const int d = p.rot + (u - turned) * V;
      store(y + d, *(const vec*)(x + d));
    } else if constexpr (HALF) {
      const int d = u * V;
      const vec a = *(const vec*)(x + d), c = *(const vec*)(x + d + r);
      vec ya, yc;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const f32x2 w = cs[e];
        ya[e] = (T)((float)a[e] * w[0] - (float)c[e] * w[1]);
        yc[e] = (T)((float)c[e] * w[0] + (float)a[e] * w[1]);
      }
      store(y + d, ya);
      store(y + d + r, yc);
    } else {
      const int d = u * 2 * P;
      T a[2 * P];
      if constexpr (V > 1) {
        *(vec*)a = *(const vec*)(x + d);
      } else {
        a[0] = x[d];
        a[1] = x[d + 1];
      }
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const f32x2 w = cs[e];
        const float f0 = (float)a[2 * e], f1 = (float)a[2 * e + 1];
        a[2 * e] = (T)(f0 * w[0] - f1 * w[1]);
        a[2 * e + 1] = (T)(f1 * w[0] + f0 * w[1]);
      }
      if constexpr (V > 1) {
        store(y + d, *(const vec*)a);
      } else {
        y[d] = a[0];
        y[d + 1] = a[1];
      }
    }
  }
}

template <typename T> static hipError_t launch(RingRotaryArgs p, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  const int r = p.rot / 2;
  const bool vec = p.D % W == 0 && (p.interleaved ? p.rot % W == 0 : r % W == 0) && p.in[0].vec && (p.heads[1] == 0 || p.in[1].vec);
  const long all = (long)p.B * p.T;
  // As many tokens as give every lane an angle, fewer where that leaves compute units without work, then fewer heads (us, so and
  // with whole workgroups, bf16, 16 + 4 heads of 128: 64 x 1 tokens 3.0, 4.4; 100 tokens 3.0, 4.4; 1000 tokens 4.2, 5.1; 4 x 1000 8.9, 9.0).
  p.tokens = r >= 256 ? 1 : 256 / r;
  while (p.tokens > 1 && (all + p.tokens - 1) / p.tokens < 1024) p.tokens /= 2;
  const int heads = p.heads[0] + p.heads[1];
  const long blocks = (all + p.tokens - 1) / p.tokens;
  int split = blocks < 512 ? (int)(512 / blocks) : 1;
  if (split > heads) split = heads;
  p.heads_per = (heads + split - 1) / split;
  const long row = blocks < (1 << 20) ? blocks : 1 << 20;      // (a launch counts fewer than 2^32 threads along x)
  const dim3 grid((unsigned)row, (unsigned)((heads + p.heads_per - 1) / p.heads_per), (unsigned)((blocks + row - 1) / row)), block(256);
  const size_t row_bytes = p.D * sizeof(T);
  const bool past = row_bytes >= 256 && 2 * row_bytes * heads * (size_t)all >= kPastCache;
  if (p.interleaved) {
    if (vec && past) hipLaunchKernelGGL((ring_rotary_kernel<T, W, false, true>), grid, block, 0, st, p);
    else if (vec) hipLaunchKernelGGL((ring_rotary_kernel<T, W, false, false>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((ring_rotary_kernel<T, 1, false, false>), grid, block, 0, st, p);
  } else {
    if (vec && past) hipLaunchKernelGGL((ring_rotary_kernel<T, W, true, true>), grid, block, 0, st, p);
    else if (vec) hipLaunchKernelGGL((ring_rotary_kernel<T, W, true, false>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((ring_rotary_kernel<T, 1, true, false>), grid, block, 0, st, p);
  }
  return hipGetLastError();
}

hipError_t ring_launch_rotary(const RingRotaryArgs& p, int type, hipStream_t st) {
  if (type == RINGATTR_F32) return launch<float>(p, st);
  if (type == RINGATTR_BF16) return launch<__bf16>(p, st);
  return launch<_Float16>(p, st);
}
