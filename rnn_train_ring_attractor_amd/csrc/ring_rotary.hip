// Rotary positions: pair m of a head's values, (a, b), is turned by the angle position * frequency[m],
//
//   (a, b) -> scale (a cos - b sin, b cos + a sin),
//
// pairs being halves apart (m, m + rot / 2) or neighbours (2m, 2m + 1); what lies behind the first `rot` values of a head is copied.
// Backwards the same with the opposite angle.  A position is a count of tokens or an angle of its own (a heading; the pairs then turn
// with its harmonics).
//
// Bound by memory: everything is read once and written once: 8 x 4096 tokens, 16 + 4 heads of 128, bf16: 336 MB in 67 us, 5.0 TB/s (a
// large copy: 5.2).  A workgroup takes a few tokens through all heads of both tensors, so a
// token's angles are found once: the number of turns without its whole part, exact to 2^-40 for every 64-bit position (at position 2^20 a product
// in 32 bits is off by 0.06 rad, at 2^40 one in 64 bits by 2e-4), then one sine and cosine in 32.
#include "ring_common.hpp"
#include "ring_kernels.hpp"
#include "ringattr.h"

namespace {

constexpr int kAngles = 1024;      // (cos, sin) that a workgroup keeps
constexpr int kTokens = 256;       // tokens that a workgroup takes at most

// n / d for n < 2^31 by a product and a shift: with 2^(s - 1) < d <= 2^s, floor(n (2^32 + m) / 2^(32 + s)) for m = floor(2^32 (2^s - d) / d) + 1
// (the excess of (2^32 + m) / 2^(32 + s) over 1 / d is at most 2^-(32 + s), which n < 2^31 does not carry past a whole number).  Divisions
// as such were most of the time of odd widths (the case below of 52 turned 308 us, 213 with products, one value at a time each).
struct Divisor {
  unsigned m, s;
  static Divisor of(unsigned d) {
    unsigned s = 0;
    while ((1ull << s) < d) ++s;
    return Divisor{(unsigned)((((1ull << s) - d) << 32) / d + 1), s};
  }
  __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, m) + n) >> s; }
};
struct Divisors { Divisor units, heads, pairs, T, last_heads; };

// A position as the sum of two numbers in 64 bits, both exact
struct Position { double high, low; };
__device__ __forceinline__ Position position_of(const RingRotaryArgs& p, long at) {
  if (p.position_type == RINGATTR_POS_F32) return {0.0, (double)((const float*)p.positions)[at]};
  if (p.position_type == RINGATTR_POS_I32) return {0.0, (double)((const int*)p.positions)[at]};
  const long long x = ((const long long*)p.positions)[at];
  return {(double)(int)(x >> 32) * 4294967296.0, (double)(unsigned)x};
}

// position * frequency / (2 pi) less whole turns.  frequency / (2 pi) = f + g with 106 bits; of the products with f whole turns are taken off
// inside the fma, ahead of its rounding.
__device__ __forceinline__ float turns(Position x, double frequency) {
  constexpr double R = 0.15915494309189535, S = -9.839338337591243e-18;          // 1 / (2 pi) = R + S
  const double f = frequency * R, g = fma(frequency, R, -f) + frequency * S;
  const double t = fma(x.high, f, -rint(x.high * f)) + fma(x.low, f, -rint(x.low * f)) + fma(x.high, g, x.low * g);
  return (float)(t - rint(t));
}

}  // namespace

// V values at a time, neighbours in memory: 16 bytes, two values, or one (any strides and widths); what is copied C at a time.
// (Results stored past the caches: 68.4 us in place of 69.6 for 336 MB from memory, 106 in place of 97 for 252 MB with a reader behind it: not done.)
template <typename T, int V, int C, bool HALF>
__global__ __launch_bounds__(256) void ring_rotary_kernel(RingRotaryArgs p, Divisors by) {
  constexpr int P = HALF ? V : (V + 1) / 2;                    // pairs of a unit
  typedef T vec __attribute__((ext_vector_type(V)));
  typedef T copied __attribute__((ext_vector_type(C)));
  __shared__ f32x2 trig[kAngles];
  __shared__ long base[2][kTokens];
  const int tid = threadIdx.x, r = p.rot / 2, D = p.D;
  const long first = ((long)blockIdx.z * gridDim.x + blockIdx.x) * p.tokens, all = (long)p.B * p.T;
  if (first >= all) return;
  const int here = (int)(all - first < p.tokens ? all - first : p.tokens);
  const unsigned b0 = (unsigned)first / (unsigned)p.T, t0 = (unsigned)first - b0 * (unsigned)p.T;
  if (tid < here) {
    const unsigned more = by.T.div(t0 + tid);
    const long b = b0 + more, t = t0 + tid - more * (unsigned)p.T;
    base[0][tid] = b * p.in[0].sb + t * p.in[0].st;
    base[1][tid] = b * p.in[1].sb + t * p.in[1].st;
  }
  for (int i = tid; i < here * r; i += 256) {
    const int tok = by.pairs.div(i), m = i - tok * r;
    const unsigned more = by.T.div(t0 + tok);
    const long b = b0 + more, t = t0 + tok - more * (unsigned)p.T;
    float s, c;
    sincospif(2.f * turns(position_of(p, b * p.pos_b + t * p.pos_t), p.frequencies[m]), &s, &c);
    trig[i] = f32x2{p.scale * c, p.inverse ? -p.scale * s : p.scale * s};
  }
  __syncthreads();
  // a row's units: P pairs each, then C values to copy
  const int turned = r / P, units = turned + (D - p.rot) / C;
  const int heads = p.heads[0] + p.heads[1], h0 = blockIdx.y * p.heads_per, h1 = min(heads, h0 + p.heads_per), nh = h1 - h0;
  for (int i = tid; i < here * nh * units; i += 256) {
    const int row = by.units.div(i), u = i - row * units, tok = (blockIdx.y + 1 == gridDim.y ? by.last_heads : by.heads).div(row);
    int h = h0 + row - tok * nh;
    const int which = h >= p.heads[0];
    if (which) h -= p.heads[0];
    const RingLinTensor& in = p.in[which];
    const T* x = (const T*)in.p + base[which][tok] + h * in.sh;
    T* y = (T*)p.out[which] + ((first + tok) * p.heads[which] + h) * D;
    const f32x2* cs = trig + tok * r + u * P;
    if (u >= turned) {
      const int d = p.rot + (u - turned) * C;
      *(copied*)(y + d) = *(const copied*)(x + d);
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
      *(vec*)(y + d) = ya;
      *(vec*)(y + d + r) = yc;
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
        *(vec*)(y + d) = *(const vec*)a;
      } else {
        y[d] = a[0];
        y[d + 1] = a[1];
      }
    }
  }
}

// The largest of 16 bytes, two values and one that rows, pairs (halves: r, else all that is turned) and addresses are whole numbers of (us,
// 8 x 4096 tokens, 16 + 4 heads of 128, bf16, halves: 64 turned 68; 52 turned, by two values 127, by one 213; 50 turned, by one and what is copied
// by two 158; heads of 127 215).
template <typename T> static int values_at_once(const RingRotaryArgs& p, int pairs) {
  for (int v = 16 / sizeof(T); v > 1; v = v > 2 ? 2 : 1) {
    bool fits = p.D % v == 0 && pairs % v == 0;
    for (int i = 0; i < (p.heads[1] ? 2 : 1); ++i)
      fits = fits && p.in[i].sb % v == 0 && p.in[i].st % v == 0 && p.in[i].sh % v == 0 &&
             (reinterpret_cast<uintptr_t>(p.in[i].p) | reinterpret_cast<uintptr_t>(p.out[i])) % (v * sizeof(T)) == 0;
    if (fits) return v;
  }
  return 1;
}

template <typename T, int V, int C> static void launch_kernel(const RingRotaryArgs& p, dim3 grid, hipStream_t st) {
  const int r = p.rot / 2, pairs = p.interleaved ? (V + 1) / 2 : V;
  // (the last heads of a grid row are fewer: their workgroups divide by their own number)
  const int heads = p.heads[0] + p.heads[1], units = r / pairs + (p.D - p.rot) / C, last = heads - ((int)grid.y - 1) * p.heads_per;
  const Divisors by = {Divisor::of(units), Divisor::of(p.heads_per), Divisor::of(r), Divisor::of(p.T), Divisor::of(last)};
  if constexpr (V == C) {                                      // (neighbours: where two values fit, a pair does)
    if (p.interleaved) {
      hipLaunchKernelGGL((ring_rotary_kernel<T, V, C, false>), grid, dim3(256), 0, st, p, by);
      return;
    }
  }
  hipLaunchKernelGGL((ring_rotary_kernel<T, V, C, true>), grid, dim3(256), 0, st, p, by);
}

template <typename T> static hipError_t launch(RingRotaryArgs p, hipStream_t st) {
  constexpr int W = 16 / sizeof(T);
  const int r = p.rot / 2, v = values_at_once<T>(p, p.interleaved ? p.rot : r), c = v > 1 ? v : values_at_once<T>(p, 2);
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
  const dim3 grid((unsigned)row, (unsigned)((heads + p.heads_per - 1) / p.heads_per), (unsigned)((blocks + row - 1) / row));
  if (v == W) launch_kernel<T, W, W>(p, grid, st);
  else if (v == 2) launch_kernel<T, 2, 2>(p, grid, st);
  else if (c == 2) launch_kernel<T, 1, 2>(p, grid, st);
  else launch_kernel<T, 1, 1>(p, grid, st);
  return hipGetLastError();
}

hipError_t ring_launch_rotary(const RingRotaryArgs& p, int type, hipStream_t st) {
  if (type == RINGATTR_F32) return launch<float>(p, st);
  if (type == RINGATTR_BF16) return launch<__bf16>(p, st);
  return launch<_Float16>(p, st);
}
