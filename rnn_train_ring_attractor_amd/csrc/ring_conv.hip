// Short causal convolution: a channel by itself, K taps up to 8,
//
//   p_t = bias + sum_k w[k] x_(t - K + 1 + k),  y_t = act(p_t);  the K - 1 inputs in front of a sequence are its state.
//
// Backwards, g_t = dy_t act'(p_t): dx_t = sum_k w[k] g_(t + K - 1 - k), dw[k] = sum_t g_t x_(t - K + 1 + k), dbias = sum_t g_t; p is found again from x.
//
// Bound by memory: rows are read once and written once (the K - 1 tokens that a piece of a sequence shares with the next one a second time, from
// L2).  A thread takes four channels (one where rows are not whole numbers of four) through a piece's tokens, the next ones on their way; inputs and
// gradients that later tokens need stay in registers.  (Eight channels of 16 bits, 16 bytes a lane, take 256 registers backwards: 188 us in place of 181, and forwards
// no less.)
#include "ring_recur.hpp"
#include "ringattr.h"

#include <type_traits>

using namespace ring_recur;

namespace {

enum { kIdentity = 0, kSilu = 1 };

struct Piece { int b, seg, c, first, last, sub; bool mine; };

// `tx` threads along the channels, the workgroup's others take pieces of p.seg_tokens tokens behind one another
template <int E> __device__ __forceinline__ Piece piece(const RingConvArgs& p, int tx, int blocks) {
  unsigned i = blockIdx.x;
  const int cb = (int)(i % blocks);
  i /= blocks;
  const int seg = (int)(i % p.nseg), b = (int)(i / p.nseg), lane = threadIdx.x & (tx - 1), sub = threadIdx.x / tx;
  const int c = (cb * tx + lane) * E;
  const long first = ((long)seg * (256 / tx) + sub) * p.seg_tokens;
  return {b, seg, c, (int)(first < p.T ? first : p.T), (int)(first + p.seg_tokens < p.T ? first + p.seg_tokens : p.T), sub, c < p.C};
}

}  // namespace

// (E > 1: rows are whole numbers of E channels, which are all there)
template <int E> constexpr bool kWide = E > 1;

// KT taps are built for; K < KT (only where KT = 8): the first KT - K are left out.  8 x 4096 tokens of 4096 channels, 4 taps, silu, bf16: 97 us, 537 MB at 5.5 TB/s;
// fp32 of 7 x 1001 of 515, one channel a thread, 8.
template <typename T, int E, int KT, int U>      // U tokens at a time
__global__ __launch_bounds__(256) void ring_conv_fwd_kernel(RingConvArgs p, int tx, int blocks) {
  const Piece a = piece<E>(p, tx, blocks);
  if (!a.mine) return;
  const int K = KT == 8 ? p.K : KT, skip = KT - K, len = length_of(p.lengths, a.b, p.T), end = min(a.last, len);
  float w[KT][E], bias[E], win[KT - 1 + U][E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    bias[e] = p.bias ? p.bias[a.c + e] : 0.f;
#pragma unroll
    for (int k = 0; k < KT; ++k) w[k][e] = k >= skip ? p.w[(size_t)(a.c + e) * K + k - skip] : 0.f;
  }
  const T* const x = (const T*)p.x.p + a.b * p.x.sb + a.c;
  const T* const start = p.start ? (const T*)p.start + (size_t)a.b * (K - 1) * p.C + a.c : nullptr;
  T* const y = (T*)p.y + (size_t)a.b * p.T * p.C + a.c;
  auto input = [&](int t) {              // x at t, or the state's where that is in front of the sequence
    Row<T, E> r;
    r.zero();
    if (t >= 0) r.load(x + t * p.x.st, kWide<E>, E);
    else if (start && t >= -(K - 1)) r.load(start + (size_t)(t + K - 1) * p.C, kWide<E>, E);
    return r;
  };
  if (a.seg == 0 && a.sub == 0 && p.end)
    for (int j = 0; j < K - 1; ++j) input(len - (K - 1) + j).store((T*)p.end + ((size_t)a.b * (K - 1) + j) * p.C + a.c, kWide<E>, E);
  if (a.first < end) {
#pragma unroll
    for (int j = 0; j < KT - 1; ++j) {
      const Row<T, E> r = input(a.first - (KT - 1) + j);
#pragma unroll
      for (int e = 0; e < E; ++e) win[j][e] = j >= skip ? (float)r.v[e] : 0.f;
    }
    Row<T, E> next[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      next[i].zero();
      if (a.first + i < end) next[i].load(x + (a.first + i) * p.x.st, kWide<E>, E);
    }
    const T* xp = x + (a.first + U) * p.x.st;
    T* yp = y + (size_t)a.first * p.C;
    auto tokens = [&](int t, auto inner) {       // inner: these tokens and the next ones are all there
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) win[KT - 1 + i][e] = (float)next[i].v[e];
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (decltype(inner)::value || t + U + i < end) next[i].load(xp + i * p.x.st, kWide<E>, E);
      xp += U * p.x.st;
      float s[U][E];
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e) s[i][e] = bias[e];
#pragma unroll
      for (int k = 0; k < KT; ++k)
        if (KT < 8 || k >= skip)
#pragma unroll
          for (int i = 0; i < U; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) s[i][e] = fmaf(w[k][e], win[i + k][e], s[i][e]);
      if (p.act == kSilu)
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
          for (int e = 0; e < E; ++e) s[i][e] = silu<sizeof(T) == 4>(s[i][e]);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        Row<T, E> out;
#pragma unroll
        for (int e = 0; e < E; ++e) out.v[e] = (T)s[i][e];
        if (decltype(inner)::value || t + i < end) out.store(yp + (size_t)i * p.C, kWide<E>, E);
      }
      yp += (size_t)U * p.C;
#pragma unroll
      for (int j = 0; j < KT - 1; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) win[j][e] = win[j + U][e];
    };
    int t = a.first;
    for (; t + 2 * U <= end; t += U) tokens(t, std::true_type{});
    for (; t < end; t += U) tokens(t, std::false_type{});
  }
  Row<T, E> none;                        // tokens that do not count
  none.zero();
  for (int t = max(a.first, end); t < a.last; ++t) none.store(y + (size_t)t * p.C, kWide<E>, E);
}

// A token at a time, its input and gradient read KT tokens (or more) ahead.  Inputs and gradients of the last KT tokens go round in registers: a piece's token t is in
// place t % KT, and so many tokens follow each other without a loop between them that places are known.  Bound by memory, in part by its
// latency: 8 x 4096 tokens of 4096 channels, 4 taps, silu, bf16: 181 us, 805 MB at 4.5 TB/s (18 more with windows that move up by one a token).
template <typename T, int E, int KT, bool SILU>
__global__ __launch_bounds__(256) void ring_conv_bwd_kernel(RingConvArgs p, int tx, int blocks) {
  constexpr int N = KT == 2 ? 4 : KT;    // tokens that follow each other
  __shared__ float sums[256 * E];
  const Piece a = piece<E>(p, tx, blocks);
  const int K = KT == 8 ? p.K : KT, skip = KT - K, len = length_of(p.lengths, a.b, p.T);
  float w[KT][E], bias[E], dw[KT][E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    bias[e] = p.bias && a.mine ? p.bias[a.c + e] : 0.f;
    db[e] = 0.f;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      w[k][e] = k >= skip && a.mine ? p.w[(size_t)(a.c + e) * K + k - skip] : 0.f;
      dw[k][e] = 0.f;
    }
  }
  if (a.mine) {
    float win[KT][E], g[KT][E];
    const T* const x = (const T*)p.x.p + a.b * p.x.sb + a.c;
    const T* const dy = (const T*)p.dy.p + a.b * p.dy.sb + a.c;
    const size_t state = (size_t)a.b * (K - 1) * p.C + a.c;
    const T* const start = p.start ? (const T*)p.start + state : nullptr;
    const T* const dend = p.dend ? (const T*)p.dend + state : nullptr;
    T* const dx = p.dx ? (T*)p.dx + (size_t)a.b * p.T * p.C + a.c : nullptr;
    T* const dstart = p.dstart ? (T*)p.dstart + state : nullptr;
#pragma unroll
    for (int j = 0; j < KT; ++j) {       // (place j has token j - KT of the piece)
      const int t = a.first - KT + j;
      Row<T, E> r;
      r.zero();
      if (j > 0 && a.first < len) {
        if (t >= 0) r.load(x + t * p.x.st, kWide<E>, E);
        else if (start && t >= -(K - 1)) r.load(start + (size_t)(t + K - 1) * p.C, kWide<E>, E);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        win[j][e] = (float)r.v[e];
        g[j][e] = 0.f;
      }
    }
    Row<T, E> nx[N], ny[N];
    // gradients of the piece's tokens, then those behind it that its last inputs take part in
    const int to = a.first < a.last || (a.first == 0 && a.sub == 0 && a.seg == 0) ? a.last + KT - 1 : a.first, full = min(a.last, len);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      nx[i].zero(), ny[i].zero();
      const int t = a.first + i;
      if (t < min(to, len)) {
        nx[i].load(x + t * p.x.st, kWide<E>, E);
        ny[i].load(dy + t * p.dy.st, kWide<E>, E);
      }
    }
    const T *xp = x + (a.first + N) * p.x.st, *yp = dy + (a.first + N) * p.dy.st;
    T* dxp = dx + (long)(a.first - KT + 1) * p.C;       // (of token t - KT + 1; used where that is one)
    auto tokens = [&](int t, auto inner) {       // inner: these tokens count in the sums, the next ones are there, gradients are complete and of the piece
      constexpr bool IN = decltype(inner)::value;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        constexpr int M = KT;
        const int s = t + i, back = s - KT + 1, at = i % M;
        const bool counts = IN || s < len;
        float q[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          win[at][e] = (float)nx[i].v[e];
          g[at][e] = (float)ny[i].v[e];
          q[e] = bias[e];
        }
        if (IN || s + N < min(to, len)) {
          nx[i].load(xp, kWide<E>, E);
          ny[i].load(yp, kWide<E>, E);
        }
        xp += p.x.st;
        yp += p.dy.st;
        if (SILU) {
#pragma unroll
          for (int k = 0; k < KT; ++k)
            if (KT < 8 || k >= skip)
#pragma unroll
              for (int e = 0; e < E; ++e) q[e] = fmaf(w[k][e], win[(at + 1 + k) % M][e], q[e]);
#pragma unroll
          for (int e = 0; e < E; ++e) g[at][e] *= silu_slope(q[e], sigmoid<sizeof(T) == 4>(q[e]));
        }
        if (!IN)
#pragma unroll
          for (int e = 0; e < E; ++e) g[at][e] = counts ? g[at][e] : 0.f;
        if (IN || (s < a.last && counts)) {
#pragma unroll
          for (int e = 0; e < E; ++e) db[e] += g[at][e];
#pragma unroll
          for (int k = 0; k < KT; ++k)
            if (KT < 8 || k >= skip)
#pragma unroll
              for (int e = 0; e < E; ++e) dw[k][e] = fmaf(g[at][e], win[(at + 1 + k) % M][e], dw[k][e]);
        }
        T* row = nullptr;
        if (IN || (back >= a.first && back < a.last)) row = dx ? dxp : nullptr;
        else if (back < 0 && back >= -(K - 1) && s < to && dstart) row = dstart + (size_t)(back + K - 1) * p.C;
        dxp += p.C;
        if (row) {
          Row<T, E> out, more;
          more.zero();
          if (!IN && dend && back < len && back >= len - (K - 1)) more.load(dend + (size_t)(back - len + K - 1) * p.C, kWide<E>, E);
          float v[E];
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = IN ? 0.f : (float)more.v[e];
#pragma unroll
          for (int k = 0; k < KT; ++k)
            if (KT < 8 || k >= skip)
#pragma unroll
              for (int e = 0; e < E; ++e) v[e] = fmaf(w[k][e], g[(at + M - k) % M][e], v[e]);
#pragma unroll
          for (int e = 0; e < E; ++e) out.v[e] = (T)(IN || back < len ? v[e] : 0.f);
          out.store(row, kWide<E>, E);
        }
      }
    };
    int t = a.first;
    for (; t < min(to, a.first + KT - 1); t += N) tokens(t, std::false_type{});
    for (; t + 2 * N <= full; t += N) tokens(t, std::true_type{});
    for (; t < to; t += N) tokens(t, std::false_type{});
  }
  if (!p.part) return;
  // the workgroup's pieces, in order
  const int subs = 256 / tx;
  float* const part = p.part + ((size_t)(a.b * p.nseg + a.seg) * p.C + a.c) * (K + 1);
#pragma unroll
  for (int k = 0; k <= KT; ++k) {
    if (k < skip) continue;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) sums[e * 256 + threadIdx.x] = k < KT ? dw[k < KT ? k : 0][e] : db[e];
    __syncthreads();
    if (a.mine && a.sub == 0)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float s = 0.f;
        for (int i = 0; i < subs; ++i) s += sums[e * 256 + i * tx + threadIdx.x];
        part[(size_t)e * (K + 1) + k - skip] = s;
      }
  }
}

// A single token: the state's rows move up by one.  64 sequences of 2048 channels: 5 us, a launch and one read behind another.
template <typename T, int E>
__global__ __launch_bounds__(64) void ring_conv_step_kernel(RingConvStep p, int blocks, bool wide) {
  const int b = (int)(blockIdx.x / blocks), c = (int)(blockIdx.x % blocks * 64 + threadIdx.x) * E, here = p.C - c;
  if (here <= 0) return;
  Row<T, E> out;
  out.zero();
  T* const y = (T*)p.y + (size_t)b * p.C + c;
  if (p.active && !p.active[b]) {
    out.store(y, wide, here);
    return;
  }
  T* const state = (T*)p.state + (size_t)b * (p.K - 1) * p.C + c;
  Row<T, E> row[8];
#pragma unroll
  for (int k = 0; k < 7; ++k)
    if (k < p.K - 1) row[k].load(state + (size_t)k * p.C, wide, here);
  Row<T, E> x;
  x.load((const T*)p.x + b * p.xs + c, wide, here);
  float s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = p.bias && e < here ? p.bias[c + e] : 0.f;
#pragma unroll
  for (int k = 0; k < 7; ++k)
    if (k < p.K - 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] = fmaf(e < here ? p.w[(size_t)(c + e) * p.K + k] : 0.f, (float)row[k].v[e], s[e]);
      if (k > 0) row[k].store(state + (size_t)(k - 1) * p.C, wide, here);
    }
  if (p.K > 1) x.store(state + (size_t)(p.K - 2) * p.C, wide, here);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s[e] = fmaf(e < here ? p.w[(size_t)(c + e) * p.K + p.K - 1] : 0.f, (float)x.v[e], s[e]);
    out.v[e] = (T)(p.act == kSilu ? silu<sizeof(T) == 4>(s[e]) : s[e]);
  }
  out.store(y, wide, here);
}

static int along(int C, int E) {         // threads along the channels
  int tx = 1;
  while (tx < 64 && tx * E < C) tx *= 2;
  return tx;
}

// Pieces are long beside the K - 1 tokens that they share, up to 256, and short enough that every compute unit has two workgroups (8 x 4096 tokens, 4096 channels,
// 4 taps, bf16, us forwards and with gradients by a piece's tokens: 64 111, 310; 128 103, 292; 256 102, 282; 512 102, 318).
static void cut(RingConvArgs& p, int tx, int blocks) {
  const int subs = 256 / tx;
  p.seg_tokens = 256;
  while (p.seg_tokens > 8 && (long)p.B * blocks * ((p.T + (long)subs * p.seg_tokens - 1) / ((long)subs * p.seg_tokens)) < 512) p.seg_tokens /= 2;
  p.nseg = (int)((p.T + (long)subs * p.seg_tokens - 1) / ((long)subs * p.seg_tokens));
  if (p.nseg < 1) p.nseg = 1;
}

template <typename T, int E> static hipError_t launch(RingConvArgs p, bool back, hipStream_t st) {
  const int tx = along(p.C, E), blocks = (p.C + tx * E - 1) / (tx * E);
  cut(p, tx, blocks);
  const dim3 grid((unsigned)((size_t)blocks * p.nseg * p.B)), block(256);
#define RING_CONV(KT)                                                                             \
  if (back && p.act == kSilu) hipLaunchKernelGGL((ring_conv_bwd_kernel<T, E, KT, true>), grid, block, 0, st, p, tx, blocks); \
  else if (back) hipLaunchKernelGGL((ring_conv_bwd_kernel<T, E, KT, false>), grid, block, 0, st, p, tx, blocks); \
  else hipLaunchKernelGGL((ring_conv_fwd_kernel<T, E, KT, (E > 1 ? 8 : 4)>), grid, block, 0, st, p, tx, blocks)
  if (p.K == 2) { RING_CONV(2); }
  else if (p.K == 3) { RING_CONV(3); }
  else if (p.K == 4) { RING_CONV(4); }
  else { RING_CONV(8); }
#undef RING_CONV
  return hipGetLastError();
}

template <typename T> static hipError_t launch_wide(const RingConvArgs& p, bool back, hipStream_t st) {
  return p.wide && p.wide_out && p.wide_state ? launch<T, 4>(p, back, st) : launch<T, 1>(p, back, st);
}

static hipError_t launch_type(const RingConvArgs& p, int type, bool back, hipStream_t st) {
  if (type == RINGATTR_F32) return launch_wide<float>(p, back, st);
  if (type == RINGATTR_BF16) return launch_wide<__bf16>(p, back, st);
  return launch_wide<_Float16>(p, back, st);
}

// (of rows read four channels at a time and one; either may be more)
static int parts_of(int B, int T, int C, bool wide) {
  const int E = wide ? 4 : 1, tx = along(C, E), blocks = (C + tx * E - 1) / (tx * E);
  RingConvArgs p = {};
  p.B = B;
  p.T = T;
  p.C = C;
  cut(p, tx, blocks);
  return p.nseg * B;
}

size_t ring_conv_bwd_bytes(int B, int T, int C, int K, bool params) {
  if (!params) return 0;
  const int a = parts_of(B, T, C, true), b = parts_of(B, T, C, false);
  return (size_t)(a > b ? a : b) * C * (K + 1) * sizeof(float);
}

hipError_t ring_conv_fwd(RingConvArgs p, int type, hipStream_t st) { return launch_type(p, type, false, st); }

hipError_t ring_conv_bwd(RingConvArgs p, int type, hipStream_t st) {
  hipError_t e = launch_type(p, type, true, st);
  if (e != hipSuccess || !p.part) return e;
  return ring_launch_sum_parts(RingSumArgs{p.part, parts_of(p.B, p.T, p.C, p.wide && p.wide_out && p.wide_state), p.K + 1, p.K, 1,
                                           (size_t)p.C * (p.K + 1), p.dw, {p.dbias, nullptr}}, st);
}

template <typename T> static hipError_t launch_step(const RingConvStep& p, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = p.C % V == 0 && p.xs % V == 0 &&
                    ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.state) | reinterpret_cast<uintptr_t>(p.y)) & 15) == 0;
  const int E = wide ? V : 1, blocks = (p.C + 64 * E - 1) / (64 * E);
  const dim3 grid((unsigned)((size_t)blocks * p.B)), block(64);
  if (wide) hipLaunchKernelGGL((ring_conv_step_kernel<T, V>), grid, block, 0, st, p, blocks, true);
  else hipLaunchKernelGGL((ring_conv_step_kernel<T, 1>), grid, block, 0, st, p, blocks, false);
  return hipGetLastError();
}

hipError_t ring_conv_step(const RingConvStep& p, int type, hipStream_t st) {
  if (type == RINGATTR_F32) return launch_step<float>(p, st);
  if (type == RINGATTR_BF16) return launch_step<__bf16>(p, st);
  return launch_step<_Float16>(p, st);
}
