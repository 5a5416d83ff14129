// What stands around a block: its output normalised, gated and added to the residual stream, which the next block's norm then reads,
//
//   unit = (x - mean) rstd over each group of neighbouring values (kind rms: without the mean),  rstd = (mean of squares + eps)^-1/2,
//   y = residual + scale unit w act(gate),   n = unit(y) next over the whole row.
//
// Backwards, t = dy + what n gives back: dresidual = t, dgate = t scale unit w act'(gate), d unit = t scale act(gate) w, dx = rstd (d unit - mean(d unit)
// - unit mean(d unit unit)); the weights' gradients are sums over rows.  Units and y are found again from what was read.
//
// Bound by memory: every tensor is read once or written once.  A row lies in the registers of one workgroup (several rows, where they are short);
// backwards a workgroup walks rows and keeps the sums of its columns until it is done.  Rounded are what is written, once each; sums, units and statistics are fp32.
#pragma once
#include "ring_recur.hpp"
#include "ringattr.h"

namespace ring_norm {

using namespace ring_recur;

enum { kIdentity = 0, kSilu = 1, kSigmoid = 2 };

// How a row lies on threads: groups of `lanes` threads (a power of two), `slots` groups side by side (a power of two), `rows` rows a workgroup.  MANY: a thread
// holds one unit of V values of each of I groups, else I units of one group.
struct Lie { int lanes, slots, rows, groups; };

// Sums of K values over `n` neighbouring threads, a power of two, the same in each.  Across waves through one of two rooms by turns: who writes into a room
// for the next but one sum has passed the barrier of the next one, which nobody reaches before this one is read.
struct Room {
  float* at;
  int turn;
};
constexpr int kRoom = 2 * 32;
template <int K> __device__ __forceinline__ void add_up(float (&v)[K], int n, Room& room) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (n > 1) v[k] = plus_dpp<kXor1>(v[k]);
    if (n > 2) v[k] = plus_dpp<kXor2>(v[k]);
    if (n > 4) v[k] = plus_dpp<0x141>(v[k]);        // mirrored within 8, 16: whole quads, whole eights
    if (n > 8) v[k] = plus_dpp<0x140>(v[k]);
    if (n > 16) v[k] = fold16(v[k], v[k]);
    if (n > 32) v[k] = fold32(v[k], v[k]);
  }
  if constexpr (K <= 2) {
    if (n > 64) {
      float* const at = room.at + room.turn * 32;
      const int w = threadIdx.x >> 6, per = n >> 6;
      room.turn ^= 1;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) at[k * 16 + w] = v[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
        v[k] = at[k * 16 + (w & -per) + (threadIdx.x & (per - 1))];
        v[k] = plus_dpp<kXor1>(v[k]);
        if (per > 2) v[k] = plus_dpp<kXor2>(v[k]);
        if (per > 4) v[k] = plus_dpp<0x141>(v[k]);
        if (per > 8) v[k] = plus_dpp<0x140>(v[k]);
      }
    }
  }
}

// Of a gate by itself NaN stays NaN, which FINE's clamped argument loses (silu multiplies by it besides)
template <bool FINE> __device__ __forceinline__ float gate_sigmoid(float x) {
  const float s = sigmoid<FINE>(x);
  return FINE && x != x ? x : s;
}

// v times act(gate)
template <typename T, int V> __device__ __forceinline__ void gate_of(float (&v)[V], const Row<T, V>& g, int act) {
  if (act == kSilu) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= silu<sizeof(T) == 4>((float)g.v[e]);
  } else if (act == kSigmoid) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= gate_sigmoid<sizeof(T) == 4>((float)g.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] *= (float)g.v[e];
  }
}

// A thread's place in a row
template <int V, int I, bool MANY> struct Spot {
  int lane, slot, row, threads;
  __device__ __forceinline__ Spot(const Lie& l) {
    threads = l.lanes * l.slots;
    lane = threadIdx.x & (l.lanes - 1);
    slot = threadIdx.x / l.lanes & (l.slots - 1);
    row = threadIdx.x / threads;
  }
  __device__ __forceinline__ int column(const Lie& l, int i, int group) const {
    const int g = MANY ? i * l.slots + slot : slot, u = MANY ? lane : i * l.lanes + lane;
    return g * group + u * V;
  }
  __device__ __forceinline__ bool there(const Lie& l, int i, int group) const {      // whether unit i is (groups are whole numbers of units)
    const int g = MANY ? i * l.slots + slot : slot, u = MANY ? lane : i * l.lanes + lane;
    return g < l.groups && u * V < group;
  }
};

// sums[i] += the sum over its group of the thread's values of unit i
template <int V, int I, bool MANY> __device__ __forceinline__ void group_sums(float (&sums)[I], const Lie& l, Room& room) {
  if constexpr (MANY) {
    add_up<I>(sums, l.lanes, room);      // (at most 64 lanes)
  } else {
    float one[1] = {sums[0]};
#pragma unroll
    for (int i = 1; i < I; ++i) one[0] += sums[i];
    add_up<1>(one, l.lanes, room);
#pragma unroll
    for (int i = 0; i < I; ++i) sums[i] = one[0];
  }
}

// v becomes (v - mean) over its groups, rstd beside it (zero where a unit is not there: what follows from it is zero then, whatever eps is); `each` is one
// over the values of a group
template <int V, int I, bool MANY>
__device__ __forceinline__ void normalise(float (&v)[I][V], float (&rstd)[I], const bool (&there)[I], const Lie& l, float each, bool layer, float eps, Room& room) {
  float s[I];
  if (layer) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      s[i] = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) s[i] += v[i][e];
    }
    group_sums<V, I, MANY>(s, l, room);
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) v[i][e] = there[i] ? v[i][e] - s[i] * each : 0.f;
  }
#pragma unroll
  for (int i = 0; i < I; ++i) {
    s[i] = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) s[i] = fmaf(v[i][e], v[i][e], s[i]);
  }
  group_sums<V, I, MANY>(s, l, room);
#pragma unroll
  for (int i = 0; i < I; ++i) rstd[i] = there[i] ? __builtin_amdgcn_rsqf(fmaf(s[i], each, eps)) : 0.f;
}

// 32768 rows of 2048, bf16, gate, residual, scale and next norm: 131 us, 671 MB at 5.1 TB/s, which is a copy's; 64 rows 4 us, a launch.
template <typename T, int V, int I, bool MANY>
__global__ __launch_bounds__(1024) void ring_norm_fwd_kernel(RingNormArgs p, Lie l) {
  __shared__ float rooms[kRoom];
  Room room = {rooms, 0};
  const Spot<V, I, MANY> at(l);
  const Lie whole = {at.threads, 1, l.rows, 1};
  const long row = ((long)blockIdx.y * gridDim.x + blockIdx.x) * l.rows + at.row;
  const bool real = row < p.rows;
  bool there[I];
  int col[I];
  float v[I][V], rstd[I];
  Row<T, V> rx[I], rg[I], rr[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    there[i] = real && at.there(l, i, p.group);
    col[i] = at.column(l, i, p.group);
    rx[i].zero(), rg[i].zero(), rr[i].zero();
    if (there[i]) {
      rx[i].load((const T*)p.x + row * p.xs + col[i], V > 1, V);
      if (p.gate) rg[i].load((const T*)p.gate + row * p.gs + col[i], V > 1, V);
      if (p.residual) rr[i].load((const T*)p.residual + row * p.rs + col[i], V > 1, V);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) v[i][e] = (float)rx[i].v[e];
  }
  normalise<V, I, MANY>(v, rstd, there, l, p.each, p.layer, p.eps, room);
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (there[i]) {
      Row<T, V> out;
      Row<float, V> w;
      w.load(p.w + col[i], V > 1, V);
#pragma unroll
      for (int e = 0; e < V; ++e) v[i][e] *= rstd[i] * w.v[e];
      if (p.gate) gate_of<T, V>(v[i], rg[i], p.act);
      if (p.scale) {
        w.load(p.scale + col[i], V > 1, V);
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] *= w.v[e];
      }
      if (p.residual)
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] += (float)rr[i].v[e];
#pragma unroll
      for (int e = 0; e < V; ++e) out.v[e] = (T)v[i][e];
      out.store((T*)p.y + row * p.C + col[i], V > 1, V);
    }
  if (!p.next) return;
  normalise<V, I, false>(v, rstd, there, whole, p.each_row, p.layer, p.eps, room);
#pragma unroll
  for (int i = 0; i < I; ++i)
    if (there[i]) {
      Row<T, V> out;
      Row<float, V> w;
      w.load(p.next + col[i], V > 1, V);
#pragma unroll
      for (int e = 0; e < V; ++e) out.v[e] = (T)(v[i][e] * rstd[i] * w.v[e]);
      out.store((T*)p.n + row * p.C + col[i], V > 1, V);
    }
}

// MOST threads a workgroup.  Up to 512 of eight values each keep the weights and read the next row ahead; others have no registers left for that.  32768 rows of
// 2048, bf16, all of it: 202 us, 1074 MB at 5.3 TB/s, a copy's (240 with sums across waves by a loop over them, which also made the code three times as long).
template <typename T, int V, int I, bool MANY, int MOST>
__global__ __launch_bounds__(MOST) void ring_norm_bwd_kernel(RingNormArgs p, Lie l) {
  constexpr bool KEEP = MOST <= 512 && I * V <= 8, FINE = sizeof(T) == 4;
  __shared__ float rooms[kRoom];
  Room room = {rooms, 0};
  extern __shared__ float sums[];        // [threads][V]: rows of a workgroup are added up
  const Spot<V, I, MANY> at(l);
  const Lie whole = {at.threads, 1, l.rows, 1};
  struct Unit { Row<T, V> x, g, r, t, n; };          // of the row: x, gate, residual, gradients of y and n
  struct Weights { Row<float, V> w, s, n; } kept[KEEP ? I : 1];
  Unit next[I];
  bool there[I];
  int col[I];
  float aw[I][V], as[I][V], an[I][V];
  auto weights = [&](int i) {
    Weights k;
    k.w.zero(), k.s.zero(), k.n.zero();
    if (there[i]) {
      k.w.load(p.w + col[i], V > 1, V);
      if (p.scale) k.s.load(p.scale + col[i], V > 1, V);
      if (p.dn) k.n.load(p.next + col[i], V > 1, V);
    }
    if (!p.scale)
#pragma unroll
      for (int e = 0; e < V; ++e) k.s.v[e] = 1.f;
    return k;
  };
  auto load = [&](long row) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      if (row >= p.rows || !there[i]) continue;
      next[i].x.load((const T*)p.x + row * p.xs + col[i], V > 1, V);
      if (p.gate) next[i].g.load((const T*)p.gate + row * p.gs + col[i], V > 1, V);
      if (p.dy) next[i].t.load((const T*)p.dy + row * p.dys + col[i], V > 1, V);
      if (p.dn) {
        next[i].n.load((const T*)p.dn + row * p.dns + col[i], V > 1, V);
        if (p.residual) next[i].r.load((const T*)p.residual + row * p.rs + col[i], V > 1, V);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < I; ++i) {
    there[i] = at.there(l, i, p.group);
    col[i] = at.column(l, i, p.group);
    next[i].x.zero(), next[i].g.zero(), next[i].r.zero(), next[i].t.zero(), next[i].n.zero();
#pragma unroll
    for (int e = 0; e < V; ++e) aw[i][e] = as[i][e] = an[i][e] = 0.f;
  }
  if constexpr (KEEP)
#pragma unroll
    for (int i = 0; i < I; ++i) kept[i] = weights(i);
  const long step = (long)gridDim.x * l.rows;
  load((long)blockIdx.x * l.rows + at.row);
  for (long first = (long)blockIdx.x * l.rows; first < p.rows; first += step) {
    const long row = first + at.row;
    const bool real = row < p.rows;
    bool here[I];
    float unit[I][V], rstd[I], total[I][V], act[I][V], sig[I][V];      // sig: the gate's sigmoid, which its slope follows from
    Unit now[I];
    if constexpr (!KEEP) {
      if (first > (long)blockIdx.x * l.rows) load(row);
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
      now[i] = next[i];
      here[i] = real && there[i];
      if (!real) now[i].x.zero(), now[i].g.zero(), now[i].r.zero(), now[i].t.zero(), now[i].n.zero();
#pragma unroll
      for (int e = 0; e < V; ++e) {
        unit[i][e] = (float)now[i].x.v[e];
        total[i][e] = (float)now[i].t.v[e];
        act[i][e] = sig[i][e] = 1.f;
      }
    }
    if constexpr (KEEP) load(row + step);
    if (p.gate)
#pragma unroll
      for (int i = 0; i < I; ++i) {
        if (p.act != kIdentity)
#pragma unroll
          for (int e = 0; e < V; ++e) sig[i][e] = gate_sigmoid<FINE>((float)now[i].g.v[e]);
        if (p.act == kSigmoid)
#pragma unroll
          for (int e = 0; e < V; ++e) act[i][e] = sig[i][e];
        else
#pragma unroll
          for (int e = 0; e < V; ++e) act[i][e] = (float)now[i].g.v[e] * sig[i][e];
      }
    normalise<V, I, MANY>(unit, rstd, here, l, p.each, p.layer, p.eps, room);
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) unit[i][e] *= rstd[i];
    if (p.dn) {
      // n = (y - mean) r next: sums of y and of the gradient, then of their squares and products, both at once
      float y[I][V], gn[I][V], s[2] = {0.f, 0.f}, m0 = 0.f;
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const Weights k = KEEP ? kept[KEEP ? i : 0] : weights(i);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          y[i][e] = fmaf(unit[i][e] * k.w.v[e] * act[i][e], k.s.v[e], (float)now[i].r.v[e]);      // (zero where there is no residual)
          gn[i][e] = (float)now[i].n.v[e] * k.n.v[e];
        }
      }
      if (p.layer) {
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            s[0] += y[i][e];
            s[1] += gn[i][e];
          }
        add_up<2>(s, at.threads, room);
        const float mean = s[0] * p.each_row;
        m0 = s[1] * p.each_row;
        s[0] = s[1] = 0.f;
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int e = 0; e < V; ++e) y[i][e] = here[i] ? y[i][e] - mean : 0.f;
      }
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[0] = fmaf(y[i][e], y[i][e], s[0]);
          s[1] = fmaf(gn[i][e], y[i][e], s[1]);
        }
      add_up<2>(s, at.threads, room);
      const float r = real ? __builtin_amdgcn_rsqf(fmaf(s[0], p.each_row, p.eps)) : 0.f, m1 = s[1] * r * p.each_row;
#pragma unroll
      for (int i = 0; i < I; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float u = y[i][e] * r;
          an[i][e] = fmaf((float)now[i].n.v[e], u, an[i][e]);
          total[i][e] = fmaf(r, fmaf(-u, m1, gn[i][e] - m0), total[i][e]);
        }
    }
    float s1[I], s0[I];
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const Weights k = KEEP ? kept[KEEP ? i : 0] : weights(i);
      Row<T, V> out;
      s1[i] = s0[i] = 0.f;
      if (here[i] && p.dresidual) {
#pragma unroll
        for (int e = 0; e < V; ++e) out.v[e] = (T)total[i][e];
        out.store((T*)p.dresidual + row * p.C + col[i], V > 1, V);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        as[i][e] = fmaf(total[i][e], unit[i][e] * k.w.v[e] * act[i][e], as[i][e]);
        total[i][e] *= k.s.v[e];
      }
      if (here[i] && p.dgate) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float q = sig[i][e];
          const float slope = p.act == kSilu ? fmaf(act[i][e], 1.f - q, q) : (p.act == kSigmoid ? q * (1.f - q) : 1.f);
          out.v[e] = (T)(total[i][e] * unit[i][e] * k.w.v[e] * slope);
        }
        out.store((T*)p.dgate + row * p.C + col[i], V > 1, V);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float g = total[i][e] * act[i][e];
        aw[i][e] = fmaf(g, unit[i][e], aw[i][e]);
        total[i][e] = g * k.w.v[e];
        s1[i] = fmaf(total[i][e], unit[i][e], s1[i]);
        s0[i] += total[i][e];
      }
    }
    if (!p.dx) continue;
    group_sums<V, I, MANY>(s1, l, room);
    if (p.layer) group_sums<V, I, MANY>(s0, l, room);
#pragma unroll
    for (int i = 0; i < I; ++i)
      if (here[i]) {
        Row<T, V> out;
        const float m1 = s1[i] * p.each, m0 = p.layer ? s0[i] * p.each : 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) out.v[e] = (T)(rstd[i] * fmaf(-unit[i][e], m1, total[i][e] - m0));
        out.store((T*)p.dx + row * p.C + col[i], V > 1, V);
      }
  }
  if (!p.part) return;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    if (k == 1 && !p.dscale) continue;
    if (k == 2 && !p.dnext) continue;
    if (k == 0 && !p.dw) continue;
#pragma unroll
    for (int i = 0; i < I; ++i) {
      float (&a)[V] = k == 0 ? aw[i] : (k == 1 ? as[i] : an[i]);
      if (l.rows > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) sums[e * blockDim.x + threadIdx.x] = a[e];
        __syncthreads();
        if (at.row == 0)
#pragma unroll
          for (int e = 0; e < V; ++e)
            for (int m = 1; m < l.rows; ++m) a[e] += sums[e * blockDim.x + m * at.threads + threadIdx.x];
      }
      if (at.row == 0)
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (there[i]) p.part[((size_t)blockIdx.x * 3 + k) * p.C + col[i] + e] = a[e];
    }
  }
}

inline int pow2(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

struct Plan { Lie lie; int I, threads; bool many; };

// Eight values a thread (four of 32 bits) up to 512 threads, whose weights stay in registers; then twice that with 512 threads; then 1024 threads, for rows of 8192
// whose groups fill little more than half of their threads.  Us of a training step's norms, bf16, 67 million values: rows of 8192 as 512 threads of two
// units 506, as 1024 of one 877; rows of 2047, value by value, as 256 threads of eight 600, as 1024 of two 1279; of 8191 as 512 of sixteen 3588, as 1024 of
// eight 4115 (both spill registers); fp32, half as many, rows of 2048 as 512 threads of one unit 323, as 256 of two 353, of 8192 as 512 of four 630, as
// 1024 of two 949.  Backwards every row over 4096 spills: 28 registers (bf16) and 240 to 317 (fp32) of whole units on 512 threads, 378 to 651 on 1024, 636 to 957 value by value.  A
// training step's norms by the row's width 2048, 4096, 5120, 6144, 8192: bf16 334, 333, 581, 540, 507; fp32 319, 334, 715, 659, 623.
inline Plan plan_of(int C, int group, int V) {
  Plan a = {};
  const int groups = C / group, units = (group + V - 1) / V;
  a.many = groups > 1 && units <= 64;
  for (a.threads = 64; a.threads <= 1024; a.threads *= 2) {
    a.lie = {0, 0, 1, groups};
    if (a.many) {
      a.lie.lanes = pow2(units);
      a.lie.slots = a.threads / a.lie.lanes;
      if (a.lie.slots > pow2(groups)) a.lie.slots = pow2(groups);
      a.I = (groups + a.lie.slots - 1) / a.lie.slots;
    } else {
      a.lie.slots = pow2(groups);
      a.lie.lanes = a.threads / a.lie.slots;
      if (a.lie.lanes < 1) continue;
      if (a.lie.lanes > pow2(units)) a.lie.lanes = pow2(units);
      a.I = (units + a.lie.lanes - 1) / a.lie.lanes;
    }
    if (a.I * V <= (V == 4 ? 4 : 8) || (a.threads == 512 && a.I * V <= 16) || a.threads == 1024) break;
  }
  // several short rows a workgroup
  const int row = a.lie.lanes * a.lie.slots;
  if (row < 256) {
    a.threads = 256;
    a.lie.rows = 256 / row;
  } else {
    a.threads = row;
  }
  return a;
}

inline int parts_of(const Plan& a, long rows) {
  const long wanted = (rows + a.lie.rows - 1) / a.lie.rows, most = 512 * 256 / a.threads;
  return (int)(wanted < most ? wanted : most);
}

template <typename T, int V, int I, bool MANY> void launch_one(const RingNormArgs& p, const Plan& a, bool back, hipStream_t st) {
  if (back) {
    const size_t room = a.threads * V * sizeof(float);
    if constexpr (I * V <= 16) {
      if (a.threads <= 512) {
        hipLaunchKernelGGL((ring_norm_bwd_kernel<T, V, I, MANY, 512>), dim3((unsigned)p.parts), dim3(a.threads), room, st, p, a.lie);
        return;
      }
    }
    if constexpr (I * V == 16) hipLaunchKernelGGL((ring_norm_bwd_kernel<T, V, I, MANY, 1024>), dim3((unsigned)p.parts), dim3(a.threads), room, st, p, a.lie);
  } else {
    const long blocks = (p.rows + a.lie.rows - 1) / a.lie.rows, row = blocks < (1 << 20) ? blocks : 1 << 20;      // (a launch counts fewer than 2^32 threads along x)
    hipLaunchKernelGGL((ring_norm_fwd_kernel<T, V, I, MANY>), dim3((unsigned)row, (unsigned)((blocks + row - 1) / row)), dim3(a.threads), 0, st, p, a.lie);
  }
}

template <typename T, int V, bool MANY> void launch_units(const RingNormArgs& p, const Plan& a, bool back, hipStream_t st) {
  if (a.I == 1) launch_one<T, V, 1, MANY>(p, a, back, st);
  else if constexpr (V == 8) launch_one<T, V, 2, MANY>(p, a, back, st);
  else if constexpr (V == 4) {
    if (a.I == 2) launch_one<T, V, 2, MANY>(p, a, back, st);
    else launch_one<T, V, 4, MANY>(p, a, back, st);
  } else {
    if (a.I == 2) launch_one<T, V, 2, MANY>(p, a, back, st);
    else if (a.I <= 4) launch_one<T, V, 4, MANY>(p, a, back, st);
    else if (a.I <= 8) launch_one<T, V, 8, MANY>(p, a, back, st);
    else launch_one<T, V, 16, MANY>(p, a, back, st);
  }
}

template <typename T> hipError_t launch(const RingNormArgs& p, bool w, bool back, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const Plan a = plan_of(p.C, p.group, w ? V : 1);
  if (w) {
    if (a.many) launch_units<T, V, true>(p, a, back, st);
    else launch_units<T, V, false>(p, a, back, st);
  } else {
    if (a.many) launch_units<T, 1, true>(p, a, back, st);
    else launch_units<T, 1, false>(p, a, back, st);
  }
  return hipGetLastError();
}

}  // namespace ring_norm
