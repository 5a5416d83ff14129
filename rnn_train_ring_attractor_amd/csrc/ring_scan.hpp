// Selective state space scan: a channel c keeps N states h[n], whose decay and input depend on the token,
//
//   d_t = softplus(delta_t + bias),  h_t = e^(d_t A[n]) h_(t-1) + d_t x_t B_t[n],  y_t = (sum_n C_t[n] h_t[n] + D x_t) silu(z_t),
//
// B and C shared by the channels of a group.  Backwards, with q_t = dy_t silu(z_t) and g_t = q_t C_t + a_(t+1) g_(t+1), a = e^(d A):
//
//   dB_t = sum_c d x g,  dC_t = sum_c q h,  dx = d sum_n g B + D q,  dd = x sum_n g B + sum_n A a g h_(t-1),  dA = sum_t d a g h_(t-1).
//
// There is no matrix product in this: a power, four multiplications and additions for each token, channel and state forwards, three times
// that backwards, in vector instructions.  A wave takes 16 channels and 16 states of each (four waves 64 channels, or fewer channels of
// more states); a lane keeps four states of a channel in registers from token to token.  A chunk's rows are read by all threads, 16
// bytes a lane, worked out once (softplus, gate) and laid into LDS, where lanes find four tokens of their channel in one access.  Sums over a
// channel's states go across lanes two values at a time (half a wave's lanes change places with those of another register, then one addition).
//
// Where there are few channels, the tokens are cut into segments: a pass finds what each adds to a state of zeros, a scan the states between
// them, and the pass behind starts from those.
#pragma once
#include "ring_recur.hpp"
#include "ringattr.h"

namespace ring_scan {

using namespace ring_recur;

constexpr int kL = 32;                // tokens of a chunk forwards
constexpr int kSave = RingScanArgs::kSave;      // tokens between states that are kept for the backward, and of a chunk there

// Where a channel's tokens lie: rows of L + 4, eight of them displaced by 8 against the next eight, so that lanes of a wave that write a token of eight
// channels each spread over the banks
template <int L> __device__ __forceinline__ int at(int c, int t) { return c * (L + 4) + (c >> 3) * 8 + t; }
template <int CH, int L> constexpr int plane() { return CH * (L + 4) + CH; }

struct Place { int seg, b, g, c0, here; };      // segment, sequence, group, first channel of the tile, channels in it

template <int CH> __device__ __forceinline__ Place place(const RingScanArgs& p) {
  const unsigned all = (unsigned)p.tiles * p.G;
  unsigned i = blockIdx.x;
  const int tile = (int)(i % all);
  i /= all;
  const int g = tile / p.tiles, first = (tile - g * p.tiles) * CH, Cg = p.C / p.G;
  return {(int)(i / p.B), (int)(i % p.B), g, g * Cg + first, min(CH, Cg - first)};
}

enum Mode { kOutputs, kState, kAdjoint };

// Outputs (and the states kept for a backward), or what a segment adds to a state of zeros, or, backwards in time, to an adjoint of zeros
template <typename T, int NL, int NB, int MODE>
__global__ __launch_bounds__(256) void ring_scan_kernel(RingScanArgs p) {
  constexpr int CH = 64 / NB, L = kL, E = CH / 8, NS = 4 * NL * NB, PL = plane<CH, L>();
  constexpr int NV = (L * NS + 255) / 256;          // values of B or C that a thread lays down
  constexpr bool REV = MODE == kAdjoint, OUT = MODE == kOutputs;
  __shared__ __attribute__((aligned(16))) float sd[PL], su[PL], sB[L * NS], sC[OUT ? L * NS : 4], sy[OUT ? NB * PL : 4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const Place at_ = place<CH>(p);
  const int seg = REV ? p.nseg - 1 - at_.seg : at_.seg, b = at_.b;
  const int len = length_of(p.lengths, b, p.T), first = seg * p.seg_tokens, last = min(first + p.seg_tokens, p.T), end = min(last, len);
  // a lane's channel and states
  const int nb = w % NB, ch = w / NB * 16 + (lane & 15), sub = lane >> 4, n0 = nb * 4 * NL + sub * NL, c = at_.c0 + ch;
  const bool mine = ch < at_.here;
  // a thread's token and channels where rows are read and written
  const int tl = tid >> 3, cl = (tid & 7) * E, cr = at_.c0 + cl, here = at_.here - cl;
  float A2[NL], h[NL], D[E], bias[E];
#pragma unroll
  for (int n = 0; n < NL; ++n) {
    A2[n] = mine && n0 + n < p.N ? (float)((double)p.A[(size_t)c * p.N + n0 + n] * 1.4426950408889634) : 0.f;
    h[n] = 0.f;
    if (OUT && mine) {
      if (seg > 0) h[n] = p.seg[(((size_t)(seg - 1) * p.B + b) * p.C + c) * NS + n0 + n];
      else if (p.s_in && n0 + n < p.N) h[n] = p.s_in[((size_t)b * p.C + c) * p.N + n0 + n];
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    D[e] = OUT && p.D && e < here ? p.D[cr + e] : 0.f;
    bias[e] = p.bias && e < here ? p.bias[cr + e] : 0.f;
  }
  float total = 0.f;                     // of d, for the segment's whole decay
  Row<T, E> rx, rd, rz, ry, kx, kz;
  T rB[NV], rC[NV];
  rx.zero(), rd.zero(), rz.zero(), ry.zero();
  const T* const Bp = (const T*)(REV ? p.Cm : p.Bm) + (size_t)b * (REV ? p.csb : p.bsb) + (size_t)at_.g * (REV ? p.csg : p.bsg);
  const T* const Cp = (const T*)p.Cm + (size_t)b * p.csb + (size_t)at_.g * p.csg;
  auto load = [&](int t0) {
    const int t = t0 + tl;
    if (t < end && here > 0) {
      rd.load((const T*)p.delta.p + b * p.delta.sb + t * p.delta.st + cr, p.wide, here);
      if (!REV) rx.load((const T*)p.x.p + b * p.x.sb + t * p.x.st + cr, p.wide, here);
      if ((OUT || REV) && p.z.p) rz.load((const T*)p.z.p + b * p.z.sb + t * p.z.st + cr, p.wide, here);
      if (REV) ry.load((const T*)p.dy.p + b * p.dy.sb + t * p.dy.st + cr, p.wide, here);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = tid + 256 * i, tk = t0 + k / NS, n = k % NS;
      const bool there = k < L * NS && tk < end && n < p.N;
      rB[i] = there ? Bp[(long)tk * (REV ? p.cst : p.bst) + n] : (T)0.f;
      if (OUT) rC[i] = there ? Cp[(long)tk * p.cst + n] : (T)0.f;
    }
  };
  auto lay = [&](int t0) {
    const bool there = t0 + tl < end;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float d = 0.f, u = 0.f;
      if (there && e < here) {
        d = (float)rd.v[e] + bias[e];
        if (p.softplus) d = softplus(d);
        if (REV) u = p.z.p ? (float)ry.v[e] * silu((float)rz.v[e]) : (float)ry.v[e];
        else u = d * (float)rx.v[e];
      }
      sd[at<L>(cl + e, tl)] = d;
      su[at<L>(cl + e, tl)] = u;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = tid + 256 * i;
      if (k < L * NS) {
        sB[k] = (float)rB[i];
        if (OUT) sC[k] = (float)rC[i];
      }
    }
  };
  const int chunks = end > first ? (end - first + L - 1) / L : 0;
  if (chunks > 0) load(first + (REV ? chunks - 1 : 0) * L);
  for (int k = 0; k < chunks; ++k) {
    const int t0 = first + (REV ? chunks - 1 - k : k) * L;
    __syncthreads();
    lay(t0);
    if (OUT) kx = rx, kz = rz;
    if (k + 1 < chunks) load(REV ? t0 - L : t0 + L);
    __syncthreads();
#pragma unroll 2
    for (int jj = 0; jj < L; jj += 4) {
      const int j = REV ? L - 4 - jj : jj;
      if (OUT && p.states && j % kSave == 0 && mine && t0 + j < end) {
        float* s = p.states + (((size_t)b * p.saved + (t0 + j) / kSave) * p.C + c) * NS + n0;
#pragma unroll
        for (int n = 0; n < NL; ++n) s[n] = h[n];
      }
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + at<L>(ch, j)), u4 = *reinterpret_cast<const f32x4*>(su + at<L>(ch, j));
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int o = REV ? 3 - i : i;
        float Bn[NL], Cn[NL];
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          Bn[n] = sB[(j + o) * NS + n0 + n];
          if (OUT) Cn[n] = sC[(j + o) * NS + n0 + n];
        }
        y[o] = 0.f;
        if (!OUT) total += d4[o];
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          const float a = __builtin_amdgcn_exp2f(d4[o] * A2[n]);
          if (REV) h[n] = a * fmaf(u4[o], Bn[n], h[n]);
          else h[n] = fmaf(a, h[n], u4[o] * Bn[n]);
          if (OUT) y[o] = fmaf(h[n], Cn[n], y[o]);
        }
      }
      if (OUT) {
        // row r of 16 lanes is left with token (0, 2, 1, 3)[r]
        const float sum = fold16(fold32(y[0], y[1]), fold32(y[2], y[3]));
        sy[nb * PL + at<L>(ch, j + ((sub & 1) << 1 | sub >> 1))] = sum;
      }
    }
    if (OUT) {
      __syncthreads();
      const int t = t0 + tl;
      if (t < last && here > 0) {
        Row<T, E> out;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float y = sy[at<L>(cl + e, tl)];
#pragma unroll
          for (int i = 1; i < NB; ++i) y += sy[i * PL + at<L>(cl + e, tl)];
          if (p.D) y = fmaf(D[e], (float)kx.v[e], y);
          if (p.z.p) y *= silu((float)kz.v[e]);
          out.v[e] = (T)(t < end ? y : 0.f);
        }
        out.store((T*)p.y + ((size_t)b * p.T + t) * p.C + cr, p.wide_out, here);
      }
    }
  }
  if (OUT) {                             // tokens that do not count
    Row<T, E> none;
    none.zero();
    for (int t = first + chunks * L + tl; t < last; t += L)
      if (here > 0) none.store((T*)p.y + ((size_t)b * p.T + t) * p.C + cr, p.wide_out, here);
    if (p.s_out && seg == p.nseg - 1 && mine) {
#pragma unroll
      for (int n = 0; n < NL; ++n)
        if (n0 + n < p.N) p.s_out[((size_t)b * p.C + c) * p.N + n0 + n] = h[n];
    }
  } else if (mine) {
    const size_t row = ((size_t)at_.seg * p.B + b) * p.C + c;
#pragma unroll
    for (int n = 0; n < NL; ++n) p.seg[row * NS + n0 + n] = h[n];
    if (n0 == 0) p.total[row] = total;
  }
}

// The gradients.  Chunks of kSave tokens against the time: forwards through a chunk from the state kept in front of it, powers and states in
// registers, then back.  A quad of lanes shares a channel: sums over its states cross the quad, sums over channels (of dB and dC) the 16 quads.
template <typename T, int NL, int NB>
__global__ __launch_bounds__(256, 2) void ring_scan_bwd_kernel(RingScanArgs p) {
  constexpr int CH = 64 / NB, L = kSave, E = CH / 16, NS = 4 * NL * NB, PL = plane<CH, L>(), CW = 4 / NB, R = 8 * NL;
  constexpr int NV = (L * NS + 255) / 256;
  __shared__ __attribute__((aligned(16))) float sd[PL], su[PL], sq[PL], sB[L * NS], sC[L * NS], so[3 * NB * PL], red[4][L * 32];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const Place at_ = place<CH>(p);
  const int seg = at_.seg, b = at_.b;
  const int len = length_of(p.lengths, b, p.T), first = seg * p.seg_tokens, last = min(first + p.seg_tokens, p.T), end = min(last, len);
  const int nb = w % NB, ch = w / NB * 16 + (lane >> 2), sub = lane & 3, n0 = nb * 4 * NL + sub * NL, c = at_.c0 + ch;
  const bool mine = ch < at_.here;
  const int tl = tid >> 4, cl = (tid & 15) * E, cr = at_.c0 + cl, here = at_.here - cl;
  float A2[NL], G[NL], dA[NL], D[E], bias[E], dD[E], dbias[E];
#pragma unroll
  for (int n = 0; n < NL; ++n) {
    A2[n] = mine && n0 + n < p.N ? (float)((double)p.A[(size_t)c * p.N + n0 + n] * 1.4426950408889634) : 0.f;
    G[n] = dA[n] = 0.f;
    if (mine) {
      if (seg < p.nseg - 1) G[n] = p.seg[(((size_t)(p.nseg - 2 - seg) * p.B + b) * p.C + c) * NS + n0 + n];
      else if (p.s_in && n0 + n < p.N) G[n] = p.s_in[((size_t)b * p.C + c) * p.N + n0 + n];
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    D[e] = p.D && e < here ? p.D[cr + e] : 0.f;
    bias[e] = p.bias && e < here ? p.bias[cr + e] : 0.f;
    dD[e] = dbias[e] = 0.f;
  }
  Row<T, E> rx, rd, rz, ry, kx, kz, ky, kd;
  rx.zero(), rd.zero(), rz.zero(), ry.zero();
  T rB[NV], rC[NV];
  const T* const Bp = (const T*)p.Bm + (size_t)b * p.bsb + (size_t)at_.g * p.bsg;
  const T* const Cp = (const T*)p.Cm + (size_t)b * p.csb + (size_t)at_.g * p.csg;
  float hk[NL];                          // the state kept in front of a chunk
  auto load = [&](int t0) {
    const int t = t0 + tl;
    if (t < end && here > 0) {
      rd.load((const T*)p.delta.p + b * p.delta.sb + t * p.delta.st + cr, p.wide, here);
      rx.load((const T*)p.x.p + b * p.x.sb + t * p.x.st + cr, p.wide, here);
      if (p.z.p) rz.load((const T*)p.z.p + b * p.z.sb + t * p.z.st + cr, p.wide, here);
      ry.load((const T*)p.dy.p + b * p.dy.sb + t * p.dy.st + cr, p.wide, here);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = tid + 256 * i, tk = t0 + k / NS, n = k % NS;
      const bool there = k < L * NS && tk < end && n < p.N;
      rB[i] = there ? Bp[(long)tk * p.bst + n] : (T)0.f;
      rC[i] = there ? Cp[(long)tk * p.cst + n] : (T)0.f;
    }
#pragma unroll
    for (int n = 0; n < NL; ++n) hk[n] = mine ? p.states[(((size_t)b * p.saved + t0 / kSave) * p.C + c) * NS + n0 + n] : 0.f;
  };
  auto lay = [&](int t0) {
    const bool there = t0 + tl < end;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float d = 0.f, u = 0.f, q = 0.f;
      if (there && e < here) {
        d = (float)rd.v[e] + bias[e];
        if (p.softplus) d = softplus(d);
        u = d * (float)rx.v[e];
        q = p.z.p ? (float)ry.v[e] * silu((float)rz.v[e]) : (float)ry.v[e];
      }
      sd[at<L>(cl + e, tl)] = d;
      su[at<L>(cl + e, tl)] = u;
      sq[at<L>(cl + e, tl)] = q;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = tid + 256 * i;
      if (k < L * NS) {
        sB[k] = (float)rB[i];
        sC[k] = (float)rC[i];
      }
    }
  };
  const int chunks = end > first ? (end - first + L - 1) / L : 0;
  const bool shared = p.part_bc != nullptr;
  if (chunks > 0) load(first + (chunks - 1) * L);
  for (int k = chunks - 1; k >= 0; --k) {
    const int t0 = first + k * L;
    __syncthreads();
    lay(t0);
    kx = rx, kz = rz, ky = ry, kd = rd;
    float h[NL];
#pragma unroll
    for (int n = 0; n < NL; ++n) h[n] = hk[n];
    if (k > 0) load(t0 - L);
    __syncthreads();
    float hs[L][NL], as[L][NL], dAc[NL];
#pragma unroll
    for (int j = 0; j < L; j += 4) {
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + at<L>(ch, j)), u4 = *reinterpret_cast<const f32x4*>(su + at<L>(ch, j));
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          hs[j + i][n] = h[n];
          as[j + i][n] = __builtin_amdgcn_exp2f(d4[i] * A2[n]);
          h[n] = fmaf(as[j + i][n], h[n], u4[i] * sB[(j + i) * NS + n0 + n]);
        }
    }
#pragma unroll
    for (int n = 0; n < NL; ++n) dAc[n] = 0.f;
#pragma unroll
    for (int j = L - 4; j >= 0; j -= 4) {
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + at<L>(ch, j)), u4 = *reinterpret_cast<const f32x4*>(su + at<L>(ch, j)),
                  q4 = *reinterpret_cast<const f32x4*>(sq + at<L>(ch, j));
#pragma unroll
      for (int i = 3; i >= 0; --i) {
        float s1 = 0.f, s2 = 0.f, y = 0.f, v[2 * NL];
        if (t0 + j + i + 1 == end)         // (behind the last token that counts no state takes part in dA, however large)
#pragma unroll
          for (int n = 0; n < NL; ++n) dAc[n] = 0.f;
#pragma unroll
        for (int n = 0; n < NL; ++n) {
          const float Bn = sB[(j + i) * NS + n0 + n], Cn = sC[(j + i) * NS + n0 + n];
          y = fmaf(Cn, h[n], y);
          v[NL + n] = q4[i] * h[n];
          const float g = fmaf(q4[i], Cn, G[n]);
          v[n] = g * u4[i];
          s1 = fmaf(g, Bn, s1);
          G[n] = as[j + i][n] * g;
          h[n] = hs[j + i][n];
          const float turn = G[n] * h[n];
          s2 = fmaf(turn, A2[n], s2);
          dAc[n] = fmaf(d4[i], turn, dAc[n]);
        }
        s1 = plus_dpp<kXor2>(plus_dpp<kXor1>(s1));
        s2 = plus_dpp<kXor2>(plus_dpp<kXor1>(s2));
        y = plus_dpp<kXor2>(plus_dpp<kXor1>(y));
        if (sub < 3) so[(sub * NB + nb) * PL + at<L>(ch, j + i)] = sub == 0 ? s1 : (sub == 1 ? s2 : y);
        if (shared) {
          // over the 16 quads: halves, rows, then within a row; a lane of row r keeps the values r >> 1 and r & 1 name
#pragma unroll
          for (int m = 0; m < NL; ++m) v[m] = fold32(v[m], v[NL + m]);
          if constexpr (NL > 1) {
#pragma unroll
            for (int m = 0; m < NL / 2; ++m) v[m] = fold16(v[m], v[NL / 2 + m]);
          } else {
            v[0] = fold16(v[0], v[0]);
          }
          constexpr int LEFT = NL > 1 ? NL / 2 : 1;
          const int r = lane >> 4, type = r >> 1, half = NL > 1 ? (r & 1) * LEFT : 0;
#pragma unroll
          for (int m = 0; m < LEFT; ++m) {
            const float sum = plus_dpp<kRor4>(plus_dpp<kRor8>(v[m]));
            if ((lane & 12) == 0) red[w][(j + i) * R + type * 4 * NL + sub * NL + half + m] = sum;
          }
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NL; ++n) dA[n] += dAc[n];
    __syncthreads();
    const int t = t0 + tl;
    if (t < last && here > 0) {
      Row<T, E> ox, od, oz;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float s1 = 0.f, s2 = 0.f, y = 0.f;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          s1 += so[i * PL + at<L>(cl + e, tl)];
          s2 += so[(NB + i) * PL + at<L>(cl + e, tl)];
          y += so[(2 * NB + i) * PL + at<L>(cl + e, tl)];
        }
        const float d = sd[at<L>(cl + e, tl)], q = sq[at<L>(cl + e, tl)], x = (float)kx.v[e];
        float dd = fmaf(s1, x, s2 * kLn2);
        if (p.softplus) dd *= sigmoid((float)kd.v[e] + bias[e]);
        const bool counts = t < end && e < here;
        ox.v[e] = (T)(counts ? fmaf(D[e], q, d * s1) : 0.f);
        od.v[e] = (T)(counts ? dd : 0.f);
        if (counts) {
          dD[e] = fmaf(q, x, dD[e]);
          dbias[e] += dd;
        }
        if (p.z.p) {
          const float z = (float)kz.v[e], s = sigmoid(z);
          oz.v[e] = (T)(counts ? (float)ky.v[e] * fmaf(D[e], x, y) * silu_slope(z, s) : 0.f);
        }
      }
      const size_t row = ((size_t)b * p.T + t) * p.C + cr;
      if (p.dx) ox.store((T*)p.dx + row, p.wide_out, here);
      if (p.ddelta) od.store((T*)p.ddelta + row, p.wide_out, here);
      if (p.dz) oz.store((T*)p.dz + row, p.wide_out, here);
    }
    if (shared) {
      const int tile = (at_.c0 - at_.g * (p.C / p.G)) / CH;
      for (int i = tid; i < L * 2 * NS; i += 256) {
        const int tk = i / (2 * NS), type = i / NS % 2, n = i % NS, block = n / (4 * NL);
        float sum = 0.f;
#pragma unroll
        for (int m = 0; m < CW; ++m) sum += red[m * NB + block][tk * R + type * 4 * NL + n % (4 * NL)];
        if (t0 + tk < end) p.part_bc[((((size_t)tile * p.B + b) * p.T + t0 + tk) * p.G + at_.g) * 2 * NS + type * NS + n] = sum;
      }
    }
  }
  Row<T, E> none;                        // tokens that do not count
  none.zero();
  for (int t = first + chunks * L + tl; t < last; t += L)
    if (here > 0) {
      const size_t row = ((size_t)b * p.T + t) * p.C + cr;
      if (p.dx) none.store((T*)p.dx + row, p.wide_out, here);
      if (p.ddelta) none.store((T*)p.ddelta + row, p.wide_out, here);
      if (p.dz) none.store((T*)p.dz + row, p.wide_out, here);
    }
  if (mine && seg == 0 && p.s_out) {
#pragma unroll
    for (int n = 0; n < NL; ++n)
      if (n0 + n < p.N) p.s_out[((size_t)b * p.C + c) * p.N + n0 + n] = G[n];
  }
  if (p.part_a) {
    float* part = p.part_a + ((size_t)seg * p.B + b) * p.C * (NS + 2);
    if (mine) {
#pragma unroll
      for (int n = 0; n < NL; ++n) part[(size_t)c * (NS + 2) + n0 + n] = dA[n];
    }
    // the 16 threads of a channel, in order
    static_assert(sizeof(red) >= 16 * CH * 2 * sizeof(float), "room for the sums");
    float* sums = &red[0][0];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      sums[tl * CH + cl + e] = dD[e];
      sums[16 * CH + tl * CH + cl + e] = dbias[e];
    }
    __syncthreads();
    if (tid < 2 * CH && tid % CH < at_.here) {
      float sum = 0.f;
      for (int i = 0; i < 16; ++i) sum += sums[tid / CH * 16 * CH + i * CH + tid % CH];
      part[(size_t)(at_.c0 + tid % CH) * (NS + 2) + NS + tid / CH] = sum;
    }
  }
}

template <typename T, int NL, int NB> hipError_t launch_sized(const RingScanArgs& p, int mode, hipStream_t st) {
  const int CH = 64 / NB;
  RingScanArgs a = p;
  a.tiles = (p.C / p.G + CH - 1) / CH;
  const int segs = mode == RING_SCAN_STATE || mode == RING_SCAN_ADJOINT ? p.nseg - 1 : p.nseg;
  const dim3 grid((unsigned)((size_t)a.tiles * p.G * p.B * segs)), block(256);
  if (mode == RING_SCAN_OUTPUTS) hipLaunchKernelGGL((ring_scan_kernel<T, NL, NB, kOutputs>), grid, block, 0, st, a);
  else if (mode == RING_SCAN_STATE) hipLaunchKernelGGL((ring_scan_kernel<T, NL, NB, kState>), grid, block, 0, st, a);
  else if (mode == RING_SCAN_ADJOINT) hipLaunchKernelGGL((ring_scan_kernel<T, NL, NB, kAdjoint>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((ring_scan_bwd_kernel<T, NL, NB>), grid, block, 0, st, a);
  return hipGetLastError();
}

template <typename T> hipError_t launch(const RingScanArgs& p, int mode, hipStream_t st) {
  if (p.N <= 4) return launch_sized<T, 1, 1>(p, mode, st);
  if (p.N <= 8) return launch_sized<T, 2, 1>(p, mode, st);
  if (p.N <= 16) return launch_sized<T, 4, 1>(p, mode, st);
  if (p.N <= 32) return launch_sized<T, 4, 2>(p, mode, st);
  return launch_sized<T, 4, 4>(p, mode, st);
}

}  // namespace ring_scan
