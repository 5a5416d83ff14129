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

#include <type_traits>

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
  if (gridDim.x % 8 == 0) i = i % 8 * (gridDim.x / 8) + i / 8;       // neighbours, which share rows, lines and pages, on one XCD
  const int tile = (int)(i % all);
  i /= all;
  const int g = tile / p.tiles, first = (tile - g * p.tiles) * CH, Cg = p.C / p.G;
  return {(int)(i / p.B), (int)(i % p.B), g, g * Cg + first, min(CH, Cg - first)};
}

// Four sums over the lanes of a quad, of which lane `sub` keeps number sub
__device__ __forceinline__ float quad_sums(const float* v, int sub) {
  // (sums first, by all lanes, then the choice)
  const float a0 = plus_dpp<kXor1>(v[0]), a1 = plus_dpp<kXor1>(v[1]), b0 = plus_dpp<kXor1>(v[2]), b1 = plus_dpp<kXor1>(v[3]);
  const float a = plus_dpp<kXor2>(sub & 1 ? a1 : a0), b = plus_dpp<kXor2>(sub & 1 ? b1 : b0);
  return sub & 2 ? b : a;
}
// Four sums over a row's quads, of which quad (0, 2, 1, 3)[i] keeps number i
__device__ __forceinline__ float row_sums(const float* v, int quad) {
  const float a0 = plus_dpp<kRor8>(v[0]), a1 = plus_dpp<kRor8>(v[1]), b0 = plus_dpp<kRor8>(v[2]), b1 = plus_dpp<kRor8>(v[3]);
  const float a = plus_dpp<kUp4>(quad & 2 ? a1 : a0), b = plus_dpp<kDown4>(quad & 2 ? b1 : b0);
  return quad & 1 ? b : a;
}

enum Mode { kOutputs, kState, kAdjoint };

template <int NL> __device__ __forceinline__ void take(float (&v)[NL], const float* p) {      // NL floats at a whole number of NL of them
  typedef float vec __attribute__((ext_vector_type(NL)));
  const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
  for (int n = 0; n < NL; ++n) v[n] = x[n];
}
template <> __device__ __forceinline__ void take<1>(float (&v)[1], const float* p) { v[0] = *p; }

// B or C of a chunk, read by 256 threads and laid down in fp32
template <typename T, int L, int NS> struct Shared {
  static constexpr int NV = (L * NS + 255) / 256;
  T v[NV];
  static __device__ __forceinline__ int place(int i, long st, int N, int tid) {      // of value i in a chunk's buffer
    const int k = tid + 256 * i;
    return k < L * NS && k % NS < N ? (int)((k / NS * st + k % NS) * (long)sizeof(T)) : kOutside;
  }
  __device__ __forceinline__ void fetch(__amdgpu_buffer_rsrc_t b, const int (&at)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Row<T, 1> x;
      x.fetch(b, at[i]);
      v[i] = x.v[0];
    }
  }
  __device__ __forceinline__ void load(const T* p, long st, int t0, int end, int N, int tid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = tid + 256 * i, t = t0 + k / NS, n = k % NS;
      const T x = p[(long)min(t, end - 1) * st + min(n, N - 1)];       // (t0 < end: there is a row)
      v[i] = t < end && n < N ? x : (T)0.f;
    }
  }
  __device__ __forceinline__ void lay(float* to, int tid) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + 256 * i < L * NS) to[tid + 256 * i] = (float)v[i];
  }
};

// Outputs (and the states kept for a backward), or what a segment adds to a state of zeros, or, backwards in time, to an adjoint of zeros.
// The first four waves go through the tokens; the other four read and work out the next chunk's rows and finish the last one's outputs meanwhile.
//
// Bound by vector instructions: a power takes a pipe 8.5 cycles, as do exchanges of lanes; a multiplication or addition takes 4.5 of one wave, of which two waves' overlap.
// A state of a token is a power and four of the others, and 2.4 instructions for its share of the rows'.  Their counters have the pipes busy to 97
// percent at four cycles each; two workgroups a unit, where there are so many and they fit, are 4 percent faster than one.  They fit where outputs take up to 128
// registers: 16-bit rows of whole 16 bytes (107 to 119), such fp32 rows of over 16 states (119 to 125; 178 to 185 otherwise), rows value by value of over 32 states (120; 135 to
// 206 otherwise).  Bf16, 16 states, gate: eight sequences of
// 2048 tokens of 2048 channels 142 us (270 MB: 51 at the rate of a copy; 3.8 T states/s), one of 32768 tokens in 16 segments 190 for what they add,
// 7 between them and 270 for the outputs.
template <typename T, int NL, int NB, int MODE, bool WIDE>
__global__ __launch_bounds__(512) void ring_scan_kernel(RingScanArgs p) {
  constexpr int CH = 64 / NB, L = kL, E = CH / 8, NS = 4 * NL * NB, PL = plane<CH, L>();
  constexpr bool REV = MODE == kAdjoint, OUT = MODE == kOutputs;
  __shared__ __attribute__((aligned(16))) float sd[2][PL], su[2][PL], sB[2][L * NS], sC[2][OUT ? L * NS : 4], sy[2][OUT ? NB * PL : 4];
  const int tid = threadIdx.x & 255, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at_ = place<CH>(p);
  const int seg = REV ? p.nseg - 1 - at_.seg : at_.seg, b = at_.b;
  const int len = length_of(p.lengths, b, p.T), first = seg * p.seg_tokens, last = min(first + p.seg_tokens, p.T), end = min(last, len);
  const int chunks = end > first ? (end - first + L - 1) / L : 0;
  auto begin = [&](int k) { return first + (REV ? chunks - 1 - k : k) * L; };
  if (w < 4) {
    const int nb = w % NB, ch = w / NB * 16 + (lane & 15), sub = lane >> 4, n0 = nb * 4 * NL + sub * NL, c = at_.c0 + ch;
    const bool mine = ch < at_.here;
    float A2[NL], h[NL], total = 0.f;      // total: of d, for the segment's whole decay
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      A2[n] = mine && n0 + n < p.N ? times_log2e(p.A[(size_t)c * p.N + n0 + n]) : 0.f;
      h[n] = 0.f;
      if (OUT && mine) {
        if (seg > 0) h[n] = p.seg[(((size_t)(seg - 1) * p.B + b) * p.C + c) * NS + n0 + n];
        else if (p.s_in && n0 + n < p.N) h[n] = p.s_in[((size_t)b * p.C + c) * p.N + n0 + n];
      }
    }
    __syncthreads();
    for (int k = 0; k < chunks; ++k) {
      const int t0 = begin(k);
      const float *d_ = sd[k & 1] + at<L>(ch, 0), *u_ = su[k & 1] + at<L>(ch, 0), *B_ = sB[k & 1] + n0, *C_ = sC[k & 1] + n0;
      float* const y_ = sy[k & 1] + (OUT ? nb * PL + at<L>(ch, (sub & 1) << 1 | sub >> 1) : 0);
      // Four tokens at a time, what the next four need on its way from LDS; powers and inputs of the four first, then the states one after another (without
      // the order, which the compiler does not find by itself, the wave waits for LDS and for every power)
      struct Four { f32x4 d, u; float B[4][NL], C[4][NL]; } g[2];
      auto fetch = [&](int j, Four& f) {
        f.d = *reinterpret_cast<const f32x4*>(d_ + j);
        f.u = *reinterpret_cast<const f32x4*>(u_ + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          take<NL>(f.B[i], B_ + (j + i) * NS);
          if (OUT) take<NL>(f.C[i], C_ + (j + i) * NS);
        }
      };
      fetch(REV ? L - 4 : 0, g[0]);
#pragma unroll
      for (int jj = 0; jj < L; jj += 4) {
        const int j = REV ? L - 4 - jj : jj;
        const Four& f = g[jj / 4 & 1];
        if (OUT && p.states && j % kSave == 0 && mine && t0 + j < end) {
          float* s = p.states + (((size_t)b * p.saved + (t0 + j) / kSave) * p.C + c) * NS + n0;
#pragma unroll
          for (int n = 0; n < NL; ++n) s[n] = h[n];
        }
        if (jj + 4 < L) fetch(REV ? j - 4 : j + 4, g[jj / 4 + 1 & 1]);
        __builtin_amdgcn_sched_barrier(0);
        float a[4][NL], v[4][NL], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!OUT) total += f.d[i];
#pragma unroll
          for (int n = 0; n < NL; ++n) a[i][n] = f.d[i] * A2[n];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NL; ++n) {
            a[i][n] = __builtin_amdgcn_exp2f(a[i][n]);
            if (!REV) v[i][n] = f.u[i] * f.B[i][n];
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int o = REV ? 3 - i : i;
#pragma unroll
          for (int n = 0; n < NL; ++n) {
            if (REV) h[n] = a[o][n] * fmaf(f.u[o], f.B[o][n], h[n]);
            else h[n] = fmaf(a[o][n], h[n], v[o][n]);
            if (OUT) y[o] = n == 0 ? h[n] * f.C[o][n] : fmaf(h[n], f.C[o][n], y[o]);
          }
        }
        // row r of 16 lanes is left with token (0, 2, 1, 3)[r]
        if (OUT) y_[j] = fold16(fold32(y[0], y[1]), fold32(y[2], y[3]));
      }
      __syncthreads();
    }
    if (!mine) return;
    if (OUT) {
      if (p.s_out && seg == p.nseg - 1) {
#pragma unroll
        for (int n = 0; n < NL; ++n)
          if (n0 + n < p.N) p.s_out[((size_t)b * p.C + c) * p.N + n0 + n] = h[n];
      }
    } else {
      const size_t row = ((size_t)at_.seg * p.B + b) * p.C + c;
#pragma unroll
      for (int n = 0; n < NL; ++n) p.seg[row * NS + n0 + n] = h[n];
      if (n0 == 0) p.total[row] = total;
    }
    return;
  }
  // a thread's token and channels where rows are read and written
  const int tl = tid >> 3, cl = (tid & 7) * E, cr = at_.c0 + cl, here = at_.here - cl;
  float D[E], bias[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    D[e] = OUT && p.D && e < here ? p.D[cr + e] : 0.f;
    bias[e] = p.bias && e < here ? p.bias[cr + e] : 0.f;
  }
  // Rows two chunks ahead: a chunk takes less time than a row from memory (one chunk ahead: 255 us in place of 168 for eight sequences of 2048 tokens, 2048
  // channels, before the rows were buffers).  Reads have no conditions, which the compiler could not count them by: what is not there is read from a place that is, and left out.
  const bool skip = p.D != nullptr;
  struct In { Row<T, E> x, d, z; Shared<T, L, NS> B, C; } in[2];
  struct { Row<T, E> x, z; } now, before;
  const int tr = here > 0 ? here : at_.here, cw = here > 0 ? cr : at_.c0;
  const T *const dp = (const T*)p.delta.p + b * p.delta.sb, *const xp = (const T*)(REV ? p.dy.p : p.x.p) + b * (REV ? p.dy.sb : p.x.sb),
          *const zp = p.z.p ? (const T*)p.z.p + b * p.z.sb : xp;
  const long xt = REV ? p.dy.st : p.x.st, zt = p.z.p ? p.z.st : xt;
  const T* const Bp = (const T*)(REV ? p.Cm : p.Bm) + (size_t)b * (REV ? p.csb : p.bsb) + (size_t)at_.g * (REV ? p.csg : p.bsg);
  const T* const Cp = (const T*)p.Cm + (size_t)b * p.csb + (size_t)at_.g * p.csg;
  const long Bt = REV ? p.cst : p.bst;
  typedef Shared<T, L, NS> Sh;
  const int dw = (int)((tl * p.delta.st + cw) * (long)sizeof(T)), xw = (int)((tl * xt + cw) * (long)sizeof(T)), zw = (int)((tl * zt + cw) * (long)sizeof(T)),
            yw = here > 0 ? (int)((tl * (long)p.C + cr) * (long)sizeof(T)) : kOutside;
  int Bw[Sh::NV], Cw[Sh::NV];
#pragma unroll
  for (int i = 0; i < Sh::NV; ++i) {
    Bw[i] = Sh::place(i, Bt, p.N, tid);
    Cw[i] = Sh::place(i, p.cst, p.N, tid);
  }
  auto load = [&](int k, In& r) {
    const int t0 = begin(min(k, chunks - 1)), rows = min(end - t0, L);
    if constexpr (WIDE) {
      r.d.fetch(buffer_of(dp + t0 * p.delta.st, p.delta.st, rows), dw);
      r.x.fetch(buffer_of(xp + t0 * xt, xt, rows), xw);
      if (OUT || REV) r.z.fetch(buffer_of(zp + t0 * zt, zt, rows), zw);
      r.B.fetch(buffer_of(Bp + t0 * Bt, Bt, rows), Bw);
      if (OUT) r.C.fetch(buffer_of(Cp + t0 * p.cst, p.cst, rows), Cw);
    } else {
      const long t = min(t0 + tl, end - 1);
      r.d.read(dp + cw + t * p.delta.st, tr);
      r.x.read(xp + cw + t * xt, tr);
      if (OUT || REV) r.z.read(zp + cw + t * zt, tr);
      r.B.load(Bp, Bt, t0, end, p.N, tid);
      if (OUT) r.C.load(Cp, p.cst, t0, end, p.N, tid);
    }
  };
  auto lay = [&](int k, const In& r) {
    const bool there = begin(k) + tl < end;
    float d[E], u[E];
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = (float)r.d.v[e] + bias[e];
    if (p.softplus)
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = softplus<sizeof(T) == 4>(d[e]);
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = REV ? (float)r.x.v[e] : d[e] * (float)r.x.v[e];
    if (REV && p.z.p)
#pragma unroll
      for (int e = 0; e < E; ++e) u[e] *= silu<sizeof(T) == 4>((float)r.z.v[e]);
    float *const d_ = sd[k & 1] + at<L>(cl, tl), *const u_ = su[k & 1] + at<L>(cl, tl);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool counts = there && e < here;
      d_[e * (L + 4)] = counts ? d[e] : 0.f;
      u_[e * (L + 4)] = counts ? u[e] : 0.f;
    }
    r.B.lay(sB[k & 1], tid);
    if (OUT) r.C.lay(sC[k & 1], tid);
  };
  auto finish = [&](int k) {
    const int t = begin(k) + tl;
    const float* const y_ = sy[k & 1] + (OUT ? at<L>(cl, tl) : 0);
    Row<T, E> out;
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      y[e] = y_[e * (L + 4)];
#pragma unroll
      for (int i = 1; i < NB; ++i) y[e] += y_[i * PL + e * (L + 4)];
      y[e] = skip ? fmaf(D[e], (float)before.x.v[e], y[e]) : y[e];
    }
    if (p.z.p)
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] *= silu<sizeof(T) == 4>((float)before.z.v[e]);
#pragma unroll
    for (int e = 0; e < E; ++e) out.v[e] = (T)(t < end ? y[e] : 0.f);
    if constexpr (WIDE) out.give(buffer_of((T*)p.y + ((size_t)b * p.T + begin(k)) * p.C, p.C, min(last - begin(k), L)), yw);
    else if (t < last && here > 0) out.store((T*)p.y + ((size_t)b * p.T + t) * p.C + cr, false, here);
  };
  auto turn = [&](int k, In& r) {                // r: of chunk k + 1
    Row<T, E> nx, nz;
    if (k + 1 < chunks) lay(k + 1, r);
    if (OUT) nx = r.x, nz = r.z;
    load(k + 3, r);
    if (OUT) {
      if (k > 0) finish(k - 1);
      before = now;
      now.x = nx, now.z = nz;
    }
    __syncthreads();
  };
  if (chunks > 0) {
    load(0, in[0]);
    load(1, in[1]);
    lay(0, in[0]);
    now.x = in[0].x, now.z = in[0].z;
    load(2, in[0]);
  }
  __syncthreads();
  for (int k = 0; k < chunks; k += 2) {
    turn(k, in[1]);
    if (k + 1 < chunks) turn(k + 1, in[0]);
  }
  if (!OUT) return;
  if (chunks > 0) finish(chunks - 1);
  Row<T, E> none;                        // tokens that do not count
  none.zero();
  for (int t = first + chunks * L + tl; t < last; t += L)
    if (here > 0) none.store((T*)p.y + ((size_t)b * p.T + t) * p.C + cr, WIDE, here);
}

// The gradients.  Chunks of kSave tokens against the time: forwards through a chunk from the state kept in front of it, powers and states in
// registers, then back.  A quad of lanes shares a channel: sums over its states cross the quad, sums over channels (of dB and dC) the 16 quads.
//
// Bound by the wave of a pipe that goes through the tokens, which never waits for the others: 19 vector instructions for a state of a token (four on the way there,
// nine on the way back, six for the sums across lanes), 4.5 cycles each and 8.5 for powers and exchanges, and 80 accesses to LDS a chunk.  Eight waves of
// two states a lane have more of both and are slower (us of a training step 647 in place of 552).  Outputs in front of the gate, one more and the sums, are
// found only where its gradient is wanted (541 us without a gate, 513 so).  93 KB of LDS and 250 registers: one workgroup a
// unit.  Eight sequences of 2048 tokens of 2048 channels, 16 states, gate, bf16: 412 us (540 MB with the sums of dB and dC: 102 at the rate of a copy).
template <typename T, int NL, int NB, bool WIDE>
__global__ __launch_bounds__(512) void ring_scan_bwd_kernel(RingScanArgs p) {
  constexpr int CH = 64 / NB, L = kSave, E = CH / 16, NS = 4 * NL * NB, PL = plane<CH, L>(), CW = 4 / NB, R = 8 * NL;
  __shared__ __attribute__((aligned(16))) float sd[2][PL], su[2][PL], sq[2][PL], sB[2][L * NS], sC[2][L * NS], so[2][3 * NB * PL], red[2][4 * L * R],
      sums[32 * CH];
  const int tid = threadIdx.x & 255, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at_ = place<CH>(p);
  const int seg = at_.seg, b = at_.b;
  const int len = length_of(p.lengths, b, p.T), first = seg * p.seg_tokens, last = min(first + p.seg_tokens, p.T), end = min(last, len);
  const int chunks = end > first ? (end - first + L - 1) / L : 0;
  const bool shared = p.part_bc != nullptr;
  auto begin = [&](int k) { return first + (chunks - 1 - k) * L; };
  float* const part = p.part_a ? p.part_a + ((size_t)seg * p.B + b) * p.C * (NS + 2) : nullptr;
  if (w < 4) {
    const int nb = w % NB, ch = w / NB * 16 + (lane >> 2), sub = lane & 3, n0 = nb * 4 * NL + sub * NL, c = at_.c0 + ch;
    const bool mine = ch < at_.here;
    float A2[NL], G[NL], dA[NL], hk[NL];   // hk: the state kept in front of the next chunk
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      A2[n] = mine && n0 + n < p.N ? times_log2e(p.A[(size_t)c * p.N + n0 + n]) : 0.f;
      G[n] = dA[n] = hk[n] = 0.f;
      if (mine) {
        if (seg < p.nseg - 1) G[n] = p.seg[(((size_t)(p.nseg - 2 - seg) * p.B + b) * p.C + c) * NS + n0 + n];
        else if (p.s_in && n0 + n < p.N) G[n] = p.s_in[((size_t)b * p.C + c) * p.N + n0 + n];
      }
    }
    auto kept = [&](int k) {
      take<NL>(hk, p.states + (((size_t)b * p.saved + begin(min(k, chunks - 1)) / kSave) * p.C + (mine ? c : at_.c0)) * NS + n0);
    };
    if (chunks > 0) kept(0);
    __syncthreads();
    const int r = lane >> 4, quad = lane >> 2 & 3;
    auto chunk = [&](int k, auto whole, auto gated) {      // gated: the outputs in front of the gate are wanted, for its gradient
      constexpr bool GATED = decltype(gated)::value;
      const int t0 = begin(k), f = k & 1;
      float h[NL], hs[L][NL], as[L][NL], dAc[NL];
#pragma unroll
      for (int n = 0; n < NL; ++n) {
        h[n] = mine ? hk[n] : 0.f;
        dAc[n] = 0.f;
      }
      kept(k + 1);
      const float *d_ = sd[f] + at<L>(ch, 0), *u_ = su[f] + at<L>(ch, 0), *q_ = sq[f] + at<L>(ch, 0), *B_ = sB[f] + n0, *C_ = sC[f] + n0;
      float* const o_ = so[f] + nb * PL + at<L>(ch, sub);
      // where a lane's sums of dB and dC lie: row r has type r >> 1 and, of four states, half r & 1; quads have values (0, 2, 1, 3) of four
      constexpr int LEFT = NL > 1 ? NL / 2 : 1, VAL = 4 * LEFT;
      const int mine4 = quad >> 1 | (quad & 1) << 1;
      float* const r_ = red[f] + w * L * R + (r >> 1) * 4 * NL + sub * NL + (NL > 1 ? (r & 1) * LEFT : 0) + mine4 / LEFT * R + mine4 % LEFT;
      // (what the next tokens need is on its way from LDS, as forwards: four tokens on the way there, two back, where the registers are full)
      struct Four { f32x4 d, u; float B[4][NL]; } g[2];
      auto fetch = [&](int j, Four& x) {
        x.d = *reinterpret_cast<const f32x4*>(d_ + j);
        x.u = *reinterpret_cast<const f32x4*>(u_ + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) take<NL>(x.B[i], B_ + (j + i) * NS);
      };
      struct Two { float B[2][NL], C[2][NL]; } two[2];
      auto fetch_two = [&](int j, Two& x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          take<NL>(x.B[i], B_ + (j + i) * NS);
          take<NL>(x.C[i], C_ + (j + i) * NS);
        }
      };
      fetch(0, g[0]);
#pragma unroll
      for (int j = 0; j < L; j += 4) {
        const Four& x = g[j / 4 & 1];
        if (j + 4 < L) fetch(j + 4, g[j / 4 + 1 & 1]);
        else fetch_two(L - 2, two[1]);
        __builtin_amdgcn_sched_barrier(0);
        float v[4][NL];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NL; ++n) as[j + i][n] = x.d[i] * A2[n];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NL; ++n) {
            as[j + i][n] = __builtin_amdgcn_exp2f(as[j + i][n]);
            v[i][n] = x.u[i] * x.B[i][n];
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NL; ++n) {
            hs[j + i][n] = h[n];
            h[n] = fmaf(as[j + i][n], h[n], v[i][n]);
          }
        __builtin_amdgcn_sched_barrier(0);
      }
      f32x4 d4, u4, q4;
      auto fetch_rows = [&](int j) {
        d4 = *reinterpret_cast<const f32x4*>(d_ + j);
        u4 = *reinterpret_cast<const f32x4*>(u_ + j);
        q4 = *reinterpret_cast<const f32x4*>(q_ + j);
      };
      fetch_rows(L - 4);
#pragma unroll
      for (int j = L - 4; j >= 0; j -= 4) {
        float s1[4], s2[4], y[4], val[VAL];
#pragma unroll
        for (int half = 1; half >= 0; --half) {
          const Two& x = two[half];
          if (j + 2 * half > 0) fetch_two(j + 2 * half - 2, two[1 - half]);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 2 * half + 1; i >= 2 * half; --i) {
            float v[2 * NL];
            const float(&Bn)[NL] = x.B[i & 1], (&Cn)[NL] = x.C[i & 1];
            // (behind the last token that counts no state takes part in dA, however large)
            if constexpr (!decltype(whole)::value)
              if (t0 + j + i + 1 == end)
#pragma unroll
                for (int n = 0; n < NL; ++n) dAc[n] = 0.f;
#pragma unroll
            for (int n = 0; n < NL; ++n) {
              if constexpr (GATED) y[i] = n == 0 ? Cn[n] * h[n] : fmaf(Cn[n], h[n], y[i]);
              v[NL + n] = q4[i] * h[n];
              const float gn = fmaf(q4[i], Cn[n], G[n]);
              v[n] = gn * u4[i];
              s1[i] = n == 0 ? gn * Bn[n] : fmaf(gn, Bn[n], s1[i]);
              G[n] = as[j + i][n] * gn;
              h[n] = hs[j + i][n];
              const float turn = G[n] * h[n];
              s2[i] = n == 0 ? turn * A2[n] : fmaf(turn, A2[n], s2[i]);
              dAc[n] = fmaf(d4[i], turn, dAc[n]);
            }
            // over the 16 quads: halves, rows
#pragma unroll
            for (int n = 0; n < NL; ++n) v[n] = fold32(v[n], v[NL + n]);
#pragma unroll
            for (int n = 0; n < LEFT; ++n) val[i * LEFT + n] = fold16(v[n], NL > 1 ? v[NL / 2 + n] : v[n]);
          }
          if (half == 0 && j > 0) fetch_rows(j - 4);
        }
        // over a quad, whose lane sub is left with token j + sub
        o_[j] = quad_sums(s1, sub);
        o_[NB * PL + j] = quad_sums(s2, sub);
        if constexpr (GATED) o_[2 * NB * PL + j] = quad_sums(y, sub);
        // over a row's quads
#pragma unroll
        for (int m = 0; m < LEFT; ++m) r_[(j + m * 4 / LEFT) * R] = row_sums(val + 4 * m, quad);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int n = 0; n < NL; ++n) dA[n] += dAc[n];
      __syncthreads();
    };
    int k = 0;
    if (chunks > 0 && begin(0) + L > end) chunk(k++, std::false_type{}, std::true_type{});
    if (p.dz)
      for (; k < chunks; ++k) chunk(k, std::true_type{}, std::true_type{});
    else
      for (; k < chunks; ++k) chunk(k, std::true_type{}, std::false_type{});
    if (mine) {
      if (part) {
#pragma unroll
        for (int n = 0; n < NL; ++n) part[(size_t)c * (NS + 2) + n0 + n] = dA[n];
      }
      if (seg == 0 && p.s_out) {
#pragma unroll
        for (int n = 0; n < NL; ++n)
          if (n0 + n < p.N) p.s_out[((size_t)b * p.C + c) * p.N + n0 + n] = G[n];
      }
    }
    __syncthreads();
    return;
  }
  const int tl = tid >> 4, cl = (tid & 15) * E, cr = at_.c0 + cl, here = at_.here - cl;
  float D[E], bias[E], dD[E], dbias[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    D[e] = p.D && e < here ? p.D[cr + e] : 0.f;
    bias[e] = p.bias && e < here ? p.bias[cr + e] : 0.f;
    dD[e] = dbias[e] = 0.f;
  }
  struct In { Row<T, E> x, d, z, y; Shared<T, L, NS> B, C; } in[2];      // of the next two chunks, as forwards
  struct Known { Row<T, E> x, z, y; float d[E], q[E], slope[E], gate[E]; } next, now, before;      // of the one just laid down, of the one under way, of the one before
  const int tr = here > 0 ? here : at_.here, cw = here > 0 ? cr : at_.c0;
  const T *const dp = (const T*)p.delta.p + b * p.delta.sb, *const xp = (const T*)p.x.p + b * p.x.sb,
          *const yp = (const T*)p.dy.p + b * p.dy.sb, *const zp = p.z.p ? (const T*)p.z.p + b * p.z.sb : xp;
  const long zt = p.z.p ? p.z.st : p.x.st;
  const T* const Bp = (const T*)p.Bm + (size_t)b * p.bsb + (size_t)at_.g * p.bsg;
  const T* const Cp = (const T*)p.Cm + (size_t)b * p.csb + (size_t)at_.g * p.csg;
  typedef Shared<T, L, NS> Sh;
  const int dw = (int)((tl * p.delta.st + cw) * (long)sizeof(T)), xw = (int)((tl * p.x.st + cw) * (long)sizeof(T)), zw = (int)((tl * zt + cw) * (long)sizeof(T)),
            yw = (int)((tl * p.dy.st + cw) * (long)sizeof(T)), ow = here > 0 ? (int)((tl * (long)p.C + cr) * (long)sizeof(T)) : kOutside;
  int Bw[Sh::NV], Cw[Sh::NV];
#pragma unroll
  for (int i = 0; i < Sh::NV; ++i) {
    Bw[i] = Sh::place(i, p.bst, p.N, tid);
    Cw[i] = Sh::place(i, p.cst, p.N, tid);
  }
  auto load = [&](int k, In& r) {
    const int t0 = begin(min(k, chunks - 1)), rows = min(end - t0, L);
    if constexpr (WIDE) {
      r.d.fetch(buffer_of(dp + t0 * p.delta.st, p.delta.st, rows), dw);
      r.x.fetch(buffer_of(xp + t0 * p.x.st, p.x.st, rows), xw);
      r.z.fetch(buffer_of(zp + t0 * zt, zt, rows), zw);
      r.y.fetch(buffer_of(yp + t0 * p.dy.st, p.dy.st, rows), yw);
      r.B.fetch(buffer_of(Bp + t0 * p.bst, p.bst, rows), Bw);
      r.C.fetch(buffer_of(Cp + t0 * p.cst, p.cst, rows), Cw);
    } else {
      const long t = min(t0 + tl, end - 1);
      r.d.read(dp + cw + t * p.delta.st, tr);
      r.x.read(xp + cw + t * p.x.st, tr);
      r.z.read(zp + cw + t * zt, tr);
      r.y.read(yp + cw + t * p.dy.st, tr);
      r.B.load(Bp, p.bst, t0, end, p.N, tid);
      r.C.load(Cp, p.cst, t0, end, p.N, tid);
    }
  };
  auto lay = [&](int k, const In& r) {
    const bool there = begin(k) + tl < end;
    float d[E], q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      d[e] = (float)r.d.v[e] + bias[e];
      q[e] = (float)r.y.v[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) next.slope[e] = next.gate[e] = 1.f;
    if (p.softplus)
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = softplus<sizeof(T) == 4>(d[e], next.slope[e]);
    if (p.z.p)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        next.gate[e] = sigmoid<sizeof(T) == 4>((float)r.z.v[e]);
        q[e] *= (float)r.z.v[e] * next.gate[e];
      }
    float *const d_ = sd[k & 1] + at<L>(cl, tl), *const u_ = su[k & 1] + at<L>(cl, tl), *const q_ = sq[k & 1] + at<L>(cl, tl);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool counts = there && e < here;
      d_[e * (L + 4)] = counts ? d[e] : 0.f;
      u_[e * (L + 4)] = counts ? d[e] * (float)r.x.v[e] : 0.f;
      q_[e * (L + 4)] = counts ? q[e] : 0.f;
      next.d[e] = d[e];
      next.q[e] = q[e];
    }
    next.x = r.x, next.z = r.z, next.y = r.y;
    r.B.lay(sB[k & 1], tid);
    r.C.lay(sC[k & 1], tid);
  };
  const int tile = (at_.c0 - at_.g * (p.C / p.G)) / CH;
  auto finish = [&](int k) {
    const int t0 = begin(k), t = t0 + tl, f = k & 1;
    const float* const o_ = so[f] + at<L>(cl, tl);
    Row<T, E> ox, od, oz;
    float s1[E], s2[E], dd[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s1[e] = s2[e] = 0.f;
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        s1[e] += o_[i * PL + e * (L + 4)];
        s2[e] += o_[(NB + i) * PL + e * (L + 4)];
      }
      dd[e] = fmaf(s1[e], (float)before.x.v[e], s2[e] * kLn2) * before.slope[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool counts = t < end && e < here;
      const float x = (float)before.x.v[e];
      ox.v[e] = (T)(counts ? fmaf(D[e], before.q[e], before.d[e] * s1[e]) : 0.f);
      od.v[e] = (T)(counts ? dd[e] : 0.f);
      dD[e] = counts ? fmaf(before.q[e], x, dD[e]) : dD[e];
      dbias[e] = counts ? dbias[e] + dd[e] : dbias[e];
    }
    if (p.dz)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float y = o_[2 * NB * PL + e * (L + 4)];
#pragma unroll
        for (int i = 1; i < NB; ++i) y += o_[(2 * NB + i) * PL + e * (L + 4)];
        const float g = (float)before.y.v[e] * fmaf(D[e], (float)before.x.v[e], y) * silu_slope((float)before.z.v[e], before.gate[e]);
        oz.v[e] = (T)(t < end && e < here ? g : 0.f);
      }
    if constexpr (WIDE) {
      const size_t row = ((size_t)b * p.T + t0) * p.C;
      const int rows = min(last - t0, L);
      if (p.dx) ox.give(buffer_of((T*)p.dx + row, p.C, rows), ow);
      if (p.ddelta) od.give(buffer_of((T*)p.ddelta + row, p.C, rows), ow);
      if (p.dz) oz.give(buffer_of((T*)p.dz + row, p.C, rows), ow);
    } else if (t < last && here > 0) {
      const size_t row = ((size_t)b * p.T + t) * p.C + cr;
      if (p.dx) ox.store((T*)p.dx + row, false, here);
      if (p.ddelta) od.store((T*)p.ddelta + row, false, here);
      if (p.dz) oz.store((T*)p.dz + row, false, here);
    }
    if (shared)
      for (int i = tid; i < L * 2 * NS; i += 256) {
        const int tk = i / (2 * NS), type = i / NS % 2, n = i % NS, block = n / (4 * NL);
        float sum = 0.f;
#pragma unroll
        for (int m = 0; m < CW; ++m) sum += red[f][((m * NB + block) * L + tk) * R + type * 4 * NL + n % (4 * NL)];
        if (t0 + tk < end) p.part_bc[((((size_t)tile * p.B + b) * p.T + t0 + tk) * p.G + at_.g) * 2 * NS + type * NS + n] = sum;
      }
  };
  auto turn = [&](int k, In& r) {                // r: of chunk k + 1
    if (k + 1 < chunks) lay(k + 1, r);
    load(k + 3, r);
    if (k > 0) finish(k - 1);
    before = now;
    now = next;
    __syncthreads();
  };
  if (chunks > 0) {
    load(0, in[0]);
    load(1, in[1]);
    lay(0, in[0]);
    now = next;
    load(2, in[0]);
  }
  __syncthreads();
  for (int k = 0; k < chunks; k += 2) {
    turn(k, in[1]);
    if (k + 1 < chunks) turn(k + 1, in[0]);
  }
  if (chunks > 0) finish(chunks - 1);
  Row<T, E> none;                        // tokens that do not count
  none.zero();
  for (int t = first + chunks * L + tl; t < last; t += L)
    if (here > 0) {
      const size_t row = ((size_t)b * p.T + t) * p.C + cr;
      if (p.dx) none.store((T*)p.dx + row, WIDE, here);
      if (p.ddelta) none.store((T*)p.ddelta + row, WIDE, here);
      if (p.dz) none.store((T*)p.dz + row, WIDE, here);
    }
  // the 16 threads of a channel, in order
#pragma unroll
  for (int e = 0; e < E; ++e) {
    sums[tl * CH + cl + e] = dD[e];
    sums[16 * CH + tl * CH + cl + e] = dbias[e];
  }
  __syncthreads();
  if (part && tid < 2 * CH && tid % CH < at_.here) {
    float sum = 0.f;
    for (int i = 0; i < 16; ++i) sum += sums[tid / CH * 16 * CH + i * CH + tid % CH];
    part[(size_t)(at_.c0 + tid % CH) * (NS + 2) + NS + tid / CH] = sum;
  }
}

template <typename T, int NL, int NB, bool WIDE> hipError_t launch_sized(const RingScanArgs& p, int mode, hipStream_t st) {
  const int CH = 64 / NB;
  RingScanArgs a = p;
  a.tiles = (p.C / p.G + CH - 1) / CH;
  const int segs = mode == RING_SCAN_STATE || mode == RING_SCAN_ADJOINT ? p.nseg - 1 : p.nseg;
  const dim3 grid((unsigned)((size_t)a.tiles * p.G * p.B * segs)), block(512);
  if (mode == RING_SCAN_OUTPUTS) hipLaunchKernelGGL((ring_scan_kernel<T, NL, NB, kOutputs, WIDE>), grid, block, 0, st, a);
  else if (mode == RING_SCAN_STATE) hipLaunchKernelGGL((ring_scan_kernel<T, NL, NB, kState, WIDE>), grid, block, 0, st, a);
  else if (mode == RING_SCAN_ADJOINT) hipLaunchKernelGGL((ring_scan_kernel<T, NL, NB, kAdjoint, WIDE>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((ring_scan_bwd_kernel<T, NL, NB, WIDE>), grid, block, 0, st, a);
  return hipGetLastError();
}

template <typename T, bool WIDE> hipError_t launch_rows(const RingScanArgs& p, int mode, hipStream_t st) {
  if (p.N <= 4) return launch_sized<T, 1, 1, WIDE>(p, mode, st);
  if (p.N <= 8) return launch_sized<T, 2, 1, WIDE>(p, mode, st);
  if (p.N <= 16) return launch_sized<T, 4, 1, WIDE>(p, mode, st);
  if (p.N <= 32) return launch_sized<T, 4, 2, WIDE>(p, mode, st);
  return launch_sized<T, 4, 4, WIDE>(p, mode, st);
}

template <typename T> hipError_t launch(const RingScanArgs& p, int mode, hipStream_t st) {
  return p.wide ? launch_rows<T, true>(p, mode, st) : launch_rows<T, false>(p, mode, st);
}

}  // namespace ring_scan
