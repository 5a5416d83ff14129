// Linear attention with a decay for each head: the passes of a forward and of a backward, and the single token.
#include "ring_linattn.hpp"
#include "ringattr.h"

#include <math.h>

using namespace ring_lin;

namespace {

constexpr int kChunk = 64;            // segments are whole numbers of these tokens
// Of so many segments the second adds what the first has added to the initial state itself; of more a scan does, a launch more but less to read
// (8 x 4096 tokens, 16 heads of 128, bf16, in four segments, us a pass of the chunk kernel: 129 behind a scan of 14; adding up itself took 35 more).
constexpr int kFold = 2;

size_t round_up(size_t x) { return (x + 255) / 256 * 256; }

hipError_t launch_pass(int type, const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  if (type == RINGATTR_F32) return ring_launch_linattn_f32(a, rev, state_only, st);
  if (type == RINGATTR_BF16) return ring_launch_linattn_bf16(a, rev, state_only, st);
  return ring_launch_linattn_f16(a, rev, state_only, st);
}

// A head's columns go to workgroups of 64 where there are no more, else of 128: in slices of 64 a wide head needs fewer segments, but
// forms its weights twice as often (us of a forward, and with its backward, each in its best number of segments, 128 and 64: 8 x 4096
// tokens, 16 heads of 128, bf16 195, 618 and 204, 708; 8 x 2000 tokens, 8 heads of 256, fp32 441, 1639 and 489, 2013; 16 x 1000 tokens, 8
// heads of 128, fp32 139, 472 and 136, 499).
int slices(int Db) { return Db <= 64 ? 1 : (Db + 127) / 128; }

void set_columns(RingLinArgs& a, int Db, bool narrow) {
  a.Db = Db;
  a.narrow = narrow || Db <= 64;
  a.slices = a.narrow ? (Db + 63) / 64 : (Db + 127) / 128;
}

RingLinArgs base(const RingLinShape& s, const float* log_decay, const int* lengths, int nseg) {
  RingLinArgs a = {};
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.B = s.B;
  a.T = s.T;
  a.H = s.H;
  a.nseg = nseg;
  a.scanned = nseg > kFold;
  const int chunks = (s.T + kChunk - 1) / kChunk;
  a.seg_tokens = nseg > 1 ? (chunks + nseg - 1) / nseg * kChunk : (s.T > 0 ? s.T : 1);
  a.intra = a.inter = a.update = 1.f;
  return a;
}

// a token's outputs of all heads are less than 16 MiB
bool out_fits(const RingLinArgs& a) { return (long)a.H * a.Db < (1 << 22); }

}  // namespace

// What the segments add to a state of zeros becomes the states behind them, in place.  A thread walks one element through them, eight
// reads ahead; bound by their memory and, of few heads, by the walk (16 heads of 128, 15 segments: 31 MB, 11 us).
__global__ __launch_bounds__(256) void ring_linattn_scan_kernel(RingLinArgs p, bool rev) {
  const int D = p.Da * p.Db, ns = p.nseg - 1;
  const int per = (D + 255) / 256, e = (int)(blockIdx.x % per) * 256 + threadIdx.x;
  const size_t bh = blockIdx.x / per;
  if (e >= D) return;
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const float g2 = (float)((double)p.log_decay[h] * 1.4426950408889634);
  float* seg = p.seg + bh * ns * D + e;
  float run = p.s_in ? p.s_in[bh * D + e] : 0.f;
#pragma unroll 8
  for (int u = 0; u < ns; ++u) {
    const int ts = (rev ? p.nseg - 1 - u : u) * p.seg_tokens, n = min(max(len - ts, 0), p.seg_tokens);
    const float local = seg[(size_t)u * D];
    if (n > 0) run = fmaf(power(g2, n), run, local);
    seg[(size_t)u * D] = run;
  }
}

// out[row][g][d] = sum over the heads that share g, in their order; bound by memory.  (Sums of heads inside the kernel that finds them
// would take a workgroup through all heads of a group, or atomics, whose order changes results.)
template <typename T>
__global__ __launch_bounds__(256) void ring_linattn_share_kernel(const float* __restrict__ in, T* __restrict__ out, int share, int D, size_t n) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
    const size_t row = i / D, d = i - row * D;                 // (row, shared head)
    const float* p = in + row * share * D + d;
    float sum = 0.f;
    for (int s = 0; s < share; ++s) sum += p[(size_t)s * D];
    out[i] = (T)sum;
  }
}

static hipError_t launch_share(int type, const float* in, void* out, int share, int D, size_t n, hipStream_t st) {
  const size_t blocks = (n + 255) / 256;
  const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192)), block(256);
  if (type == RINGATTR_F32) hipLaunchKernelGGL(ring_linattn_share_kernel<float>, grid, block, 0, st, in, (float*)out, share, D, n);
  else if (type == RINGATTR_BF16) hipLaunchKernelGGL(ring_linattn_share_kernel<__bf16>, grid, block, 0, st, in, (__bf16*)out, share, D, n);
  else hipLaunchKernelGGL(ring_linattn_share_kernel<_Float16>, grid, block, 0, st, in, (_Float16*)out, share, D, n);
  return hipGetLastError();
}

// A single token: S = lambda S + k v^T in place, o = scale q S.  A workgroup takes `tc` lanes of V columns each of one state; its other
// lanes share the rows.  Nothing but the state moves: read once, written once: bound by memory, 93 us for 256 x 16 heads of 128 (537 MB,
// 5.8 TB/s); few heads are cut into narrower slices (us, cut and in whole rows: 8 heads of 64 3.1, 5.2; 16 of 128
// 3.6, 7.5; 16 x 16 of 128 7.1, 8.9), as long as that makes no more than about 1024 workgroups.
template <typename T, int V>
__global__ __launch_bounds__(256) void ring_linattn_step_kernel(RingLinStep p, RingLinShape s, int tc) {
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ vec part[256];
  const int tid = threadIdx.x, lane = tid & (tc - 1), tr = tid / tc, nr = 256 / tc;
  const int ns = (s.Dv + tc * V - 1) / (tc * V);
  const int slice = blockIdx.x % ns;
  const size_t bh = blockIdx.x / ns;
  const int h = (int)(bh % s.H), b = (int)(bh / s.H), share = s.H / s.G;
  const int c = (slice * tc + lane) * V;
  T* out = (T*)p.out + bh * s.Dv + c;
  if (p.active && !p.active[b]) {
    if (tr == 0 && c < s.Dv)
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = (T)0.f;
    return;
  }
  const T* q = rows_of<T>(p.q, b, h, 1);
  const T* k = rows_of<T>(p.k, b, h, share);
  const T* v = rows_of<T>(p.v, b, h, share);
  const float lam = power((float)((double)p.log_decay[h] * 1.4426950408889634), 1);
  vec o, x;
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = x[e] = 0.f;
  if (c < s.Dv) {
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = (float)v[c + e];
    float* S = p.state + bh * s.Dk * s.Dv + c;
#pragma unroll 8
    for (int a = tr; a < s.Dk; a += nr) {
      vec* at = reinterpret_cast<vec*>(S + (size_t)a * s.Dv);
      const float ka = (float)k[a], qa = (float)q[a];
      vec y = *at;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        y[e] = fmaf(ka, x[e], lam * y[e]);
        o[e] = fmaf(qa, y[e], o[e]);
      }
      *at = y;
    }
  }
  part[tid] = o;
  __syncthreads();
  for (int half = nr / 2; half > 0; half /= 2) {
    if (tr < half) part[tid] += part[tid + half * tc];
    __syncthreads();
  }
  if (tr == 0 && c < s.Dv)
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = (T)(s.scale * part[tid][e]);
}

template <typename T> static hipError_t launch_step(const RingLinShape& s, const RingLinStep& a, hipStream_t st) {
  const bool vec = s.Dv % 4 == 0 && (reinterpret_cast<uintptr_t>(a.state) & 15) == 0;
  const int width = vec ? (s.Dv + 3) / 4 : s.Dv;               // lanes that a row of the state takes
  const long heads = (long)s.B * s.H;
  int tc = 8;
  while (tc < width && tc < 64 && heads * ((width + tc - 1) / tc) > 1024) tc *= 2;
  const dim3 grid((unsigned)(heads * ((width + tc - 1) / tc))), block(256);
  if (vec) hipLaunchKernelGGL((ring_linattn_step_kernel<T, 4>), grid, block, 0, st, a, s, tc);
  else hipLaunchKernelGGL((ring_linattn_step_kernel<T, 1>), grid, block, 0, st, a, s, tc);
  return hipGetLastError();
}

hipError_t ring_linattn_step(const RingLinShape& s, const RingLinStep& a, hipStream_t st) {
  if (s.type == RINGATTR_F32) return launch_step<float>(s, a, st);
  if (s.type == RINGATTR_BF16) return launch_step<__bf16>(s, a, st);
  return launch_step<_Float16>(s, a, st);
}

// Into how many segments the tokens are cut so that there is work for all compute units: the number with the least expected time of a
// forward.  What it is made of, in us, as measured (P: 64, 128 or 256, what the kernels round a head's widths up to):
//   a chunk of 32 tokens, a workgroup alone on its compute unit: bf16 1.2, 2.0, 3.5; fp32 products 2.8, 6.2, 12
//   two workgroups on a compute unit: 1.2 of one's time with P = 64, 1.86 with P = 128 (1.6 where a quarter of them have two); with P = 256
//   they follow each other
//   but no less than the rows take from memory, at 5 TB/s
//   the pass over states: 0.34 (bf16) or 0.4 of a chunk, and 6 or (P > 64) 10 for its launch and what the pass behind reads of it
//   the scan (more than kFold segments): 3 or 5, 0.2 a segment, and its states at 5 TB/s
// us of a forward with its final state, and with its backward, by segments, the rule's choice in brackets:
//   8 x 4096 tokens, 16 heads of 128, bf16    1: 282, 937   [2: 214, 625]    3: 211, 712    4: 196, 628    8: 228, 707
//   1 x 32768 tokens, 16 heads of 128, bf16   1: 2219, 7301  8: 390, 1178  [16: 227, 677]  32: 220, 680   64: 243, 746
//   1 x 8192 tokens, 8 heads of 128, bf16     1: 551, 1833   8: 107, 312    16: 68, 191   [32: 55, 147]   64: 63, 178
//   8 x 2048 tokens, 16 heads of 64, bf16     1: 81, 262     2: 66, 189     3: 61, 180    [4: 51, 149]    8: 52, 159
//   8 x 2000 tokens, 8 heads of 256, fp32     1: 686, 2792  [2: 455, 1637]  4: 532, 1858    8: 621, 2109
//   3 x 4096 tokens, 8 heads of 256, bf16     1: 502, 1868   4: 196, 633   [5: 162, 536]    8: 207, 697   16: 221, 698
//   20 x 4096 tokens, 16 heads of 128, bf16  [1: 430, 1612]  2: 457, 1531   4: 496, 1605
//   2 x 1000 tokens, 4 heads of 64, fp32      1: 91, 308     8: 28, 146   [16: 26, 145]
static int segments(const RingLinShape& s) {
  const int units = (s.T + kChunk - 1) / kChunk;
  const int widest = s.Dk > s.Dv ? s.Dk : s.Dv, P = widest <= 64 ? 64 : (widest <= 128 ? 128 : 256);
  const double heads = (double)s.B * s.H, groups = heads * slices(s.Dv);
  const bool bf16 = s.type == RINGATTR_BF16;
  const double chunk = bf16 ? 0.45 + 0.0118 * P : 0.047 * P;
  const double rows = heads * s.T * (s.Dk + s.Dv) * (s.type == RINGATTR_F32 ? 4 : 2) / 5e6;      // Y and Z once
  auto rounds = [&](double work) {                             // in times of a workgroup alone
    const double two = P == 64 ? 1.2 : (P == 128 ? 1.86 : 2.0), full = floor(work / 512), rest = work - 512 * full;
    return full * two + (rest == 0 ? 0.0 : (rest <= 256 ? 1.0 : (rest <= 384 && P == 128 ? 1.6 : two)));
  };
  auto no_less = [](double a, double b) { return a > b ? a : b; };
  int best = 1;
  double time = 0.0;
  for (int n = 1; n <= 64 && n <= units; ++n) {
    const int per = (units + n - 1) / n;
    if ((units + per - 1) / per != n) continue;
    double t = no_less(2 * per * chunk * rounds(groups * n), 2 * rows);
    if (n > 1) t += no_less((bf16 ? 0.68 : 0.8) * per * chunk * rounds(groups * (n - 1)), rows * (n - 1) / n) + (P == 64 ? 6 : 10);
    if (n > kFold) t += (P == 64 ? 3 : 5) + 0.2 * n + heads * n * s.Dk * s.Dv * 8 / 5e6;
    if (n == 1 || t < time) {
      time = t;
      best = n;
    }
  }
  return best;
}

static size_t states_bytes(const RingLinShape& s) {
  return round_up((size_t)s.B * s.H * (segments(s) - 1) * s.Dk * s.Dv * sizeof(float));
}

size_t ring_linattn_fwd_bytes(const RingLinShape& s) { return states_bytes(s); }

size_t ring_linattn_bwd_bytes(const RingLinShape& s, bool have_states) {
  size_t n = (have_states ? 1 : 2) * states_bytes(s);
  if (s.G != s.H) n += round_up((size_t)s.B * s.T * s.H * s.Dk * sizeof(float)) + round_up((size_t)s.B * s.T * s.H * s.Dv * sizeof(float));
  return n;
}

static hipError_t launch_two(int type, const RingLinArgs& a, hipStream_t st) {
  if (type == RINGATTR_F32) return ring_launch_linattn_pair_f32(a, st);
  if (type == RINGATTR_BF16) return ring_launch_linattn_pair_bf16(a, st);
  return ring_launch_linattn_pair_f16(a, st);
}

// What the segments of Y and Z add to a state (natural states, [Dk][Dv]), or the states behind them, into a.seg.  64 columns a
// workgroup: nothing is formed twice for it, and there are fewer segments here than in the pass behind (us: 8 x 2000 tokens, 8 heads of
// 256, fp32 220 -> 139; 8 x 4096 tokens, 16 heads of 128, bf16 68 -> 61; one sequence of 32768 71 -> 72).  fp32 products take chunks of
// twice the tokens (139 -> 121; bf16 72 -> 77).
static hipError_t segment_states(const RingLinShape& s, RingLinArgs a, bool rev, hipStream_t st) {
  if (a.nseg == 1) return hipSuccess;
  a.Da = s.Dk;
  a.sa = s.Dv;
  a.sb = 1;
  set_columns(a, s.Dv, true);
  hipError_t e = launch_pass(s.type, a, rev, true, st);
  if (e != hipSuccess || !a.scanned) return e;
  const unsigned per = (unsigned)((s.Dk * s.Dv + 255) / 256);
  hipLaunchKernelGGL(ring_linattn_scan_kernel, dim3((unsigned)((size_t)per * s.B * s.H)), dim3(256), 0, st, a, rev);
  return hipGetLastError();
}

hipError_t ring_linattn_fwd(const RingLinShape& s, const RingLinTensor& q, const RingLinTensor& k, const RingLinTensor& v,
                            const float* log_decay, const float* s_in, const int* lengths, void* o, float* s_out, void* ws, hipStream_t st) {
  const int nseg = segments(s), epv = s.type == RINGATTR_F32 ? 4 : 8;
  RingLinArgs a = base(s, log_decay, lengths, nseg);
  a.X = q;
  a.Y = k;
  a.Z = v;
  a.xs = 1;
  a.ys = a.zs = s.H / s.G;
  a.s_in = s_in;
  a.s_out = s_out;
  a.seg = (float*)ws;
  hipError_t e = segment_states(s, a, false, st);
  if (e != hipSuccess) return e;
  a.Da = s.Dk;
  a.sa = s.Dv;
  a.sb = 1;
  set_columns(a, s.Dv, false);
  a.out = o;
  a.out_vec = a.Db % epv == 0 && out_fits(a);
  a.intra = a.inter = s.scale;
  return launch_pass(s.type, a, false, false, st);
}

hipError_t ring_linattn_bwd(const RingLinShape& s, const RingLinTensor& q, const RingLinTensor& k, const RingLinTensor& v,
                            const float* log_decay, const float* s_in, const int* lengths, const float* states,
                            const RingLinTensor& go, const float* gs, void* gq, void* gk, void* gv, float* gs_in, void* ws, hipStream_t st) {
  const int nseg = segments(s), share = s.H / s.G, epv = s.type == RINGATTR_F32 ? 4 : 8;
  unsigned char* w = (unsigned char*)ws;
  const size_t each = states_bytes(s);
  float *seg_r = (float*)w, *seg_f = states ? const_cast<float*>(states) : (float*)(w + each);
  w += (states ? 1 : 2) * each;
  float *part_k = (float*)w, *part_v = (float*)(w + round_up((size_t)s.B * s.T * s.H * s.Dk * sizeof(float)));
  hipError_t e;
  auto launch_shares = [&]() {
    hipError_t f = gk ? launch_share(s.type, part_k, gk, share, s.Dk, (size_t)s.B * s.T * s.G * s.Dk, st) : hipSuccess;
    return f != hipSuccess || !gv ? f : launch_share(s.type, part_v, gv, share, s.Dv, (size_t)s.B * s.T * s.G * s.Dv, st);
  };
  // dv and dk read the same rows and go backwards together where one kernel does both
  const bool together = gk && gv && s.Dk <= 128 && s.Dv <= 128 && (s.Dk <= 64) == (s.Dv <= 64);
  RingLinArgs f = base(s, log_decay, lengths, nseg), r = f;
  f.s_in = s_in;
  f.seg = seg_f;
  f.Y = k;
  f.Z = v;
  f.ys = f.zs = share;
  r.s_in = gs;
  r.seg = seg_r;
  r.Y = q;
  r.Z = go;
  r.ys = r.zs = 1;
  r.update = s.scale;
  r.s_out = gs_in;
  if (gq) {
    if (!states) {
      e = segment_states(s, f, false, st);
      if (e != hipSuccess) return e;
    }
    // dq: do against v weighs k, the state transposed
    f.X = go;
    f.xs = 1;
    f.Y = v;
    f.Z = k;
    f.Da = s.Dv;
    f.sa = 1;
    f.sb = s.Dv;
    set_columns(f, s.Dk, false);
    f.out = gq;
    f.out_vec = f.Db % epv == 0 && out_fits(f);
    f.intra = f.inter = s.scale;
    e = launch_pass(s.type, f, false, false, st);
    if (e != hipSuccess) return e;
  }
  if (!gk && !gv) return hipSuccess;
  e = segment_states(s, r, true, st);
  if (e != hipSuccess) return e;
  // dv: k against q weighs do
  r.X = k;
  r.xs = share;
  r.Da = s.Dk;
  r.sa = s.Dv;
  r.sb = 1;
  set_columns(r, s.Dv, false);
  r.intra = s.scale;
  r.out = share > 1 ? (void*)part_v : gv;
  r.out_f32 = share > 1;
  r.out_vec = r.Db % epv == 0 && out_fits(r);
  if (together) {
    r.X2 = v;
    r.x2s = share;
    r.out2 = share > 1 ? (void*)part_k : gk;
    r.out_vec = r.out_vec && r.Da % epv == 0 && (long)s.H * r.Da < (1 << 22);
    e = launch_two(s.type, r, st);
    if (e != hipSuccess || share == 1) return e;
    return launch_shares();
  }
  if (gv) {
    e = launch_pass(s.type, r, true, false, st);
    if (e != hipSuccess) return e;
  }
  // dk: v against do weighs q, the state transposed
  if (!gk) return share > 1 ? launch_shares() : hipSuccess;
  r.X = v;
  r.Y = go;
  r.Z = q;
  r.Da = s.Dv;
  r.sa = 1;
  r.sb = s.Dv;
  set_columns(r, s.Dk, false);
  r.s_out = nullptr;
  r.out = share > 1 ? (void*)part_k : gk;
  r.out_vec = r.Db % epv == 0 && out_fits(r);
  e = launch_pass(s.type, r, true, false, st);
  if (e != hipSuccess || share == 1) return e;
  return launch_shares();
}
