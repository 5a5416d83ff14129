// Selective state space scan: the passes of a forward and of a backward, sums over parts, and the single token.
#include "ring_recur.hpp"
#include "ringattr.h"

using namespace ring_recur;

namespace {

constexpr int kChunk = 32;            // segments are whole numbers of these tokens

size_t round_up(size_t x) { return (x + 255) / 256 * 256; }
int padded(int N) { return N <= 4 ? 4 : (N <= 8 ? 8 : (N <= 16 ? 16 : (N <= 32 ? 32 : 64))); }
int tile(int N) { return N <= 16 ? 64 : (N <= 32 ? 32 : 16); }        // channels of a workgroup
int tiles_of(const RingScanShape& s) { return (s.C / s.G + tile(s.N) - 1) / tile(s.N); }
int saved_of(const RingScanShape& s) { return (s.T + RingScanArgs::kSave - 1) / RingScanArgs::kSave; }

// Segments that the tokens are cut into: none where every compute unit has a workgroup without, otherwise so many that each has two (us, bf16, 16 states, 2048
// channels: one sequence of 32768 tokens by workgroups 256 472, 384 557, 512 424, 768 433; with gradients four of 2048 tokens, none 540, four
// segments 396; eight, none 549, two 661).  Measured on 16-bit rows of whole 16 bytes, whose outputs have two workgroups a unit; gradients, and outputs
// of most other rows (at ring_scan_kernel), have one, and so many workgroups are two rounds there, a few more three.  Just over 256 without segments leave most units idle in a second round.
int segments(const RingScanShape& s) {
  const long groups = (long)tiles_of(s) * s.G * s.B;
  const int units = (s.T + kChunk - 1) / kChunk;
  long n = groups >= 256 ? 1 : (512 + groups - 1) / groups;
  if (n > units / 2) n = units / 2;
  if (n < 1) n = 1;
  const int per = (int)((units + n - 1) / n);
  return (units + per - 1) / per;
}

size_t seg_bytes(const RingScanShape& s, int nseg) {
  const size_t rows = (size_t)(nseg - 1) * s.B * s.C;
  return round_up(rows * padded(s.N) * sizeof(float)) + round_up(rows * sizeof(float));
}
size_t shared_bytes(const RingScanShape& s) {
  return round_up((size_t)tiles_of(s) * s.B * s.T * s.G * 2 * padded(s.N) * sizeof(float));
}

void set_segments(RingScanArgs& a, const RingScanShape& s, int nseg, void* ws) {
  const int units = (s.T + kChunk - 1) / kChunk;
  a.nseg = nseg;
  a.seg_tokens = (units + nseg - 1) / nseg * kChunk;
  a.saved = saved_of(s);
  a.seg = (float*)ws;
  a.total = (float*)((char*)ws + round_up((size_t)(nseg - 1) * s.B * s.C * padded(s.N) * sizeof(float)));
}

hipError_t launch_pass(int type, const RingScanArgs& a, int mode, hipStream_t st) {
  if (type == RINGATTR_F32) return ring_launch_scan_f32(a, mode, st);
  if (type == RINGATTR_BF16) return ring_launch_scan_bf16(a, mode, st);
  return ring_launch_scan_f16(a, mode, st);
}

}  // namespace

// What the segments add to a state of zeros becomes the states behind them, in place; a segment's whole decay is the power of its sum of d.  Where that may be a power that 32
// bits do not hold and its product with the state a number all the same, whole powers go into the exponent: zero and infinity stay what they are, as
// they do under the tokens one by one.
// A thread walks one state through them, a segment's reads behind the last one's write: bound by latency (16 segments of 2048 channels of 16 states: 7 us; of 630 of 11, 5).
__global__ __launch_bounds__(256) void ring_scan_between_kernel(float* seg, const float* total, const float* A, const float* s_in, int B, int C, int N,
                                                                int NS, int ns) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, rows = (size_t)B * C;
  if (i >= rows * NS) return;
  const size_t row = i / NS;
  const int n = (int)(i - row * NS), c = (int)(row % C);
  const float A2 = n < N ? times_log2e(A[(size_t)c * N + n]) : 0.f;
  float run = s_in && n < N ? s_in[row * N + n] : 0.f;
#pragma unroll 4
  for (int u = 0; u < ns; ++u) {
    const float local = seg[u * rows * NS + i], x = total[u * rows + row] * A2;
    const bool far = fabsf(x) >= 126.f;
    const float y = far ? __builtin_amdgcn_fmed3f(x, -1000.f, 1000.f) : x, whole = far ? truncf(y) : 0.f;
    run = fmaf(__builtin_amdgcn_exp2f(y - whole), ldexpf(run, (int)whole), local);
    seg[u * rows * NS + i] = run;
  }
}

static hipError_t between(const RingScanShape& s, RingScanArgs a, int mode, hipStream_t st) {
  if (a.nseg == 1) return hipSuccess;
  hipError_t e = launch_pass(s.type, a, mode, st);
  if (e != hipSuccess) return e;
  const size_t n = (size_t)s.B * s.C * padded(s.N);
  hipLaunchKernelGGL(ring_scan_between_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a.seg, a.total, a.A, a.s_in, s.B, s.C, s.N,
                     padded(s.N), a.nseg - 1);
  return hipGetLastError();
}

size_t ring_scan_states_bytes(const RingScanShape& s) { return round_up((size_t)s.B * saved_of(s) * s.C * padded(s.N) * sizeof(float)); }
size_t ring_scan_fwd_bytes(const RingScanShape& s) { return seg_bytes(s, segments(s)); }
size_t ring_scan_bwd_bytes(const RingScanShape& s, bool shared, bool params) {
  const int nseg = segments(s);
  return seg_bytes(s, nseg) + (shared ? shared_bytes(s) : 0) +
         (params ? round_up((size_t)nseg * s.B * s.C * (padded(s.N) + 2) * sizeof(float)) : 0);
}

hipError_t ring_scan_fwd(const RingScanShape& s, RingScanArgs a, void* ws, hipStream_t st) {
  set_segments(a, s, segments(s), ws);
  hipError_t e = between(s, a, RING_SCAN_STATE, st);
  return e == hipSuccess ? launch_pass(s.type, a, RING_SCAN_OUTPUTS, st) : e;
}

// What parts become, in one launch.  The first `columns` workgroups: sums of the parameters' parts, bound by latency.  The others: dB and dC [B,T,G,N] from the sums over the
// tiles of a group's channels, in their order; rows that do not count are zero; bound by memory (32 tiles of 16384 tokens, 16 states: 67 MB, just written and in the
// last cache in part).  14 us there, 4 for 4 tiles of 3885 tokens (as two launches 18, 9).
template <typename T, int W>
__global__ __launch_bounds__(256) void ring_scan_join_kernel(const float* __restrict__ part, T* dB, T* dC, const int* lengths, int tiles, int B, int Tn, int G, int N,
                                                             int NS, unsigned columns, RingSumArgs p) {
  __shared__ float sums[256];
  if (blockIdx.x < columns) return sum_parts<W>(p, blockIdx.x, sums);
  const size_t rows = (size_t)B * Tn * G, all = rows * 2 * NS;
  for (size_t i = (size_t)(blockIdx.x - columns) * 256 + threadIdx.x; i < all; i += (size_t)(gridDim.x - columns) * 256) {
    const size_t row = i / (2 * NS);
    const int k = (int)(i - row * 2 * NS), n = k % NS;
    T* out = k < NS ? dB : dC;
    if (n >= N || !out) continue;
    const int b = (int)(row / ((size_t)Tn * G)), t = (int)(row / G % Tn);
    float sum = 0.f;
    if (t < length_of(lengths, b, Tn))
#pragma unroll 4
      for (int m = 0; m < tiles; ++m) sum += part[m * all + i];
    out[row * N + n] = (T)sum;
  }
}

template <typename T> static hipError_t launch_join(const RingScanShape& s, const RingScanArgs& a, const RingScanGrads& g, int nseg, hipStream_t st) {
  const int per = padded(s.N) + 2;
  const RingSumArgs p = {a.part_a, nseg * s.B, per, s.N, 2, a.part_a ? (size_t)s.C * per : 0, g.A, {g.D, g.bias}};
  const size_t blocks = a.part_bc ? ((size_t)s.B * s.T * s.G * 2 * padded(s.N) + 255) / 256 : 0;
  const unsigned columns = sum_blocks(p);
  const dim3 grid(columns + (unsigned)(blocks < (1 << 22) ? blocks : 1 << 22)), block(256);
  if (grid.x == 0) return hipSuccess;
  T *const dB = (T*)g.B, *const dC = (T*)g.C;
  const int tiles = tiles_of(s), NS = padded(s.N);
  if (sum_ways(p) > 1) hipLaunchKernelGGL((ring_scan_join_kernel<T, kWays>), grid, block, 0, st, a.part_bc, dB, dC, a.lengths, tiles, s.B, s.T, s.G, s.N, NS, columns, p);
  else hipLaunchKernelGGL((ring_scan_join_kernel<T, 1>), grid, block, 0, st, a.part_bc, dB, dC, a.lengths, tiles, s.B, s.T, s.G, s.N, NS, columns, p);
  return hipGetLastError();
}

hipError_t ring_scan_bwd(const RingScanShape& s, RingScanArgs a, const RingScanGrads& g, void* ws, hipStream_t st) {
  const int nseg = segments(s);
  set_segments(a, s, nseg, ws);
  char* at = (char*)ws + seg_bytes(s, nseg);
  if (g.B || g.C) {
    a.part_bc = (float*)at;
    at += shared_bytes(s);
  }
  if (g.A || g.D || g.bias) a.part_a = (float*)at;
  hipError_t e = between(s, a, RING_SCAN_ADJOINT, st);
  if (e == hipSuccess) e = launch_pass(s.type, a, RING_SCAN_GRADIENTS, st);
  if (e != hipSuccess) return e;
  if (s.type == RINGATTR_F32) return launch_join<float>(s, a, g, nseg, st);
  return s.type == RINGATTR_BF16 ? launch_join<__bf16>(s, a, g, nseg, st) : launch_join<_Float16>(s, a, g, nseg, st);
}

// A single token.  A lane takes V states of a channel, 2^log_lanes of them a channel; bound by the states, read and written once (bf16, 16 states, gate: 256
// sequences of 4096 channels, 143 MB in 28 us, 5.1 TB/s; 34 with places found by divisions of 64 bits, which kept the vector pipes busy; one sequence of 1024
// channels 4 us, a launch).
// ONE: a workgroup takes channels of one sequence, whose rows scalar addresses find; otherwise (channels with fewer lanes than that) 2^log_row lanes are a sequence.
template <typename T, int V, bool ONE>
__global__ __launch_bounds__(256) void ring_scan_step_kernel(RingScanStep p, RingScanShape s, int log_lanes, int log_row, int blocks) {
  typedef float vec __attribute__((ext_vector_type(V)));
  const int b = ONE ? (int)(blockIdx.x / blocks) : (int)(blockIdx.x * (256 >> log_row) + (threadIdx.x >> log_row));
  const int i = ONE ? (int)(blockIdx.x - b * blocks) * 256 + (int)threadIdx.x : (int)threadIdx.x & ((1 << log_row) - 1), lanes = 1 << log_lanes;
  const int c = i >> log_lanes, n = (i & (lanes - 1)) * V;
  if (b >= s.B || c >= s.C) return;              // (whole channels: a channel's lanes go together)
  const int g = s.G == 1 ? 0 : c / (s.C / s.G);
  T* const out = (T*)p.y + (size_t)b * s.C + c;
  if (p.active && !p.active[b]) {
    if (n == 0) *out = (T)0.f;
    return;
  }
  const float x = (float)((const T*)p.x + b * p.xs)[c];
  float d = (float)((const T*)p.delta + b * p.ds)[c], z = 0.f;
  if (p.z) z = (float)((const T*)p.z + b * p.zs)[c];
  if (p.bias) d += p.bias[c];
  if (p.softplus) d = softplus<sizeof(T) == 4>(d);
  float y = 0.f;
  if (n < s.N) {
    const int k = c * s.N + n;
    vec* const at = reinterpret_cast<vec*>(p.state + (size_t)b * s.C * s.N + k);
    const vec A = *reinterpret_cast<const vec*>(p.A + k);
    const T* const B = (const T*)p.Bm + b * p.bsb + g * p.bsg + n;
    const T* const C = (const T*)p.Cm + b * p.csb + g * p.csg + n;
    vec h = *at;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      h[e] = fmaf(__builtin_amdgcn_exp2f(d * times_log2e(A[e])), h[e], d * x * (float)B[e]);
      y = fmaf(h[e], (float)C[e], y);
    }
    *at = h;
  }
  for (int half = lanes / 2; half > 0; half /= 2) y += __shfl_xor(y, half);
  if (n == 0) {
    if (p.D) y = fmaf(p.D[c], x, y);
    if (p.z) y *= silu<sizeof(T) == 4>(z);
    *out = (T)y;
  }
}

template <typename T, int V> static void launch_step_of(const RingScanShape& s, const RingScanStep& a, hipStream_t st) {
  int log_lanes = 0, log_row = 0;
  while (V << log_lanes < s.N) ++log_lanes;
  while (1 << log_row < s.C << log_lanes) ++log_row;
  const int blocks = ((s.C << log_lanes) + 255) / 256, per = log_row < 8 ? 256 >> log_row : 1;
  if (log_row >= 8) hipLaunchKernelGGL((ring_scan_step_kernel<T, V, true>), dim3((unsigned)((size_t)blocks * s.B)), dim3(256), 0, st, a, s, log_lanes, log_row, blocks);
  else hipLaunchKernelGGL((ring_scan_step_kernel<T, V, false>), dim3((unsigned)((s.B + per - 1) / per)), dim3(256), 0, st, a, s, log_lanes, log_row, blocks);
}

template <typename T> static hipError_t launch_step(const RingScanShape& s, const RingScanStep& a, hipStream_t st) {
  if (s.N % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.state) | reinterpret_cast<uintptr_t>(a.A)) & 15) == 0) launch_step_of<T, 4>(s, a, st);
  else launch_step_of<T, 1>(s, a, st);
  return hipGetLastError();
}

hipError_t ring_scan_step(const RingScanShape& s, const RingScanStep& a, hipStream_t st) {
  if (s.type == RINGATTR_F32) return launch_step<float>(s, a, st);
  if (s.type == RINGATTR_BF16) return launch_step<__bf16>(s, a, st);
  return launch_step<_Float16>(s, a, st);
}
