// Linear attention with a decay for each head, in chunks of tokens.
//
//   S_t = lambda S_{t-1} + k_t v_t^T,   o_t = scale q_t S_t,   lambda = exp(log_decay[h])
//
// The leak of the ring's time loop on a matrix of associations in place of a row of neurons.  Unrolled over a chunk of tokens
// l = 0..n-1 with the state S in front of it:
//
//   o_l = scale (lambda^(l+1) q_l S + sum_{j<=l} lambda^(l-j) (q_l . k_j) v_j),   S' = lambda^n S + sum_j lambda^(n-1-j) k_j v_j^T
//
// and every gradient is the same sum with other operands, forwards or backwards in time (R: the state's gradient):
//
//   dq = scale (sums over j <= l of lambda^(l-j) (do_l . v_j) k_j),      state S^T
//   dk = sums over i >= l of lambda^(i-l) (v_l . do_i) scale q_i,        state R^T,  R = dL/dS behind the chunk
//   dv = sums over i >= l of lambda^(i-l) (k_l . q_i) scale do_i,        state R
//
// so one kernel does all four: rows X against rows Y give weights, the weights collect rows Z, and S collects Y Z^T.  Backwards in
// time (REV) a row sees itself and those behind it, the powers are mirrored, and what is left of the state in front of the sequence
// is the gradient of the initial state.
#pragma once
#include "ring_common.hpp"
#include "ring_kernels.hpp"

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

namespace ring_lin {

// bf16 operands go to the matrix units as they are, and what is computed on the way enters them so (half a step of bf16 is 2^-9 to 2^-8):
//   weights, and the state in a product with a row: a sum of two bf16 numbers, 2^-15.  Each term of an output passes one of them, so that
//     an output's error is its own rounding, 0.0017 of its size (with one number 0.0023; a forward of 8 x 4096 tokens, 16 heads of 128,
//     takes 213 us so and 189 with one)
//   a decayed row that goes into the state: a sum of two, 2^-16, because a state collects the errors of all that came before
//   the same where the state is itself a result: a sum of three, 2^-24, as exact as fp32 sums (EXACT)
// The state is kept in 32 bits throughout.  fp32 and fp16 go to the fp32 matrix units: fp16 because weights and states can pass its range.
template <typename T> struct Type;
template <> struct Type<__bf16> { static constexpr bool BF = true; static constexpr unsigned EXPONENT = 0x7f80u; typedef bf16x4 V4; typedef unsigned short Bits; };
template <> struct Type<float> { static constexpr bool BF = false; static constexpr unsigned EXPONENT = 0x7f800000u; typedef f32x4 V4; typedef unsigned Bits; };
template <> struct Type<_Float16> { static constexpr bool BF = false; static constexpr unsigned EXPONENT = 0x7c00u; typedef f16x4 V4; typedef unsigned short Bits; };

__device__ __forceinline__ float power(float g2, int e) { return e == 0 ? 1.f : __builtin_amdgcn_exp2f(g2 * (float)e); }

// (by bits: left to itself the compiler converts the second of each pair once more instead)
__device__ __forceinline__ f32x4 widen(bf16x4 x) {
  const u32x2 b = __builtin_bit_cast(u32x2, x);
  return f32x4{__builtin_bit_cast(float, b[0] << 16), __builtin_bit_cast(float, b[0] & 0xffff0000u), __builtin_bit_cast(float, b[1] << 16),
               __builtin_bit_cast(float, b[1] & 0xffff0000u)};
}
__device__ __forceinline__ f32x4 widen(f16x4 x) { return __builtin_convertvector(x, f32x4); }
__device__ __forceinline__ f32x4 widen(f32x4 x) { return x; }
__device__ __forceinline__ bf16x4 narrow(f32x4 x) { return __builtin_convertvector(x, bf16x4); }
// x as the sum of two bf16 numbers, 2^-15 of it left out at most: x cut off behind its first 8 bits (cut off, so that the largest finite
// numbers stay finite), then what is left, rounded
struct Halves { bf16x4 high, low; };
__device__ __forceinline__ Halves halves(f32x4 x) {
  const u32x4 b = __builtin_bit_cast(u32x4, x);
  const u32x2 high = {__builtin_amdgcn_perm(b[1], b[0], 0x07060302u), __builtin_amdgcn_perm(b[3], b[2], 0x07060302u)};
  return {__builtin_bit_cast(bf16x4, high), narrow(x - __builtin_bit_cast(f32x4, b & 0xffff0000u))};
}
__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

__device__ __forceinline__ bool nonfinite(float x) { return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u; }

// The largest magnitude of a number of values, by their bits
template <typename T> struct Magnitude {
  typedef typename Type<T>::Bits bits __attribute__((ext_vector_type(2)));
  bits most = {0, 0};
  __device__ __forceinline__ void add(typename Type<T>::V4 x) {
    struct Two { bits b[2]; };
    const Two two = __builtin_bit_cast(Two, x);
    constexpr typename Type<T>::Bits M = (typename Type<T>::Bits)~((typename Type<T>::Bits)1 << (8 * sizeof(T) - 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) most = __builtin_elementwise_max(most, two.b[i] & M);
  }
  __device__ __forceinline__ bool nonfinite() const { return most[0] >= Type<T>::EXPONENT || most[1] >= Type<T>::EXPONENT; }
};

// Place of operand row m (0..15) of tile i among tiles of 16.  Two tiles of 16-bit values go together: a lane's four of each are eight
// neighbours, 16 bytes of one read or store.
template <typename T, bool PAIR> __device__ __forceinline__ int place(int i, int m) {
  return PAIR && sizeof(T) == 2 ? 32 * (i >> 1) + 8 * (m >> 2) + 4 * (i & 1) + (m & 3) : 16 * i + m;
}

// A tile of ROWS x COLS values in LDS, rows one behind the other.  A row's 16-byte granules change places by an exclusive or with a
// function of the row, such that what one instruction reads lies in all banks: 16 rows at one place (`rows`), 8 rows at two
// neighbouring places by the transposing read of 16-bit values, 4 rows at four by single words (`columns`).
template <typename T, int ROWS, int COLS> struct Tile16 {
  static constexpr int EPV = 16 / sizeof(T), GPR = COLS / EPV, RB = COLS * sizeof(T), BYTES = ROWS * RB;
  typedef typename Type<T>::V4 V4;

  static __device__ __forceinline__ int turn(int row) {
    if (sizeof(T) == 4) return row & 15;
    if (GPR >= 16) return ((row << 1) | ((row >> 3) & 1)) & 15;
    const int k = (row >> 1) & 7;
    return ((k << 1) | (k >> 2)) & 7;
  }
  // byte address of (row, col)
  static __device__ __forceinline__ int at(int row, int col) {
    return row * RB + (((col / EPV) ^ turn(row)) * 16) + (col % EPV) * (int)sizeof(T);
  }

  // Lane (g, l): row 16 t + l, the EPV columns from 4 EPV s + EPV g on.  first: the address at t = 0, s = 0, from which the others
  // follow.
  typedef T V16 __attribute__((ext_vector_type(16 / sizeof(T))));
  static __device__ __forceinline__ int rows_first(int g, int l) { return at(l, EPV * g); }
  static __device__ __forceinline__ V16 rows(const char* tile, int first, int t, int s) {
    return *reinterpret_cast<const V16*>(tile + (first ^ (s * 64)) + t * 16 * RB);
  }
  // Element e of lane (g, l): row 16 t + 4 g + e, column place(s, l).
  template <bool PAIR> static __device__ __forceinline__ int columns_first(int g, int l, int r) {
    if (sizeof(T) == 2) return PAIR ? at(4 * g + (l >> 2), 8 * (l & 3)) : at(4 * g + (l >> 2), 4 * (l & 3));
    return at(4 * g + r, l);
  }
  template <bool PAIR> static __device__ __forceinline__ V4 columns(const char* tile, const int (&first)[4], int t, int s) {
    const int x = PAIR && sizeof(T) == 2 ? ((s >> 1) * 64) | ((s & 1) * 8) : s * 16 * (int)sizeof(T);
    if constexpr (sizeof(T) == 2) {
      const char* p = tile + (first[0] ^ x) + t * 16 * RB;
      return __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
    } else {
      V4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = *reinterpret_cast<const float*>(tile + (first[r] ^ x) + t * 16 * RB);
      return v;
    }
  }
};

// Global memory -> LDS without registers: a wave's instruction fills 64 granules one behind the other, each lane from where it likes.
// What is loaded is there behind a wait for vmcnt and a barrier (nobody else keeps count: the compiler does not see these loads).  It
// says nothing about memory to the compiler, so that reads of the other buffer pass it by: every use of what it writes, and every
// use of what was there, is on the other side of such a wait and barrier, which do.
// base and lds are the same in all lanes.  (The wait states are for a base that a vector instruction has just put into its scalar
// registers: the compiler does not look into the statement.)
__device__ __forceinline__ void load_to_lds(const void* base, unsigned off, unsigned lds) {
  const unsigned long long a = (unsigned long long)(uintptr_t)base;
  const unsigned low = __builtin_amdgcn_readfirstlane((unsigned)a), high = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
  const unsigned long long s = (unsigned long long)high << 32 | low;
  unsigned kept;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
               : "=&s"(kept) : "s"(lds), "v"(off), "s"(s));
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}

// Fills a tile: rows 0..n-1 of `cols` values from base on, token stride st; what is not loaded is left as it is.
template <typename T, int ROWS, int COLS, int NT, bool VEC> struct Filler {
  typedef Tile16<T, ROWS, COLS> Tl;
  // (the first FT threads fill it: granules of a thread, rows between them)
  static constexpr int FT = ROWS * Tl::GPR < NT ? ROWS * Tl::GPR : NT, EPV = Tl::EPV, GPR = Tl::GPR, NU = ROWS * GPR / FT, RS = FT / GPR;
  static_assert(ROWS * GPR % FT == 0 && FT % GPR == 0 && FT % 64 == 0, "");
  unsigned off[NU];                                            // byte offsets of the thread's granules in a whole chunk

  __device__ __forceinline__ void init(long st, int tid) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int row = tid / GPR + u * RS, c = ((tid % GPR) ^ Tl::turn(row)) * EPV;
      off[u] = (unsigned)row * (unsigned)st * (unsigned)sizeof(T) + (unsigned)c * (unsigned)sizeof(T);
    }
  }
  // WHOLE: all rows and columns are there
  template <bool WHOLE> __device__ __forceinline__ void fill(char* tile, const T* base, long st, int n, int cols, int tid) const {
    if (FT < NT && tid >= FT) return;
    if constexpr (VEC) {
      const unsigned lds = __builtin_amdgcn_readfirstlane(lds_address(tile) + (tid >> 6) * 1024);
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int row = tid / GPR + u * RS, c = ((tid % GPR) ^ Tl::turn(row)) * EPV;
        if (WHOLE || (row < n && c < cols)) load_to_lds(base, off[u], lds + u * FT * 16);
      }
    } else {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int row = tid / GPR + u * RS, c = ((tid % GPR) ^ Tl::turn(row)) * EPV;
        T v[EPV];
#pragma unroll
        for (int e = 0; e < EPV; ++e) v[e] = row < n && c + e < cols ? base[(long)row * st + c + e] : (T)0.f;
        if (row < n) *reinterpret_cast<u32x4*>(tile + (tid + u * FT) * 16) = *reinterpret_cast<const u32x4*>(v);
      }
    }
  }
  static __device__ __forceinline__ void clear(char* tile, int from, int tid) {
    if (FT < NT && tid >= FT) return;
#pragma unroll
    for (int u = 0; u < NU; ++u)
      if (tid / GPR + u * RS >= from) *reinterpret_cast<u32x4*>(tile + (tid + u * FT) * 16) = u32x4{0, 0, 0, 0};
  }
};

template <typename T> __device__ __forceinline__ const T* rows_of(const RingLinTensor& t, int b, int h, int share) {
  return reinterpret_cast<const T*>(t.p) + (long)b * t.sb + (long)(h / share) * t.sh;
}

// Waits until no more than N of the wave's accesses to memory are on their way, the last N that it issued
template <int N> __device__ __forceinline__ void wait_for_memory() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// A workgroup: one head of one sequence, WC = 16 NC NW columns of Z and of the state, one segment of the tokens.  Its waves share the
// chunk's rows in LDS (two buffers: the next chunk's are on their way while one is worked on); each keeps 16 NC columns of the state
// in registers, where they are an operand as they lie: the matrix units put rows 4g..4g+3 of column l into lane (g, l) and take them
// as contraction indices from there.  The weights are formed transposed for the same reason, by every wave for itself.
//
// What bounds it.  bf16, a state of 128 x 128: a chunk of 32 tokens is 84 matrix instructions of 16 clocks a wave (EXACT: 100), more
// clocks than that of vector instructions (a third of them split the state), which hardly overlap them, and a chain from the rows through the
// weights to the outputs: 2.0 us a chunk in a chip with few workgroups (EXACT: 2.2).  8 x 4096 tokens, 16 heads, 537 MB a pass: 129 us with
// 512 workgroups (4.2 TB/s; a large copy 5.2), 156 with 256, EXACT 179 and 197; one sequence of 32768 tokens, EXACT, 180.  Before weights and
// states were two numbers (153 there) chunks of 64 tokens took 165, eight waves of 16 columns 166, two chunks on their way at once 165.  fp32
// and fp16 multiply at 32 clocks for an eighth of the contraction, in chunks of 16 tokens (fp16: 32), and are bound by that: 8 x 2000 tokens,
// 8 heads of 256, fp32, 33.6 GFLOP a pass without the weights: 390 to 416 us, 81 to 86 TFLOP/s (154 in a large matrix product).  States alone,
// one sequence of 32768 tokens: 252 MB, 68 us (3.7 TB/s).
template <typename T, int DA, int NC, int NW, int CT, bool VEC, bool REV, bool STATE_ONLY, bool EXACT, bool PAIR = false>
__global__ __launch_bounds__(64 * NW, (DA <= 128 || NW == 8 ? 2 : 1)) void ring_linattn_kernel(RingLinArgs p) {
  constexpr int GW = PAIR ? NW / 2 : NW, WC = 16 * NC * GW, NT = 64 * NW, CH = 16 * CT, DT = DA / 16;
  static_assert(!PAIR || (WC == DA && !STATE_ONLY), "");
  // States alone are collected against the time, each chunk with its distance: nothing is multiplied from chunk to chunk, and the pass
  // behind, which goes with the time, finds the rows that were read last in the last cache.
  constexpr bool DOWN = REV != STATE_ONLY;
  constexpr bool BF = Type<T>::BF;
  typedef typename Type<T>::V4 V4;
  typedef Tile16<T, CH, DA> TA;
  typedef Tile16<T, CH, WC> TZ;
  typedef Filler<T, CH, DA, NT, VEC> FA;
  typedef Filler<T, CH, WC, NT, VEC> FZ;
  constexpr int XB = STATE_ONLY ? 0 : TA::BYTES, BUF = XB + TA::BYTES + TZ::BYTES + (PAIR ? TA::BYTES : 0);
  // The weights of fp32 products: each wave forms a part of the contraction and the parts are added up in LDS (with bf16 products there
  // is nothing to gain: what the products take less is what the exchange takes).
  constexpr int STEPS = DA / (64 / (int)sizeof(T)), TPS = DT / STEPS;          // steps of 64 bytes a row, tiles of the state in each
  constexpr bool SHARED = !BF && !STATE_ONLY && STEPS % GW == 0;
  __shared__ __align__(16) char lds[2 * BUF];
  __shared__ __align__(16) f32x4 shares[SHARED ? NW * CT * CT * 64 : 1];

  const int tid = threadIdx.x, wave = tid >> 6, l = tid & 15, g = (tid >> 4) & 3;
  // PAIR: the second half of the waves runs the second pass: rows X2 against rows Z weigh rows Y, the state transposed
  const int second = PAIR ? __builtin_amdgcn_readfirstlane(wave / GW) : 0, w = PAIR ? wave % GW : wave;
  const int Da = second ? p.Db : p.Da, Db = second ? p.Da : p.Db;
  // `order` counts the segments as they follow each other; the pass over states has no use for the last
  const int per = STATE_ONLY ? p.nseg - 1 : p.nseg, order = blockIdx.x % per, seg = REV ? p.nseg - 1 - order : order;
  const int slice = blockIdx.x / per % p.slices, head = blockIdx.x / (per * p.slices);
  const int c0 = slice * WC, h = head % p.H, b = head / p.H;
  const int cw = 16 * NC * w;                                  // the wave's columns within the workgroup's
  const int T_ = p.T;
  const int len = p.lengths ? min(max(p.lengths[b], 0), T_) : T_;
  const int t0 = seg * p.seg_tokens, t1 = min(T_, t0 + p.seg_tokens), te = min(len, t1), nch = (t1 - t0 + CH - 1) / CH;
  const int full = te > t0 ? (te - t0 + CH - 1) / CH : 0;      // chunks with tokens that count
  const float g2 = (float)((double)p.log_decay[h] * 1.4426950408889634);
  const size_t bh = (size_t)b * p.H + h;

  const T* X = STATE_ONLY ? nullptr : rows_of<T>(p.X, b, h, p.xs);
  const T* Y = rows_of<T>(p.Y, b, h, p.ys);
  const T* Z = rows_of<T>(p.Z, b, h, p.zs) + c0;
  const T* X2 = PAIR ? rows_of<T>(p.X2, b, h, p.x2s) : nullptr;
  const int cols = Db - c0;

  // The state in front: a scan has left it, or it is the initial one and, of two segments, what the first has added to it.
  const bool wide = p.Da == DA && (PAIR ? p.Db == DA : cols >= WC);            // (nothing to leave out)
  f32x4 S[DT][NC];
  const size_t D = (size_t)p.Da * p.Db;
  auto add_state = [&](const float* s, float f) {
    const int sa = (int)(second ? p.sb : p.sa), sb = (int)(second ? p.sa : p.sb);
    int a0 = place<T, true>(0, 4 * g), b0 = cw + place<T, NC == 2>(0, l);
    asm volatile("" : "+v"(a0), "+v"(b0));                     // (64 addresses are not to be kept from one call to the next)
    s += (size_t)c0 * sb;
    const unsigned at = (unsigned)(a0 * sa + b0 * sb);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int da = place<T, true>(d, 0) + r, db = place<T, NC == 2>(ct, 0);
          float x;
          if (wide) {
            x = (s + (da * sa + db * sb))[at];
          } else {
            x = s[(unsigned)(min(a0 + da, Da - 1) * sa + min(b0 + db, cols - 1) * sb)];
            x = a0 + da < Da && b0 + db < cols ? x : 0.f;
          }
          S[d][ct][r] = fmaf(f, S[d][ct][r], x);
        }
      if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);       // (not all on their way at once)
    }
  };
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int ct = 0; ct < NC; ++ct) S[d][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (!STATE_ONLY) {
    const float* const segs = p.nseg > 1 ? p.seg + bh * (p.nseg - 1) * D : nullptr;
    const float* const front = p.scanned && order > 0 ? segs + (order - 1) * D : (p.s_in ? p.s_in + bh * D : nullptr);
    if (front) add_state(front, 0.f);
    if (!p.scanned && order > 0) {
      const int n = min(max(len - (REV ? p.seg_tokens : 0), 0), p.seg_tokens);                   // the first segment's tokens
      add_state(segs, power(g2, n));
    }
  }

  // powers of the decay: by distance within a pair of tiles, and for the rows of a chunk of n.  None that no token has: with a decay above one it
  // could be infinite, and a row of zeros times it no longer zero.
  float near[CT][4], inner[CT], outer[CT][4], whole = 1.f;
#pragma unroll
  for (int d = 0; d < CT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int e = 16 * d + (REV ? 4 * g + r - l : l - 4 * g - r);
      near[d][r] = e < 0 || e >= te - t0 ? 0.f : p.intra * power(g2, e);
    }
  int n_now = -1;

  auto put = [&](const f32x4 (&O)[NC][CT], int t, int rows) {
    const size_t at = ((size_t)b * T_ + t) * p.H + h, size = p.out_f32 || sizeof(T) == 4 ? 4 : sizeof(T);
    char* const base = (char*)(second ? p.out2 : p.out) + (at * Db + c0) * size;
    const unsigned step = (unsigned)(p.H * Db) * (unsigned)size;                                   // (VEC: within 24 bits)
#pragma unroll
    for (int it = 0; it < CT; ++it) {
      const int row = 16 * it + l, c = cw + place<T, NC == 2>(0, 4 * g);
      if (row >= rows || c >= cols) continue;
      char* const o = (VEC ? base + __umul24((unsigned)row, step) : base + (size_t)row * p.H * Db * size) + c * (int)size;
      if (p.out_f32 || sizeof(T) == 4) {
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          const int more = place<T, NC == 2>(ct, 0);
          if (VEC) {
            if (c + more < cols) *reinterpret_cast<f32x4*>(o + 4 * more) = O[ct][it];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c + more + r < cols) reinterpret_cast<float*>(o)[more + r] = O[ct][it][r];
          }
        }
      } else {
        typedef T vec_t __attribute__((ext_vector_type(4 * NC)));
        vec_t q;
#pragma unroll
        for (int e = 0; e < 4 * NC; ++e) q[e] = (T)O[e / 4][it][e % 4];
        if (VEC) {
          *reinterpret_cast<vec_t*>(o) = q;
        } else {
#pragma unroll
          for (int e = 0; e < 4 * NC; ++e)
            if (c + e < cols) reinterpret_cast<T*>(o)[e] = q[e];
        }
      }
    }
  };

  if constexpr (!STATE_ONLY) {                                 // chunks without tokens that count
    f32x4 zero[NC][CT];
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int it = 0; it < CT; ++it) zero[ct][it] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c = full; c < nch; ++c) put(zero, t0 + c * CH, min(CH, t1 - t0 - c * CH));
  }

  FA fx, fy, f2;
  FZ fz;
  if (!STATE_ONLY) fx.init(p.X.st, tid);
  fy.init(p.Y.st, tid);
  fz.init(p.Z.st, tid);
  if (PAIR) f2.init(p.X2.st, tid);
  auto fetch = [&](int c, int buf) {
    const int t = t0 + c * CH, n = min(CH, te - t);
    char* const tile = lds + buf * BUF;
    const T *x = STATE_ONLY ? nullptr : X + (long)t * p.X.st, *y = Y + (long)t * p.Y.st, *zz = Z + (long)t * p.Z.st;
    const T* x2 = PAIR ? X2 + (long)t * p.X2.st : nullptr;
    if (VEC && wide && n == CH) {
      if constexpr (PAIR) f2.template fill<true>(tile + XB + TA::BYTES + TZ::BYTES, x2, p.X2.st, n, p.Db, tid);
      if (!STATE_ONLY) fx.template fill<true>(tile, x, p.X.st, n, p.Da, tid);
      fy.template fill<true>(tile + XB, y, p.Y.st, n, p.Da, tid);
      fz.template fill<true>(tile + XB + TA::BYTES, zz, p.Z.st, n, p.Db - c0, tid);
    } else {
      if constexpr (PAIR) f2.template fill<false>(tile + XB + TA::BYTES + TZ::BYTES, x2, p.X2.st, n, p.Db, tid);
      if (!STATE_ONLY) fx.template fill<false>(tile, x, p.X.st, n, p.Da, tid);
      fy.template fill<false>(tile + XB, y, p.Y.st, n, p.Da, tid);
      fz.template fill<false>(tile + XB + TA::BYTES, zz, p.Z.st, n, p.Db - c0, tid);
    }
  };
  int rows1 = TA::rows_first(g, l), cols1[4], cz1[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    cols1[r] = TA::template columns_first<true>(g, l, r);
    cz1[r] = TZ::template columns_first<NC == 2>(g, l, r);
  }
  if (full > 0) {
    if (VEC && !wide) {                                        // columns that no load fills
#pragma unroll
      for (int buf = 0; buf < 2; ++buf) {
        if (!STATE_ONLY) FA::clear(lds + buf * BUF, 0, tid);
        FA::clear(lds + buf * BUF + XB, 0, tid);
        FZ::clear(lds + buf * BUF + XB + TA::BYTES, 0, tid);
        if (PAIR) FA::clear(lds + buf * BUF + XB + TA::BYTES + TZ::BYTES, 0, tid);
      }
      lds_barrier();
    }
    fetch(DOWN ? full - 1 : 0, 0);
  }
  bool stored = false;
  for (int i = 0; i < full; ++i) {
    const int c = DOWN ? full - 1 - i : i, t = t0 + c * CH, n = min(CH, te - t), buf = i & 1;
    char *const tile = lds + buf * BUF, *const ty = tile + XB, *const tz = ty + TA::BYTES, *const t2 = tz + TZ::BYTES;
    char *const lx = second ? t2 : tile, *const ly = second ? tz : ty, *const lz = second ? ty : tz;
    // the chunk's rows are there; the outputs of the one before, stored behind the loads, need not be (a store for each of its tiles)
    if (VEC && !STATE_ONLY && stored) wait_for_memory<CT>();
    else wait_for_memory<0>();
    lds_barrier();
    if (n < CH) {                                              // (the last chunk of a sequence)
      if (!STATE_ONLY) FA::clear(tile, n, tid);
      FA::clear(ty, n, tid);
      FZ::clear(tz, n, tid);
      if (PAIR) FA::clear(t2, n, tid);
      lds_barrier();
    }
    if (i + 1 < full) fetch(DOWN ? c - 1 : c + 1, buf ^ 1);
    if (n != n_now) {
      n_now = n;
      whole = power(g2, n);
#pragma unroll
      for (int it = 0; it < CT; ++it) {
        inner[it] = p.inter * power(g2, REV ? max(n - 1 - 16 * it - l, 0) : 16 * it + l + 1);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * it + 4 * g + r;
          outer[it][r] = p.update * power(g2, REV ? min(j, n - 1) + 1 : max(n - 1 - j, 0));
        }
      }
    }
    // The rows Z.  A value there that is infinite or NaN must not reach rows that do not see it, which the products within the tiles
    // multiply by zero: it is taken out, and what it gives is added at the end, one by one.
    V4 z[NC][CT];
    bool bad = false;
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int jt = 0; jt < CT; ++jt) {
        z[ct][jt] = TZ::template columns<NC == 2>(lz, cz1, jt, NC * w + ct);
      }
    if (!STATE_ONLY) {
      Magnitude<T> most;
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) most.add(z[ct][jt]);
      bad = __any(most.nonfinite());
    }
    if (!STATE_ONLY && bad)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int jt = 0; jt < CT; ++jt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (nonfinite((float)z[ct][jt][e])) z[ct][jt][e] = (T)0.f;

    f32x4 O[NC][CT];
    if constexpr (!STATE_ONLY) {
      f32x4 P[CT][CT];                                         // [tile of Y's rows][tile of X's rows]
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int it = 0; it < CT; ++it) O[ct][it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int jt = 0; jt < CT; ++jt)
#pragma unroll
        for (int it = 0; it < CT; ++it) P[jt][it] = f32x4{0.f, 0.f, 0.f, 0.f};
      // O = S X^T, what the state in front gives, and P = Y X^T, the weights; rows are read a step ahead
      typename TA::V16 xr[2][CT], yr[2][CT];
      if constexpr (SHARED) {
#pragma unroll
        for (int q = 0; q < STEPS / GW; ++q) {
          const int s = w * (STEPS / GW) + q;
          typename TA::V16 x[CT], y[CT];
#pragma unroll
          for (int it = 0; it < CT; ++it) {
            x[it] = TA::rows(lx, rows1, it, s);
            y[it] = TA::rows(ly, rows1, it, s);
          }
#pragma unroll
          for (int e = 0; e < 16 / (int)sizeof(T); ++e)
#pragma unroll
            for (int it = 0; it < CT; ++it)
#pragma unroll
              for (int jt = 0; jt < CT; ++jt)
                if (REV ? jt >= it : jt <= it) P[jt][it] = mfma4((float)y[jt][e], (float)x[it][e], P[jt][it]);
        }
#pragma unroll
        for (int it = 0; it < CT; ++it)
#pragma unroll
          for (int jt = 0; jt < CT; ++jt)
            if (REV ? jt >= it : jt <= it) shares[((wave * CT + jt) * CT + it) * 64 + (tid & 63)] = P[jt][it];
      }
      auto read = [&](int s) {
#pragma unroll
        for (int it = 0; it < CT; ++it) {
          xr[s & 1][it] = TA::rows(lx, rows1, it, s);
          if (!SHARED) yr[s & 1][it] = TA::rows(ly, rows1, it, s);
        }
      };
      read(0);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        if (s + 1 < STEPS) read(s + 1);
        if constexpr (BF) {
#pragma unroll
          for (int jt = 0; jt < CT; ++jt)
#pragma unroll
            for (int it = 0; it < CT; ++it)
              if (REV ? jt >= it : jt <= it) P[jt][it] = mfma16(yr[s & 1][jt], xr[s & 1][it], P[jt][it]);
#pragma unroll
          for (int ct = 0; ct < NC; ++ct) {
            const Halves a0 = halves(S[2 * s][ct]), a1 = halves(S[2 * s + 1][ct]);
            const bf16x8 high = join(a0.high, a1.high), low = join(a0.low, a1.low);
            S[2 * s][ct] *= whole;
            S[2 * s + 1][ct] *= whole;
#pragma unroll
            for (int it = 0; it < CT; ++it) O[ct][it] = mfma16(high, xr[s & 1][it], O[ct][it]);
#pragma unroll
            for (int it = 0; it < CT; ++it) O[ct][it] = mfma16(low, xr[s & 1][it], O[ct][it]);
          }
        } else {
#pragma unroll
          for (int q = 0; q < TPS; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float x[CT], y[CT];
#pragma unroll
              for (int it = 0; it < CT; ++it) {
                x[it] = (float)xr[s & 1][it][4 * q + r];
                y[it] = SHARED ? 0.f : (float)yr[s & 1][it][4 * q + r];
              }
#pragma unroll
              for (int it = 0; it < CT; ++it)
#pragma unroll
                for (int jt = 0; jt < CT; ++jt)
                  if (!SHARED && (REV ? jt >= it : jt <= it)) P[jt][it] = mfma4(y[jt], x[it], P[jt][it]);
#pragma unroll
              for (int ct = 0; ct < NC; ++ct)
#pragma unroll
                for (int it = 0; it < CT; ++it) O[ct][it] = mfma4(S[TPS * s + q][ct][r], x[it], O[ct][it]);
            }
#pragma unroll
          for (int q = 0; q < TPS; ++q)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) S[TPS * s + q][ct] *= whole;
        }
      }
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int it = 0; it < CT; ++it) O[ct][it] *= inner[it];
      if constexpr (SHARED) {
        lds_barrier();
#pragma unroll
        for (int it = 0; it < CT; ++it)
#pragma unroll
          for (int jt = 0; jt < CT; ++jt)
            if (REV ? jt >= it : jt <= it) {
              f32x4 part[GW];
#pragma unroll
              for (int v = 0; v < GW; ++v) part[v] = shares[(((second * GW + v) * CT + jt) * CT + it) * 64 + (tid & 63)];
#pragma unroll
              for (int v = GW / 2; v > 0; v /= 2)
#pragma unroll
                for (int x = 0; x < v; ++x) part[x] += part[x + v];
              P[jt][it] = part[0];
            }
      }
      // what is not to be seen is left out, not multiplied by zero: it may be anything
#pragma unroll
      for (int jt = 0; jt < CT; ++jt)
#pragma unroll
        for (int it = 0; it < CT; ++it)
          if (REV ? jt >= it : jt <= it)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float f = near[REV ? jt - it : it - jt][r];
              P[jt][it][r] = jt == it && (REV ? 4 * g + r < l : 4 * g + r > l) ? 0.f : P[jt][it][r] * f;
            }
      if constexpr (BF) {
#pragma unroll
        for (int jp = 0; jp < CT; jp += 2)
#pragma unroll
          for (int it = 0; it < CT; ++it)
            if (REV ? jp + 1 >= it : jp <= it) {
              const Halves a0 = halves(P[jp][it]), a1 = halves(P[jp + 1][it]);
              const bf16x8 high = join(a0.high, a1.high), low = join(a0.low, a1.low);
#pragma unroll
              for (int ct = 0; ct < NC; ++ct) O[ct][it] = mfma16(join(z[ct][jp], z[ct][jp + 1]), high, O[ct][it]);
#pragma unroll
              for (int ct = 0; ct < NC; ++ct) O[ct][it] = mfma16(join(z[ct][jp], z[ct][jp + 1]), low, O[ct][it]);
            }
      } else {
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
          f32x4 v[NC];
#pragma unroll
          for (int ct = 0; ct < NC; ++ct) v[ct] = widen(z[ct][jt]);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int it = 0; it < CT; ++it)
              if (REV ? jt >= it : jt <= it)
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) O[ct][it] = mfma4(v[ct][r], P[jt][it][r], O[ct][it]);
        }
      }
    }
    if constexpr (!STATE_ONLY) {
      if (bad)
#pragma clang loop unroll(disable)
        for (int j = 0; j < n; ++j) {
          int here = 0;                                        // (nothing of this rare turn is to be prepared outside of it)
          asm volatile("" : "+v"(here));
          float zo[NC][4], zs[NC];                             // row j in the lane's columns of O, of S
          bool any = false;
#pragma unroll
          for (int ct = 0; ct < NC; ++ct) {
#pragma unroll
            for (int r = 0; r < 4; ++r) zo[ct][r] = (float)*reinterpret_cast<const T*>(lz + here + TZ::at(j, cw + place<T, NC == 2>(ct, 4 * g + r)));
            zs[ct] = (float)*reinterpret_cast<const T*>(lz + here + TZ::at(j, cw + place<T, NC == 2>(ct, l)));
            any |= nonfinite(zs[ct]);
          }
          if (!__any(any)) continue;
#pragma unroll
          for (int it = 0; it < CT; ++it) {
            const int row = 16 * it + l, e = REV ? j - row : row - j;
            float dot = 0.f;
#pragma clang loop unroll(disable) vectorize(disable)
            for (int a = 0; a < DA; ++a)
              dot = fmaf((float)*reinterpret_cast<const T*>(lx + here + TA::at(row, a)),
                         (float)*reinterpret_cast<const T*>(ly + here + TA::at(j, a)), dot);
            dot *= e < 0 ? 0.f : p.intra * power(g2, e);
#pragma unroll
            for (int ct = 0; ct < NC; ++ct)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (e >= 0 && row < n && nonfinite(zo[ct][r])) O[ct][it][r] += dot * zo[ct][r];
          }
          const float f = p.update * power(g2, REV ? j + 1 : n - 1 - j);
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float y = f * (float)*reinterpret_cast<const T*>(ly + here + TA::at(j, place<T, true>(d, 4 * g + r)));
#pragma unroll
              for (int ct = 0; ct < NC; ++ct)
                if (nonfinite(zs[ct])) S[d][ct][r] = fmaf(y, zs[ct], S[d][ct][r]);
            }
        }
      // rows that do not count come from rows of zeros, but zero times what is not finite is not zero
      if (n < CH)
#pragma unroll
        for (int it = 0; it < CT; ++it)
          if (16 * it + l >= n)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) O[ct][it] = f32x4{0.f, 0.f, 0.f, 0.f};
      // What the wait at the next chunk's front counts on: its loads go out ahead of these stores.  The loads say nothing about memory to the
      // compiler; statements like them it leaves in order, and the stores in order with this one.
      asm volatile("" ::: "memory");
      put(O, t, min(CH, t1 - t));
      stored = n == CH && __builtin_amdgcn_readfirstlane(cw) + 16 * NC <= cols;      // (the same in all lanes: a barrier depends on it)
    }
    // the state behind the chunk; Y's columns are read AHEAD tiles ahead
    const float apart = power(g2, REV ? t - t0 : te - t - n);  // (STATE_ONLY: the tokens between the chunk and the state)
    constexpr int AHEAD = 2;
    V4 yc[AHEAD + 1][CT];
    auto turned = [&](int d) {
#pragma unroll
      for (int jt = 0; jt < CT; ++jt) yc[d % (AHEAD + 1)][jt] = TA::template columns<true>(ly, cols1, jt, d);
    };
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) turned(d);
    if constexpr (BF) {
      constexpr int PARTS = EXACT ? 3 : 2;
      bf16x8 part[NC][CT / 2][PARTS];
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int jp = 0; jp < CT; jp += 2) {
          bf16x4 k[2][PARTS];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            f32x4 v = widen(z[ct][jp + q]);
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] *= STATE_ONLY ? outer[jp + q][r] * apart : outer[jp + q][r];
#pragma unroll
            for (int m = 0; m < PARTS; ++m) {
              k[q][m] = narrow(v);
              if (m + 1 < PARTS) v -= widen(k[q][m]);
            }
          }
#pragma unroll
          for (int m = 0; m < PARTS; ++m) part[ct][jp / 2][m] = join(k[0][m], k[1][m]);
        }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if (d + AHEAD < DT) turned(d + AHEAD);
#pragma unroll
        for (int jp = 0; jp < CT; jp += 2)
#pragma unroll
          for (int m = 0; m < PARTS; ++m)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct)
              S[d][ct] = mfma16(join(yc[d % (AHEAD + 1)][jp], yc[d % (AHEAD + 1)][jp + 1]), part[ct][jp / 2][m], S[d][ct]);
      }
    } else {
      f32x4 v[NC][CT];
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
          v[ct][jt] = widen(z[ct][jt]);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[ct][jt][r] *= STATE_ONLY ? outer[jt][r] * apart : outer[jt][r];
        }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if (d + AHEAD < DT) turned(d + AHEAD);
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
          const f32x4 y = widen(yc[d % (AHEAD + 1)][jt]);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) S[d][ct] = mfma4(y[r], v[ct][jt][r], S[d][ct]);
        }
      }
    }
  }

  float* const s = STATE_ONLY ? p.seg + (bh * (p.nseg - 1) + order) * D : (order == p.nseg - 1 && p.s_out && !second ? p.s_out + bh * D : nullptr);
  if (s) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int a = place<T, true>(d, 4 * g + r), c = cw + place<T, NC == 2>(ct, l);
          if (a < Da && c < cols) s[(size_t)a * p.sa + (size_t)(c0 + c) * p.sb] = S[d][ct][r];
        }
  }
}

// EXACT: a state here is a result (only bf16 rows have another way to one that is not)
template <typename T, int DA, int NC, int NW, bool VEC, bool REV> hipError_t launch_sized(const RingLinArgs& a, bool state_only, hipStream_t st) {
  constexpr bool BF = Type<T>::BF;
  constexpr int CT = sizeof(T) == 4 ? 1 : 2, CTS = BF ? CT : 2 * CT;           // tiles of a chunk; for states alone (see segment_states)
  const dim3 grid((unsigned)((long)(state_only ? a.nseg - 1 : a.nseg) * a.slices * a.H * a.B)), block(64 * NW);
  const bool exact = !BF || a.s_out;
  if (state_only) {
    if constexpr (NC == 1 && NW == 4) {                        // (see segment_states)
      if (exact) hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, NW, CTS, VEC, REV, true, true>), grid, block, 0, st, a);
      else hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, NW, CTS, VEC, REV, true, !BF>), grid, block, 0, st, a);
    }
  } else {
    if (exact) hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, NW, CT, VEC, REV, false, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, NW, CT, VEC, REV, false, !BF>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}

// Wide heads (a state of 256 rows): four waves of 32 columns fill the registers, one wave a SIMD.  fp32 products take eight waves of 16
// instead, two a SIMD (8 x 2000 tokens, 8 heads of 256: 435 -> 389 us); bf16 products would form the weights twice as often.
// Up to 128 rows four waves of 32 columns, so that the weights are formed once for 128 columns.
template <typename T, bool VEC, bool REV> hipError_t launch_access(const RingLinArgs& a, bool state_only, hipStream_t st) {
  if (a.narrow) {
    if (a.Da <= 64) return launch_sized<T, 64, 1, 4, VEC, REV>(a, state_only, st);
    if (a.Da <= 128) return launch_sized<T, 128, 1, 4, VEC, REV>(a, state_only, st);
    return launch_sized<T, 256, 1, 4, VEC, REV>(a, state_only, st);
  }
  if (a.Da <= 64) return launch_sized<T, 64, 2, 4, VEC, REV>(a, state_only, st);
  if (a.Da <= 128) return launch_sized<T, 128, 2, 4, VEC, REV>(a, state_only, st);
  return launch_sized<T, 256, Type<T>::BF ? 2 : 1, Type<T>::BF ? 4 : 8, VEC, REV>(a, state_only, st);
}

// Two passes at once, backwards in time: heads whose dk and dv go with the same kernel
template <typename T, int DA, int NC, bool VEC> hipError_t launch_two(const RingLinArgs& a, hipStream_t st) {
  constexpr bool BF = Type<T>::BF;
  constexpr int CT = sizeof(T) == 4 ? 1 : 2;
  const dim3 grid((unsigned)((long)a.nseg * a.H * a.B)), block(512);
  if (!BF || a.s_out) hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, 8, CT, VEC, true, false, true, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, 8, CT, VEC, true, false, !BF, true>), grid, block, 0, st, a);
  return hipGetLastError();
}

template <typename T> hipError_t launch_pair(const RingLinArgs& a, hipStream_t st) {
  const bool vec = a.X.vec && a.Y.vec && a.Z.vec && a.X2.vec && a.out_vec;
  if (a.Da <= 64) return vec ? launch_two<T, 64, 1, true>(a, st) : launch_two<T, 64, 1, false>(a, st);
  return vec ? launch_two<T, 128, 2, true>(a, st) : launch_two<T, 128, 2, false>(a, st);
}

template <typename T> hipError_t launch(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  const bool vec = a.Y.vec && a.Z.vec && (state_only || (a.X.vec && a.out_vec));
  if (rev) return vec ? launch_access<T, true, true>(a, state_only, st) : launch_access<T, false, true>(a, state_only, st);
  return vec ? launch_access<T, true, false>(a, state_only, st) : launch_access<T, false, false>(a, state_only, st);
}

}  // namespace ring_lin
