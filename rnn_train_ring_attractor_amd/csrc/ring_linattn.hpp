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

// What is in memory as T is multiplied as C.  bf16 operands go to the matrix units as they are; what is computed on the way (weights,
// decayed rows, the state) enters as the sum of two or three bf16 numbers, 16 or 24 bits, so that only the results are rounded to
// bf16 and the state, which is kept in 32 bits, stays as exact as fp32 sums are.  fp32 and fp16 go to the fp32 matrix units: fp16
// because the weights and the state can pass its range.
template <typename T> struct Type;
template <> struct Type<__bf16> { typedef __bf16 C; static constexpr int EPV = 8, PAD = 16; static constexpr bool BF = true; };
template <> struct Type<float> { typedef float C; static constexpr int EPV = 4, PAD = 4; static constexpr bool BF = false; };
template <> struct Type<_Float16> { typedef float C; static constexpr int EPV = 8, PAD = 4; static constexpr bool BF = false; };

__device__ __forceinline__ float power(float g2, int e) { return e == 0 ? 1.f : __builtin_amdgcn_exp2f(g2 * (float)e); }

// (by bits: left to itself the compiler converts the second of each pair once more instead)
__device__ __forceinline__ f32x4 widen(bf16x4 x) {
  const u32x2 b = __builtin_bit_cast(u32x2, x);
  return f32x4{__builtin_bit_cast(float, b[0] << 16), __builtin_bit_cast(float, b[0] & 0xffff0000u), __builtin_bit_cast(float, b[1] << 16),
               __builtin_bit_cast(float, b[1] & 0xffff0000u)};
}
__device__ __forceinline__ bf16x4 narrow(f32x4 x) { return __builtin_convertvector(x, bf16x4); }
__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Column of operand row m (0..15) of column tile ct of a wave: with two tiles, a lane's four values of both are eight neighbours.
template <int NC> __device__ __forceinline__ int column(int ct, int m) {
  return NC == 2 ? 8 * (m >> 2) + 4 * ct + (m & 3) : m;
}

// Rows of a tile, columns col0..col0+15 in the order of `column`: element e of lane (g, l) is row 4g + e, the lane's own column.
template <int LD, int NC>
__device__ __forceinline__ bf16x4 read_columns(const __bf16* tile, int row0, int col0, int ct, int g, int l) {
  const __bf16* p = tile + (row0 + 4 * g + (l >> 2)) * LD + col0 + (NC == 2 ? 8 * (l & 3) + 4 * ct : 4 * (l & 3));
  return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}
template <int LD, int NC>
__device__ __forceinline__ f32x4 read_columns(const float* tile, int row0, int col0, int ct, int g, int l) {
  const float* p = tile + (row0 + 4 * g) * LD + col0 + column<NC>(ct, l);
  return f32x4{p[0], p[LD], p[2 * LD], p[3 * LD]};
}
// Element e of lane (g, l): row row0 + l, column col0 + 4g + e.
template <int LD> __device__ __forceinline__ bf16x4 read_rows(const __bf16* tile, int row0, int col0, int g, int l) {
  return *reinterpret_cast<const bf16x4*>(tile + (row0 + l) * LD + col0 + 4 * g);
}
template <int LD> __device__ __forceinline__ f32x4 read_rows(const float* tile, int row0, int col0, int g, int l) {
  return *reinterpret_cast<const f32x4*>(tile + (row0 + l) * LD + col0 + 4 * g);
}

__device__ __forceinline__ bool nonfinite(float x) { return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) == 0x7f800000u; }
template <typename T> __device__ constexpr unsigned exponent() { return sizeof(T) == 4 ? 0x7f800000u : (Type<T>::BF ? 0x7f80u : 0x7c00u); }
template <typename T> __device__ __forceinline__ bool words_nonfinite(u32x4 w) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    constexpr unsigned E = exponent<T>();
    bad |= (w[i] & E) == E;
    if (sizeof(T) == 2) bad |= (w[i] & (E << 16)) == (E << 16);
  }
  return bad;
}

// One tile of ROWS x COLS values, global -> registers -> LDS.  Rows from `n` on and columns from `cols` on become zero on the way into
// LDS; until then their place is taken by the last row and columns that there are, so that no load hangs on a branch (a value that is
// merged behind one is waited for there).  VEC: 16-byte loads (RingLinTensor::vec).
template <typename T, int ROWS, int COLS, int NT, bool VEC> struct Stage {
  typedef typename Type<T>::C C;
  static constexpr int EPV = Type<T>::EPV, UPR = COLS / EPV, UNITS = ROWS * UPR, NU = (UNITS + NT - 1) / NT, LD = COLS + Type<T>::PAD;
  static constexpr int RS = NT / UPR;                          // rows from a thread's unit to its next; its columns stay
  static_assert(NT % UPR == 0, "");
  u32x4 r[NU];

  // rows 0..last from base on, token stride st
  __device__ __forceinline__ void load(const T* base, long st, int last, int cols, int tid) {
    const int row = tid / UPR, c = (tid % UPR) * EPV;
    if constexpr (VEC) {
      const unsigned stb = (unsigned)st * (unsigned)sizeof(T), cb = (unsigned)(min(c, cols - EPV) * (int)sizeof(T));
#pragma unroll
      for (int u = 0; u < NU; ++u)
        r[u] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(base) + (__umul24((unsigned)min(row + u * RS, last), stb) + cb));
    } else {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const T* p = base + (long)min(row + u * RS, last) * st;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int e = 0; e < EPV; ++e) r[u][e] = __builtin_bit_cast(unsigned, p[min(c + e, cols - 1)]);
        } else {
#pragma unroll
          for (int e = 0; e < EPV; e += 2)
            r[u][e / 2] = __builtin_bit_cast(unsigned short, p[min(c + e, cols - 1)]) |
                          (unsigned)__builtin_bit_cast(unsigned short, p[min(c + e + 1, cols - 1)]) << 16;
        }
      }
    }
  }
  __device__ __forceinline__ void mask(int n, int cols, int tid) {
    const int row = tid / UPR, c = (tid % UPR) * EPV;
    if (n >= ROWS && cols >= COLS) return;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const bool in = row + u * RS < n;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (VEC) {
          r[u][e] = in && c < cols ? r[u][e] : 0u;
        } else if constexpr (sizeof(T) == 4) {
          r[u][e] = in && c + e < cols ? r[u][e] : 0u;
        } else {
          r[u][e] &= (in && c + 2 * e < cols ? 0xffffu : 0u) | (in && c + 2 * e + 1 < cols ? 0xffff0000u : 0u);
        }
      }
    }
  }
  __device__ __forceinline__ void store(C* tile, int tid) const {
    const int row = tid / UPR, c = (tid % UPR) * EPV;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (UNITS % NT != 0 && row + u * RS >= ROWS) continue;
      C* p = tile + (row + u * RS) * LD + c;
      if constexpr (sizeof(C) == sizeof(T)) {
        *reinterpret_cast<u32x4*>(p) = r[u];
      } else {
        const f16x8 h = __builtin_bit_cast(f16x8, r[u]);
        *reinterpret_cast<f32x4*>(p) = f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{(float)h[4], (float)h[5], (float)h[6], (float)h[7]};
      }
    }
  }
  __device__ __forceinline__ void clean() {                    // values that are not finite become zero
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        constexpr unsigned E = exponent<T>();
        if constexpr (sizeof(T) == 4) {
          if ((r[u][e] & E) == E) r[u][e] = 0;
        } else {
          if ((r[u][e] & E) == E) r[u][e] &= 0xffff0000u;
          if ((r[u][e] & (E << 16)) == (E << 16)) r[u][e] &= 0xffffu;
        }
      }
  }
  __device__ __forceinline__ bool bad() const {
    bool b = false;
#pragma unroll
    for (int u = 0; u < NU; ++u) b |= words_nonfinite<T>(r[u]);
    return b;
  }
};

template <typename T> __device__ __forceinline__ const T* rows_of(const RingLinTensor& t, int b, int h, int share) {
  return reinterpret_cast<const T*>(t.p) + (long)b * t.sb + (long)(h / share) * t.sh;
}

// A workgroup: one head of one sequence, WC = 16 NC NW columns of Z and of the state, one segment of the tokens.  Its waves share the
// chunk's rows in LDS; each keeps 16 NC columns of the state in registers, where they are an operand as they lie: the matrix units put
// rows 4g..4g+3 of column l into lane (g, l) and take them as contraction indices from there.  The weights are formed transposed
// for the same reason, by every wave for itself (the kernel is bound by memory: a chunk of 128-wide bf16 rows moves in about four times what
// its products take).
template <typename T, int DA, int NC, int CT, bool VEC, bool REV, bool STATE_ONLY>
__global__ __launch_bounds__(256, (DA <= 128 ? 2 : 1)) void ring_linattn_kernel(RingLinArgs p) {
  constexpr int NW = 4, NT = 64 * NW, WC = 16 * NC * NW, CH = 16 * CT, DT = DA / 16;
  constexpr bool BF = Type<T>::BF;
  typedef typename Type<T>::C C;
  typedef Stage<T, CH, DA, NT, VEC> SA;
  typedef Stage<T, CH, WC, NT, VEC> SZ;
  __shared__ __align__(16) C ldsX[STATE_ONLY ? 8 : CH * SA::LD];
  __shared__ __align__(16) C ldsY[CH * SA::LD];
  __shared__ __align__(16) C ldsZ[CH * SZ::LD];
  __shared__ int flag[2];

  const int tid = threadIdx.x, w = tid >> 6, l = tid & 15, g = (tid >> 4) & 3;
  const int seg = blockIdx.x % p.nseg, slice = blockIdx.x / p.nseg % p.slices, head = blockIdx.x / (p.nseg * p.slices);
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
  const int cols = p.Db - c0;

  f32x4 S[DT][NC];
  {
    const float* s = p.nseg > 1 && !STATE_ONLY ? p.seg + (bh * p.nseg + seg) * p.Da * p.Db : (p.s_in ? p.s_in + bh * p.Da * p.Db : nullptr);
    if (STATE_ONLY) s = nullptr;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int a = 16 * d + 4 * g + r, c = cw + column<NC>(ct, l);
          S[d][ct][r] = s && a < p.Da && c < cols ? s[(size_t)a * p.sa + (size_t)(c0 + c) * p.sb] : 0.f;
        }
  }

  // powers of the decay: by distance within a pair of tiles, and for the rows of a chunk of n
  float near[CT][4], inner[CT], outer[CT][4], whole = 1.f;
#pragma unroll
  for (int d = 0; d < CT; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int e = 16 * d + (REV ? 4 * g + r - l : l - 4 * g - r);
      near[d][r] = e < 0 ? 0.f : p.intra * power(g2, e);
    }
  int n_now = -1;

  // O = inner S X^T, what the state in front gives, and P = Y X^T, the weights
  auto from_state = [&](f32x4 (&O)[NC][CT], f32x4 (&P)[CT][CT]) {
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int it = 0; it < CT; ++it) O[ct][it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DT; s += 2) {
      if constexpr (BF) {
        bf16x8 x[CT];
#pragma unroll
        for (int it = 0; it < CT; ++it)
          x[it] = join(read_rows<SA::LD>(ldsX, 16 * it, 16 * s, g, l), read_rows<SA::LD>(ldsX, 16 * it, 16 * s + 16, g, l));
#pragma unroll
          for (int jt = 0; jt < CT; ++jt) {
            const bf16x8 y = join(read_rows<SA::LD>(ldsY, 16 * jt, 16 * s, g, l), read_rows<SA::LD>(ldsY, 16 * jt, 16 * s + 16, g, l));
#pragma unroll
            for (int it = 0; it < CT; ++it)
              if (REV ? jt >= it : jt <= it) P[jt][it] = mfma16(y, x[it], P[jt][it]);
          }
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          const bf16x4 a0 = narrow(S[s][ct]), a1 = narrow(S[s + 1][ct]);
          const bf16x8 hi = join(a0, a1), lo = join(narrow(S[s][ct] - widen(a0)), narrow(S[s + 1][ct] - widen(a1)));
#pragma unroll
          for (int it = 0; it < CT; ++it) O[ct][it] = mfma16(hi, x[it], O[ct][it]);
#pragma unroll
          for (int it = 0; it < CT; ++it) O[ct][it] = mfma16(lo, x[it], O[ct][it]);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          f32x4 x[CT];
#pragma unroll
          for (int it = 0; it < CT; ++it) x[it] = read_rows<SA::LD>(ldsX, 16 * it, 16 * (s + q), g, l);
#pragma unroll
            for (int jt = 0; jt < CT; ++jt) {
              const f32x4 y = read_rows<SA::LD>(ldsY, 16 * jt, 16 * (s + q), g, l);
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int it = 0; it < CT; ++it)
                  if (REV ? jt >= it : jt <= it) P[jt][it] = mfma4(y[r], x[it][r], P[jt][it]);
            }
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct)
#pragma unroll
              for (int it = 0; it < CT; ++it) O[ct][it] = mfma4(S[s + q][ct][r], x[it][r], O[ct][it]);
        }
      }
    }
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int it = 0; it < CT; ++it) O[ct][it] *= inner[it];
  };
  auto put = [&](const f32x4 (&O)[NC][CT], int t, int rows) {
    const int c = cw + (NC == 2 ? 8 * g : 4 * g);
    const size_t at = ((size_t)b * T_ + t) * p.H + h, size = p.out_f32 || sizeof(T) == 4 ? 4 : sizeof(T);
    char* const base = (char*)p.out + (at * p.Db + c0) * size;
    const unsigned step = (unsigned)(p.H * p.Db) * (unsigned)size, first = (unsigned)c * (unsigned)size;     // (VEC: within 24 bits)
#pragma unroll
    for (int it = 0; it < CT; ++it) {
      const int row = 16 * it + l;
      if (row >= rows || c >= cols) continue;
      char* const o = VEC ? base + (__umul24((unsigned)row, step) + first) : base + ((size_t)row * step + first);
      if (p.out_f32 || sizeof(T) == 4) {
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          if (VEC) {
            if (c + 4 * ct < cols) reinterpret_cast<f32x4*>(o)[ct] = O[ct][it];
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (c + 4 * ct + r < cols) reinterpret_cast<float*>(o)[4 * ct + r] = O[ct][it][r];
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

  SA rx, ry;
  SZ rz;
  auto fetch = [&](int c) {
    const int t = t0 + c * CH, last = min(CH, te - t) - 1;
    if (!STATE_ONLY) rx.load(X + (long)t * p.X.st, p.X.st, last, p.Da, tid);
    ry.load(Y + (long)t * p.Y.st, p.Y.st, last, p.Da, tid);
    rz.load(Z + (long)t * p.Z.st, p.Z.st, last, cols, tid);
  };
  if (tid < 2) flag[tid] = 0;
  __syncthreads();
  if (full > 0) fetch(REV ? full - 1 : 0);
  for (int i = 0; i < full; ++i) {
    const int c = REV ? full - 1 - i : i, t = t0 + c * CH, n = min(CH, te - t);
    if (!STATE_ONLY) {
      rx.mask(n, p.Da, tid);
      rx.store(ldsX, tid);
    }
    ry.mask(n, p.Da, tid);
    ry.store(ldsY, tid);
    rz.mask(n, cols, tid);
    if (!STATE_ONLY) {
      if (rz.bad()) {
        rz.clean();
        flag[i & 1] = 1;
      }
      if (tid == 0) flag[(i + 1) & 1] = 0;
    }
    rz.store(ldsZ, tid);
    lds_barrier();
    fetch(i + 1 < full ? (REV ? c - 1 : c + 1) : c);           // (the last one's again: nothing reads it)
    if (n != n_now) {                                          // (whole chunks, but for the last of a sequence)
      n_now = n;
      whole = power(g2, n);
#pragma unroll
      for (int it = 0; it < CT; ++it) {
        inner[it] = p.inter * power(g2, REV ? max(n - 1 - 16 * it - l, 0) : 16 * it + l + 1);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = 16 * it + 4 * g + r;
          outer[it][r] = p.update * power(g2, REV ? j + 1 : max(n - 1 - j, 0));
        }
      }
    }
    if constexpr (!STATE_ONLY) {
      f32x4 O[NC][CT], P[CT][CT];                              // P: [tile of Y's rows][tile of X's rows]
#pragma unroll
      for (int jt = 0; jt < CT; ++jt)
#pragma unroll
        for (int it = 0; it < CT; ++it) P[jt][it] = f32x4{0.f, 0.f, 0.f, 0.f};
      const bool bad = flag[i & 1] != 0;
      from_state(O, P);
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
        for (int jp = 0; jp < CT; jp += 2) {
          bf16x8 z[NC];
#pragma unroll
          for (int ct = 0; ct < NC; ++ct)
            z[ct] = join(read_columns<SZ::LD, NC>(ldsZ, 16 * jp, cw, ct, g, l), read_columns<SZ::LD, NC>(ldsZ, 16 * jp + 16, cw, ct, g, l));
#pragma unroll
          for (int it = 0; it < CT; ++it)
            if (REV ? jp + 1 >= it : jp <= it) {
              const bf16x4 a0 = narrow(P[jp][it]), a1 = narrow(P[jp + 1][it]);
              const bf16x8 hi = join(a0, a1), lo = join(narrow(P[jp][it] - widen(a0)), narrow(P[jp + 1][it] - widen(a1)));
#pragma unroll
              for (int ct = 0; ct < NC; ++ct) O[ct][it] = mfma16(z[ct], hi, O[ct][it]);
#pragma unroll
              for (int ct = 0; ct < NC; ++ct) O[ct][it] = mfma16(z[ct], lo, O[ct][it]);
            }
        }
      } else {
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
          f32x4 z[NC];
#pragma unroll
          for (int ct = 0; ct < NC; ++ct) z[ct] = read_columns<SZ::LD, NC>(ldsZ, 16 * jt, cw, ct, g, l);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int it = 0; it < CT; ++it)
              if (REV ? jt >= it : jt <= it)
#pragma unroll
                for (int ct = 0; ct < NC; ++ct) O[ct][it] = mfma4(z[ct][r], P[jt][it][r], O[ct][it]);
        }
      }
      // A value of Z that is infinite or NaN must not reach rows that do not see it, which the products within the tiles multiply by
      // zero: such values are zero in LDS and what they give is added here, one by one.
      if (bad)
        for (int j = 0; j < n; ++j) {
          float z[NC][4], zs[NC];                              // of the lane's columns of O, of its columns of S
          const T* row = Z + (long)(t + j) * p.Z.st;
          bool any = false;
#pragma unroll
          for (int ct = 0; ct < NC; ++ct) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int col = cw + column<NC>(ct, 4 * g + r);
              z[ct][r] = col < cols ? (float)row[col] : 0.f;
            }
            const int col = cw + column<NC>(ct, l);
            zs[ct] = col < cols ? (float)row[col] : 0.f;
            any |= nonfinite(zs[ct]);
          }
          if (!__any(any)) continue;
#pragma unroll
          for (int it = 0; it < CT; ++it) {
            const int i = 16 * it + l, e = REV ? j - i : i - j;
            float dot = 0.f;
            for (int a = 0; a < DA; ++a) dot = fmaf((float)ldsX[i * SA::LD + a], (float)ldsY[j * SA::LD + a], dot);
            dot *= e < 0 ? 0.f : p.intra * power(g2, e);
#pragma unroll
            for (int ct = 0; ct < NC; ++ct)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (e >= 0 && i < n && nonfinite(z[ct][r])) O[ct][it][r] += dot * z[ct][r];
          }
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int ct = 0; ct < NC; ++ct)
                if (nonfinite(zs[ct])) S[d][ct][r] = fmaf((float)ldsY[j * SA::LD + 16 * d + 4 * g + r], zs[ct], S[d][ct][r]);
        }
      put(O, t, min(CH, t1 - t));
    }
    // the state behind the chunk
    if constexpr (BF) {
      bf16x8 z[NC][CT / 2][3];
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int jp = 0; jp < CT; jp += 2) {
          bf16x4 part[2][3];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            f32x4 v = widen(read_columns<SZ::LD, NC>(ldsZ, 16 * (jp + q), cw, ct, g, l));
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] *= outer[jp + q][r];
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              part[q][k] = narrow(v);
              v -= widen(part[q][k]);
            }
          }
#pragma unroll
          for (int k = 0; k < 3; ++k) z[ct][jp / 2][k] = join(part[0][k], part[1][k]);
        }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) S[d][ct] *= whole;
#pragma unroll
        for (int jp = 0; jp < CT; jp += 2) {
          const bf16x8 y = join(read_columns<SA::LD, 1>(ldsY, 16 * jp, 16 * d, 0, g, l), read_columns<SA::LD, 1>(ldsY, 16 * jp + 16, 16 * d, 0, g, l));
#pragma unroll
          for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) S[d][ct] = mfma16(y, z[ct][jp / 2][k], S[d][ct]);
        }
      }
    } else {
      f32x4 z[NC][CT];
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
          z[ct][jt] = read_columns<SZ::LD, NC>(ldsZ, 16 * jt, cw, ct, g, l);
#pragma unroll
          for (int r = 0; r < 4; ++r) z[ct][jt][r] *= outer[jt][r];
        }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) S[d][ct] *= whole;
#pragma unroll
        for (int jt = 0; jt < CT; ++jt) {
          const f32x4 y = read_columns<SA::LD, 1>(ldsY, 16 * jt, 16 * d, 0, g, l);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) S[d][ct] = mfma4(y[r], z[ct][jt][r], S[d][ct]);
        }
      }
    }
    lds_barrier();                                             // the tiles are free for the next chunk
  }

  float* s = STATE_ONLY ? p.seg + (bh * p.nseg + seg) * p.Da * p.Db : (p.s_out ? p.s_out + bh * p.Da * p.Db : nullptr);
  if (!STATE_ONLY && p.nseg > 1) s = nullptr;                  // (the scan over segments writes it)
  if (s) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int ct = 0; ct < NC; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int a = 16 * d + 4 * g + r, c = cw + column<NC>(ct, l);
          if (a < p.Da && c < cols) s[(size_t)a * p.sa + (size_t)(c0 + c) * p.sb] = S[d][ct][r];
        }
  }
}

template <typename T, int DA, int NC, bool VEC> hipError_t launch_sized(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  constexpr int CT = 2;
  const dim3 grid((unsigned)((long)a.nseg * a.slices * a.H * a.B)), block(256);
  if (state_only) {
    if (rev) hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, VEC, true, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, VEC, false, true>), grid, block, 0, st, a);
  } else {
    if (rev) hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, VEC, true, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, VEC, false, false>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}

template <typename T, bool VEC> hipError_t launch_access(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  if (a.Db <= 64) {
    if (a.Da <= 64) return launch_sized<T, 64, 1, VEC>(a, rev, state_only, st);
    if (a.Da <= 128) return launch_sized<T, 128, 1, VEC>(a, rev, state_only, st);
    return launch_sized<T, 256, 1, VEC>(a, rev, state_only, st);
  }
  if (a.Da <= 64) return launch_sized<T, 64, 2, VEC>(a, rev, state_only, st);
  if (a.Da <= 128) return launch_sized<T, 128, 2, VEC>(a, rev, state_only, st);
  return launch_sized<T, 256, 2, VEC>(a, rev, state_only, st);
}

template <typename T> hipError_t launch(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  const bool vec = a.Y.vec && a.Z.vec && (state_only || (a.X.vec && a.out_vec));
  return vec ? launch_access<T, true>(a, rev, state_only, st) : launch_access<T, false>(a, rev, state_only, st);
}

}  // namespace ring_lin
