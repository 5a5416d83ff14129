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

__device__ __forceinline__ f32x4 widen(bf16x4 x) { return __builtin_convertvector(x, f32x4); }
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
template <typename T> __device__ __forceinline__ bool words_nonfinite(u32x4 w) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    constexpr unsigned E = sizeof(T) == 4 ? 0x7f800000u : (Type<T>::BF ? 0x7f80u : 0x7c00u);
    bad |= (w[i] & E) == E;
    if (sizeof(T) == 2) bad |= (w[i] & (E << 16)) == (E << 16);
  }
  return bad;
}

// One tile of ROWS x COLS values, global -> registers -> LDS.
template <typename T, int ROWS, int COLS, int NT> struct Stage {
  typedef typename Type<T>::C C;
  static constexpr int EPV = Type<T>::EPV, UPR = COLS / EPV, UNITS = ROWS * UPR, NU = (UNITS + NT - 1) / NT, LD = COLS + Type<T>::PAD;
  u32x4 r[NU];

  // n rows of `cols` values from base on, token stride st
  __device__ __forceinline__ void load(const T* base, long st, int n, int cols, bool vec, int tid) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int idx = tid + u * NT, row = idx / UPR, c = (idx % UPR) * EPV;
      r[u] = u32x4{0, 0, 0, 0};
      if (row < n && c < cols) {
        const T* p = base + (long)row * st + c;
        if (vec) {
          r[u] = *reinterpret_cast<const u32x4*>(p);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int e = 0; e < EPV; ++e)
            if (c + e < cols) r[u][e] = __builtin_bit_cast(unsigned, p[e]);
        } else {
#pragma unroll
          for (int e = 0; e < EPV; ++e)
            if (c + e < cols) r[u][e / 2] |= (unsigned)__builtin_bit_cast(unsigned short, p[e]) << (16 * (e & 1));
        }
      }
    }
  }
  __device__ __forceinline__ void store(C* tile, int tid) const {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int idx = tid + u * NT, row = idx / UPR, c = (idx % UPR) * EPV;
      if (UNITS % NT == 0 || idx < UNITS) {
        C* p = tile + row * LD + c;
        if constexpr (sizeof(C) == sizeof(T)) {
          *reinterpret_cast<u32x4*>(p) = r[u];
        } else {
          const f16x8 h = __builtin_bit_cast(f16x8, r[u]);
          *reinterpret_cast<f32x4*>(p) = f32x4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
          *reinterpret_cast<f32x4*>(p + 4) = f32x4{(float)h[4], (float)h[5], (float)h[6], (float)h[7]};
        }
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
template <typename T, int DA, int NC, int CT, bool REV, bool STATE_ONLY>
__global__ __launch_bounds__(256, (DA <= 128 ? 2 : 1)) void ring_linattn_kernel(RingLinArgs p) {
  constexpr int NW = 4, NT = 64 * NW, WC = 16 * NC * NW, CH = 16 * CT, DT = DA / 16;
  constexpr bool BF = Type<T>::BF;
  typedef typename Type<T>::C C;
  typedef Stage<T, CH, DA, NT> SA;
  typedef Stage<T, CH, WC, NT> SZ;
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
  const int t0 = seg * p.seg_tokens, t1 = min(T_, t0 + p.seg_tokens), nch = (t1 - t0 + CH - 1) / CH;
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

  SA rx, ry;
  SZ rz;
  auto fetch = [&](int c) {
    const int t = t0 + c * CH, n = min(max(len - t, 0), min(CH, t1 - t));
    if (n <= 0) return;
    if (!STATE_ONLY) rx.load(X + (long)t * p.X.st, p.X.st, n, p.Da, p.X.vec, tid);
    ry.load(Y + (long)t * p.Y.st, p.Y.st, n, p.Da, p.Y.vec, tid);
    rz.load(Z + (long)t * p.Z.st, p.Z.st, n, cols, p.Z.vec, tid);
  };
  if (tid < 2) flag[tid] = 0;
  __syncthreads();
  fetch(REV ? nch - 1 : 0);
  for (int i = 0; i < nch; ++i) {
    const int c = REV ? nch - 1 - i : i, t = t0 + c * CH;
    const int rows = min(CH, t1 - t), n = min(max(len - t, 0), rows);
    f32x4 O[NC][CT];
#pragma unroll
    for (int ct = 0; ct < NC; ++ct)
#pragma unroll
      for (int it = 0; it < CT; ++it) O[ct][it] = f32x4{0.f, 0.f, 0.f, 0.f};

    if (n > 0) {
      if (!STATE_ONLY) {
        rx.store(ldsX, tid);
        if (rz.bad()) flag[i & 1] = 1;
        if (tid == 0) flag[(i + 1) & 1] = 0;
      }
      ry.store(ldsY, tid);
      rz.store(ldsZ, tid);
      __syncthreads();
    }
    if (i + 1 < nch) fetch(REV ? c - 1 : c + 1);
    if (n > 0) {
      if (n != n_now) {                                        // (whole chunks, but for the last of a sequence)
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
        f32x4 P[CT][CT];                                       // [tile of Y's rows][tile of X's rows]
#pragma unroll
        for (int jt = 0; jt < CT; ++jt)
#pragma unroll
          for (int it = 0; it < CT; ++it) P[jt][it] = f32x4{0.f, 0.f, 0.f, 0.f};
        // weights, and what the state in front gives
#pragma unroll
        for (int s = 0; s < DT; s += 2) {
          if constexpr (BF) {
            bf16x8 x[CT];
#pragma unroll
            for (int it = 0; it < CT; ++it)
              x[it] = join(read_rows<SA::LD>(ldsX, 16 * it, 16 * s, g, l), read_rows<SA::LD>(ldsX, 16 * it, 16 * s + 16, g, l));
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) {
              const bf16x4 a0 = narrow(S[s][ct]), a1 = narrow(S[s + 1][ct]);
              const bf16x4 b0 = narrow(S[s][ct] - widen(a0)), b1 = narrow(S[s + 1][ct] - widen(a1));
              const bf16x8 hi = join(a0, a1), lo = join(b0, b1);
#pragma unroll
              for (int it = 0; it < CT; ++it) {
                O[ct][it] = mfma16(hi, x[it], O[ct][it]);
                O[ct][it] = mfma16(lo, x[it], O[ct][it]);
              }
            }
#pragma unroll
            for (int jt = 0; jt < CT; ++jt) {
              const bf16x8 y = join(read_rows<SA::LD>(ldsY, 16 * jt, 16 * s, g, l), read_rows<SA::LD>(ldsY, 16 * jt, 16 * s + 16, g, l));
#pragma unroll
              for (int it = 0; it < CT; ++it)
                if (REV ? jt >= it : jt <= it) P[jt][it] = mfma16(y, x[it], P[jt][it]);
            }
          } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              f32x4 x[CT];
#pragma unroll
              for (int it = 0; it < CT; ++it) x[it] = read_rows<SA::LD>(ldsX, 16 * it, 16 * (s + q), g, l);
#pragma unroll
              for (int ct = 0; ct < NC; ++ct)
#pragma unroll
                for (int it = 0; it < CT; ++it)
#pragma unroll
                  for (int r = 0; r < 4; ++r) O[ct][it] = mfma4(S[s + q][ct][r], x[it][r], O[ct][it]);
#pragma unroll
              for (int jt = 0; jt < CT; ++jt) {
                const f32x4 y = read_rows<SA::LD>(ldsY, 16 * jt, 16 * (s + q), g, l);
#pragma unroll
                for (int it = 0; it < CT; ++it)
                  if (REV ? jt >= it : jt <= it)
#pragma unroll
                    for (int r = 0; r < 4; ++r) P[jt][it] = mfma4(y[r], x[it][r], P[jt][it]);
              }
            }
          }
        }
#pragma unroll
        for (int ct = 0; ct < NC; ++ct)
#pragma unroll
          for (int it = 0; it < CT; ++it) O[ct][it] *= inner[it];
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
        // A row of Z with infinities or NaN must not reach rows that do not see it: there the products within tiles on the
        // diagonal, which multiply it by zero, go without its non-finite values, which are added one by one.
        const bool bad = flag[i & 1] != 0;
#pragma unroll
        for (int ct = 0; ct < NC; ++ct) {
          if constexpr (BF) {
#pragma unroll
            for (int jp = 0; jp < CT; jp += 2) {
              bf16x4 z0 = read_columns<SZ::LD, NC>(ldsZ, 16 * jp, cw, ct, g, l), z1 = read_columns<SZ::LD, NC>(ldsZ, 16 * jp + 16, cw, ct, g, l);
              if (bad)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if (nonfinite((float)z0[e])) z0[e] = (__bf16)0.f;
                  if (nonfinite((float)z1[e])) z1[e] = (__bf16)0.f;
                }
              const bf16x8 z = join(z0, z1);
#pragma unroll
              for (int it = 0; it < CT; ++it)
                if (REV ? jp + 1 >= it : jp <= it) {
                  const bf16x4 a0 = narrow(P[jp][it]), a1 = narrow(P[jp + 1][it]);
                  O[ct][it] = mfma16(z, join(a0, a1), O[ct][it]);
                  O[ct][it] = mfma16(z, join(narrow(P[jp][it] - widen(a0)), narrow(P[jp + 1][it] - widen(a1))), O[ct][it]);
                }
            }
          } else {
#pragma unroll
            for (int jt = 0; jt < CT; ++jt) {
              f32x4 z = read_columns<SZ::LD, NC>(ldsZ, 16 * jt, cw, ct, g, l);
              if (bad)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (nonfinite(z[e])) z[e] = 0.f;
#pragma unroll
              for (int it = 0; it < CT; ++it)
                if (REV ? jt >= it : jt <= it)
#pragma unroll
                  for (int r = 0; r < 4; ++r) O[ct][it] = mfma4(z[r], P[jt][it][r], O[ct][it]);
            }
          }
        }
        if (bad) {
          for (int j = 0; j < n; ++j) {
            float z[NC][4];
            bool any = false;
#pragma unroll
            for (int ct = 0; ct < NC; ++ct)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                z[ct][r] = (float)ldsZ[j * SZ::LD + cw + column<NC>(ct, 4 * g + r)];
                any |= nonfinite(z[ct][r]);
              }
            if (!__any(any)) continue;
#pragma unroll
            for (int it = 0; it < CT; ++it) {
              const int row = 16 * it + l, e = REV ? j - row : row - j;
              float dot = 0.f;
              for (int a = 0; a < DA; ++a) dot = fmaf((float)ldsX[row * SA::LD + a], (float)ldsY[j * SA::LD + a], dot);
              if (e < 0) continue;
              dot *= p.intra * power(g2, e);
#pragma unroll
              for (int ct = 0; ct < NC; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                  if (nonfinite(z[ct][r])) O[ct][it][r] += dot * z[ct][r];
            }
          }
        }
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
            for (int ct = 0; ct < NC; ++ct)
#pragma unroll
              for (int k = 0; k < 3; ++k) S[d][ct] = mfma16(y, z[ct][jp / 2][k], S[d][ct]);
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
            for (int ct = 0; ct < NC; ++ct)
#pragma unroll
              for (int r = 0; r < 4; ++r) S[d][ct] = mfma4(y[r], z[ct][jt][r], S[d][ct]);
          }
        }
      }
      __syncthreads();                                         // the tiles are free for the next chunk
    }
    if constexpr (!STATE_ONLY) {
      const bool wide = p.out_vec;
#pragma unroll
      for (int it = 0; it < CT; ++it) {
        const int row = 16 * it + l, c = cw + (NC == 2 ? 8 * g : 4 * g);
        if (row >= rows || c >= cols) continue;
        const size_t at = (((size_t)b * T_ + t + row) * p.H + h) * p.Db + c0 + c;
        float v[4 * NC];
#pragma unroll
        for (int ct = 0; ct < NC; ++ct)
#pragma unroll
          for (int r = 0; r < 4; ++r) v[4 * ct + r] = O[ct][it][r];
        if (p.out_f32 || sizeof(T) == 4) {
          float* o = (float*)p.out + at;
          if (wide) {
#pragma unroll
            for (int ct = 0; ct < NC; ++ct) *reinterpret_cast<f32x4*>(o + 4 * ct) = O[ct][it];
          } else {
#pragma unroll
            for (int e = 0; e < 4 * NC; ++e)
              if (c + e < cols) o[e] = v[e];
          }
        } else {
          T* o = (T*)p.out + at;
          typedef T vec_t __attribute__((ext_vector_type(4 * NC)));
          vec_t q;
#pragma unroll
          for (int e = 0; e < 4 * NC; ++e) q[e] = (T)v[e];
          if (wide) {
            *reinterpret_cast<vec_t*>(o) = q;
          } else {
#pragma unroll
            for (int e = 0; e < 4 * NC; ++e)
              if (c + e < cols) o[e] = q[e];
          }
        }
      }
    }
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

template <typename T, int DA, int NC> hipError_t launch_sized(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  constexpr int CT = 2;
  const dim3 grid((unsigned)((long)a.nseg * a.slices * a.H * a.B)), block(256);
  if (state_only) {
    if (rev) hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, true, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, false, true>), grid, block, 0, st, a);
  } else {
    if (rev) hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, true, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((ring_linattn_kernel<T, DA, NC, CT, false, false>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}

template <typename T> hipError_t launch(const RingLinArgs& a, bool rev, bool state_only, hipStream_t st) {
  if (a.Db <= 64) {
    if (a.Da <= 32) return launch_sized<T, 32, 1>(a, rev, state_only, st);
    if (a.Da <= 64) return launch_sized<T, 64, 1>(a, rev, state_only, st);
    if (a.Da <= 128) return launch_sized<T, 128, 1>(a, rev, state_only, st);
    return launch_sized<T, 256, 1>(a, rev, state_only, st);
  }
  if (a.Da <= 32) return launch_sized<T, 32, 2>(a, rev, state_only, st);
  if (a.Da <= 64) return launch_sized<T, 64, 2>(a, rev, state_only, st);
  if (a.Da <= 128) return launch_sized<T, 128, 2>(a, rev, state_only, st);
  return launch_sized<T, 256, 2>(a, rev, state_only, st);
}

}  // namespace ring_lin
