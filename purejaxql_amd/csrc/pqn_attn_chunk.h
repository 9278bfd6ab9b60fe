// pqn_attn_chunk.h -- the chunked scan of pqn_attn.hip (see there for the operator), included by one source file per element type.
#pragma once
#include <type_traits>

#include "pqn_vec.h"

struct da_pass {
  const void *q, *k, *v;
  void *o;
  long long qs[3], ks[3], vs[3], os[3];   // strides over (time, row, head) in elements
  const float *s_in;
  float *s_out;
  int s_rs, s_cs;                         // element strides of the state's first (q, k) and second (v, o) index
  const uint8_t *reset;                   // flag of the border before step i at reset[i * reset_ts + row]
  long long reset_ts;
  float o_scale, s_scale;                 // on the outputs; on what a step adds to the state
  int a, b;                               // width of q, k; width of v, o
  int late;                               // 0: a border (decay, reset) lies before every step.  1 (backward scans): before every step
                                          // but the first, and one more behind the last step, before the state goes out
};
struct da_args {
  da_pass pass[3];
  int t_len, m, heads;
  const float *decay;
};

// ---- the recurrence, chunk by chunk ------------------------------------------------------------------------------------------
// Within a chunk of L steps the outputs are masked matrix products, and the state crosses chunks:
//   o_t  = o_scale (decay^(t+1) S^T q_t + sum_{j <= t} decay^(t-j) (q_t . k_j) v_j)        S <- decay^n S + sum_j decay^(n-1-j) k_j v_j^T
// (terms across an episode's end fall out).  A workgroup holds one (row, head)'s whole state in accumulators, a wave 32 columns of it.
// Everything is computed transposed so that no operand leaves the registers to change its layout: P^T = K Q^T leaves 4 neighbouring
// j of one t in a lane, O^T = S^T Q^T + V^T P^T takes the state's accumulators as they lie as its left operand, and S += K^T (w V)
// shares V's fragments with it.  The columns of q, k, v are assigned to accumulator rows so that a lane's 8 values of two stacked
// 16 x 16 tiles are 8 neighbouring columns (da_col): one 16-byte read of Q, one 16-byte store of O.
//
// bf16: v_mfma_f32_16x16x32_bf16 with the state (S^T Q^T) and the weighted products (V^T P^T) rounded to bf16 as operands -- the
// output is rounded to bf16 anyway -- and w V split in two bf16 pieces (16 significant bits), because the state is an f32 result that
// is carried on.  f32: v_mfma_f32_16x16x4_f32 throughout, four of them per 16 values of k.
//
// Bound: HBM.  A chunk of 64 steps of 128 + 128 columns moves 64 KB (about 7300 cycles of a CU's share of the bandwidth) and costs
// about 2000 cycles of MFMA, 2400 of LDS and 2000 of VALU per workgroup; two workgroups share a CU, and the next chunk's loads are
// in flight in registers while a chunk is computed.
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef pqn_bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short da_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) da_s16x4 da_lds_s16x4;

// column of row (or lane) r of tile `tile`, tiles counted over 16 columns each
template <typename T>
PQN_D int da_col(int tile, int r) {
  if constexpr (sizeof(T) == 2) return 32 * (tile >> 1) + 8 * (r >> 2) + 4 * (tile & 1) + (r & 3);
  else return 16 * tile + r;
}

// A matrix of W columns in LDS, one row per step.  bf16: rows of W / 8 slots of 16 B, slot s of row r at s ^ swz(r): both the 16-byte
// reads of 8 rows at one column and the transposing reads (4 rows x 4 slots per 16 lanes) touch every bank once.  f32: rows padded by
// 16 B, which serves the 16-byte reads along a row and the 4-byte reads down a column alike.
template <typename T, int W>
struct DaTile {
  static constexpr int EV = 16 / (int)sizeof(T);
  static constexpr int LD = sizeof(T) == 2 ? W : W + 4;
  static constexpr int SHIFT = W >= 128 ? 0 : W == 64 ? 1 : 2;   // rows that share the 64 banks: 1, 2, 4
  PQN_D static int at(int row, int col) {
    if constexpr (sizeof(T) == 2) {
      const int swz = (((row & 3) >> SHIFT) << 2) | ((row >> 2) & 3);
      return row * LD + ((((col >> 3) ^ swz) << 3) | (col & 7));
    } else return row * LD + col;
  }
  // operand with the row index on the lanes (row0 + lane & 15), k along the columns from col0
  template <typename F>
  PQN_D static F rows(const T *m, int row0, int col0) {
    const int lane = threadIdx.x & 63;
    return *(const F *)(m + at(row0 + (lane & 15), col0 + (lane >> 4) * EV));
  }
  // operand with the column index on the lanes (columns da_col(tile, lane & 15) behind col0), k down the rows from row0
  template <typename F>
  PQN_D static F cols(const T *m, int row0, int col0, int tile) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    F f;
    if constexpr (sizeof(T) == 2) {
      const int c = col0 + 32 * (tile >> 1) + 8 * (i & 3) + 4 * (tile & 1), r = row0 + 8 * g + (i >> 2);
      const da_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_lds_s16x4 *)(m + at(r, c)));
      const da_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_lds_s16x4 *)(m + at(r + 4, c)));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      f = __builtin_bit_cast(F, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) f[s] = m[at(row0 + 4 * g + s, col0 + 16 * tile + i)];
    }
    return f;
  }
};

PQN_D f32x4_t da_mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
PQN_D f32x4_t da_mfma(f32x4_t a, f32x4_t b, f32x4_t c) {   // k = 4 (lane >> 4) + s in both operands
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
  return c;
}

// rows first + r (r < n) of one (row, head)'s tensor, on their way to a DaTile<T, W> of L rows
template <typename T, int W, int L, int NTHR>
struct DaLoad {
  static constexpr int EV = 16 / (int)sizeof(T), VPR = W / EV, N = L * VPR / NTHR, STEP = NTHR / VPR;
  static_assert(NTHR % VPR == 0 && L % STEP == 0, "whole rows per pass");
  u32x4_t r[N];
  PQN_D void load(const T *p, long long stride, int n, int width, bool vec) {
    const int row0 = threadIdx.x / VPR, c = (threadIdx.x % VPR) * EV;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = row0 + i * STEP;
      r[i] = u32x4_t{0u, 0u, 0u, 0u};
      if (row < n && c < width) {
        const T *src = p + row * stride + c;
        if (vec) r[i] = *(const u32x4_t *)src;
        else {
          pqn_pack<T, EV> v;
#pragma unroll
          for (int e = 0; e < EV; ++e) v.v[e] = c + e < width ? src[e] : (T)0.f;
          r[i] = __builtin_bit_cast(u32x4_t, v);
        }
      }
    }
  }
  PQN_D void store(T *lds) const {
    const int row0 = threadIdx.x / VPR, c = (threadIdx.x % VPR) * EV;
#pragma unroll
    for (int i = 0; i < N; ++i) *(u32x4_t *)(lds + DaTile<T, W>::at(row0 + i * STEP, c)) = r[i];
  }
  PQN_D static void zero_behind(T *lds, int n) {
    const int row0 = threadIdx.x / VPR, c = (threadIdx.x % VPR) * EV;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (row0 + i * STEP >= n) *(u32x4_t *)(lds + DaTile<T, W>::at(row0 + i * STEP, c)) = u32x4_t{0u, 0u, 0u, 0u};
  }
  PQN_D bool not_finite() const {
    if constexpr (sizeof(T) == 2) {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, r[i][j] & 0x7fff7fffu));
      return m.x >= 0x7f80 || m.y >= 0x7f80;
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, r[i][j] & 0x7fffffffu);
      return m >= 0x7f800000u;
    }
  }
};

struct da_split {       // the time axis in `parts` parts of `len` steps, one workgroup each; parts = 1: not cut
  int parts, len, vec;  // vec: every row of every tensor of the launch starts on 16 bytes and is whole 16-byte accesses
  float *state;         // [pass][row, head][parts - 1][a_pad * b_pad], in the order of the accumulators: the state behind part p ...
  int *cut;             // ... and whether an episode ends inside it
  long long pass_stride, cut_stride;
};

// STATE: only what the part adds to the state (its first step onwards from zero, the first part from the state that came in)
template <typename T, int AP, int NW, int L, bool STATE>
__global__ __launch_bounds__(64 * NW) void da_chunk_kernel(da_args A, da_split X, int passes) {
  constexpr int NTHR = 64 * NW, BP = 32 * NW, KB = sizeof(T) == 2 ? 32 : 16, NF = AP / KB, NS = AP / 16, NJ = L / KB, NT = L / 16;
  typedef typename std::conditional<sizeof(T) == 2, bf16x8_t, f32x4_t>::type F;
  typedef DaTile<T, AP> TA;
  typedef DaTile<T, BP> TB;
  typedef DaTile<T, L> TP;
  __shared__ __attribute__((aligned(16))) T Qs[STATE ? 8 : L * TA::LD], Ks[L * TA::LD], Vs[L * TB::LD], Ps[STATE ? 8 : L * TP::LD];
  __shared__ __attribute__((aligned(16))) float pw[L + 4], wv[L];
  __shared__ int bad[NW];
  // the passes of one (row, head) meet in one XCD's L2: workgroups go round the 8 XCDs
  const long long nunits = (long long)A.m * A.heads * (STATE ? X.parts - 1 : X.parts);
  const long long block = blockIdx.x, unit = block / (8 * passes) * 8 + block % 8;
  const int pass = (int)(block / 8 % passes);
  if (unit >= nunits) return;
  const da_pass &P = A.pass[pass];
  const int parts = STATE ? X.parts - 1 : X.parts;
  const long long mh = unit / parts;
  const int part = (int)(unit % parts);
  const int h = (int)(mh % A.heads), row = (int)(mh / A.heads);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, ln = lane & 15;
  const int t_first = part * X.len, t_end = min(A.t_len, t_first + X.len);
  const double decay = (double)A.decay[h];
  for (int i = threadIdx.x; i <= L; i += NTHR) pw[i] = (float)pqn_powi(decay, i);   // every power rounded once
  if constexpr (!STATE)
    for (int i = threadIdx.x; i < L * TP::LD; i += NTHR) Ps[i] = (T)0.f;             // tiles above the diagonal stay zero
  const T *qp = (const T *)P.q + row * P.qs[1] + h * P.qs[2];
  const T *kp = (const T *)P.k + row * P.ks[1] + h * P.ks[2];
  const T *vp = (const T *)P.v + row * P.vs[1] + h * P.vs[2];
  T *op = (T *)P.o + row * P.os[1] + h * P.os[2];
  f32x4_t s[NS][2];
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) s[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const long long so = mh * ((long long)P.a * P.b);
  const int dv0 = 32 * wave;
  float *xs = X.state + pass * X.pass_stride + (mh * (X.parts - 1)) * (long long)(AP * BP) + wave * (AP * 32) + lane * 4;
  if (part == 0) {
    if (P.s_in)
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int ra = da_col<T>(i, 4 * g + e), cb = dv0 + da_col<T>(c, ln);
            if (ra < P.a && cb < P.b) s[i][c][e] = P.s_in[so + (long long)ra * P.s_rs + (long long)cb * P.s_cs];
          }
  } else if constexpr (!STATE) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) s[i][c] = *(const f32x4_t *)(xs + (long long)(part - 1) * (AP * BP) + (i * 2 + c) * 256);
  }
  DaLoad<T, AP, L, NTHR> rq, rk;
  DaLoad<T, BP, L, NTHR> rv;
  int flag = 0;
  auto fetch = [&](int t) {
    const int n = min(L, t_end - t);
    if constexpr (!STATE) rq.load(qp + t * P.qs[0], P.qs[0], n, P.a, X.vec);
    rk.load(kp + t * P.ks[0], P.ks[0], n, P.a, X.vec);
    rv.load(vp + t * P.vs[0], P.vs[0], n, P.b, X.vec);
    flag = 0;
    if (P.reset && lane < n && (t + lane > 0 || !P.late)) flag = P.reset[(t + lane) * P.reset_ts + row];
  };
  if (t_first < t_end) fetch(t_first);
  bool any_cut = false;
  for (int t0 = t_first; t0 < t_end;) {
    int n = min(L, t_end - t0);
    __syncthreads();                                   // the chunk before has been read
    if constexpr (!STATE) rq.store(Qs);
    rk.store(Ks);
    rv.store(Vs);
    const bool nf = __any(rk.not_finite() || rv.not_finite());
    if (lane == 0) bad[wave] = nf;
    const unsigned long long cuts_all = __ballot(flag != 0);
    __syncthreads();
    int off = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) off |= bad[w];
    // A NaN or infinity in k or v times a weight of zero is no zero: such a chunk is taken one step at a time, where nothing is masked.
    if (off && n > 1) {
      n = 1;
      decltype(rk)::zero_behind(Ks, 1);
      decltype(rv)::zero_behind(Vs, 1);
      __syncthreads();
    }
    const unsigned long long cuts = cuts_all & (n == 64 ? ~0ull : (1ull << n) - 1ull);
    if (t0 + n < t_end) fetch(t0 + n);
    const int first = (t0 == 0 && P.late) ? 0 : 1;     // borders up to and including step 0 of this chunk
    const int last_cut = cuts ? 63 - __clzll(cuts) : -1;
    if (wave == 0 && lane < L) wv[lane] = lane < n && lane >= last_cut ? pw[n - 1 - lane] * P.s_scale : 0.f;
    if constexpr (!STATE) {
      // P^T tiles on and below the diagonal, dealt to the waves
#pragma unroll
      for (int tt = 0; tt < NT; ++tt)
#pragma unroll
        for (int jt = 0; jt <= tt; ++jt) {
          if ((tt * (tt + 1) / 2 + jt) % NW != wave || 16 * tt >= n) continue;
          f32x4_t p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int f = 0; f < NF; ++f) p = da_mfma(TA::template rows<F>(Ks, 16 * jt, f * KB), TA::template rows<F>(Qs, 16 * tt, f * KB), p);
          const int t = 16 * tt + ln;
          const unsigned long long upto = cuts & ((2ull << t) - 1ull);
          const int from = upto ? 63 - __clzll(upto) : 0;      // first step of t's episode in this chunk
          float o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = 16 * jt + 4 * g + e;
            o[e] = j <= t && j >= from ? p[e] * (pw[max(t - j, 0)] * P.s_scale) : 0.f;
          }
          pqn_store<T, 4>(Ps + TP::at(t, 16 * jt + 4 * g), o);
        }
    }
    __syncthreads();
    F vf[2][NJ];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < NJ; ++j) vf[c][j] = TB::template cols<F>(Vs, j * KB, dv0, c);
    if constexpr (!STATE) {
      F sf[NF][2];
#pragma unroll
      for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              sf[f][c][e] = (T)s[2 * f][c][e];
              sf[f][c][4 + e] = (T)s[2 * f + 1][c][e];
            }
          } else sf[f][c] = s[f][c];
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        if (16 * tt >= n) continue;
        f32x4_t o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          const F qf = TA::template rows<F>(Qs, 16 * tt, f * KB);
#pragma unroll
          for (int c = 0; c < 2; ++c) o[c] = da_mfma(sf[f][c], qf, o[c]);
        }
        const int t = 16 * tt + ln;
        const bool carried = (cuts & ((2ull << t) - 1ull)) == 0;
        const float w = pw[t + first];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][e] = carried ? o[c][e] * w : 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (j * KB >= 16 * (tt + 1)) continue;
          const F pf = TP::template rows<F>(Ps, 16 * tt, j * KB);
#pragma unroll
          for (int c = 0; c < 2; ++c) o[c] = da_mfma(vf[c][j], pf, o[c]);
        }
        if (t < n) {
          T *dst = op + (t0 + t) * P.os[0];
          if constexpr (sizeof(T) == 2) {
            const int col = dv0 + 8 * g;
            float v8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v8[e] = o[e >> 2][e & 3] * P.o_scale;
            if (X.vec) {
              if (col < P.b) pqn_store<T, 8>(dst + col, v8);
            } else
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (col + e < P.b) dst[col + e] = (T)v8[e];
          } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int col = dv0 + 16 * c + 4 * g;
              float v4[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v4[e] = o[c][e] * P.o_scale;
              if (X.vec) {
                if (col < P.b) pqn_store<T, 4>(dst + col, v4);
              } else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (col + e < P.b) dst[col + e] = (T)v4[e];
            }
          }
        }
      }
    }
    // the state behind the chunk
    const float fade = cuts ? 0.f : pw[n - 1 + first];
    any_cut = any_cut || cuts != 0;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][c][e] = cuts ? 0.f : s[i][c][e] * fade;
    F lo[2][NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      constexpr int EV = 16 / (int)sizeof(T);
      float w[EV];
#pragma unroll
      for (int e = 0; e < EV; e += 4) *(f32x4_t *)(w + e) = *(const f32x4_t *)(wv + j * KB + g * EV + e);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          const float x = w[e] == 0.f ? 0.f : pqn_to_f32((T)vf[c][j][e]) * w[e];
          vf[c][j][e] = (T)x;
          if constexpr (sizeof(T) == 2) lo[c][j][e] = (T)(x - pqn_to_f32((T)vf[c][j][e]));
        }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (j * KB >= n) continue;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const F kf = TA::template cols<F>(Ks, j * KB, 0, i);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          s[i][c] = da_mfma(kf, vf[c][j], s[i][c]);
          if constexpr (sizeof(T) == 2) s[i][c] = da_mfma(kf, lo[c][j], s[i][c]);
        }
      }
    }
    t0 += n;
  }
  if constexpr (STATE) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) *(f32x4_t *)(xs + (long long)part * (AP * BP) + (i * 2 + c) * 256) = s[i][c];
    if (threadIdx.x == 0) X.cut[pass * X.cut_stride + mh * (X.parts - 1) + part] = any_cut;
  } else if (P.s_out && part == X.parts - 1) {
    const bool cut = P.late && P.reset && P.reset[A.t_len * P.reset_ts + row];
    const float fade = P.late ? pw[1] : 1.f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ra = da_col<T>(i, 4 * g + e), cb = dv0 + da_col<T>(c, ln);
          if (ra < P.a && cb < P.b) P.s_out[so + (long long)ra * P.s_rs + (long long)cb * P.s_cs] = cut ? 0.f : s[i][c][e] * fade;
        }
  }
}


// widths as the kernel is built for them: rows of the state padded to AP, 32 columns a wave
inline int da_ap(int a) { return a <= 32 ? 32 : a <= 64 ? 64 : 128; }
inline int da_nw(int a, int b) {
  const int nw = b <= 32 ? 1 : b <= 64 ? 2 : 4;
  return a > 64 && nw < 2 ? 2 : nw;               // a wave alone would hold 128 registers of loads in flight
}
int da_launch_chunk_f32(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st);
int da_launch_chunk_bf16(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st);

template <typename T, int L>
static int da_launch_chunk(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st) {
  const int ap = da_ap(A.pass[0].a), nw = da_nw(A.pass[0].a, A.pass[0].b);
  const long long units = (long long)A.m * A.heads * (state ? X.parts - 1 : X.parts), grid = (units + 7) / 8 * 8 * passes;
  PQN_REQUIRE(grid < (1ll << 31), "pqn_decay_attn: %d x %d rows and heads are more than one launch covers", A.m, A.heads);
#define DA_GO(AP, NW)                                                                               \
  if (ap == AP && nw == NW) {                                                                       \
    if (state) da_chunk_kernel<T, AP, NW, L, true><<<(unsigned)grid, 64 * NW, 0, st>>>(A, X, passes);  \
    else da_chunk_kernel<T, AP, NW, L, false><<<(unsigned)grid, 64 * NW, 0, st>>>(A, X, passes);       \
    return pqn_check_launch("pqn_decay_attn");                                                      \
  }
  DA_GO(32, 1)
  DA_GO(32, 2)
  DA_GO(32, 4)
  DA_GO(64, 1)
  DA_GO(64, 2)
  DA_GO(64, 4)
  DA_GO(128, 2)
  DA_GO(128, 4)
#undef DA_GO
  pqn_set_error("pqn_decay_attn: no kernel for widths %d, %d", A.pass[0].a, A.pass[0].b);
  return PQN_E_UNSUPPORTED;
}
