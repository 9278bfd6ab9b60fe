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
  int s_vec;                              // 2: pairs of columns lie on 8 bytes; 4: fours of rows on 16; 0: neither
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
// 16 x 16 tiles are 8 neighbouring columns (da_row, da_col): one 16-byte read of Q, one 16-byte store of O.
//
// bf16: v_mfma_f32_16x16x32_bf16.  What is f32 and an operand -- the state (S^T Q^T), the weighted products (V^T P^T), w V -- is three bf16
// pieces, which hold it exactly: sums and states are f32 and an output is rounded once.  With the state and the weights as one bf16 number
// each (2.5e-3 rms on the outputs instead of 1.7e-3, their own rounding) calls of 128 steps x 2048 rows of 128 x 128 took 123 / 266 us, now
// 137 / 321 (in turn, one session):
// 111 matrix instructions a chunk and wave instead of 71, and some 300 vector instructions.  f32: v_mfma_f32_16x16x4_f32 throughout, four
// of them per 16 values of k.
//
// Bound: HBM and the vector and matrix work together where there are rows enough.  A chunk of 32 steps of 128 + 128 bf16 columns moves 32 KB
// (about 3900 cycles of a CU's share of the bandwidth) and costs a wave 111 matrix instructions of 16 cycles beside its vector work; f32
// doubles the bytes and costs four times the instructions at 32 cycles each, about as much as the bytes.  Chunks of 32 steps and not 64:
// half the registers in flight, two waves a SIMD.  Of the 48 kernels of a type six (bf16) and nine (f32) still spill, 8 to 116 bytes a
// lane -- f32 heads of 32 in one chunk 36 at three waves a SIMD, 128 x 64 and 128 x 96 up to 80 --, bf16 and f32 heads of 128 x 128 on 16
// bytes do not.  Next chunk's loads are in flight in registers while a chunk is computed.
// Measured, forward / gradient (the kernels' least under a trace): bf16, 128 steps x 2048 rows of 128 x 128: 140 / 353 us (floors 106 / 171 by
// the bytes at 5.08 TB/s); f32, 32 steps x 16384 rows of 32 x 32: 117 / 270 us (79 / 132; the three scans of the gradient read the window
// nearly twice); whole calls of f32, 1001 steps x 35 rows of 48 x 80: 52 / 126 us (latency: three launches a scan, parts three chunks deep).
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef pqn_bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short da_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) da_s16x4 da_lds_s16x4;

// The state's accumulator tiles: row r of tile i is row da_row(i, r) of the state -- a lane's 8 values of two stacked bf16 tiles are 8
// neighbouring rows -- and lane r of tile c (of a wave's two) is column da_col(c, r) of the wave's 32: the two tiles' values of a lane
// lie side by side, for 8-byte accesses to the state and 8 neighbouring outputs in a lane.
template <typename T>
PQN_D int da_row(int tile, int r) {
  if constexpr (sizeof(T) == 2) return 32 * (tile >> 1) + 8 * (r >> 2) + 4 * (tile & 1) + (r & 3);
  else return 16 * tile + r;
}
PQN_D int da_col(int c, int r) { return 2 * r + c; }

// A matrix of W columns in LDS, one row per step.  bf16: rows of W / 8 slots of 16 B, slot s of row r at s ^ swz(r): both the 16-byte
// reads of 8 rows at one column and the transposing reads (4 rows x 4 slots per 16 lanes) touch every bank once.  f32: rows padded by
// 16 B, which serves the 16-byte reads along a row and the 4-byte reads down a column alike.
template <typename T, int W>
struct DaTile {
  static constexpr int EV = 16 / (int)sizeof(T);
  static constexpr int LD = sizeof(T) == 2 ? (W == 96 ? 128 : W) : W + 4;   // bf16: a power of two of slots
  static constexpr int SHIFT = W >= 96 ? 0 : W == 64 ? 1 : 2;   // rows that share the 64 banks: 1, 2, 4
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
  // operand with the column index on the lanes (columns da_row(tile, lane & 15)), k down the rows from row0.  bf16: a lane's 8 values are
  // rows 4 g + e and 16 + 4 g + e (e < 4), the order in which two 16 x 16 accumulators lie in a lane
  template <typename F>
  PQN_D static F cols(const T *m, int row0, int tile) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    if constexpr (sizeof(T) == 2) return turned<F>(m, row0 + 4 * g + (i >> 2), 32 * (tile >> 1) + 8 * (i & 3) + 4 * (tile & 1));
    else {
      F f;
#pragma unroll
      for (int s = 0; s < 4; ++s) f[s] = m[at(row0 + 4 * g + s, 16 * tile + i)];
      return f;
    }
  }
  // the same for both tiles of the 32 columns from col0 in the order of da_col.  bf16: such a tile's slots hold their 8 columns as the
  // even ones, then the odd ones (DaLoad, PAIRS), so that a transposing read finds a tile's four neighbours side by side
  template <typename F>
  PQN_D static void pairs(const T *m, int row0, int col0, F (&f)[2]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int c = 0; c < 2; ++c) f[c] = turned<F>(m, row0 + 4 * g + (i >> 2), col0 + 8 * (i & 3) + 4 * c);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const pqn_pack<float, 2> v = *(const pqn_pack<float, 2> *)(m + at(row0 + 4 * g + s, col0 + 2 * i));
        f[0][s] = v.v[0];
        f[1][s] = v.v[1];
      }
    }
  }
  template <typename F>
  PQN_D static F turned(const T *m, int r, int c) {
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const da_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_lds_s16x4 *)(m + at(r, c)));
    const da_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((da_lds_s16x4 *)(m + at(r + 16, c)));
    return __builtin_bit_cast(F, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// c += a b.  bf16 as asm, volatile and with the accumulator tied: the builtin lets the compiler give this instruction a destination
// that partly overlaps its accumulator input, which has given results that differed between runs.  `s_nop 1` covers an operand that a
// vector instruction has just written; a result is read by the next product of its chain or behind da_drain, and by nothing else.
PQN_D void da_mfma(bf16x8_t a, bf16x8_t b, f32x4_t &c) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
PQN_D void da_mfma2(bf16x8_t a0, bf16x8_t a1, bf16x8_t b0, bf16x8_t b1, f32x4_t (&c)[2]) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %2, %4, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %3, %5, %1"
               : "+v"(c[0]), "+v"(c[1])
               : "v"(a0), "v"(a1), "v"(b0), "v"(b1));
}
// both of c by a and the three pieces of b
PQN_D void da_mfma6(bf16x8_t a, const bf16x8_t (&b)[2][3], f32x4_t (&c)[2]) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %2, %3, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %2, %6, %1\n\t"
               "v_mfma_f32_16x16x32_bf16 %0, %2, %4, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %2, %7, %1\n\t"
               "v_mfma_f32_16x16x32_bf16 %0, %2, %5, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %2, %8, %1"
               : "+v"(c[0]), "+v"(c[1])
               : "v"(a), "v"(b[0][0]), "v"(b[0][1]), "v"(b[0][2]), "v"(b[1][0]), "v"(b[1][1]), "v"(b[1][2]));
}
// the three pieces of a by b, both of a by the three pieces of b
PQN_D void da_mfma6(const bf16x8_t (&a)[2][3], bf16x8_t b, f32x4_t (&c)[2]) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %2, %8, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %5, %8, %1\n\t"
               "v_mfma_f32_16x16x32_bf16 %0, %3, %8, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %6, %8, %1\n\t"
               "v_mfma_f32_16x16x32_bf16 %0, %4, %8, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %7, %8, %1"
               : "+v"(c[0]), "+v"(c[1])
               : "v"(a[0][0]), "v"(a[0][1]), "v"(a[0][2]), "v"(a[1][0]), "v"(a[1][1]), "v"(a[1][2]), "v"(b));
}
PQN_D void da_mfma6(const bf16x8_t (&a)[2], const bf16x8_t (&b)[3], f32x4_t (&c)[2]) {
  asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %2, %4, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %3, %4, %1\n\t"
               "v_mfma_f32_16x16x32_bf16 %0, %2, %5, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %3, %5, %1\n\t"
               "v_mfma_f32_16x16x32_bf16 %0, %2, %6, %0\n\tv_mfma_f32_16x16x32_bf16 %1, %3, %6, %1"
               : "+v"(c[0]), "+v"(c[1])
               : "v"(a[0]), "v"(a[1]), "v"(b[0]), "v"(b[1]), "v"(b[2]));
}
// waits for the products before it and hands on their results: the one wait for all of x
template <typename F, int N>
PQN_D void da_drain(f32x4_t (&x)[N][2]) {
  if constexpr (std::is_same<F, bf16x8_t>::value) {
    asm volatile("s_nop 7\n\ts_nop 7" : "+v"(x[0][0]), "+v"(x[0][1]));
#pragma unroll
    for (int i = 1; i < N; ++i) asm volatile("" : "+v"(x[i][0]), "+v"(x[i][1]));
  }
}
template <typename F>
PQN_D void da_drain(f32x4_t (&c)[2]) {
  if constexpr (std::is_same<F, bf16x8_t>::value) asm volatile("s_nop 7\n\ts_nop 7" : "+v"(c[0]), "+v"(c[1]));
}
template <typename F>
PQN_D void da_drain(f32x4_t &c) {
  if constexpr (std::is_same<F, bf16x8_t>::value) asm volatile("s_nop 7\n\ts_nop 7" : "+v"(c));
}
// f32: the builtin, whose results the compiler waits for; k = 4 (lane >> 4) + s in both operands
PQN_D void da_mfma(f32x4_t a, f32x4_t b, f32x4_t &c) {
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
}
PQN_D void da_mfma2(f32x4_t a0, f32x4_t a1, f32x4_t b0, f32x4_t b1, f32x4_t (&c)[2]) {
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    c[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a0[s], b0[s], c[0], 0, 0, 0);
    c[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(a1[s], b1[s], c[1], 0, 0, 0);
  }
}

// Rows of one (row, head)'s tensor on their way to a DaTile<T, W> of L rows.  load() only requests: every lane reads some row and column
// that exists, without a branch, so that all requests are in flight together; store() puts zeros into the rows from n on.  Columns
// from `width` on are never written: the tile starts out as zeros.
// PAIRS: the slots' even columns before their odd ones (DaTile::pairs; bf16 only)
template <typename T, int W, int L, int NTHR, bool VEC, bool PAIRS>
struct DaLoad {
  static constexpr int EV = 16 / (int)sizeof(T), VPR = W / EV, STEP = NTHR / VPR, N = (L + STEP - 1) / STEP;
  // threads behind the last whole row of a pass do the next pass's first row as well, the same values to the same place
  static constexpr bool EVEN = NTHR % VPR == 0 && L % STEP == 0;
  u32x4_t r[N];
  const T *p;                       // this lane's first row and column of the chunk
  long long stride;
  int width;
  PQN_D static int row0() { return threadIdx.x / VPR; }
  PQN_D static int col() { return threadIdx.x % VPR * EV; }
  PQN_D static bool inside(int row) { return EVEN || row < L; }
  PQN_D void start(const T *first, long long stride_, int width_) {
    stride = stride_;
    width = width_;
    p = first + row0() * stride + (col() < width ? col() : 0);
  }
  PQN_D void advance(int n) { p += n * stride; }
  PQN_D void fetch(int i, const T *src) {
    if constexpr (VEC) r[i] = *(const u32x4_t *)src;
    else {
      const int c = col() < width ? col() : 0;
      pqn_pack<T, EV> v;
#pragma unroll
      for (int e = 0; e < EV; ++e) v.v[e] = src[min(c + e, width - 1) - c];
      r[i] = __builtin_bit_cast(u32x4_t, v);
    }
  }
  PQN_D void load(int n) {          // n >= 1
    if (n == L && EVEN) {
#pragma unroll
      for (int i = 0; i < N; ++i) fetch(i, p + i * STEP * stride);
    } else
#pragma unroll
      for (int i = 0; i < N; ++i) fetch(i, p + (min(row0() + i * STEP, n - 1) - row0()) * stride);
  }
  PQN_D void store(T *lds, int n) {
    const int c = col();
    if (c >= width) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = u32x4_t{0u, 0u, 0u, 0u};          // not_finite() looks at these too
      return;
    }
    if (n < L) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (row0() + i * STEP >= n) r[i] = u32x4_t{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = row0() + i * STEP;
      if constexpr (!VEC) {
        pqn_pack<T, EV> v = __builtin_bit_cast(pqn_pack<T, EV>, r[i]);
#pragma unroll
        for (int e = 0; e < EV; ++e) v.v[e] = c + e < width ? v.v[e] : (T)0.f;
        r[i] = __builtin_bit_cast(u32x4_t, v);
      }
      u32x4_t x = r[i];
      if constexpr (PAIRS && sizeof(T) == 2)
        x = u32x4_t{__builtin_amdgcn_perm(r[i][1], r[i][0], 0x05040100u), __builtin_amdgcn_perm(r[i][3], r[i][2], 0x05040100u),
                    __builtin_amdgcn_perm(r[i][1], r[i][0], 0x07060302u), __builtin_amdgcn_perm(r[i][3], r[i][2], 0x07060302u)};
      if (inside(row)) *(u32x4_t *)(lds + DaTile<T, W>::at(row, c)) = x;
    }
  }
  PQN_D static void zero_behind(T *lds, int n) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = row0() + i * STEP;
      if (row >= n && inside(row)) *(u32x4_t *)(lds + DaTile<T, W>::at(row, col())) = u32x4_t{0u, 0u, 0u, 0u};
    }
  }
  PQN_D bool not_finite() const {                                          // of what store() has put down
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

// two floats to bf16, one instruction; the value of a bf16 pair's halves
typedef pqn_bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
PQN_D uint32_t da_pair(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), bf16x2_t)); }
PQN_D float da_low(uint32_t p) { return __uint_as_float(p << 16); }
PQN_D float da_high(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// f32 numbers as the sum of three bf16 ones, exactly: the leading 8 bits of what is left, three times (cut off, not rounded: the largest
// floats stay finite).  da_cut3 takes one piece of a pair off it.
PQN_D uint32_t da_cut3(float &a, float &b) {
  const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
  a -= __uint_as_float(ua & 0xffff0000u);
  b -= __uint_as_float(ub & 0xffff0000u);
  return __builtin_amdgcn_perm(ub, ua, 0x07060302u);
}
PQN_D void da_pieces(f32x4_t a, f32x4_t b, bf16x8_t (&x)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    u32x4_t u;
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = da_cut3(v[2 * e], v[2 * e + 1]);
    x[k] = __builtin_bit_cast(bf16x8_t, u);
    a = f32x4_t{v[0], v[1], v[2], v[3]};
    b = f32x4_t{v[4], v[5], v[6], v[7]};
  }
}

struct da_split {       // the time axis in `parts` parts of `len` steps, one workgroup each; parts = 1: not cut
  int parts, len;
  int vec;              // every row of every tensor of the launch starts on 16 bytes and is whole 16-byte accesses
  float *state;         // [pass][row, head][parts - 1][a_pad * b_pad], in the order of the accumulators: the state behind part p ...
  int *cut;             // ... and whether an episode ends inside it
  long long pass_stride, cut_stride;
};

// A wave's 32 columns of a state in memory, to or from its accumulators: two columns an access where they lie side by side, four rows
// where those do (a transposed state).  Reads go out without a branch between them: a row or column that does not exist reads the
// first and counts as zero.  WHOLE: all of them exist.
template <typename T, int NS, bool WHOLE>
PQN_D void da_state_in(f32x4_t (&s)[NS][2], const float *mem, const da_pass &P, int dv0) {
  const int lane = threadIdx.x & 63, g = lane >> 4, col = dv0 + 2 * (lane & 15);
  if (P.s_vec == 2) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = da_row<T>(i, 4 * g) + e;
        const bool in = WHOLE || (row < P.a && col < P.b);
        const pqn_pack<float, 2> v = *(const pqn_pack<float, 2> *)(mem + (in ? (long long)row * P.s_rs + col : 0ll));
        s[i][0][e] = in ? v.v[0] : 0.f;
        s[i][1][e] = in ? v.v[1] : 0.f;
      }
  } else if (P.s_vec == 4) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = da_row<T>(i, 4 * g);
        const bool in = WHOLE || (row < P.a && col + c < P.b);
        const f32x4_t v = *(const f32x4_t *)(mem + (in ? row + (long long)(col + c) * P.s_cs : 0ll));
        s[i][c] = in ? v : f32x4_t{0.f, 0.f, 0.f, 0.f};
      }
  } else {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int row = da_row<T>(i, 4 * g) + e;
          const bool in = WHOLE || (row < P.a && col + c < P.b);
          const float v = mem[in ? (long long)row * P.s_rs + (long long)(col + c) * P.s_cs : 0ll];
          s[i][c][e] = in ? v : 0.f;
        }
  }
}
template <typename T, int NS, bool WHOLE>
PQN_D void da_state_out(const f32x4_t (&s)[NS][2], float *mem, const da_pass &P, int dv0) {
  const int lane = threadIdx.x & 63, g = lane >> 4, col = dv0 + 2 * (lane & 15);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int row = da_row<T>(i, 4 * g);
    if (P.s_vec == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (WHOLE || (row + e < P.a && col < P.b))
          *(pqn_pack<float, 2> *)(mem + (long long)(row + e) * P.s_rs + col) = pqn_pack<float, 2>{{s[i][0][e], s[i][1][e]}};
    } else {                       // a state that goes out is never transposed
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (row + e < P.a && col + c < P.b) mem[(long long)(row + e) * P.s_rs + (long long)(col + c) * P.s_cs] = s[i][c][e];
    }
  }
}

// What a workgroup does: MAIN a part of the time axis; STATE only what the part adds to the state (its first step onwards from zero, the
// first part from the state that came in); ONE a window that is one chunk, with nothing in flight beside the computation and so with
// registers for twice the waves.
enum { DA_MAIN, DA_STATE, DA_ONE };
template <typename T, int AP, int NW, int L, bool VEC, int MODE>
__global__ __launch_bounds__(64 * NW, MODE == DA_ONE && AP == 32 ? 3 : 2) void da_chunk_kernel(da_args A, da_split X, int passes) {
  constexpr bool B16 = sizeof(T) == 2, STATE = MODE == DA_STATE;
  constexpr int NTHR = 64 * NW, BP = 32 * NW, KB = B16 ? 32 : 16, NF = AP / KB, NS = AP / 16, NJ = L / KB, NT = L / 16;
  constexpr int EV = 16 / (int)sizeof(T), PER = KB / 16, OUT = B16 ? 1 : 2;
  constexpr int PIECES = B16 ? 3 : 1;   // operands that an f32 number is in a product
  // The weights between the steps of a chunk: the waves share the tiles out and exchange them through LDS.  A wave alone keeps them in
  // its registers, where they lie as the next product's operand already.
  constexpr bool SHARE = NW > 1 && !STATE;
  // ONE: Q takes V's place in LDS once V lies in registers, and more workgroups share a CU.
  constexpr bool ALIAS = MODE == DA_ONE;
  typedef typename std::conditional<B16, bf16x8_t, f32x4_t>::type F;
  typedef DaTile<T, AP> TA;
  typedef DaTile<T, BP> TB;
  typedef DaTile<T, L> TP;
  __shared__ __attribute__((aligned(16))) T Qs[STATE || ALIAS ? 8 : L * TA::LD], Ks[L * TA::LD], Ps[SHARE ? PIECES * L * TP::LD : 8];
  __shared__ __attribute__((aligned(16))) T Vs[L * (ALIAS && TA::LD > TB::LD ? TA::LD : TB::LD)];
  T *const Q = ALIAS ? Vs : Qs;
  __shared__ __attribute__((aligned(16))) float pw[L + 4];
  __shared__ int bad[NW];
  // the passes of one (row, head) meet in one XCD's L2: workgroups go round the 8 XCDs.  32-bit divisions: the launch has checked
  const uint32_t parts = STATE ? X.parts - 1 : X.parts;
  const uint32_t block = blockIdx.x, unit = block / (8u * passes) * 8u + block % 8u, pass = block / 8u % (uint32_t)passes;
  if (unit >= (uint32_t)A.m * (uint32_t)A.heads * parts) return;
  const da_pass &P = A.pass[pass];
  const uint32_t mh32 = unit / parts;
  const int part = (int)(unit - mh32 * parts), row = (int)(mh32 / (uint32_t)A.heads), h = (int)(mh32 - (uint32_t)row * A.heads);
  const long long mh = mh32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, ln = lane & 15;
  const int t_first = part * X.len, t_end = min(A.t_len, t_first + X.len);
  DaLoad<T, AP, L, NTHR, VEC, false> rq, rk;
  DaLoad<T, BP, L, NTHR, VEC, true> rv;
  if constexpr (!STATE) rq.start((const T *)P.q + t_first * P.qs[0] + row * P.qs[1] + h * P.qs[2], P.qs[0], P.a);
  rk.start((const T *)P.k + t_first * P.ks[0] + row * P.ks[1] + h * P.ks[2], P.ks[0], P.a);
  rv.start((const T *)P.v + t_first * P.vs[0] + row * P.vs[1] + h * P.vs[2], P.vs[0], P.b);
  int flag = 0;
  auto fetch = [&](int t) {
    const int n = min(L, t_end - t);
    rk.load(n);
    rv.load(n);
    if constexpr (!STATE) rq.load(n);
    if (P.reset) flag = P.reset[max(t + min(lane, n - 1), P.late) * P.reset_ts + row];
  };
  if (t_first < t_end) fetch(t_first);
  f32x4_t s[NS][2];
#pragma unroll
  for (int i = 0; i < NS; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) s[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const long long so = mh * ((long long)P.a * P.b);
  const int dv0 = 32 * wave;
  const bool whole = P.a == AP && P.b == BP;
  float *xs = X.state + pass * X.pass_stride + (mh * (X.parts - 1)) * (long long)(AP * BP) + wave * (AP * 32) + lane * 4;
  if (part == 0) {
    if (P.s_in) whole ? da_state_in<T, NS, true>(s, P.s_in + so, P, dv0) : da_state_in<T, NS, false>(s, P.s_in + so, P, dv0);
  } else if constexpr (!STATE) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) s[i][c] = *(const f32x4_t *)(xs + (long long)(part - 1) * (AP * BP) + (i * 2 + c) * 256);
  }
  const double decay = (double)A.decay[h];
  for (int i = threadIdx.x; i <= L; i += NTHR) pw[i] = (float)pqn_powi(decay, i);   // every power rounded once
  if (P.a < AP || P.b < BP) {
    for (int i = threadIdx.x; i < L * TA::LD; i += NTHR) {
      if constexpr (!STATE && !ALIAS) Qs[i] = (T)0.f;
      Ks[i] = (T)0.f;
    }
    for (int i = threadIdx.x; i < L * TB::LD; i += NTHR) Vs[i] = (T)0.f;
  }
  T *op = STATE ? nullptr : (T *)P.o + t_first * P.os[0] + row * P.os[1] + h * P.os[2] + ln * P.os[0] + dv0 + 8 * g;
  typedef pqn_pack<T, EV> Out;
  Out held[NT][OUT];                   // a chunk's outputs, step 16 tt + ln, 8 columns from 8 g
  int n_held = 0;
  auto write_out = [&]() {
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
      if (16 * tt + ln >= n_held) continue;
#pragma unroll
      for (int c = 0; c < OUT; ++c) {
        T *dst = op + 16 * tt * P.os[0] + 4 * c;
        const int col = dv0 + 8 * g + 4 * c;
        if constexpr (VEC) {
          if (col < P.b) *(pqn_pack<T, EV> *)dst = held[tt][c];
        } else
#pragma unroll
          for (int e = 0; e < EV; ++e)
            if (col + e < P.b) dst[e] = held[tt][c].v[e];
      }
    }
    op += n_held * P.os[0];
  };
  // What depends on the decay alone for a whole chunk without an episode's end is made once: the weights between steps, of the state
  // on the outputs and of the steps on the state behind them.  `usual` says that they are those.
  float wt[NT][NT][4], wu[NJ][EV];
  bool usual = false, any_cut = false;
  auto weigh_steps = [&](int tt, int jt, unsigned long long cuts) {      // of steps 16 jt + 4 g + e on step 16 tt + ln
    const int t = 16 * tt + ln;
    const unsigned long long upto = cuts & ((2ull << t) - 1ull);
    const int from = upto ? 63 - __clzll(upto) : 0;                      // first step of t's episode in this chunk
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = 16 * jt + 4 * g + e;
      wt[tt][jt][e] = j <= t && j >= from ? pw[max(t - j, 0)] * (P.s_scale * P.o_scale) : 0.f;
    }
  };
  auto weigh_state = [&](int j, int n, unsigned long long cuts) {
    const int last_cut = cuts ? 63 - __clzll(cuts) : 0;
#pragma unroll
    for (int e = 0; e < EV; ++e) {
      const int at = j * KB + 4 * g + (e & 3) + 16 * (e >> 2);
      wu[j][e] = at < n && at >= last_cut ? pw[max(n - 1 - at, 0)] * P.s_scale : 0.f;
    }
  };
  __syncthreads();                                     // pw
  for (int t0 = t_first; t0 < t_end;) {
    int n = min(L, t_end - t0);
    const int n_loaded = n;
    if (MODE == DA_ONE && t0 > 0) fetch(t0);           // only where a chunk is taken step by step
    rk.store(Ks, n);
    rv.store(Vs, n);
    if constexpr (!STATE && !ALIAS) rq.store(Qs, n);
    const bool nf = __any(rk.not_finite() || rv.not_finite());
    if (lane == 0) bad[wave] = nf;
    const unsigned long long cuts_all = __ballot(flag != 0 && lane < n && (t0 + lane > 0 || !P.late));
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
    const unsigned long long cuts = cuts_all & ((1ull << n) - 1ull);
    // Outputs leave one chunk late, in front of the next requests: memory operations end in order, so the wait for a chunk's inputs
    // would otherwise be one for the stores behind them as well.
    if constexpr (MODE == DA_MAIN) write_out();
    if (t0 + n < t_end) {
      rk.advance(n);
      rv.advance(n);
      if constexpr (!STATE) rq.advance(n);
      if constexpr (MODE != DA_ONE) fetch(t0 + n);
    }
    const int first = (t0 == 0 && P.late) ? 0 : 1;     // borders up to and including step 0 of this chunk
    const bool plain = n == L && !cuts && first;
    if (MODE != DA_ONE && !(plain && usual)) {         // ONE makes them where they are needed
      if constexpr (!STATE)
#pragma unroll
        for (int tt = 0; tt < NT; ++tt)
#pragma unroll
          for (int jt = 0; jt <= tt; ++jt)
            if (!SHARE || (tt * (tt + 1) / 2 + jt) % NW == wave) weigh_steps(tt, jt, cuts);
#pragma unroll
      for (int j = 0; j < NJ; ++j) weigh_state(j, n, cuts);
    }
    usual = plain;
    auto weights = [&](int tt, int jt, const F (&qf)[NF]) {
      f32x4_t p = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < NF; ++f) da_mfma(TA::template rows<F>(Ks, 16 * jt, f * KB), qf[f], p);
      da_drain<F>(p);
      if constexpr (MODE == DA_ONE) weigh_steps(tt, jt, cuts);
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = wt[tt][jt][e] == 0.f ? 0.f : p[e] * wt[tt][jt][e];   // a later step's product may overflow
      return p;
    };
    F vf[NJ][2];
#pragma unroll
    for (int j = 0; j < NJ; ++j) TB::template pairs<F>(Vs, j * KB, dv0, vf[j]);
    if constexpr (ALIAS) {
      __syncthreads();                                 // V has been read
      if (P.a < AP) {
        for (int i = threadIdx.x; i < L * TA::LD; i += NTHR) Q[i] = (T)0.f;
        __syncthreads();
      }
      rq.store(Q, n_loaded);
      __syncthreads();
    }
    if constexpr (SHARE) {
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        if (16 * tt >= n) continue;
#pragma unroll
        for (int jt = 0; jt < (tt / PER + 1) * PER; ++jt) {      // whole operands: with zeros above the diagonal
          if ((tt * (tt + 1) / 2 + min(jt, tt)) % NW != wave) continue;
          f32x4_t p = {0.f, 0.f, 0.f, 0.f};
          if (jt <= tt) {
            F qf[NF];
#pragma unroll
            for (int f = 0; f < NF; ++f) qf[f] = TA::template rows<F>(Q, 16 * tt, f * KB);
            p = weights(tt, jt, qf);
          }
          if constexpr (B16) {                                   // in the order of DaTile::cols
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
              uint32_t *dst = (uint32_t *)(Ps + k * L * TP::LD + TP::at(16 * tt + ln, 32 * (jt >> 1) + 8 * g + 4 * (jt & 1)));
              float v[4] = {p[0], p[1], p[2], p[3]};
              dst[0] = da_cut3(v[0], v[1]);
              dst[1] = da_cut3(v[2], v[3]);
              p = f32x4_t{v[0], v[1], v[2], v[3]};
            }
          } else *(f32x4_t *)(Ps + TP::at(16 * tt + ln, 16 * jt + 4 * g)) = p;
        }
      }
      __syncthreads();
    }
    if constexpr (!STATE) {
      f32x4_t os[B16 ? NT : 1][2];                               // bf16: the state is cut in pieces once for all steps
      if constexpr (B16) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) os[tt][0] = os[tt][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int f = 0; f < NF; ++f) {
          F sp[2][PIECES];
#pragma unroll
          for (int c = 0; c < 2; ++c) da_pieces(s[2 * f][c], s[2 * f + 1][c], sp[c]);
#pragma unroll
          for (int tt = 0; tt < NT; ++tt)
            if (16 * tt < n) da_mfma6(sp, TA::template rows<F>(Q, 16 * tt, f * KB), os[tt]);
        }
        da_drain<F>(os);
      }
#pragma unroll
      for (int tt = 0; tt < NT; ++tt) {
        if (16 * tt >= n) continue;
        f32x4_t (&o)[2] = os[B16 ? tt : 0];
        F qf[NF];
        if constexpr (!B16 || !SHARE)
#pragma unroll
          for (int f = 0; f < NF; ++f) qf[f] = TA::template rows<F>(Q, 16 * tt, f * KB);
        if constexpr (!B16) {
          o[0] = o[1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int f = 0; f < NF; ++f) da_mfma2(s[f][0], s[f][1], qf[f], qf[f], o);
        }
        const float wc = pw[16 * tt + ln + first] * P.o_scale;
        if (cuts) {                                              // a choice, not a product: the state may be NaN
          const bool carried = (cuts & ((2ull << (16 * tt + ln)) - 1ull)) == 0;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][e] = carried ? o[c][e] : 0.f;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][e] *= wc;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (j * KB >= 16 * (tt + 1)) continue;
          F pf[PIECES];
          if constexpr (SHARE)
#pragma unroll
            for (int k = 0; k < PIECES; ++k) pf[k] = TP::template rows<F>(Ps + k * L * TP::LD, 16 * tt, j * KB);
          else {
            f32x4_t p[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              if (PER * j + i > tt) p[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
              else p[i] = weights(tt, PER * j + i, qf);
            }
            if constexpr (B16) da_pieces(p[0], p[1], pf);
            else pf[0] = p[0];
          }
          if constexpr (B16) da_mfma6(vf[j], pf, o);
          else da_mfma2(vf[j][0], vf[j][1], pf[0], pf[0], o);
        }
        da_drain<F>(o);
        if constexpr (B16)
          held[tt][0] = __builtin_bit_cast(Out, (u32x4_t{da_pair(o[0][0], o[1][0]), da_pair(o[0][1], o[1][1]), da_pair(o[0][2], o[1][2]),
                                                         da_pair(o[0][3], o[1][3])}));
        else
#pragma unroll
          for (int c = 0; c < OUT; ++c)
            held[tt][c] = __builtin_bit_cast(Out, (f32x4_t{o[0][2 * c], o[1][2 * c], o[0][2 * c + 1], o[1][2 * c + 1]}));
      }
      n_held = n;
      if constexpr (MODE == DA_ONE) write_out();
    }
    // the state behind the chunk
    const float fade = pw[n - 1 + first];
    any_cut = any_cut || cuts != 0;
    if (cuts) {
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) s[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    } else {
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][c][e] *= fade;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (j * KB >= n) continue;
      if constexpr (MODE == DA_ONE) weigh_state(j, n, cuts);
      F x[2][PIECES];                                  // w v is its pieces' sum exactly
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (B16) {
          const u32x4_t v = __builtin_bit_cast(u32x4_t, vf[j][c]);
          u32x4_t u[3];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float lo = da_low(v[e]) * wu[j][2 * e], hi = da_high(v[e]) * wu[j][2 * e + 1];
#pragma unroll
            for (int k = 0; k < 3; ++k) {
              u[k][e] = da_pair(lo, hi);
              lo -= da_low(u[k][e]);
              hi -= da_high(u[k][e]);
            }
          }
#pragma unroll
          for (int k = 0; k < 3; ++k) x[c][k] = __builtin_bit_cast(F, u[k]);
        } else
#pragma unroll
          for (int e = 0; e < 4; ++e) x[c][0][e] = vf[j][c][e] * wu[j][e];
      }
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const F kf = TA::template cols<F>(Ks, j * KB, i);
        if constexpr (B16) da_mfma6(kf, x, s[i]);
        else da_mfma2(kf, kf, x[0][0], x[1][0], s[i]);
      }
    }
    da_drain<F>(s);
    t0 += n;
    __syncthreads();                                   // the chunk has been read
  }
  if constexpr (MODE == DA_MAIN) write_out();
  if constexpr (STATE) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) *(f32x4_t *)(xs + (long long)part * (AP * BP) + (i * 2 + c) * 256) = s[i][c];
    if (threadIdx.x == 0) X.cut[pass * X.cut_stride + mh * (X.parts - 1) + part] = any_cut;
  } else if (P.s_out && part == X.parts - 1) {
    if (P.late) {
      const bool cut = P.reset && P.reset[A.t_len * P.reset_ts + row];
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][c][e] = cut ? 0.f : s[i][c][e] * pw[1];
    }
    whole ? da_state_out<T, NS, true>(s, P.s_out + so, P, dv0) : da_state_out<T, NS, false>(s, P.s_out + so, P, dv0);
  }
}

// widths as the kernel is built for them: rows of the state padded to AP, 32 columns a wave.  96 beside the powers of two: 200 steps x 800
// rows of 96 x 96, forward / gradient, f32 142 / 334 us, padded to 128 175 / 418, bf16 75 / 173 and 89 / 209.  Tensors whose rows are not
// whole 16-byte accesses go element by element, in fewer forms.
inline int da_ap(int a, int vec) { return a <= 32 && vec ? 32 : a <= 64 ? 64 : a <= 96 && vec ? 96 : 128; }
inline int da_nw(int a, int b, int vec) {
  const int nw = b <= 32 ? 1 : b <= 64 ? 2 : b <= 96 && vec ? 3 : 4;
  return !vec ? a > 64 || nw == 4 ? 4 : 2 : a > 64 && nw < 2 ? 2 : nw;    // a wave alone would hold 128 registers of loads in flight
}
// the kernel for passes of unequal widths is the one that holds the widest
inline int da_widest(const da_args &A, int passes, int da_pass::*width) {
  int w = 0;
  for (int p = 0; p < passes; ++p) w = A.pass[p].*width > w ? A.pass[p].*width : w;
  return w;
}
int da_launch_chunk_f32(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st);
int da_launch_chunk_bf16(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st);

template <typename T, int L>
static int da_launch_chunk(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st) {
  const int a = da_widest(A, passes, &da_pass::a), ap = da_ap(a, X.vec), nw = da_nw(a, da_widest(A, passes, &da_pass::b), X.vec);
  const long long units = (long long)A.m * A.heads * (state ? X.parts - 1 : X.parts), grid = (units + 7) / 8 * 8 * passes;
  PQN_REQUIRE(pqn_one_launch(grid, 64 * nw), "pqn_decay_attn: %d x %d rows and heads are more than one launch covers", A.m, A.heads);
#define DA_GO(AP, NW, VEC)                                                                                                   \
  if (ap == AP && nw == NW && (X.vec != 0) == VEC) {                                                                         \
    if (state) da_chunk_kernel<T, AP, NW, L, VEC, DA_STATE><<<(unsigned)grid, 64 * NW, 0, st>>>(A, X, passes);               \
    else if (VEC && A.t_len <= L) da_chunk_kernel<T, AP, NW, L, true, DA_ONE><<<(unsigned)grid, 64 * NW, 0, st>>>(A, X, passes); \
    else da_chunk_kernel<T, AP, NW, L, VEC, DA_MAIN><<<(unsigned)grid, 64 * NW, 0, st>>>(A, X, passes);                      \
    return pqn_check_launch("pqn_decay_attn");                                                                               \
  }
  DA_GO(32, 1, true)
  DA_GO(32, 2, true)
  DA_GO(32, 3, true)
  DA_GO(32, 4, true)
  DA_GO(64, 1, true)
  DA_GO(64, 2, true)
  DA_GO(64, 3, true)
  DA_GO(64, 4, true)
  DA_GO(96, 2, true)
  DA_GO(96, 3, true)
  DA_GO(96, 4, true)
  DA_GO(128, 2, true)
  DA_GO(128, 3, true)
  DA_GO(128, 4, true)
  DA_GO(64, 2, false)
  DA_GO(64, 4, false)
  DA_GO(128, 4, false)
#undef DA_GO
  pqn_set_error("pqn_decay_attn: no kernel for widths of up to %d", a);
  return PQN_E_UNSUPPORTED;
}
