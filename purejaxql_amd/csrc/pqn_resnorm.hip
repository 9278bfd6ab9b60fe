// pqn_resnorm.hip -- the norms around a residual block with the block's gate and residual scale, forward and gradient, one pass over
// the rows each (pqn_residual_norm, pqn_residual_norm_grad in include/pqn_hotpath.h).
//
//   z = Norm(f)      n = z * post_scale + post_bias      y = x + res_scale * act(g) * n      u = Norm(y)      h = u * pre_scale + pre_bias
//
// A row lives in the registers of one wave (up to 512 columns) or of one workgroup from its load to its store, so the forward reads
// x, f, g once and writes y, h once, and the gradient reads x, f, g, dy, dh once and writes dx, df, dg once; both norms' statistics are
// taken twice over the registers (mean, then the centred sum of squares), in f32.  The gradient recomputes y in f32 from x, f, g
// instead of reading a stored y: the same bytes, and no rounding between the two halves.
//
// Bound: HBM.  Waves walk over rows with the parameters in registers and the next row's loads in flight; 8 columns per thread keep
// the gradient's row tensors, parameters and five column sums within the registers of two waves per SIMD (160 to 244 at 512 to 4096 columns;
// over 4096, 1024 threads with 128 registers, of which silu in 16 bits spills up to 20 bytes a lane and f32 up to 100).  Measured, forward /
// gradient (the kernels' least under a trace): 131072 x 1024 bf16 with a gate and all parameters 270 / 439 + 9 us (column sums), 5.0 / 4.9
// TB/s; 4099 x 4095 f32, element by element, 63 / 115 + 13 us, 5.3 / 4.7 TB/s; 128 x 128 f32 3.2 us, latency (12.8 with the call).
#include <type_traits>

#include "pqn_vec.h"

static constexpr int RN_MAX_D = 8192;

struct rn_args {
  long long n;
  int d;
  int rms, gate_act, has_post, has_pre;
  float eps;
  const void *x, *f, *g;
  long long xs, fs, gs;                   // row strides in elements
  const float *res_scale, *post_scale, *post_bias, *pre_scale, *pre_bias;
  void *y, *h;
  const void *dy, *dh;
  long long dys, dhs;
  void *dx, *df, *dg;
  float *partials;                        // [gridDim.x][RN_PARAMS][d]
  struct RnStat *stats;                   // rows of more than RN_WIDE columns: [n]
};
struct RnStat {                           // of a row: f's and y's mean and 1 / sqrt(var + eps); mean(dh' u), mean(dh') of y's norm
  float mean_f, inv_f, mean_y, inv_y, a, b;
};
static constexpr int RN_WIDE = 4096;
enum { RN_RES = 0, RN_POST_SCALE, RN_POST_BIAS, RN_PRE_SCALE, RN_PRE_BIAS, RN_PARAMS };

// K sums at once over the NT threads that hold a row, the same in every thread.  `turn` alternates between two places in LDS, so
// that one barrier per sum is enough: a place is written again behind the barrier of the sum in between.
template <int NT, int K>
PQN_D void rn_row_sum(float (&v)[K], float *lds, int &turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = pqn_wave_sum(v[k]);
  if constexpr (NT > 64) {
    constexpr int NW = NT / 64;
    float *at = lds + turn * 2 * NW;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) at[k * NW + (threadIdx.x >> 6)] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = at[k * NW];
#pragma unroll
      for (int w = 1; w < NW; ++w) s += at[k * NW + w];
      v[k] = s;
    }
  }
}

// Thread `lane` of the NT holds NV accesses of VW columns, the i-th from (i NT + lane) VW on.  LOOSE: the rows start anywhere and their
// width is no multiple of VW; the access that would end behind the row ends at its last column instead, and what it shares with the one
// before is that one's.  For rows of more than RN_WIDE columns, whose kernels have no registers for an address and a condition per
// element: 2799 x 5394 bf16, forward / gradient 65 / 166 us, element by element 101 / 362; 18326 x 1163 60 / 157 and 56 / 145.
template <typename T, int NT, int VW, int NV, bool LOOSE>
struct RnRow {
  static constexpr int E = VW * NV;
  template <typename U>
  using PackOf = typename std::conditional<LOOSE, pqn_loose<U, VW>, pqn_pack<U, VW>>::type;
  typedef PackOf<T> Pack;
  int d, lane;
  PQN_D int first(int i) const { return (i * NT + lane) * VW; }
  PQN_D int at(int i) const {                        // where the access is made
    const int c = first(i);
    return LOOSE ? min(c, d - VW) : c < d ? c : 0;
  }
  PQN_D bool own(int i, int j) const { return LOOSE ? at(i) + j >= first(i) : first(i) < d; }
  PQN_D void fetch(Pack (&r)[NV], const void *base, long long off) const {
    const T *p = (const T *)base + off;
#pragma unroll
    for (int i = 0; i < NV; ++i) r[i] = *(const Pack *)(p + at(i));
  }
  PQN_D void open(float (&x)[E], const Pack (&r)[NV]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VW; ++j) x[i * VW + j] = own(i, j) ? pqn_to_f32(r[i].v[j]) : 0.f;
  }
  template <typename U>
  PQN_D void store(U *p, const float (&r)[E]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = first(i);
      if (LOOSE ? c + VW <= d : c < d) {
        PackOf<U> x;
#pragma unroll
        for (int j = 0; j < VW; ++j) x.v[j] = (U)r[i * VW + j];
        *(PackOf<U> *)(p + c) = x;
      } else if (LOOSE && c < d) {
#pragma unroll
        for (int j = 0; j < VW; ++j)
          if (own(i, j)) p[at(i) + j] = (U)r[i * VW + j];
      }
    }
  }
  PQN_D void store(void *base, long long off, const float (&r)[E]) const { store((T *)base + off, r); }
  PQN_D void param(float (&r)[E], const float *p, float absent) const {
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = absent;
    if (!p) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const PackOf<float> x = *(const PackOf<float> *)(p + at(i));
#pragma unroll
      for (int j = 0; j < VW; ++j) r[i * VW + j] = own(i, j) ? x.v[j] : absent;
    }
  }
  // r -> (r - mean) * inv in place; returns inv = 1 / sqrt(var + eps).  rms: mean = 0
  PQN_D float normalise(float (&r)[E], int rms, float eps, float *lds, int &turn, float *mean_out = nullptr) const {
    const float per = 1.0f / (float)d;
    if (!rms) {
      float s[1] = {0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) s[0] += r[e];
      rn_row_sum<NT>(s, lds, turn);
      const float mean = s[0] * per;
      if (mean_out) *mean_out = mean;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VW; ++j) r[i * VW + j] = own(i, j) ? r[i * VW + j] - mean : 0.f;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) q[0] = fmaf(r[e], r[e], q[0]);
    rn_row_sum<NT>(q, lds, turn);
    const float inv = 1.0f / sqrtf(fmaf(q[0], per, eps));
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] *= inv;
    return inv;
  }
  // gradient of the normalisation: dz -> d(input), z = the normalised row; ab: mean(dz z), mean(dz)
  PQN_D void normalise_back(float (&dz)[E], const float (&z)[E], float inv, int rms, float *lds, int &turn, float *ab = nullptr) const {
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s[0] = fmaf(dz[e], z[e], s[0]);
      s[1] += dz[e];
    }
    rn_row_sum<NT>(s, lds, turn);
    const float per = 1.0f / (float)d, a = s[0] * per, b = rms ? 0.f : s[1] * per;
    if (ab) {
      ab[0] = a;
      ab[1] = b;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VW; ++j) dz[i * VW + j] = own(i, j) ? (fmaf(-z[i * VW + j], a, dz[i * VW + j]) - b) * inv : 0.f;
  }
};

// act(g) and its slope; the sigmoid from v_exp_f32 and v_rcp_f32, each within an ulp
PQN_D void rn_act(int kind, float g, float &act, float &slope) {
  act = 1.f;
  slope = 0.f;
  if (kind == PQN_GATE_NONE) return;
  const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g));
  if (kind == PQN_GATE_SIGMOID) {
    act = s;
    slope = s * (1.0f - s);
  } else {
    act = g * s;
    slope = s * fmaf(g, 1.0f - s, 1.0f);
  }
}

// A wave per row (NT = 64, four to a workgroup) or a workgroup per row, walking over the rows.
template <typename T, int NT, int VW, int NV, bool LOOSE, int ACT>
__global__ __launch_bounds__(NT > 64 ? NT : 256) void rn_fwd_kernel(rn_args A) {
  using Row = RnRow<T, NT, VW, NV, LOOSE>;
  constexpr int E = Row::E, RPB = NT > 64 ? 1 : 4;
  constexpr bool KEEP = NT < 1024;        // the parameters stay in registers, and the next row is in flight
  __shared__ float lds[NT > 64 ? 4 * NT / 64 : 1];
  const int lane = NT > 64 ? threadIdx.x : threadIdx.x & 63;
  const int d = A.d;
  const Row rw = {d, lane};
  int turn = 0;
  long long row = (long long)blockIdx.x * RPB + (NT > 64 ? 0 : threadIdx.x >> 6);
  const long long step = (long long)gridDim.x * RPB;
  if (row >= A.n) return;                 // whole waves / workgroups
  typename Row::Pack fx[NV], ff[NV], fg[NV];
  auto fetch = [&](long long r) {
    rw.fetch(ff, A.f, r * A.fs);
    if constexpr (ACT != PQN_GATE_NONE) rw.fetch(fg, A.g, r * A.gs);
    rw.fetch(fx, A.x, r * A.xs);
  };
  float ps[E], pb[E], rs[E], qs[E], qb[E];
  auto params_in = [&]() {
    rw.param(ps, A.post_scale, 1.f);
    rw.param(pb, A.post_bias, 0.f);
    rw.param(rs, A.res_scale, 1.f);
  };
  auto params_out = [&]() {
    rw.param(qs, A.pre_scale, 1.f);
    rw.param(qb, A.pre_bias, 0.f);
  };
  if constexpr (KEEP) {
    fetch(row);
    params_in();
    params_out();
  }
  for (; row < A.n; row += step) {
    float z[E], y[E], g[E];
    if constexpr (!KEEP) fetch(row);
    rw.open(z, ff);
    rw.open(y, fx);
    if constexpr (ACT != PQN_GATE_NONE) rw.open(g, fg);
    if (KEEP && row + step < A.n) fetch(row + step);
    if (A.has_post) rw.normalise(z, A.rms, A.eps, lds, turn);
    if constexpr (!KEEP) params_in();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float act, slope;
      rn_act(ACT, g[e], act, slope);
      y[e] = fmaf(rs[e], act * fmaf(z[e], ps[e], pb[e]), y[e]);
    }
    rw.store(A.y, row * d, y);
    if (A.has_pre) {
      rw.normalise(y, A.rms, A.eps, lds, turn);
      if constexpr (!KEEP) params_out();
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] = fmaf(y[e], qs[e], qb[e]);
      rw.store(A.h, row * d, y);
    }
  }
}

// The parameter gradients are summed over a thread's rows in registers and leave the workgroup as one partial row per parameter,
// summed in a fixed order by rn_param_kernel (the same result in every run).  NT = 1024 has no registers for the sums: it leaves the
// row's statistics instead, and rn_sums_kernel reads the rows a second time.
template <typename T, int NT, int VW, int NV, bool LOOSE, int ACT>
__global__ __launch_bounds__(NT > 64 ? NT : 256) void rn_bwd_kernel(rn_args A) {
  using Row = RnRow<T, NT, VW, NV, LOOSE>;
  constexpr int E = Row::E, RPB = NT > 64 ? 1 : 4;
  constexpr bool KEEP = NT < 1024, SUMS = KEEP;
  __shared__ float lds[NT > 64 ? 4 * NT / 64 : 1];
  __shared__ float fold[NT > 64 ? 1 : 3 * 64 * E];
  const int lane = NT > 64 ? threadIdx.x : threadIdx.x & 63, wave = NT > 64 ? 0 : threadIdx.x >> 6;
  const int d = A.d;
  const Row rw = {d, lane};
  int turn = 0;
  float sum[SUMS ? RN_PARAMS : 1][E];
  if constexpr (SUMS)
#pragma unroll
    for (int k = 0; k < RN_PARAMS; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) sum[k][e] = 0.f;
  long long row = (long long)blockIdx.x * RPB + wave;
  const long long step = (long long)gridDim.x * RPB;
  typename Row::Pack fx[NV], ff[NV], fg[NV], fy[NV], fh[NV];
  auto fetch = [&](long long r) {
    rw.fetch(ff, A.f, r * A.fs);
    if constexpr (ACT != PQN_GATE_NONE) rw.fetch(fg, A.g, r * A.gs);
    rw.fetch(fx, A.x, r * A.xs);
    if (A.dh) rw.fetch(fh, A.dh, r * A.dhs);
    if (A.dy) rw.fetch(fy, A.dy, r * A.dys);
  };
  if (KEEP && row < A.n) fetch(row);
  float ps[E], pb[E], rs[E], qs[E];
  auto params = [&]() {
    rw.param(ps, A.post_scale, 1.f);
    rw.param(pb, A.post_bias, 0.f);
    rw.param(rs, A.res_scale, 1.f);
  };
  if constexpr (KEEP) {
    params();
    rw.param(qs, A.pre_scale, 1.f);
  }
  for (; row < A.n; row += step) {
    float z[E], y[E], e_[E], g[E], dh[E];
    if constexpr (!KEEP) fetch(row);
    rw.open(z, ff);
    rw.open(y, fx);
    if constexpr (ACT != PQN_GATE_NONE) rw.open(g, fg);
    if (A.dh) rw.open(dh, fh);
    if (A.dy) rw.open(e_, fy);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) e_[e] = 0.f;
    if (KEEP && row + step < A.n) fetch(row + step);
    if constexpr (!KEEP) params();
    float inv_f = 1.f, act[E], slope[E];
    RnStat st = {0.f, 1.f, 0.f, 1.f, 0.f, 0.f};
    if (A.has_post) inv_f = rw.normalise(z, A.rms, A.eps, lds, turn, &st.mean_f);
    st.inv_f = inv_f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      rn_act(ACT, g[e], act[e], slope[e]);
      y[e] = fmaf(rs[e], act[e] * fmaf(z[e], ps[e], pb[e]), y[e]);
    }
    if (A.dh) {
      const float inv_y = rw.normalise(y, A.rms, A.eps, lds, turn, &st.mean_y);
      st.inv_y = inv_y;
      if constexpr (!KEEP) rw.param(qs, A.pre_scale, 1.f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (SUMS) {
          sum[RN_PRE_SCALE][e] = fmaf(dh[e], y[e], sum[RN_PRE_SCALE][e]);
          sum[RN_PRE_BIAS][e] += dh[e];
        }
        dh[e] *= qs[e];
      }
      rw.normalise_back(dh, y, inv_y, A.rms, lds, turn, &st.a);
#pragma unroll
      for (int e = 0; e < E; ++e) e_[e] += dh[e];
    }
    rw.store(A.dx, row * d, e_);
    if constexpr (!KEEP) params();          // read and made again rather than held
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (!KEEP) rn_act(ACT, g[e], act[e], slope[e]);
      const float n = fmaf(z[e], ps[e], pb[e]), da = e_[e] * rs[e], dn = da * act[e];
      if constexpr (ACT != PQN_GATE_NONE) g[e] = da * n * slope[e];
      if constexpr (SUMS) {
        sum[RN_RES][e] = fmaf(e_[e], act[e] * n, sum[RN_RES][e]);
        sum[RN_POST_SCALE][e] = fmaf(dn, z[e], sum[RN_POST_SCALE][e]);
        sum[RN_POST_BIAS][e] += dn;
      }
      e_[e] = dn * ps[e];
    }
    if constexpr (ACT != PQN_GATE_NONE) rw.store(A.dg, row * d, g);
    if (A.has_post) rw.normalise_back(e_, z, inv_f, A.rms, lds, turn);
    rw.store(A.df, row * d, e_);
    if (!SUMS && threadIdx.x == 0) A.stats[row] = st;
  }
  if constexpr (!SUMS) return;
  float *out = A.partials + (size_t)blockIdx.x * RN_PARAMS * d;
#pragma unroll
  for (int k = 0; k < (SUMS ? RN_PARAMS : 0); ++k) {
    if constexpr (NT == 64) {              // waves 1 .. 3 hand their sums to wave 0
      __syncthreads();
      if (wave > 0)
#pragma unroll
        for (int e = 0; e < E; ++e) fold[((wave - 1) * E + e) * 64 + lane] = sum[k][e];
      __syncthreads();
      if (wave == 0)
#pragma unroll
        for (int e = 0; e < E; ++e)
          sum[k][e] = ((sum[k][e] + fold[e * 64 + lane]) + fold[(E + e) * 64 + lane]) + fold[(2 * E + e) * 64 + lane];
    }
    if (wave == 0) rw.store(out + (size_t)k * d, sum[k]);
  }
}

// The parameter gradients of wide rows: a thread's VW columns over the rows of its slice, from the statistics that rn_bwd_kernel left.
template <typename T, int VW, bool LOOSE, int ACT>
__global__ __launch_bounds__(256) void rn_sums_kernel(rn_args A) {
  const int d = A.d, mine = (blockIdx.x * 256 + threadIdx.x) * VW;
  if (mine >= d) return;
  const int c = LOOSE ? min(mine, d - VW) : mine;            // as in RnRow
  typedef typename std::conditional<LOOSE, pqn_loose<T, VW>, pqn_pack<T, VW>>::type Pack;
  auto load = [&](float (&r)[VW], const void *base, long long off) {
    const Pack x = *(const Pack *)((const T *)base + off + c);
#pragma unroll
    for (int e = 0; e < VW; ++e) r[e] = pqn_to_f32(x.v[e]);
  };
  float ps[VW], pb[VW], rs[VW], qs[VW], sum[RN_PARAMS][VW];
  auto param = [&](float (&r)[VW], const float *p, float absent) {
#pragma unroll
    for (int e = 0; e < VW; ++e) r[e] = p ? p[c + e] : absent;
  };
  param(ps, A.post_scale, 1.f);
  param(pb, A.post_bias, 0.f);
  param(rs, A.res_scale, 1.f);
  param(qs, A.pre_scale, 1.f);
#pragma unroll
  for (int k = 0; k < RN_PARAMS; ++k)
#pragma unroll
    for (int e = 0; e < VW; ++e) sum[k][e] = 0.f;
  for (long long row = blockIdx.y; row < A.n; row += gridDim.y) {
    float x[VW], f[VW], g[VW], dy[VW], dh[VW];
    load(f, A.f, row * A.fs);
    load(x, A.x, row * A.xs);
    if constexpr (ACT != PQN_GATE_NONE) load(g, A.g, row * A.gs);
    if (A.dh) load(dh, A.dh, row * A.dhs);
    if (A.dy) load(dy, A.dy, row * A.dys);
    const RnStat st = A.stats[row];
#pragma unroll
    for (int e = 0; e < VW; ++e) {
      float act, slope;
      rn_act(ACT, g[e], act, slope);
      const float z = (f[e] - st.mean_f) * st.inv_f, n = fmaf(z, ps[e], pb[e]);
      float grad = A.dy ? dy[e] : 0.f;
      if (A.dh) {
        const float u = (fmaf(rs[e], act * n, x[e]) - st.mean_y) * st.inv_y;
        sum[RN_PRE_SCALE][e] = fmaf(dh[e], u, sum[RN_PRE_SCALE][e]);
        sum[RN_PRE_BIAS][e] += dh[e];
        grad += (fmaf(-u, st.a, dh[e] * qs[e]) - st.b) * st.inv_y;
      }
      const float dn = grad * rs[e] * act;
      sum[RN_RES][e] = fmaf(grad, act * n, sum[RN_RES][e]);
      sum[RN_POST_SCALE][e] = fmaf(dn, z, sum[RN_POST_SCALE][e]);
      sum[RN_POST_BIAS][e] += dn;
    }
  }
  float *out = A.partials + (size_t)blockIdx.y * RN_PARAMS * d + c;
#pragma unroll
  for (int k = 0; k < RN_PARAMS; ++k)
#pragma unroll
    for (int e = 0; e < VW; ++e)
      if (c + e >= mine) out[(size_t)k * d + e] = sum[k][e];
}

// column sums of the partials: COLS columns x 1024 / COLS row groups per workgroup, fixed order
struct rn_param_out {
  float *p[RN_PARAMS];
};
template <int COLS>
__global__ __launch_bounds__(1024) void rn_param_kernel(const float *__restrict__ partials, int parts, int d, rn_param_out out) {
  constexpr int ROWS = 1024 / COLS;
  __shared__ float s[ROWS][COLS + 1];
  const int k = blockIdx.y, cc = threadIdx.x % COLS, c = blockIdx.x * COLS + cc, r = threadIdx.x / COLS;
  if (!out.p[k]) return;
  float a = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int i = r; i < parts; i += ROWS) a += partials[((size_t)i * RN_PARAMS + k) * d + c];
  }
  s[r][cc] = a;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  for (int col = threadIdx.x >> 6; col < COLS; col += 16) {       // a wave per column
    a = pqn_wave_sum(lane < ROWS ? s[lane % ROWS][col] : 0.f);
    if (lane == 0 && blockIdx.x * COLS + col < d) out.p[k][blockIdx.x * COLS + col] = a;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Threads per row: as few as hold it at 8 columns each -- a wave up to 512 columns (no barrier then), then 128 to 1024 threads, the
// last without the registers for parameters and a row in flight.  Vector accesses of up to 16 B where width, strides and pointers allow
// them, else one element per lane and access, or (over RN_WIDE columns) accesses that start anywhere (RnRow).
static int rn_threads(int d) { return d <= 512 ? 64 : d <= 1024 ? 128 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024; }
// Workgroups: enough to fill the chip (8 waves per SIMD asked for by the forward, 2 by the gradient with its sums in registers), each
// walking over its rows; the gradient leaves a partial row per workgroup and parameter, wide rows one per slice of rn_sums_kernel.
static int rn_blocks(long long n, int d, bool grad) {
  const int nt = rn_threads(d);
  const long long want = nt == 64 ? (n + 3) / 4 : n;
  const long long cap = grad && nt < 1024 ? (nt <= 128 ? 1024 : 512) : 65536 / (nt == 64 ? 256 : nt) * 8;
  return (int)(want < cap ? want : cap);
}
static int rn_parts(long long n, int d) { return d <= RN_WIDE ? rn_blocks(n, d, true) : (int)(n < 256 ? n : 256); }

template <typename T, bool BWD, int ACT>
static int rn_launch_act(const rn_args &A, bool vec, hipStream_t st) {
  constexpr int VW = 16 / (int)sizeof(T);
  const int nt = rn_threads(A.d);
  const unsigned grid = rn_blocks(A.n, A.d, BWD);
#define RN_GO(NT, W, NVV, LOOSE)                                                                                  \
  do {                                                                                                            \
    if constexpr (BWD) rn_bwd_kernel<T, NT, W, NVV, LOOSE, ACT><<<grid, NT > 64 ? NT : 256, 0, st>>>(A);          \
    else rn_fwd_kernel<T, NT, W, NVV, LOOSE, ACT><<<grid, NT > 64 ? NT : 256, 0, st>>>(A);                        \
    return pqn_check_launch(BWD ? "pqn_residual_norm_grad" : "pqn_residual_norm");                                \
  } while (0)
  if (vec) {
    if (A.d <= 128) RN_GO(64, 2, 1, false);
    if (A.d <= 256) RN_GO(64, 4, 1, false);
    if (nt == 64) RN_GO(64, VW, 8 / VW, false);
    if (nt == 128) RN_GO(128, VW, 8 / VW, false);
    if (nt == 256) RN_GO(256, VW, 8 / VW, false);
    if (nt == 512) RN_GO(512, VW, 8 / VW, false);
    RN_GO(1024, VW, 8 / VW, false);
  }
  if (A.d <= 128) RN_GO(64, 1, 2, false);
  if (nt == 64) RN_GO(64, 1, 8, false);
  if (nt == 128) RN_GO(128, 1, 8, false);
  if (nt == 256) RN_GO(256, 1, 8, false);
  if (nt == 512) RN_GO(512, 1, 8, false);
  RN_GO(1024, VW, 8 / VW, true);
#undef RN_GO
}
template <typename T>
static int rn_launch_sums(const rn_args &A, bool vec, hipStream_t st) {
  constexpr int VW = 16 / (int)sizeof(T);
  const dim3 grid((A.d + 256 * VW - 1) / (256 * VW), rn_parts(A.n, A.d));
#define RN_GO(ACT)                                                       \
  if (A.gate_act == ACT) {                                               \
    if (vec) rn_sums_kernel<T, VW, false, ACT><<<grid, 256, 0, st>>>(A); \
    else rn_sums_kernel<T, VW, true, ACT><<<grid, 256, 0, st>>>(A);      \
  }
  RN_GO(PQN_GATE_NONE)
  RN_GO(PQN_GATE_SIGMOID)
  RN_GO(PQN_GATE_SILU)
#undef RN_GO
  return pqn_check_launch("pqn_residual_norm_grad");
}
template <typename T, bool BWD>
static int rn_launch(const rn_args &A, bool vec, hipStream_t st) {
  if (A.gate_act == PQN_GATE_SILU) return rn_launch_act<T, BWD, PQN_GATE_SILU>(A, vec, st);
  if (A.gate_act == PQN_GATE_SIGMOID) return rn_launch_act<T, BWD, PQN_GATE_SIGMOID>(A, vec, st);
  return rn_launch_act<T, BWD, PQN_GATE_NONE>(A, vec, st);
}

// 16-byte accesses: whole rows of them, all starting on 16 bytes (parameters too)
static bool rn_vec_ok(const pqn_residual_norm_t *a, const void *const *ptrs, int np, const int64_t *strides, int ns) {
  const int es = pqn_dtype_size(a->dtype), vw = 16 / es;
  if (a->d % vw) return false;
  for (int i = 0; i < np; ++i)
    if ((uintptr_t)ptrs[i] & 15) return false;
  const void *params[] = {a->res_scale, a->post_scale, a->post_bias, a->pre_scale, a->pre_bias, a->workspace};
  for (const void *p : params)
    if ((uintptr_t)p & 15) return false;
  for (int i = 0; i < ns; ++i)
    if (strides[i] % vw) return false;
  return true;
}

static int rn_check(const pqn_residual_norm_t *a, const char *who) {
  PQN_REQUIRE(a, "%s: NULL argument block", who);
  PQN_REQUIRE(pqn_dtype_known(a->dtype), "%s: unknown dtype %d", who, a->dtype);
  PQN_REQUIRE(a->n >= 0 && a->d > 0, "%s: n must be >= 0 and d > 0 (n=%lld d=%d)", who, (long long)a->n, a->d);
  PQN_REQUIRE(a->d <= RN_MAX_D, "%s: rows of up to %d columns (d=%d)", who, RN_MAX_D, a->d);
  PQN_REQUIRE(a->n <= 0x7fffffffll, "%s: up to 2^31 - 1 rows (n=%lld)", who, (long long)a->n);
  PQN_REQUIRE(a->norm == PQN_NORM_LAYER || a->norm == PQN_NORM_RMS, "%s: unknown norm %d", who, a->norm);
  PQN_REQUIRE(a->gate_act == PQN_GATE_NONE || a->gate_act == PQN_GATE_SIGMOID || a->gate_act == PQN_GATE_SILU,
              "%s: unknown gate activation %d", who, a->gate_act);
  PQN_REQUIRE(a->eps >= 0.f, "%s: eps must be >= 0", who);
  PQN_REQUIRE(a->post || (!a->post_scale && !a->post_bias), "%s: post_scale / post_bias without the norm after the block", who);
  PQN_REQUIRE(a->pre || (!a->pre_scale && !a->pre_bias), "%s: pre_scale / pre_bias without the norm before the next block", who);
  if (a->n > 0) {
    PQN_REQUIRE(a->x && a->f, "%s: NULL x or f", who);
    PQN_REQUIRE((a->gate != nullptr) == (a->gate_act != PQN_GATE_NONE), "%s: gate and gate_act go together", who);
  }
  return PQN_OK;
}

static rn_args rn_fill(const pqn_residual_norm_t *a) {
  rn_args A = {};
  A.n = a->n; A.d = a->d; A.rms = a->norm == PQN_NORM_RMS; A.gate_act = a->gate_act;
  A.has_post = a->post; A.has_pre = a->pre; A.eps = a->eps;
  A.x = a->x; A.f = a->f; A.g = a->gate; A.xs = a->x_stride; A.fs = a->f_stride; A.gs = a->gate_stride;
  A.res_scale = a->res_scale; A.post_scale = a->post_scale; A.post_bias = a->post_bias;
  A.pre_scale = a->pre_scale; A.pre_bias = a->pre_bias;
  A.y = a->y; A.h = a->h;
  A.dy = a->dy; A.dh = a->dh; A.dys = a->dy_stride; A.dhs = a->dh_stride;
  A.dx = a->dx; A.df = a->df; A.dg = a->dgate;
  A.partials = a->workspace;
  A.stats = (RnStat *)(a->workspace + (a->n > 0 ? (int64_t)rn_parts(a->n, a->d) * RN_PARAMS * a->d : 0));
  return A;
}

extern "C" int pqn_residual_norm(const pqn_residual_norm_t *a, void *stream) {
  const int rc = rn_check(a, "pqn_residual_norm");
  if (rc != PQN_OK) return rc;
  if (a->n == 0) return PQN_OK;
  PQN_REQUIRE(a->y && (a->h != nullptr) == (a->pre != 0), "pqn_residual_norm: y is an output, and h is one exactly where pre is set");
  const void *ptrs[] = {a->x, a->f, a->gate, a->y, a->h};
  const int64_t strides[] = {a->x_stride, a->f_stride, a->gate ? a->gate_stride : 0};
  const bool vec = rn_vec_ok(a, ptrs, 5, strides, 3);
  return pqn_with_dtype(a->dtype, [&](auto t) { return rn_launch<decltype(t), false>(rn_fill(a), vec, (hipStream_t)stream); });
}

extern "C" int64_t pqn_residual_norm_workspace_floats(int64_t n, int32_t d) {
  if (n <= 0 || d <= 0 || d > RN_MAX_D) return 0;
  return (int64_t)rn_parts(n, d) * RN_PARAMS * d + (d > RN_WIDE ? n * (int64_t)(sizeof(RnStat) / 4) : 0);
}

extern "C" int pqn_residual_norm_grad(const pqn_residual_norm_t *a, void *stream) {
  const int rc = rn_check(a, "pqn_residual_norm_grad");
  if (rc != PQN_OK) return rc;
  rn_param_out out = {{a->dres_scale, a->dpost_scale, a->dpost_bias, a->dpre_scale, a->dpre_bias}};
  bool any = false;
  for (int k = 0; k < RN_PARAMS; ++k) any = any || out.p[k];
  if (a->n > 0) {
    PQN_REQUIRE(a->dx && a->df && (a->dgate != nullptr) == (a->gate != nullptr), "pqn_residual_norm_grad: dx, df (and dgate with a gate) are outputs");
    PQN_REQUIRE(a->workspace, "pqn_residual_norm_grad: NULL workspace");
    PQN_REQUIRE(a->dy || a->dh, "pqn_residual_norm_grad: dy and dh are both NULL");
    PQN_REQUIRE(!a->dh || a->pre, "pqn_residual_norm_grad: dh without the norm before the next block");
    const void *ptrs[] = {a->x, a->f, a->gate, a->dy, a->dh, a->dx, a->df, a->dgate};
    const int64_t strides[] = {a->x_stride, a->f_stride, a->gate ? a->gate_stride : 0, a->dy ? a->dy_stride : 0, a->dh ? a->dh_stride : 0};
    const bool vec = rn_vec_ok(a, ptrs, 8, strides, 5);
    const int r = pqn_with_dtype(a->dtype, [&](auto t) {
      const int rc = rn_launch<decltype(t), true>(rn_fill(a), vec, (hipStream_t)stream);
      return rc == PQN_OK && any && a->d > RN_WIDE ? rn_launch_sums<decltype(t)>(rn_fill(a), vec, (hipStream_t)stream) : rc;
    });
    if (r != PQN_OK) return r;
  }
  if (!any) return PQN_OK;
  // few columns are shared out finely, or too few workgroups read.  us with 16 / 64 columns a workgroup: d = 1024, 1024 parts 9 / 23;
  // d = 4095, 512 parts 20 / 14
  const int parts = a->n > 0 ? rn_parts(a->n, a->d) : 0;
  if (a->d <= 2048) rn_param_kernel<16><<<dim3((a->d + 15) / 16, RN_PARAMS), 1024, 0, (hipStream_t)stream>>>(a->workspace, parts, a->d, out);
  else rn_param_kernel<64><<<dim3((a->d + 63) / 64, RN_PARAMS), 1024, 0, (hipStream_t)stream>>>(a->workspace, parts, a->d, out);
  return pqn_check_launch("pqn_residual_norm_grad");
}
