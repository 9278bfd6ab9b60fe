// pqn_attn.hip -- linear attention with a decay per head over time-major windows, cut at episode ends, forward and gradient
// (pqn_decay_attn, pqn_decay_attn_grad in include/pqn_hotpath.h).
//
//   S_t = decay_h (1 - reset_t) S_{t-1} + k_t v_t^T          o_t = scale S_t^T q_t            (S_-1 = the state that came in)
//
// The gradient is three scans of the same form.  With R_t = scale q_t do_t^T + decay_h (1 - reset_{t+1}) R_{t+1}, R_T-1 also holding
// the gradient of the state that went out:
//   dq_t = scale S_t do_t                 a forward scan with (do, v, k) for (q, k, v) and S transposed
//   dk_t = R_t v_t                        a backward scan with (v, do, q) and R transposed
//   dv_t = R_t^T k_t                      a backward scan with (k, q, do)
//   d(state that came in) = decay_h (1 - reset_0) R_0
// so one kernel serves the forward and, over three argument sets in one launch, the gradient; a backward scan is a forward one over
// negative time strides.
#include "pqn_attn_chunk.h"

// ---- the recurrence, step by step ------------------------------------------------------------------------------------------
// A wave owns 32 columns of one (row, head)'s state in registers for the whole scan: 8 lanes x 4 columns across, 8 lane groups down
// the rows, RPT rows per lane.  A step reads q, k, v once and reduces o over the lane groups by shuffles; no shared memory.  Bound: the
// state's bytes (HBM) for a step of many rows, latency for few: 128 rows x 4 heads of 32, f32, one step 4.8 us (10.5 with the call).
template <int RPT, bool VEC>
PQN_D void da_state_io(float (&s)[RPT][4], float *mem, const da_pass &P, int r0, int c0, bool write) {
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = r0 + 8 * i;
    if (r >= P.a) continue;
    float *p = mem + (long long)r * P.s_rs + (long long)c0 * P.s_cs;
    if constexpr (VEC) {
      if (c0 < P.b) {
        if (write) pqn_store<float, 4>(p, s[i]);
        else pqn_load<float, 4>(s[i], p);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c0 + j < P.b) {
          if (write) p[(long long)j * P.s_cs] = s[i][j];
          else s[i][j] = p[(long long)j * P.s_cs];
        }
    }
  }
}

template <typename T, int RPT, bool VEC>
__global__ __launch_bounds__(256) void da_recur_kernel(da_args A) {
  const da_pass &P = A.pass[blockIdx.y];
  const uint32_t cb = (P.b + 31) >> 5;                            // 1 .. 4; at most 2^28 (row, head) pairs: 32 bits
  const uint32_t unit = blockIdx.x * 4u + (threadIdx.x >> 6);
  if (unit >= (uint32_t)A.m * (uint32_t)A.heads * cb) return;     // whole waves
  const int lane = threadIdx.x & 63;
  const uint32_t mh32 = unit / cb;
  const int row = (int)(mh32 / (uint32_t)A.heads), h = (int)(mh32 - (uint32_t)row * A.heads);
  const long long mh = mh32;
  const int c0 = (int)(unit - mh32 * cb) * 32 + (lane & 7) * 4, r0 = lane >> 3;
  const float decay = A.decay[h];
  const T *q = (const T *)P.q + row * P.qs[1] + h * P.qs[2];
  const T *k = (const T *)P.k + row * P.ks[1] + h * P.ks[2];
  const T *v = (const T *)P.v + row * P.vs[1] + h * P.vs[2];
  T *o = (T *)P.o + row * P.os[1] + h * P.os[2];
  const long long so = mh * ((long long)P.a * P.b);
  float s[RPT][4];
#pragma unroll
  for (int i = 0; i < RPT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
  if (P.s_in) da_state_io<RPT, VEC>(s, const_cast<float *>(P.s_in) + so, P, r0, c0, false);
  for (int t = 0; t < A.t_len; ++t) {
    float kr[RPT], qr[RPT], vc[4];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = r0 + 8 * i;
      kr[i] = r < P.a ? pqn_to_f32(k[t * P.ks[0] + r]) : 0.f;
      qr[i] = r < P.a ? pqn_to_f32(q[t * P.qs[0] + r]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) vc[j] = c0 + j < P.b ? pqn_to_f32(v[t * P.vs[0] + c0 + j]) * P.s_scale : 0.f;
    if (t > 0 || !P.late) {
      const bool cut = P.reset && P.reset[t * P.reset_ts + row];
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = cut ? 0.f : s[i][j] * decay;   // a choice, not a product: what a reset drops may be NaN
    }
    float out[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fmaf(kr[i], vc[j], s[i][j]);
        out[j] = fmaf(qr[i], s[i][j], out[j]);
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int d = 8; d < 64; d <<= 1) out[j] += __shfl_xor(out[j], d, 64);
      if (r0 == 0 && c0 + j < P.b) o[t * P.os[0] + c0 + j] = (T)(out[j] * P.o_scale);
    }
  }
  if (P.s_out) {
    if (P.late && A.t_len > 0) {
      const bool cut = P.reset && P.reset[A.t_len * P.reset_ts + row];
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = cut ? 0.f : s[i][j] * decay;
    }
    da_state_io<RPT, VEC>(s, P.s_out + so, P, r0, c0, true);
  }
}

// the parts' states in order: part p's own, from zero, becomes the state behind it, S_p = decay^len S_{p-1} + own unless it was cut
__global__ __launch_bounds__(256) void da_join_kernel(da_args A, da_split X, int size) {
  const uint32_t block = blockIdx.x, per = (uint32_t)(size + 1023) / 1024u;
  const long long mh = block / per;
  const int e = (int)(block % per) * 1024 + threadIdx.x * 4, pass = blockIdx.y;
  if (e >= size) return;
  float *p = X.state + pass * X.pass_stride + mh * (X.parts - 1) * (long long)size + e;
  const int *cut = X.cut + pass * X.cut_stride + mh * (X.parts - 1);
  const float fade = (float)pqn_powi((double)A.decay[(uint32_t)mh % (uint32_t)A.heads], X.len);
  f32x4_t s = *(const f32x4_t *)p;
  const int last = X.parts - 2;
  constexpr int AHEAD = 8;                                        // states requested together: the walk waits once for so many
  for (int i0 = 1; i0 <= last; i0 += AHEAD) {
    f32x4_t own[AHEAD];
    int ends[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      own[i] = *(const f32x4_t *)(p + (long long)min(i0 + i, last) * size);
      ends[i] = cut[min(i0 + i, last)];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (i0 + i > last) break;
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = ends[i] ? own[i][j] : fmaf(s[j], fade, own[i][j]);
      *(f32x4_t *)(p + (long long)(i0 + i) * size) = s;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
template <typename T>
static int da_launch_recur(const da_args &A, int passes, hipStream_t st) {
  int amax = 0, cbmax = 0;
  bool vec = true;
  for (int p = 0; p < passes; ++p) {
    const da_pass &P = A.pass[p];
    amax = P.a > amax ? P.a : amax;
    cbmax = (P.b + 31) / 32 > cbmax ? (P.b + 31) / 32 : cbmax;
    vec = vec && P.s_cs == 1 && P.b % 4 == 0 && (((uintptr_t)P.s_in | (uintptr_t)P.s_out) & 15) == 0;
  }
  const long long units = (long long)A.m * A.heads * cbmax, blocks = (units + 3) / 4;
  PQN_REQUIRE(pqn_one_launch(blocks, 256), "pqn_decay_attn: %d x %d rows and heads are more than one launch covers", A.m, A.heads);
  const dim3 grid((unsigned)blocks, passes);
#define DA_GO(RPT)                                                          \
  do {                                                                      \
    if (vec) da_recur_kernel<T, RPT, true><<<grid, 256, 0, st>>>(A);        \
    else da_recur_kernel<T, RPT, false><<<grid, 256, 0, st>>>(A);           \
    return pqn_check_launch("pqn_decay_attn");                              \
  } while (0)
  if (amax <= 32) DA_GO(4);
  if (amax <= 64) DA_GO(8);
  DA_GO(16);
#undef DA_GO
}

static bool da_vec(const pqn_decay_attn_t *a, int grad) {
  const int ev = 16 / pqn_dtype_size(a->dtype);
  uintptr_t at = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (grad ? (uintptr_t)a->dout | (uintptr_t)a->dq | (uintptr_t)a->dk_out | (uintptr_t)a->dv_out : (uintptr_t)a->out);
  bool vec = a->dk % ev == 0 && a->dv % ev == 0 && (at & 15) == 0;
  for (int i = 0; i < 3; ++i)
    vec = vec && a->q_stride[i] % ev == 0 && a->k_stride[i] % ev == 0 && a->v_stride[i] % ev == 0 && (!grad || a->dout_stride[i] % ev == 0);
  return vec;
}

// Windows of up to this many steps go step by step, longer ones by chunks; a single step of the forward always does, so that a row acts
// alike (to the bit) whatever number of rows acts beside it.  Measured on both sides, us forward / gradient: 4096 x 4 heads of 32, f32, 2
// steps 32 / 89 against 49 / 111 by chunks, 4 steps 39 / 114 against 47 / 116, 6 steps 50 / 149 against 47 / 124; 1024 x 8 heads of 64, f32,
// 1 step 51 / 144 against 77 / 190; 1024 x 8 heads of 128, 1 step, f32 218 / 595 against 239 / 539, bf16 218 / 674 against 209 / 440; bf16
// steps in place of 1024 x 8 heads: 128 x 128 225 against 212, 72 x 128 133 against 198, 128 x 32 54 against 110; 256 x 8 of 96 x 96 32 and
// 41.  Off 16 bytes chunks load element by element: 1000 x 4 heads of 127, 3 steps f32 213 / 400 against 238 / 560, 2 steps bf16 219 / 408
// against 229 / 600, 4 steps bf16 277 / 585 against 232 / 607; 4000 x 8 heads of 33 and 65, 3 steps bf16 329 / 1176 against 675 / 2695.
static bool da_by_steps(const pqn_decay_attn_t *a, bool grad) {
  const int w = a->dk > a->dv ? a->dk : a->dv;
  return a->t_len <= (w <= 32 ? 4 : !da_vec(a, grad) ? 3 : w <= 64 || !grad || (long long)a->m * a->heads < 2048 ? 1 : 0);
}
// The time axis is cut where rows x heads alone give the chip too few waves: parts of at least DA_MIN_PART steps (each costs a second
// reading of k and v and a state written and read), as many as make DA_FILL waves, in whole chunks: 1001 steps x 35 rows of 48 and 80 columns
// go in 11 parts of 96.  Measured there, f32, forward / gradient: parts of at least 64 52 / 126 us, 128 52 / 147, 256 91 / 213; 16001 x 16
// rows of 64 and 128, bf16: 1024 waves 165 / 451, 2048 109 / 300, 4096 112 / 331; 5000 x 8 of 128 and 128, bf16: 55 / 125, 51 / 88, 51 / 102.
static constexpr int DA_MIN_PART = 64, DA_FILL = 2048;

static da_split da_cut(int t_len, long long rows, int passes, int a, int b, int vec) {
  da_split X = {};
  const int nw = da_nw(a, b, vec);
  const long long waves = rows * passes * (nw == 3 ? 4 : nw);     // a CU holds as many workgroups of three waves as of four
  long long want = (DA_FILL + waves - 1) / (waves > 0 ? waves : 1);
  const long long most = t_len / DA_MIN_PART;
  if (want > most) want = most;
  if (want < 1) want = 1;
  X.len = (int)(((t_len + want - 1) / want + 31) / 32 * 32);      // whole chunks
  X.parts = X.len > 0 ? (t_len + X.len - 1) / X.len : 1;
  if (X.parts < 1) X.parts = 1;
  X.vec = vec;
  return X;
}
// workspace of one launch of `passes` scans: the parts' states, then their cut flags
static int da_state_size(const da_split &X, int a, int b) { return da_ap(a, X.vec) * 32 * da_nw(a, b, X.vec); }
static long long da_ws_bytes(const da_split &X, long long rows, int passes, int a, int b) {
  if (X.parts <= 1) return 0;
  return passes * (rows * (X.parts - 1) * 4ll * da_state_size(X, a, b) + (rows * (X.parts - 1) * 4 + 15) / 16 * 16);
}

// the passes, chunked, in one launch each of: the parts' states, their join, the scan
static int da_run_chunks(da_args &A, int passes, int dtype, int vec, void *workspace, hipStream_t st) {
  const long long rows = (long long)A.m * A.heads;
  const int a = da_widest(A, passes, &da_pass::a), b = da_widest(A, passes, &da_pass::b);
  da_split X = da_cut(A.t_len, rows, passes, a, b, vec);
  const int size = da_state_size(X, a, b);
  for (int p = 0; p < passes; ++p) {
    da_pass &P = A.pass[p];
    const uintptr_t at = (uintptr_t)P.s_in | (uintptr_t)P.s_out;
    P.s_vec = P.s_cs == 1 && P.b % 2 == 0 && at % 8 == 0 ? 2 : P.s_rs == 1 && P.a % 4 == 0 && at % 16 == 0 ? 4 : 0;
  }
  X.pass_stride = rows * (X.parts - 1) * size;
  X.cut_stride = (rows * (X.parts - 1) * 4 + 15) / 16 * 4;
  X.state = (float *)workspace;
  X.cut = (int *)(X.state + passes * X.pass_stride);
  auto go = [&](bool state) {
    return dtype == PQN_DTYPE_F32 ? da_launch_chunk_f32(A, X, passes, state, st) : da_launch_chunk_bf16(A, X, passes, state, st);
  };
  if (X.parts > 1) {
    int rc = go(true);
    if (rc != PQN_OK) return rc;
    if (X.parts > 2) {
      da_join_kernel<<<dim3((unsigned)(rows * ((size + 1023) / 1024)), passes), 256, 0, st>>>(A, X, size);
      rc = pqn_check_launch("pqn_decay_attn");
      if (rc != PQN_OK) return rc;
    }
  }
  return go(false);
}

static int da_check(const pqn_decay_attn_t *a, const char *who) {
  PQN_REQUIRE(a, "%s: NULL argument block", who);
  PQN_REQUIRE(a->dtype == PQN_DTYPE_F32 || a->dtype == PQN_DTYPE_BF16, "%s: dtype %d is neither f32 nor bf16", who, a->dtype);
  PQN_REQUIRE(a->t_len >= 0 && a->m >= 0 && a->heads > 0, "%s: t_len, m must be >= 0 and heads > 0 (%d, %d, %d)", who, a->t_len, a->m, a->heads);
  PQN_REQUIRE(a->t_len <= (1 << 30), "%s: up to 2^30 steps (t_len=%d)", who, a->t_len);
  PQN_REQUIRE(a->dk > 0 && a->dk <= PQN_ATTN_MAX_D && a->dv > 0 && a->dv <= PQN_ATTN_MAX_D, "%s: head widths of 1 .. %d (dk=%d dv=%d)", who,
              PQN_ATTN_MAX_D, a->dk, a->dv);
  PQN_REQUIRE((long long)a->m * a->heads <= (1ll << 28), "%s: up to 2^28 (row, head) pairs (m=%d heads=%d)", who, a->m, a->heads);
  PQN_REQUIRE(a->decay || a->m == 0, "%s: NULL decay", who);
  PQN_REQUIRE((a->q && a->k && a->v) || a->t_len == 0 || a->m == 0, "%s: NULL q, k or v", who);
  return PQN_OK;
}

static void da_strides(long long (&to)[3], const int64_t *from, bool reverse) {
  to[0] = reverse ? -from[0] : from[0];
  to[1] = from[1];
  to[2] = from[2];
}
// a tensor over (time, row, head): its first element in scan order and its strides
static const void *da_first(const void *p, const int64_t *s, int t_len, int es, bool reverse) {
  return (reverse && t_len > 0) ? (const char *)p + (long long)(t_len - 1) * s[0] * es : p;
}

static da_pass da_make(const pqn_decay_attn_t *a, const void *q, const int64_t *qs, const void *k, const int64_t *ks, const void *v,
                       const int64_t *vs, void *o, int wq, int wv, bool reverse) {
  const int es = pqn_dtype_size(a->dtype);
  da_pass P = {};
  const int64_t os[3] = {(int64_t)a->m * a->heads * wv, (int64_t)a->heads * wv, wv};
  P.q = da_first(q, qs, a->t_len, es, reverse);
  P.k = da_first(k, ks, a->t_len, es, reverse);
  P.v = da_first(v, vs, a->t_len, es, reverse);
  P.o = const_cast<void *>(da_first(o, os, a->t_len, es, reverse));
  da_strides(P.qs, qs, reverse);
  da_strides(P.ks, ks, reverse);
  da_strides(P.vs, vs, reverse);
  da_strides(P.os, os, reverse);
  P.a = wq;
  P.b = wv;
  // backward scans meet the border between steps t and t + 1 in front of their step T - 1 - t: flag t + 1 = T - i
  P.reset = a->reset ? a->reset + (reverse ? (long long)a->t_len * a->m : 0) : nullptr;
  P.reset_ts = reverse ? -(long long)a->m : a->m;
  P.late = reverse;
  P.o_scale = reverse ? 1.f : a->scale;
  P.s_scale = reverse ? a->scale : 1.f;
  return P;
}

extern "C" int64_t pqn_decay_attn_workspace_bytes(const pqn_decay_attn_t *a, int32_t grad) {
  if (da_check(a, "pqn_decay_attn_workspace_bytes") != PQN_OK || da_by_steps(a, grad != 0) || a->m == 0) return 0;
  const long long rows = (long long)a->m * a->heads;
  // of both forms, so that the answer goes by sizes alone and not by the tensors' addresses and strides
  auto need = [&](int passes, int wa, int wb) {
    const long long x = da_ws_bytes(da_cut(a->t_len, rows, passes, wa, wb, 0), rows, passes, wa, wb);
    const long long y = da_ws_bytes(da_cut(a->t_len, rows, passes, wa, wb, 1), rows, passes, wa, wb);
    return x > y ? x : y;
  };
  if (!grad) return need(1, a->dk, a->dv);
  const int w = a->dk > a->dv ? a->dk : a->dv;
  const long long all = need(3, w, w), one = need(2, a->dv, a->dk), two = need(1, a->dk, a->dv);   // together, or one after the other
  return all > one ? (all > two ? all : two) : one > two ? one : two;
}

extern "C" int pqn_decay_attn(const pqn_decay_attn_t *a, void *stream) {
  const int rc = da_check(a, "pqn_decay_attn");
  if (rc != PQN_OK) return rc;
  if (a->m == 0 || (a->t_len == 0 && !a->state_out)) return PQN_OK;
  PQN_REQUIRE(a->out || a->t_len == 0, "pqn_decay_attn: NULL out");
  PQN_REQUIRE(((uintptr_t)a->workspace & 15) == 0, "pqn_decay_attn: the workspace must be 16-byte aligned");
  PQN_REQUIRE(!a->state_out || a->state_out != a->state_in || a->t_len <= 1, "pqn_decay_attn: in place only for a window of one step");
  da_args A = {};
  A.t_len = a->t_len; A.m = a->m; A.heads = a->heads; A.decay = a->decay;
  da_pass &P = A.pass[0];
  P = da_make(a, a->q, a->q_stride, a->k, a->k_stride, a->v, a->v_stride, a->out, a->dk, a->dv, false);
  P.s_in = a->state_in;
  P.s_out = a->state_out;
  P.s_rs = a->dv;
  P.s_cs = 1;
  if (!da_by_steps(a, false)) {
    const int vec = da_vec(a, 0);
    PQN_REQUIRE(a->workspace || pqn_decay_attn_workspace_bytes(a, 0) == 0, "pqn_decay_attn: NULL workspace");
    return da_run_chunks(A, 1, a->dtype, vec, a->workspace, (hipStream_t)stream);
  }
  return a->dtype == PQN_DTYPE_F32 ? da_launch_recur<float>(A, 1, (hipStream_t)stream) : da_launch_recur<pqn_bf16>(A, 1, (hipStream_t)stream);
}

extern "C" int pqn_decay_attn_grad(const pqn_decay_attn_t *a, void *stream) {
  const int rc = da_check(a, "pqn_decay_attn_grad");
  if (rc != PQN_OK) return rc;
  if (a->m == 0 || (a->t_len == 0 && !a->dstate_in)) return PQN_OK;
  PQN_REQUIRE((a->dout && a->dq && a->dk_out && a->dv_out) || a->t_len == 0, "pqn_decay_attn_grad: NULL dout, dq, dk or dv");
  PQN_REQUIRE(((uintptr_t)a->workspace & 15) == 0, "pqn_decay_attn_grad: the workspace must be 16-byte aligned");
  PQN_REQUIRE(!a->dstate_in || a->dstate_in != a->dstate_out, "pqn_decay_attn_grad: dstate_in must not be dstate_out");
  da_args A = {};
  A.t_len = a->t_len; A.m = a->m; A.heads = a->heads; A.decay = a->decay;
  da_pass &Q = A.pass[0], &K = A.pass[1], &V = A.pass[2];
  Q = da_make(a, a->dout, a->dout_stride, a->v, a->v_stride, a->k, a->k_stride, a->dq, a->dv, a->dk, false);
  Q.s_in = a->state_in;
  Q.s_rs = 1;
  Q.s_cs = a->dv;
  K = da_make(a, a->v, a->v_stride, a->dout, a->dout_stride, a->q, a->q_stride, a->dk_out, a->dv, a->dk, true);
  K.s_in = a->dstate_out;
  K.s_rs = 1;
  K.s_cs = a->dv;
  V = da_make(a, a->k, a->k_stride, a->q, a->q_stride, a->dout, a->dout_stride, a->dv_out, a->dk, a->dv, true);
  V.s_in = a->dstate_out;
  V.s_out = a->dstate_in;
  V.s_rs = a->dv;
  V.s_cs = 1;
  if (!da_by_steps(a, true)) {
    const int vec = da_vec(a, 1);
    PQN_REQUIRE(a->workspace || pqn_decay_attn_workspace_bytes(a, 1) == 0, "pqn_decay_attn_grad: NULL workspace");
    // dq and dk have states of [dv][dk], dv of [dk][dv].  One launch of the kernel that holds both where that is nearly the kernel of
    // each, or where there is little to do in several launches (the time axis is cut) and they are more than the padding.  Measured on
    // both sides, together / one after the other, us: 300 steps x 6 rows, 32 and 128 columns, f32 49 / 80, bf16 37 / 63; 1001 x 35, 48
    // and 80, f32 136 / 126, bf16 80 / 88; 5000 x 8, 64 and 128, bf16 88 / 102; 4000 x 160, 32 and 64, f32 813 / 595, bf16 416 / 344;
    // 32 x 512, 80 and 48, f32 51 / 48 (not cut); 300 x 480, 128 and 96, bf16 177 / 205.
    const int w = a->dk > a->dv ? a->dk : a->dv, least = a->dk + a->dv - w;
    const bool same = da_ap(least, vec) == da_ap(w, vec) && da_nw(least, w, vec) == da_nw(w, w, vec) && da_nw(w, least, vec) == da_nw(w, w, vec);
    const bool alike = same || least > 64 || (least > 32 && w <= 64);
    const long long rows = (long long)a->m * a->heads;
    if (alike || (a->t_len * rows <= (a->dtype == PQN_DTYPE_F32 ? 1 << 14 : 1 << 16) && da_cut(a->t_len, rows, 3, w, w, vec).parts > 1))
      return da_run_chunks(A, 3, a->dtype, vec, a->workspace, (hipStream_t)stream);
    int rc = da_run_chunks(A, 2, a->dtype, vec, a->workspace, (hipStream_t)stream);      // dq, dk: states of [dv][dk]
    if (rc != PQN_OK) return rc;
    A.pass[0] = A.pass[2];                                                          // dv: [dk][dv]
    return da_run_chunks(A, 1, a->dtype, vec, a->workspace, (hipStream_t)stream);
  }
  return a->dtype == PQN_DTYPE_F32 ? da_launch_recur<float>(A, 3, (hipStream_t)stream) : da_launch_recur<pqn_bf16>(A, 3, (hipStream_t)stream);
}
