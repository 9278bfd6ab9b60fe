// pqn_logprob.hip -- log probabilities of taken actions under the softmax of their logits, with the entropy, the logsumexp and the
// top alternatives, and the gradient (pqn_action_logprobs, pqn_action_logprobs_grad in include/pqn_hotpath.h).
//
//   x_j = logit_j / temperature where allowed      lse = log sum e^x      logp = x_a - lse      H = -sum p log p = lse - sum p x
//
// One pass over the logits: every lane keeps the running maximum m of what it has seen, s = sum e^(x - m) and t = sum (x - m) e^(x - m),
// so H = log s - t / s without a second look (t is shifted like s when m grows: t' = e^(m - m') (t + (m - m') s)).  The K best logits
// come out of the same pass: a key is the logit's order-preserving bits above the complement of its index, so keys are distinct and
// ties go to the lowest index whatever the order of the work.
#include "pqn_vec.h"

typedef unsigned long long u64;
static constexpr int LP_MAX_TOP = PQN_LOGPROB_MAX_TOP;

struct lp_args {
  int n, a, top;
  float inv_temp;
  const void *logits;
  long long ls;                      // row stride of the logits in elements
  const uint8_t *mask;
  long long ms;                      // row stride of the mask
  const int32_t *action;
  float *logp, *entropy, *lse, *top_logp;
  int32_t *top_action;
  // few rows: a row is cut into `splits` parts of `part` columns, one workgroup each, joined by lp_join_kernel
  int splits, part;
  float *rec;                        // [n][splits][4 + 2 * LP_MAX_TOP] words: m, s, t, nan | keys
};
static constexpr int LP_REC = 4 + 2 * LP_MAX_TOP;

// order-preserving bits; 0 = "nothing" (a masked, infinite-negative or NaN logit is never an alternative)
PQN_D uint32_t lp_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
PQN_D float lp_unorder(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
PQN_D u64 lp_key(float logit, int j) {
  return logit > -INFINITY ? ((u64)lp_order(logit) << 32) | (uint32_t)~j : 0ull;   // false for NaN too
}
PQN_D u64 lp_max(u64 a, u64 b) { return a > b ? a : b; }
template <int G>
PQN_D u64 lp_group_max(u64 k) {
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1) k = lp_max(k, (u64)__shfl_xor((long long)k, d, 64));
  return k;
}

// (m, s, t) of a set of values; empty: m = -inf, s = t = 0
struct LpSum {
  float m, s, t;
};
PQN_D LpSum lp_join(const LpSum &a, const LpSum &b) {
  const float m = a.m > b.m ? a.m : (b.m > a.m ? b.m : a.m);   // equal (both may be infinite): either
  // a part at -inf holds nothing (s = t = 0); equal maxima need no shift, which also keeps inf - inf out
  const float da = a.m == m ? 0.f : a.m - m, db = b.m == m ? 0.f : b.m - m;
  const float ea = expf(da), eb = expf(db);
  LpSum r;
  r.m = m;
  r.s = a.s * ea + b.s * eb;
  r.t = (a.s > 0.f ? ea * (a.t + (ea > 0.f ? da * a.s : 0.f)) : 0.f) + (b.s > 0.f ? eb * (b.t + (eb > 0.f ? db * b.s : 0.f)) : 0.f);
  return r;
}
template <int G>
PQN_D LpSum lp_group_join(LpSum v) {
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1) {
    LpSum o = {__shfl_xor(v.m, d, 64), __shfl_xor(v.s, d, 64), __shfl_xor(v.t, d, 64)};
    // lanes d apart join the same two parts in the same order: bit-identical in every lane
    v = (threadIdx.x & d) ? lp_join(o, v) : lp_join(v, o);
  }
  return v;
}

// what a row's sums say; bad = a NaN or +inf among the allowed logits
struct LpRow {
  float lse, entropy;
};
PQN_D LpRow lp_row(const LpSum &v, bool bad) {
  LpRow r;
  if (bad) r.lse = r.entropy = NAN;
  else if (!(v.s > 0.f)) r.lse = -INFINITY, r.entropy = 0.f;          // nothing allowed
  else {
    const float ls = logf(v.s);
    r.lse = v.m + ls;
    r.entropy = fmaxf(ls - v.t / v.s, 0.f);
  }
  return r;
}
template <typename T>
PQN_D float lp_logit(const lp_args &A, long long row, int j) {   // -inf where not allowed
  if (A.mask && !A.mask[row * A.ms + j]) return -INFINITY;
  return pqn_to_f32(((const T *)A.logits)[row * A.ls + j]);
}
template <typename T>
PQN_D void lp_write_row(const lp_args &A, long long row, const LpRow &r) {
  A.lse[row] = r.lse;
  A.entropy[row] = r.entropy;
  const int act = A.action[row];
  float lp = 0.f;                                                      // an id outside 0 .. a-1: no action, nothing is read
  if (act >= 0 && act < A.a) {
    const float l = lp_logit<T>(A, row, act);
    lp = (r.lse != r.lse) ? NAN : l > -INFINITY ? l * A.inv_temp - r.lse : -INFINITY;
  }
  A.logp[row] = lp;
}
PQN_D void lp_write_top(const lp_args &A, long long row, int i, u64 key, float lse) {
  A.top_action[row * A.top + i] = key ? (int32_t)~(uint32_t)key : -1;
  A.top_logp[row * A.top + i] = key ? lp_unorder((uint32_t)(key >> 32)) * A.inv_temp - lse : -INFINITY;
}

// A row in the registers of G lanes, E logits each (a <= G * E): 64 / G rows per wave, no shared memory.
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void lp_rows_kernel(lp_args A) {
  const int lane = threadIdx.x & (G - 1);
  const long long row0 = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
  const bool live = row0 < A.n;                    // rows behind the last one shuffle along with a copy of it
  const long long row = live ? row0 : A.n - 1;
  float x[E];
  bool bad = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = e * G + lane;
    x[e] = j < A.a ? lp_logit<T>(A, row, j) : -INFINITY;
    bad = bad || !(x[e] < INFINITY);
  }
  LpSum v = {-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) v.m = fmaxf(v.m, x[e]);
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1) v.m = fmaxf(v.m, __shfl_xor(v.m, d, 64));
  v.m *= A.inv_temp;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float z = x[e] * A.inv_temp - v.m, p = x[e] > -INFINITY ? expf(z) : 0.f;
    v.s += p;
    v.t += p > 0.f ? z * p : 0.f;
  }
  float nbad = bad ? 1.f : 0.f;
  v.s = pqn_group_sum<G>(v.s);
  v.t = pqn_group_sum<G>(v.t);
  nbad = pqn_group_sum<G>(nbad);
  const LpRow r = lp_row(v, nbad > 0.f);
  if (live && lane == 0) lp_write_row<T>(A, row, r);
  if (A.top > 0) {
    u64 key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = lp_key(x[e], e * G + lane);
    for (int i = 0; i < A.top; ++i) {
      u64 best = key[0];
#pragma unroll
      for (int e = 1; e < E; ++e) best = lp_max(best, key[e]);
      best = lp_group_max<G>(best);
      if (live && lane == 0) lp_write_top(A, row, i, best, r.lse);
#pragma unroll
      for (int e = 0; e < E; ++e) key[e] = key[e] == best ? 0ull : key[e];
    }
  }
}

// The K best keys of a wave, key i in lane i; lanes from K on hold nothing
PQN_D void lp_insert(u64 &list, u64 key, int top) {
  const int lane = threadIdx.x & 63;
  const int at = __popcll(__ballot(list > key));               // keys above the new one, all in the first lanes
  const u64 up = (u64)__shfl_up((long long)list, 1, 64);
  list = lane < at ? list : lane == at ? key : up;
  if (lane >= top) list = 0ull;
}

// A workgroup per row (or part of a row), VW logits per lane and access.  NT threads.
template <typename T, int NT, int VW>
__global__ __launch_bounds__(NT) void lp_long_kernel(lp_args A) {
  constexpr int NW = NT / 64;
  __shared__ u64 keys[NW * LP_MAX_TOP];
  __shared__ float sums[NW][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long row = blockIdx.x / A.splits;
  const int part = blockIdx.x % A.splits;
  const int c0 = part * A.part, c1 = min(A.a, c0 + A.part);
  const T *p = (const T *)A.logits + row * A.ls;
  const uint8_t *mk = A.mask ? A.mask + row * A.ms : nullptr;
  LpSum v = {-INFINITY, 0.f, 0.f};
  u64 list = 0ull, least = 0ull;                                // least = the list's last key: what a newcomer has to beat
  float least_x = -INFINITY;
  bool bad = false;
  for (int base = c0; base < c1; base += NT * VW) {
    const int j = base + threadIdx.x * VW;
    float x[VW];
    if (j + VW <= c1) pqn_load<T, VW>(x, p + j);
    else
#pragma unroll
      for (int e = 0; e < VW; ++e) x[e] = j + e < c1 ? pqn_to_f32(p[j + e]) : -INFINITY;
    if (mk)
#pragma unroll
      for (int e = 0; e < VW; ++e)
        if (j + e < c1 && !mk[j + e]) x[e] = -INFINITY;
    float top = x[0];
#pragma unroll
    for (int e = 0; e < VW; ++e) {
      bad = bad || !(x[e] < INFINITY);
      top = fmaxf(top, x[e]);
    }
    const float m = fmaxf(v.m, top * A.inv_temp);
    if (m > -INFINITY) {
      const float dm = v.m == m ? 0.f : v.m - m, em = expf(dm);
      v.t = v.s > 0.f ? em * (v.t + (em > 0.f ? dm * v.s : 0.f)) : 0.f;
      v.s *= em;
      v.m = m;
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        const float z = x[e] * A.inv_temp - m, q = x[e] > -INFINITY ? expf(z) : 0.f;
        v.s += q;
        v.t += q > 0.f ? z * q : 0.f;
      }
    }
    if (A.top > 0 && __any(top >= least_x && top > -INFINITY)) {
      u64 key[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) key[e] = lp_key(x[e], j + e);
      for (;;) {
        u64 best = key[0];
#pragma unroll
        for (int e = 1; e < VW; ++e) best = lp_max(best, key[e]);
        best = lp_group_max<64>(best);
        if (best <= least) break;                                // 0 <= least: ends when nothing is left
        lp_insert(list, best, A.top);
        least = (u64)__shfl((long long)list, A.top - 1, 64);
#pragma unroll
        for (int e = 0; e < VW; ++e) key[e] = key[e] == best ? 0ull : key[e];
      }
      least_x = least ? lp_unorder((uint32_t)(least >> 32)) : -INFINITY;
    }
  }
  v = lp_group_join<64>(v);
  const bool wbad = __any(bad);
  if (lane == 0) {
    sums[wave][0] = v.m;
    sums[wave][1] = v.s;
    sums[wave][2] = v.t;
    sums[wave][3] = wbad ? 1.f : 0.f;
  }
  if (lane < A.top) keys[wave * A.top + lane] = list;
  __syncthreads();
  if (wave != 0) return;
  v = {sums[0][0], sums[0][1], sums[0][2]};
  bool any_bad = sums[0][3] > 0.f;
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    v = lp_join(v, {sums[w][0], sums[w][1], sums[w][2]});
    any_bad = any_bad || sums[w][3] > 0.f;
  }
  // the best of the NW lists
  u64 mine[(NW * LP_MAX_TOP + 63) / 64];
  constexpr int ML = (NW * LP_MAX_TOP + 63) / 64;
#pragma unroll
  for (int i = 0; i < ML; ++i) mine[i] = i * 64 + lane < NW * A.top ? keys[i * 64 + lane] : 0ull;
  const LpRow r = lp_row(v, any_bad);
  float *rec = A.rec + ((size_t)row * A.splits + part) * LP_REC;
  if (lane == 0) {
    if (A.splits == 1) lp_write_row<T>(A, row, r);
    else {
      rec[0] = v.m;
      rec[1] = v.s;
      rec[2] = v.t;
      rec[3] = any_bad ? 1.f : 0.f;
    }
  }
  for (int i = 0; i < A.top; ++i) {
    u64 best = mine[0];
#pragma unroll
    for (int k = 1; k < ML; ++k) best = lp_max(best, mine[k]);
    best = lp_group_max<64>(best);
    if (lane == 0) {
      if (A.splits == 1) lp_write_top(A, row, i, best, r.lse);
      else ((u64 *)(rec + 4))[i] = best;
    }
#pragma unroll
    for (int k = 0; k < ML; ++k) mine[k] = mine[k] == best ? 0ull : mine[k];
  }
}

// joins the parts of a row: one wave per row
template <typename T>
__global__ __launch_bounds__(64) void lp_join_kernel(lp_args A) {
  const long long row = blockIdx.x;
  const int lane = threadIdx.x;
  const float *rec = A.rec + (size_t)row * A.splits * LP_REC;
  LpSum v = {-INFINITY, 0.f, 0.f};
  bool bad = false;
  for (int i = lane; i < A.splits; i += 64) {
    v = lp_join(v, {rec[i * LP_REC], rec[i * LP_REC + 1], rec[i * LP_REC + 2]});
    bad = bad || rec[i * LP_REC + 3] > 0.f;
  }
  v = lp_group_join<64>(v);
  const LpRow r = lp_row(v, __any(bad));
  if (lane == 0) lp_write_row<T>(A, row, r);
  u64 floor = ~0ull;                        // keys are distinct: the next best is the largest one below the last
  for (int i = 0; i < A.top; ++i) {
    u64 best = 0ull;
    for (int e = lane; e < A.splits * A.top; e += 64) {
      const u64 k = ((const u64 *)(rec + (size_t)(e / A.top) * LP_REC + 4))[e % A.top];
      if (k < floor) best = lp_max(best, k);
    }
    best = lp_group_max<64>(best);
    if (lane == 0) lp_write_top(A, row, i, best, r.lse);
    floor = best;
  }
}

// ---- gradient ------------------------------------------------------------------------------------------------------------
// d/dx_j = dlogp (1[j = action] - p_j) - dentropy p_j (log p_j + H) + dlse p_j, over the temperature.  Elementwise over the logits:
// a lane's VW logits in one access, the row's five scalars once per lane.
struct lp_grad_args {
  lp_args A;
  const float *dlogp, *dentropy, *dlse;
  void *dlogits;                     // [n][a]
  int blocks;                        // workgroups per row
};
template <typename T, int VW>
__global__ __launch_bounds__(256) void lp_grad_kernel(lp_grad_args G) {
  const lp_args &A = G.A;
  long long row;
  int j;
  if (G.blocks > 0) {
    row = blockIdx.x / G.blocks;
    j = ((int)(blockIdx.x % G.blocks) * 256 + threadIdx.x) * VW;
    if (j >= A.a) return;
  } else {                            // narrow rows: a flat index over the whole matrix
    const long long e = ((long long)blockIdx.x * 256 + threadIdx.x) * VW;
    row = e / A.a;
    j = (int)(e - row * A.a);
    if (row >= A.n) return;
  }
  const float lse = A.lse[row], h = A.entropy[row];
  const int act = A.action[row];
  float dlp = G.dlogp ? G.dlogp[row] : 0.f;
  const float dh = G.dentropy ? G.dentropy[row] : 0.f, dl = G.dlse ? G.dlse[row] : 0.f;
  const T *p = (const T *)A.logits + row * A.ls + j;
  T *o = (T *)G.dlogits + row * A.a + j;
  // an id outside the row, or an action that is not allowed, has a constant log probability
  if (act < 0 || act >= A.a || (A.mask && !A.mask[row * A.ms + act]) ||
      !(pqn_to_f32(((const T *)A.logits)[row * A.ls + act]) > -INFINITY)) dlp = 0.f;
  float x[VW], g[VW];
  pqn_load<T, VW>(x, p);
#pragma unroll
  for (int e = 0; e < VW; ++e) {
    const bool in = (!A.mask || A.mask[row * A.ms + j + e]) && x[e] != -INFINITY && lse != -INFINITY;
    const float lp = x[e] * A.inv_temp - lse, q = expf(lp);
    const float c = dl - dlp - (q > 0.f ? dh * (lp + h) : 0.f);
    g[e] = in ? ((act == j + e ? dlp : 0.f) + q * c) * A.inv_temp : 0.f;
  }
  pqn_store<T, VW>(o, g);
}

// ---------------------------------------------------------------------------------------------------------------------------
static int lp_check(const pqn_action_logprobs_t *a, const char *who) {
  PQN_REQUIRE(a, "%s: NULL argument block", who);
  PQN_REQUIRE(pqn_dtype_known(a->dtype), "%s: unknown dtype %d", who, a->dtype);
  PQN_REQUIRE(a->n >= 0 && a->a > 0, "%s: n must be >= 0 and a > 0 (n=%d a=%d)", who, a->n, a->a);
  PQN_REQUIRE(a->a <= (1 << 30), "%s: up to 2^30 columns (a=%d)", who, a->a);
  PQN_REQUIRE(a->top >= 0 && a->top <= LP_MAX_TOP && a->top <= a->a, "%s: top must be in 0 .. min(a, %d) (top=%d a=%d)", who, LP_MAX_TOP, a->top, a->a);
  PQN_REQUIRE(a->temperature > 0.f && a->temperature < INFINITY && 1.0f / a->temperature < INFINITY, "%s: temperature must be positive and finite", who);
  if (a->n > 0) PQN_REQUIRE(a->logits && a->action && a->lse && a->entropy, "%s: NULL logits, action, lse or entropy", who);
  return PQN_OK;
}
static lp_args lp_fill(const pqn_action_logprobs_t *a) {
  lp_args A = {};
  A.n = a->n; A.a = a->a; A.top = a->top; A.inv_temp = 1.0f / a->temperature;
  A.logits = a->logits; A.ls = a->logits_stride; A.mask = a->mask; A.ms = a->mask_stride;
  A.action = a->action; A.logp = a->logp; A.entropy = a->entropy; A.lse = a->lse;
  A.top_logp = a->top_logp; A.top_action = a->top_action;
  A.rec = (float *)a->workspace;
  A.splits = 1;
  A.part = a->a;
  return A;
}

// Rows of up to LP_ROW_MAX logits live in a wave's registers.  Longer rows take a workgroup each, or several where there are too few
// rows to fill the chip (a part keeps at least LP_MIN_PART logits, below which the join costs more than it gives).
static constexpr int LP_ROW_MAX = 1024, LP_NT = 256, LP_MIN_PART = 4096, LP_FILL = 1024;
static int lp_splits(int n, int a) {
  if (a <= LP_ROW_MAX) return 1;
  const int want = (LP_FILL + n - 1) / n, most = (a + LP_MIN_PART - 1) / LP_MIN_PART;
  return want < most ? want : most;
}
// columns per part: whole accesses of 8, so that a part starts as well aligned as its row
static int lp_part(int a, int splits) { return ((a + splits - 1) / splits + 7) / 8 * 8; }

template <typename T>
static int lp_launch(lp_args A, hipStream_t st) {
  if (A.a <= LP_ROW_MAX) {
#define LP_GO(G, E)                                                                       \
  do {                                                                                    \
    lp_rows_kernel<T, G, E><<<(unsigned)(((long long)A.n * G + 255) / 256), 256, 0, st>>>(A); \
    return pqn_check_launch("pqn_action_logprobs");                                       \
  } while (0)
    if (A.a <= 8) LP_GO(8, 1);
    if (A.a <= 16) LP_GO(8, 2);
    if (A.a <= 32) LP_GO(16, 2);
    if (A.a <= 64) LP_GO(32, 2);
    if (A.a <= 128) LP_GO(64, 2);
    if (A.a <= 256) LP_GO(64, 4);
    if (A.a <= 512) LP_GO(64, 8);
    LP_GO(64, 16);
#undef LP_GO
  }
  A.splits = lp_splits(A.n, A.a);
  A.part = lp_part(A.a, A.splits);
  A.splits = (A.a + A.part - 1) / A.part;
  constexpr int VW = 16 / (int)sizeof(T);
  const bool vec = ((uintptr_t)A.logits & 15) == 0 && A.ls % VW == 0;
  const unsigned grid = (unsigned)((long long)A.n * A.splits);
  if (vec) lp_long_kernel<T, LP_NT, VW><<<grid, LP_NT, 0, st>>>(A);
  else lp_long_kernel<T, LP_NT, 1><<<grid, LP_NT, 0, st>>>(A);
  const int rc = pqn_check_launch("pqn_action_logprobs");
  if (rc != PQN_OK || A.splits == 1) return rc;
  lp_join_kernel<T><<<(unsigned)A.n, 64, 0, st>>>(A);
  return pqn_check_launch("pqn_action_logprobs");
}

extern "C" int64_t pqn_action_logprobs_workspace_bytes(int32_t n, int32_t a) {
  if (n <= 0 || a <= 0 || a > (1 << 30)) return 0;
  const int s = lp_splits(n, a);
  return s > 1 ? (int64_t)n * s * LP_REC * 4 : 0;
}

extern "C" int pqn_action_logprobs(const pqn_action_logprobs_t *a, void *stream) {
  const int rc = lp_check(a, "pqn_action_logprobs");
  if (rc != PQN_OK) return rc;
  if (a->n == 0) return PQN_OK;
  PQN_REQUIRE(a->logp, "pqn_action_logprobs: NULL logp");
  PQN_REQUIRE(a->top == 0 || (a->top_logp && a->top_action), "pqn_action_logprobs: NULL top_logp or top_action with top > 0");
  PQN_REQUIRE(a->workspace || pqn_action_logprobs_workspace_bytes(a->n, a->a) == 0, "pqn_action_logprobs: NULL workspace");
  PQN_REQUIRE(((uintptr_t)a->workspace & 7) == 0, "pqn_action_logprobs: the workspace must be 8-byte aligned");
  return pqn_with_dtype(a->dtype, [&](auto t) { return lp_launch<decltype(t)>(lp_fill(a), (hipStream_t)stream); });
}

extern "C" int pqn_action_logprobs_grad(const pqn_action_logprobs_t *a, void *stream) {
  const int rc = lp_check(a, "pqn_action_logprobs_grad");
  if (rc != PQN_OK) return rc;
  if (a->n == 0) return PQN_OK;
  PQN_REQUIRE(a->dlogits, "pqn_action_logprobs_grad: NULL dlogits");
  PQN_REQUIRE(a->dlogp || a->dentropy || a->dlse, "pqn_action_logprobs_grad: dlogp, dentropy and dlse are all NULL");
  return pqn_with_dtype(a->dtype, [&](auto t) {
    typedef decltype(t) T;
    constexpr int VW = 16 / (int)sizeof(T);
    lp_grad_args G = {lp_fill(a), a->dlogp, a->dentropy, a->dlse, a->dlogits, 0};
    // 16-B accesses where the rows keep their alignment; below one workgroup's span of columns the rows are packed end to end
    const bool vec = a->a % VW == 0 && a->logits_stride % VW == 0 && (((uintptr_t)a->logits | (uintptr_t)a->dlogits) & 15) == 0;
    const int w = vec ? VW : 1, span = 256 * w;
    G.blocks = a->a >= span ? (a->a + span - 1) / span : 0;
    const long long grid = G.blocks ? (long long)a->n * G.blocks : ((long long)a->n * a->a / w + 255) / 256;
    PQN_REQUIRE(grid < (1ll << 31), "pqn_action_logprobs_grad: %d x %d logits are more than one launch covers", a->n, a->a);
    if (vec) lp_grad_kernel<T, VW><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(G);
    else lp_grad_kernel<T, 1><<<(unsigned)grid, 256, 0, (hipStream_t)stream>>>(G);
    return pqn_check_launch("pqn_action_logprobs_grad");
  });
}
