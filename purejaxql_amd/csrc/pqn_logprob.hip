// pqn_logprob.hip -- log probabilities of taken actions under the softmax of their logits, with the entropy, the logsumexp and the
// top alternatives, and the gradient (pqn_action_logprobs, pqn_action_logprobs_grad in include/pqn_hotpath.h).
//
//   x_j = logit_j / temperature where allowed      lse = log sum e^x      logp = x_a - lse      H = -sum p log p = lse - sum p x
//
// One pass over the logits: every lane keeps the running maximum m of what it has seen, s = sum e^(x - m) and t = sum (x - m) e^(x - m),
// so H = log s - t / s without a second look (t is shifted like s when m grows: t' = e^(m - m') (t + (m - m') s)).  Powers of two
// throughout: x is scaled by log2 e / temperature once and v_exp_f32 taken as it is.  The K best logits come out of the same pass: a key
// is the logit's order-preserving bits above the complement of its index, so keys are distinct and ties go to the lowest index whatever
// the order of the work.
//
// Bound: HBM for many logits (about 9 vector operations and one v_exp_f32 a logit, below the time its bytes take), latency for few.
// Measured, forward / gradient in turn (the kernels' least under a trace): 4096 x 32000 bf16, five alternatives 74 / 81 + 4 us (52 and 103 by
// their bytes at 5.08 TB/s: part of the gradient's reads come from the last-level cache); 131072 x 17 f32 with masks and three alternatives
// 8.5 / 7.7 us (vector work of joining 17 logits over lanes); 8 x 100003 bf16, eight alternatives, 7.6 us and 5.8 us for joining 25 parts a
// row (latency).
#include <type_traits>

#include "pqn_vec.h"

typedef unsigned long long u64;
static constexpr int LP_MAX_TOP = PQN_LOGPROB_MAX_TOP;

struct lp_args {
  int n, a, top;
  float inv_temp, scale;             // 1 / temperature, log2 e / temperature
  const void *logits;
  long long ls;                      // row stride of the logits in elements
  const uint8_t *mask;
  long long ms;                      // row stride of the mask
  const int32_t *action;
  float *logp, *entropy, *lse, *top_logp;
  int32_t *top_action;
  // few rows: a row is cut into `splits` parts of `part` columns, one workgroup each, joined by lp_join_kernel
  int splits, part;
  float *rec;                        // [n][splits][4 + 2 * LP_MAX_TOP] words: m, s, t, - | keys
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
// the best key of a group: the upper halves first, the lower ones among their best
template <int G>
PQN_D u64 lp_group_max(u64 k) {
  const uint32_t hi = (uint32_t)(k >> 32);
  if constexpr (G == 64) {
    const uint32_t best = pqn_wave_max(hi);
    return ((u64)best << 32) | pqn_wave_max(hi == best ? (uint32_t)k : 0u);
  } else {
    const uint32_t best = pqn_group_max<G>(hi);
    return ((u64)best << 32) | pqn_group_max<G>(hi == best ? (uint32_t)k : 0u);
  }
}

// (m, s, t) of a set of logits: m the largest, s = sum 2^z, t = sum z 2^z with z = (logit - m) log2 e / temperature -- the difference
// first: a type's lowest value times log2 e is no float.  Empty: m = -inf, s = t = 0.  A NaN or +inf among them leaves s NaN.
struct LpSum {
  float m, s, t;
};
static constexpr float LP_LOG2E = 1.44269504f, LP_LN2 = 0.693147181f;
PQN_D float lp_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// the sums seen from a larger maximum; 2^-1000 is 0, and so is its share of t
PQN_D void lp_shift(LpSum &v, float m, float scale) {
  const float d = v.m == m ? 0.f : fmaxf((v.m - m) * scale, -1000.f), e = lp_exp2(d);   // equal: no shift, which keeps inf - inf out
  v.t = e * fmaf(d, v.s, v.t);
  v.s *= e;
  v.m = m;
}
PQN_D LpSum lp_join(LpSum a, LpSum b, float scale) {
  const float m = fmaxf(a.m, b.m);
  lp_shift(a, m, scale);
  lp_shift(b, m, scale);
  return {m, a.s + b.s, a.t + b.t};
}
// one more logit, none of them above m
PQN_D void lp_add(LpSum &v, float x, float scale) {
  const float z = (x - v.m) * scale, q = lp_exp2(z);
  v.s += q;
  v.t = fmaf(fmaxf(z, -1000.f), q, v.t);
}
template <int G>
PQN_D LpSum lp_group_join(LpSum v, float scale) {
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1) {
    LpSum o = {__shfl_xor(v.m, d, 64), __shfl_xor(v.s, d, 64), __shfl_xor(v.t, d, 64)};
    // lanes d apart join the same two parts in the same order: bit-identical in every lane
    v = (threadIdx.x & d) ? lp_join(o, v, scale) : lp_join(v, o, scale);
  }
  return v;
}

// what a row's sums say
struct LpRow {
  float lse, entropy, m, log_s;      // lse = m / temperature + log_s
};
PQN_D LpRow lp_row(const LpSum &v, float inv_temp) {
  LpRow r = {NAN, NAN, v.m, 0.f};
  if (v.s != v.s) return r;
  if (!(v.s > 0.f)) r.lse = -INFINITY, r.entropy = 0.f;          // nothing allowed
  else {
    const float l = log2f(v.s);
    r.log_s = LP_LN2 * l;
    r.lse = fmaf(v.m, inv_temp, r.log_s);
    r.entropy = fmaxf(LP_LN2 * (l - v.t / v.s), 0.f);
  }
  return r;
}
template <typename T>
PQN_D float lp_logit(const lp_args &A, long long row, int j) {   // -inf where not allowed
  if (A.mask && !A.mask[row * A.ms + j]) return -INFINITY;
  return pqn_to_f32(((const T *)A.logits)[row * A.ls + j]);
}
// from the difference to the largest logit: logit / temperature and lse may be beyond the largest float, or large and nearly equal
PQN_D float lp_logp(float logit, const LpRow &r, float inv_temp) {
  return (r.lse != r.lse) ? NAN : logit > -INFINITY ? fmaf(logit - r.m, inv_temp, -r.log_s) : -INFINITY;
}
template <typename T>
PQN_D void lp_write_row(const lp_args &A, long long row, const LpRow &r) {
  A.lse[row] = r.lse;
  A.entropy[row] = r.entropy;
  const int act = A.action[row];
  // an id outside 0 .. a-1: no action, nothing is read
  A.logp[row] = act >= 0 && act < A.a ? lp_logp(lp_logit<T>(A, row, act), r, A.inv_temp) : 0.f;
}
// a row over G lanes, element e * G + lane at e: every request first, then the choices
template <typename T, int G, int E>
PQN_D void lp_row_load(const lp_args &A, long long row, int lane, float (&x)[E]) {
  const T *p = (const T *)A.logits + row * A.ls;
  T raw[E];
  uint8_t on[E];
#pragma unroll
  for (int e = 0; e < E; ++e) raw[e] = p[min(e * G + lane, A.a - 1)];
  if (A.mask) {
    const uint8_t *mk = A.mask + row * A.ms;
#pragma unroll
    for (int e = 0; e < E; ++e) on[e] = mk[min(e * G + lane, A.a - 1)];
  } else
#pragma unroll
    for (int e = 0; e < E; ++e) on[e] = 1;
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = (on[e] != 0) & (e * G + lane < A.a) ? pqn_to_f32(raw[e]) : -INFINITY;
}
PQN_D void lp_write_top(const lp_args &A, long long row, int i, u64 key, const LpRow &r) {
  A.top_action[row * A.top + i] = key ? (int32_t)~(uint32_t)key : -1;
  A.top_logp[row * A.top + i] = key ? lp_logp(lp_unorder((uint32_t)(key >> 32)), r, A.inv_temp) : -INFINITY;
}

// A row in the registers of G lanes, E logits each (a <= G * E): 64 / G rows per wave, no shared memory.
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void lp_rows_kernel(lp_args A) {
  const int lane = threadIdx.x & (G - 1);
  const long long row0 = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
  const bool live = row0 < A.n;                    // rows behind the last one shuffle along with a copy of it
  const long long row = live ? row0 : A.n - 1;
  const int act = A.action[row];
  float x[E];
  lp_row_load<T, G, E>(A, row, lane, x);
  LpSum v = {-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) v.m = fmaxf(v.m, x[e]);
  v.m = pqn_group_fmax<G>(v.m);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (!(x[e] == -INFINITY)) lp_add(v, x[e], A.scale);
  v.s = pqn_group_sum<G>(v.s);
  v.t = pqn_group_sum<G>(v.t);
  const LpRow r = lp_row(v, A.inv_temp);
  // the taken action's logit is in the register of one of the lanes; an id outside the row is in none
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (live && e * G + lane == act && act < A.a) A.logp[row] = lp_logp(x[e], r, A.inv_temp);
  if (live && lane == 0) {
    A.lse[row] = r.lse;
    A.entropy[row] = r.entropy;
    if (act < 0 || act >= A.a) A.logp[row] = 0.f;
  }
  if (A.top > 0) {
    u64 key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = lp_key(x[e], e * G + lane);
    for (int i = 0; i < A.top; ++i) {
      u64 best = key[0];
#pragma unroll
      for (int e = 1; e < E; ++e) best = lp_max(best, key[e]);
      best = lp_group_max<G>(best);
      if (live && lane == 0) lp_write_top(A, row, i, best, r);
#pragma unroll
      for (int e = 0; e < E; ++e) key[e] = key[e] == best ? 0ull : key[e];
    }
  }
}

// The K best keys of a wave, key i in lane i; lanes from K on hold nothing
PQN_D void lp_insert(u64 &list, u64 key, int top) {
  const int lane = threadIdx.x & 63;
  const int at = __popcll(__ballot(list > key));               // keys above the new one, all in the first lanes
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)list, 0x138, 0xf, 0xf, true);           // wave_shr:1
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(list >> 32), 0x138, 0xf, 0xf, true);
  list = lane < at ? list : lane == at ? key : ((u64)hi << 32) | lo;
  if (lane >= top) list = 0ull;
}
// the wave's best of its lanes' VW logits, by order bits o (0 = none) and index j0 + e, and out of the running with it
template <int VW>
PQN_D u64 lp_take(uint32_t (&o)[VW], uint32_t j0) {
  uint32_t mine = o[0];
#pragma unroll
  for (int e = 1; e < VW; ++e) mine = max(mine, o[e]);
  const uint32_t best = pqn_wave_max(mine);
  uint32_t at = ~0u;
#pragma unroll
  for (int e = VW - 1; e >= 0; --e) at = o[e] == best ? j0 + e : at;
  at = pqn_wave_min(at);
#pragma unroll
  for (int e = 0; e < VW; ++e) o[e] = j0 + e == at ? 0u : o[e];
  return best ? ((u64)best << 32) | (uint32_t)~at : 0ull;
}

// A workgroup per row (or part of a row), which it holds in registers: N accesses of VW logits a thread, all requested at once; the
// row's first and last logits that fill no whole access one to a thread.  Three looks at the registers: the largest of every access,
// the sums under the thread's own maximum, and the alternatives.  For those, a bar: the K-th largest of a wave's 64 thread maxima is
// no larger than the wave's K-th logit, so the largest of the waves' bars sorts out all but some K logits; their keys are collected in
// LDS, in whatever order (they are distinct), and the first wave takes the K best.  Where LP_CAND do not hold them (many equal logits),
// they go through a list of K keys per wave instead, an access of the wave at a time.
static constexpr int LP_CAND = 256;
typedef uint32_t lp_u32x4 __attribute__((ext_vector_type(4)));
// logit e of an access, kept packed
template <typename T>
PQN_D float lp_get(const lp_u32x4 &r, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r[e]);
  else if constexpr (std::is_same<T, pqn_bf16>::value) return __uint_as_float(e & 1 ? r[e >> 1] & 0xffff0000u : r[e >> 1] << 16);
  else return (float)__builtin_bit_cast(T, (uint16_t)(e & 1 ? r[e >> 1] >> 16 : r[e >> 1]));
}
// ... and put to -inf
template <typename T>
PQN_D void lp_forbid(lp_u32x4 &r, int e, bool no) {
  if constexpr (sizeof(T) == 4) r[e] = no ? 0xff800000u : r[e];
  else {
    const uint32_t inf = std::is_same<T, pqn_bf16>::value ? 0xff80u : 0xfc00u, u = r[e >> 1];
    r[e >> 1] = no ? (e & 1 ? (u & 0xffffu) | inf << 16 : (u & 0xffff0000u) | inf) : u;
  }
}

template <typename T, int NT, int N>
__global__ __launch_bounds__(NT, 4) void lp_long_kernel(lp_args A) {
  constexpr int NW = NT / 64, VW = 16 / (int)sizeof(T);
  static_assert(NW * LP_MAX_TOP <= LP_CAND, "the waves' lists fit");
  __shared__ u64 keys[LP_CAND];
  __shared__ int found;
  __shared__ float sums[NW][3];
  __shared__ uint32_t bar[NW];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long row = blockIdx.x / A.splits;
  const int part = blockIdx.x % A.splits;
  const int c0 = part * A.part, c1 = min(A.a, c0 + A.part);
  const T *p = (const T *)A.logits + row * A.ls;
  const uint8_t *mk = A.mask ? A.mask + row * A.ms : nullptr;
  const int head = min(c1 - c0, (int)((16 - ((uintptr_t)(p + c0) & 15)) & 15) / (int)sizeof(T));
  const int body = c0 + head, end = body + (c1 - body) / VW * VW, rest = head + (c1 - end);
  auto first = [&](int i) { return body + (i * NT + (int)threadIdx.x) * VW; };
  lp_u32x4 r[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r[i] = lp_u32x4{0u, 0u, 0u, 0u};
    if (body + i * NT * VW < end) r[i] = *(const lp_u32x4 *)(p + (first(i) < end ? first(i) : body));
  }
  const bool has_rest = (int)threadIdx.x < rest;
  const int jr = !has_rest ? c0 : (int)threadIdx.x < head ? c0 + threadIdx.x : end + (threadIdx.x - head);
  float xr[1] = {pqn_to_f32(p[jr])};
  xr[0] = has_rest && (!mk || mk[jr] != 0) ? xr[0] : -INFINITY;
  if (mk) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (body + i * NT * VW < end) {
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          const bool no = mk[min(first(i) + e, c1 - 1)] == 0;
          lp_forbid<T>(r[i], e, no);
        }
      }
  }
  float top[N], m = xr[0];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    top[i] = -INFINITY;
    if (body + i * NT * VW < end) {
#pragma unroll
      for (int e = 0; e < VW; ++e) top[i] = fmaxf(top[i], lp_get<T>(r[i], e));
      top[i] = first(i) < end ? top[i] : -INFINITY;
    }
    m = fmaxf(m, top[i]);
  }
  LpSum v = {m, 0.f, 0.f};
  const bool any = m > -INFINITY;
  if (any && has_rest) lp_add(v, xr[0], A.scale);
  v.s += has_rest && xr[0] != xr[0] ? NAN : 0.f;                     // also where there is nothing else
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (body + i * NT * VW < end && first(i) < end) {
      if (any) {
#pragma unroll
        for (int e = 0; e < VW; ++e) lp_add(v, lp_get<T>(r[i], e), A.scale);
      } else {
#pragma unroll
        for (int e = 0; e < VW; ++e) v.s += lp_get<T>(r[i], e) != lp_get<T>(r[i], e) ? NAN : 0.f;
      }
    }
  v = lp_group_join<64>(v, A.scale);
  if (lane == 0) {
    sums[wave][0] = v.m;
    sums[wave][1] = v.s;
    sums[wave][2] = v.t;
  }
  int count = 0;
  bool lists = false;
  if (A.top > 0) {
    uint32_t mine = m > -INFINITY ? lp_order(m) : 0u, least = 0u;
    for (int i = 0; i < A.top; ++i) {
      least = pqn_wave_max(mine);
      const int at = __ffsll(__ballot(mine == least)) - 1;           // one thread of the best
      mine = lane == at ? 0u : mine;
    }
    if (lane == 0) bar[wave] = least;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) least = max(least, bar[w]);
    const float above = lp_unorder(max(least, 1u << 23));            // least = 0: every number (order 2^23 is the lowest float's)
    auto offer = [&](float x, int j) {
      if (x >= above) {                                              // false for NaN
        const int at = atomicAdd(&found, 1);
        if (at < LP_CAND) keys[at] = lp_key(x, j);
      }
    };
    offer(xr[0], jr);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (top[i] >= above) {
#pragma unroll
        for (int e = 0; e < VW; ++e) offer(lp_get<T>(r[i], e), first(i) + e);
      }
    __syncthreads();
    count = found;
  }
  if (count > LP_CAND) {
    u64 list = 0ull;
    uint32_t least = 0u;
#pragma unroll
    for (int w = 0; w < NW; ++w) least = max(least, bar[w]);
    auto look = [&](const auto &x, float best_x, int j) {
      constexpr int W = sizeof(x) / sizeof(float);
      const uint32_t best_o = best_x > -INFINITY ? lp_order(best_x) : 0u;
      if (!__any(best_o >= max(least, 1u))) return;
      uint32_t o[W];
#pragma unroll
      for (int e = 0; e < W; ++e) o[e] = best_o && x[e] > -INFINITY ? lp_order(x[e]) : 0u;
      for (;;) {
        const u64 best = lp_take(o, (uint32_t)j);
        const u64 last = ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(list >> 32), A.top - 1) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)list, A.top - 1);
        if (best <= last || (uint32_t)(best >> 32) < least) break;   // 0 <= last: ends when nothing is left
        lp_insert(list, best, A.top);
      }
    };
    look(xr, xr[0], jr);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (body + i * NT * VW < end) {
        float x[VW];
#pragma unroll
        for (int e = 0; e < VW; ++e) x[e] = lp_get<T>(r[i], e);
        look(x, top[i], first(i));
      }
    if (lane < A.top) keys[wave * A.top + lane] = list;
    count = NW * A.top;
    lists = true;
  }
  __syncthreads();
  if (wave != 0) return;
  v = {sums[0][0], sums[0][1], sums[0][2]};
#pragma unroll
  for (int w = 1; w < NW; ++w) v = lp_join(v, {sums[w][0], sums[w][1], sums[w][2]}, A.scale);
  const LpRow rw = lp_row(v, A.inv_temp);
  float *rec = A.rec + ((size_t)row * A.splits + part) * LP_REC;
  if (lane == 0) {
    if (A.splits == 1) lp_write_row<T>(A, row, rw);
    else {
      rec[0] = v.m;
      rec[1] = v.s;
      rec[2] = v.t;
    }
  }
  auto put = [&](int i, u64 key) {
    if (A.splits == 1) lp_write_top(A, row, i, key, rw);
    else ((u64 *)(rec + 4))[i] = key;
  };
  if (count <= 64 && !lists) {                    // distinct keys, one to a lane: a key's place is the number of those above it
    const u64 mine = lane < count ? keys[lane] : 0ull;
    int place = 0;
    for (int j = 0; j < count; ++j) {
      const u64 other = ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(mine >> 32), j) << 32) |
                        (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, j);
      place += other > mine;
    }
    if (lane >= count) place = lane;              // empty places
    if (place < A.top) put(place, mine);
    return;
  }
  constexpr int ML = LP_CAND / 64;
  u64 mine[ML];
#pragma unroll
  for (int i = 0; i < ML; ++i) mine[i] = i * 64 + lane < count ? keys[i * 64 + lane] : 0ull;
  for (int i = 0; i < A.top; ++i) {
    u64 best = mine[0];
#pragma unroll
    for (int k = 1; k < ML; ++k) best = lp_max(best, mine[k]);
    best = lp_group_max<64>(best);
    if (lane == 0) put(i, best);
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
  for (int i = lane; i < A.splits; i += 64) v = lp_join(v, {rec[i * LP_REC], rec[i * LP_REC + 1], rec[i * LP_REC + 2]}, A.scale);
  v = lp_group_join<64>(v, A.scale);
  const LpRow r = lp_row(v, A.inv_temp);
  if (lane == 0) lp_write_row<T>(A, row, r);
  // the first KEEP keys of a lane stay in its registers: one look at the usual number of parts
  constexpr int KEEP = 8;
  const uint32_t count = A.splits * A.top, per = A.top;
  auto at = [&](uint32_t e) { return ((const u64 *)(rec + (size_t)(e / per) * LP_REC + 4))[e % per]; };
  u64 key[KEEP];
#pragma unroll
  for (int j = 0; j < KEEP; ++j) key[j] = lane + 64u * j < count ? at(lane + 64u * j) : 0ull;
  u64 floor = ~0ull;                        // keys are distinct: the next best is the largest one below the last
  for (int i = 0; i < A.top; ++i) {
    u64 best = 0ull;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) best = key[j] < floor ? lp_max(best, key[j]) : best;
    for (uint32_t e = lane + 64u * KEEP; e < count; e += 64) {
      const u64 k = at(e);
      if (k < floor) best = lp_max(best, k);
    }
    best = lp_group_max<64>(best);
    if (lane == 0) lp_write_top(A, row, i, best, r);
    floor = best;
  }
}

// ---- gradient ------------------------------------------------------------------------------------------------------------
// d/dx_j = dlogp (1[j = action] - p_j) - dentropy p_j (log p_j + H) + dlse p_j, over the temperature.
// log p_j = x_j - lse puts every p_j of a row off by e^(the rounding of lse): nothing beside the sum's own rounding where |lse| <= LP_NEAR
// (2^-24 * 32, a sum over A logits some (64 + A / 64) 2^-24), 28 % for logits / temperature of 4e6.  So rows of larger ones take
// log p_j = (logit_j - m) / temperature - log_s from the largest logit and the sum of the powers, made again: from registers in narrow
// rows, by reading a wide row a second time.  us, |lse| <= 32 / above (of the forward's lse alone): 4096 x 32000 bf16
// 100 / 154 (97), 60000 x 1100 bf16 85 / 215 (76), 512 x 130000 f32 99 / 235 (97), 8 x 100003 bf16 9 / 22 (9), 60000 x 1000 f32 82 / 86 (86).
static constexpr float LP_NEAR = 32.f;
struct lp_grad_args {
  lp_args A;
  const float *dlogp, *dentropy, *dlse;
  void *dlogits;                     // [n][a]
  int blocks, far;                   // wide rows: workgroups per row; those of them that work on a row beyond LP_NEAR
};
// the largest of a set of logits and s = sum 2^((logit - m) log2 e / temperature); empty: -inf and 0
struct LpPowers {
  float m, s;
};
// A logsumexp beyond the largest float (or of nothing) has no gradient of its own: a row that is given one has none at all.  logp and entropy
// are finite there, and so are their gradients.
PQN_D bool lp_none(float lse, float dl) { return fabsf(lse) == INFINITY && dl != 0.f; }
PQN_D bool lp_again(float lse, float dl) { return fabsf(lse) > LP_NEAR && !lp_none(lse, dl); }   // false for NaN: so is every gradient
PQN_D float lp_rescale(float m, float to, float scale) { return m == to ? 1.f : lp_exp2((m - to) * scale); }
struct LpGrad {                      // a row's scalars
  float m, base, h, dlp, dh, dl, inv_temp;      // log p = (logit - m) / temperature - base
  int act;
  bool none, again;
  template <typename T>
  PQN_D void open(const lp_grad_args &G, long long row) {
    const lp_args &A = G.A;
    m = 0.f;
    base = A.lse[row];
    h = A.entropy[row];
    act = A.action[row];
    dlp = G.dlogp ? G.dlogp[row] : 0.f;
    dh = G.dentropy ? G.dentropy[row] : 0.f;
    dl = G.dlse ? G.dlse[row] : 0.f;
    none = lp_none(base, dl);
    again = lp_again(base, dl);
    inv_temp = A.inv_temp;
    // an id outside the row, or an action that is not allowed, has a constant log probability
    if (act < 0 || act >= A.a || lp_logit<T>(A, row, act) == -INFINITY) dlp = 0.f;
  }
  PQN_D void sums(LpPowers v) {
    m = v.m;
    base = LP_LN2 * log2f(v.s);
  }
  PQN_D float at(float x, int j) const {               // x: the logit, -inf where not allowed
    const float lp = fmaf(x - m, inv_temp, -base), q = lp_exp2(lp * LP_LOG2E);
    const float c = dl - dlp - dh * (fmaxf(lp, -1000.f) + h);          // q is 0 below
    const float g = ((act == j ? dlp : 0.f) + q * c) * inv_temp;
    return x == -INFINITY || none ? 0.f : g;
  }
};
// narrow rows: the lanes as in lp_rows_kernel
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void lp_grad_rows_kernel(lp_grad_args P) {
  const lp_args &A = P.A;
  const int lane = threadIdx.x & (G - 1);
  const long long row0 = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
  const bool live = row0 < A.n;                    // rows behind the last one go along with a copy of it
  const long long row = live ? row0 : A.n - 1;
  LpGrad R;
  R.open<T>(P, row);
  T *o = (T *)P.dlogits + row * A.a;
  float x[E];
  lp_row_load<T, G, E>(A, row, lane, x);
  if (__any(R.again)) {                            // whole waves, for the exchanges
    LpPowers v = {-INFINITY, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) v.m = fmaxf(v.m, x[e]);
    v.m = pqn_group_fmax<G>(v.m);
#pragma unroll
    for (int e = 0; e < E; ++e) v.s += x[e] == -INFINITY ? 0.f : lp_exp2((x[e] - v.m) * A.scale);
    v.s = pqn_group_sum<G>(v.s);
    if (R.again) R.sums(v);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = e * G + lane;
    if (live && j < A.a) o[j] = (T)R.at(x[e], j);
  }
}
// A wide row's columns: whole accesses of the logits lie on 16 bytes, from `head` to `end`; the first and last elements go one to a thread.
// The gradients' accesses start anywhere.
template <typename T>
struct LpWide {
  static constexpr int VW = 16 / (int)sizeof(T);
  const T *x;
  const uint8_t *mk;
  T *o;
  int head, end, jr;
  bool has_rest;
  float xr;
  PQN_D LpWide(const lp_grad_args &P, long long row) {
    const lp_args &A = P.A;
    x = (const T *)A.logits + row * A.ls;
    mk = A.mask ? A.mask + row * A.ms : nullptr;
    o = (T *)P.dlogits + row * A.a;
    head = min(A.a, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
    end = head + (A.a - head) / VW * VW;
    has_rest = (int)threadIdx.x < head + (A.a - end);
    jr = (int)threadIdx.x < head ? threadIdx.x : end + (threadIdx.x - head);
    xr = !has_rest || (mk && !mk[jr]) ? -INFINITY : pqn_to_f32(x[jr]);
  }
  // the sums of the whole row, the same in every thread; eight accesses requested together
  PQN_D LpPowers sums(float scale, LpPowers *part) const {
    constexpr int BATCH = 8;
    LpPowers v = {fmaxf(xr, -INFINITY), 0.f};        // not a NaN
    v.s = xr == -INFINITY ? 0.f : lp_exp2((xr - v.m) * scale);
    for (int j0 = head; j0 < end; j0 += 256 * VW * BATCH) {
      lp_u32x4 r[BATCH];
      auto at = [&](int i) { return j0 + (i * 256 + (int)threadIdx.x) * VW; };
      auto some = [&](int i) { return j0 + i * 256 * VW < end; };
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        r[i] = lp_u32x4{0u, 0u, 0u, 0u};
        if (some(i)) r[i] = *(const lp_u32x4 *)(x + (at(i) < end ? at(i) : head));
      }
      float top = v.m;
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (!some(i)) continue;
#pragma unroll
        for (int e = 0; e < VW; ++e) {
          if (mk) lp_forbid<T>(r[i], e, mk[min(at(i) + e, end - 1)] == 0);
          lp_forbid<T>(r[i], e, at(i) >= end);
          top = fmaxf(top, lp_get<T>(r[i], e));
        }
      }
      v.s *= lp_rescale(v.m, top, scale);
      v.m = top;
      const float m = top == -INFINITY ? 0.f : top;  // nothing yet: 2^-inf, or NaN
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (!some(i)) continue;
#pragma unroll
        for (int e = 0; e < VW; ++e) v.s += lp_exp2((lp_get<T>(r[i], e) - m) * scale);
      }
    }
    const float m = pqn_group_fmax<64>(v.m), s = pqn_wave_sum(v.s * lp_rescale(v.m, m, scale));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = {m, s};
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) v.m = fmaxf(v.m, part[w].m);
    v.s = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) v.s += part[w].s * lp_rescale(part[w].m, v.m, scale);
    return v;
  }
  PQN_D void rest(const LpGrad &R) const {
    if (has_rest) o[jr] = (T)R.at(xr, jr);
  }
  // span b, SPAN accesses a thread.  Each is requested where it is used: the four at once measured slower (16000 x 4000 bf16 52 us against 45,
  // 8192 x 8000 f32 with a mask 149 against 130).
  static constexpr int SPAN = 4;
  PQN_D void write(const LpGrad &R, int b) const {
#pragma unroll
    for (int i = 0; i < SPAN; ++i) {
      const int j = head + ((b * SPAN + i) * 256 + (int)threadIdx.x) * VW;
      if (j >= end) break;
      float v[VW];
      pqn_load<T, VW>(v, x + j);
      pqn_loose<T, VW> g;
#pragma unroll
      for (int e = 0; e < VW; ++e) g.v[e] = (T)R.at(mk && !mk[j + e] ? -INFINITY : v[e], j + e);
      *(pqn_loose<T, VW> *)(o + j) = g;
    }
  }
};
// `blocks` workgroups to a row, a span each.  Rows beyond LP_NEAR are left to lp_grad_far_kernel, or (ALONE) `far` of the workgroups make the
// row's sums, each for itself, and take the spans in turn.
template <typename T, bool ALONE>
__global__ __launch_bounds__(256) void lp_grad_kernel(lp_grad_args P) {
  const long long row = blockIdx.x / P.blocks;
  const int block = blockIdx.x % P.blocks;
  LpGrad R;
  R.open<T>(P, row);
  if (R.again && !(ALONE && block < P.far)) return;           // the workgroup's row: the same in every thread
  const LpWide<T> W(P, row);
  int step = P.blocks;
  if constexpr (ALONE) {
    __shared__ LpPowers part[4];
    if (R.again) {
      R.sums(W.sums(P.A.scale, part));
      step = P.far;
    }
  }
  if (block == 0) W.rest(R);
  for (int b = block; b < P.blocks; b += step) W.write(R, b);
}
// rows beyond LP_NEAR, a workgroup to each: it looks for them among every gridDim.x-th row, 64 at a time
template <typename T>
__global__ __launch_bounds__(256) void lp_grad_far_kernel(lp_grad_args P) {
  __shared__ LpPowers part[4];
  const int lane = threadIdx.x & 63;
  for (long long row0 = blockIdx.x; row0 < P.A.n; row0 += 64ll * gridDim.x) {
    const long long mine = row0 + (long long)lane * gridDim.x;
    const bool in = mine < P.A.n;
    unsigned long long todo = __ballot(in && lp_again(P.A.lse[in ? mine : 0], P.dlse ? P.dlse[in ? mine : 0] : 0.f));   // the same in every wave
    while (todo) {
      const long long row = row0 + (long long)(__ffsll(todo) - 1) * gridDim.x;
      todo &= todo - 1;
      LpGrad R;
      R.open<T>(P, row);
      const LpWide<T> W(P, row);
      R.sums(W.sums(P.A.scale, part));
      W.rest(R);
      for (int b = 0; b < P.blocks; ++b) W.write(R, b);
      __syncthreads();                             // `part` has been read
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
static float lp_scale(float temperature) { return (float)(1.4426950408889634 / (double)temperature); }
static int lp_check(const pqn_action_logprobs_t *a, const char *who) {
  PQN_REQUIRE(a, "%s: NULL argument block", who);
  PQN_REQUIRE(pqn_dtype_known(a->dtype), "%s: unknown dtype %d", who, a->dtype);
  PQN_REQUIRE(a->n >= 0 && a->a > 0, "%s: n must be >= 0 and a > 0 (n=%d a=%d)", who, a->n, a->a);
  PQN_REQUIRE(a->a <= (1 << 30), "%s: up to 2^30 columns (a=%d)", who, a->a);
  PQN_REQUIRE(a->top >= 0 && a->top <= LP_MAX_TOP && a->top <= a->a, "%s: top must be in 0 .. min(a, %d) (top=%d a=%d)", who, LP_MAX_TOP, a->top, a->a);
  PQN_REQUIRE(a->temperature > 0.f && a->temperature < INFINITY && lp_scale(a->temperature) < INFINITY,
              "%s: temperature must be positive, finite and at least 4.24e-39 (log2 e over it is a float)", who);
  if (a->n > 0) PQN_REQUIRE(a->logits && a->action && a->lse && a->entropy, "%s: NULL logits, action, lse or entropy", who);
  return PQN_OK;
}
static lp_args lp_fill(const pqn_action_logprobs_t *a) {
  lp_args A = {};
  A.n = a->n; A.a = a->a; A.top = a->top; A.inv_temp = 1.0f / a->temperature;
  A.scale = lp_scale(a->temperature);
  A.logits = a->logits; A.ls = a->logits_stride; A.mask = a->mask; A.ms = a->mask_stride;
  A.action = a->action; A.logp = a->logp; A.entropy = a->entropy; A.lse = a->lse;
  A.top_logp = a->top_logp; A.top_action = a->top_action;
  A.rec = (float *)a->workspace;
  A.splits = 1;
  A.part = a->a;
  return A;
}

// Rows of up to LP_ROW_MAX logits live in a wave's registers (lp_rows_kernel or lp_long_kernel), longer ones in a workgroup's, up to 16
// accesses a thread (32768 16-bit or 16384 f32 logits); beyond that, or where there are too few rows to fill the chip, a row is cut (a
// part keeps at least LP_MIN_PART logits, below which the join costs more than it gives).
static constexpr int LP_ROW_MAX = 1024, LP_NT = 256, LP_MIN_PART = 4096, LP_FILL = 1024, LP_MOST = 16;
static int lp_splits(int n, int a, int vw) {
  if (a <= LP_ROW_MAX) return 1;
  const int want = (LP_FILL + n - 1) / n, most = (a + LP_MIN_PART - 1) / LP_MIN_PART, cap = LP_NT * vw * LP_MOST;
  const int least = (a + cap - 1) / cap, s = want < most ? want : most;
  return s > least ? s : least;
}
// columns per part: whole accesses of 8, so that a part starts as well aligned as its row
static int lp_part(int a, int splits) { return ((a + splits - 1) / splits + 7) / 8 * 8; }

// the lanes and logits per lane that hold a row of up to LP_ROW_MAX logits: rather logits than lanes, whose joining is the most of the
// work (131072 rows of 17 f32 logits with masks and three alternatives: 9.0 us by 4 lanes x 6, 15.3 by 16 x 2; gradient 8.6 and 11.4)
#define LP_ROW_SHAPES(GO, a) \
  if (a <= 8) GO(4, 2);      \
  if (a <= 16) GO(4, 4);     \
  if (a <= 24) GO(4, 6);     \
  if (a <= 32) GO(8, 4);     \
  if (a <= 64) GO(16, 4);    \
  if (a <= 128) GO(32, 4);   \
  if (a <= 256) GO(64, 4);   \
  if (a <= 512) GO(64, 8);   \
  GO(64, 16);

template <typename T>
static int lp_launch(lp_args A, hipStream_t st) {
  // By the rows kernel an alternative costs a search over all of a lane's logits, by the long one only the collected: 60000 x 1000 f32 in
  // us, rows / long, no alternatives 38 / 50, 4 88 / 60, 8 136 / 76; x 300, none 21 / 37, 4 50 / 50; x 500, 16 128 / 76.
  if (A.a <= 256 || (A.a <= 512 && A.top <= 3) || (A.a <= LP_ROW_MAX && A.top <= 1)) {
#define LP_GO(G, E)                                                                           \
  do {                                                                                        \
    PQN_REQUIRE(pqn_one_launch(((long long)A.n * G + 255) / 256, 256),                        \
                "pqn_action_logprobs: %d x %d logits are more than one launch covers", A.n, A.a); \
    lp_rows_kernel<T, G, E><<<(unsigned)(((long long)A.n * G + 255) / 256), 256, 0, st>>>(A); \
    return pqn_check_launch("pqn_action_logprobs");                                           \
  } while (0)
    LP_ROW_SHAPES(LP_GO, A.a)
#undef LP_GO
  }
  constexpr int VW = 16 / (int)sizeof(T);
  A.splits = lp_splits(A.n, A.a, VW);
  A.part = lp_part(A.a, A.splits);
  A.splits = (A.a + A.part - 1) / A.part;
  const long long grid = (long long)A.n * A.splits;
  PQN_REQUIRE(pqn_one_launch(grid, LP_NT), "pqn_action_logprobs: %d x %d logits are more than one launch covers", A.n, A.a);
  const int each = (A.part + LP_NT * VW - 1) / (LP_NT * VW);
  // few accesses: a wave or two to a row, with less to join.  16000 x 4000 bf16, 8 alternatives, 128 / 256 threads 52 / 69 us; 60000 x
  // 1100, 64 / 256 threads 88 / 195
  const int wave = (A.part + 64 * VW - 1) / (64 * VW);
  if (A.splits == 1 && wave <= 2) lp_long_kernel<T, 64, 2><<<(unsigned)grid, 64, 0, st>>>(A);
  else if (A.splits == 1 && wave <= 4) lp_long_kernel<T, 64, 4><<<(unsigned)grid, 64, 0, st>>>(A);
  else if (A.splits == 1 && wave <= 8) lp_long_kernel<T, 128, 4><<<(unsigned)grid, 128, 0, st>>>(A);
  else if (each <= 1) lp_long_kernel<T, LP_NT, 1><<<(unsigned)grid, LP_NT, 0, st>>>(A);
  else if (each <= 2) lp_long_kernel<T, LP_NT, 2><<<(unsigned)grid, LP_NT, 0, st>>>(A);
  else if (each <= 4) lp_long_kernel<T, LP_NT, 4><<<(unsigned)grid, LP_NT, 0, st>>>(A);
  else lp_long_kernel<T, LP_NT, LP_MOST><<<(unsigned)grid, LP_NT, 0, st>>>(A);
  const int rc = pqn_check_launch("pqn_action_logprobs");
  if (rc != PQN_OK || A.splits == 1) return rc;
  lp_join_kernel<T><<<(unsigned)A.n, 64, 0, st>>>(A);
  return pqn_check_launch("pqn_action_logprobs");
}

template <typename T>
static int lp_launch_grad(lp_grad_args P, hipStream_t st) {
  const lp_args &A = P.A;
  if (A.a <= LP_ROW_MAX) {
#define LP_GO(G, E)                                                                                \
  do {                                                                                             \
    PQN_REQUIRE(pqn_one_launch(((long long)A.n * G + 255) / 256, 256),                             \
                "pqn_action_logprobs_grad: %d x %d logits are more than one launch covers", A.n, A.a); \
    lp_grad_rows_kernel<T, G, E><<<(unsigned)(((long long)A.n * G + 255) / 256), 256, 0, st>>>(P); \
    return pqn_check_launch("pqn_action_logprobs_grad");                                           \
  } while (0)
    LP_ROW_SHAPES(LP_GO, A.a)
#undef LP_GO
  }
  constexpr int span = 256 * LpWide<T>::SPAN * (16 / (int)sizeof(T));
  P.blocks = (A.a + span - 1) / span;
  const long long grid = (long long)A.n * P.blocks;
  PQN_REQUIRE(pqn_one_launch(grid, 256), "pqn_action_logprobs_grad: %d x %d logits are more than one launch covers", A.n, A.a);
  // Few workgroups: rows beyond LP_NEAR in the same launch, several workgroups to each though every one reads all of the row
  if (grid <= LP_FILL) {
    const int far = LP_FILL / A.n;
    P.far = far < 32 ? far : 32;
    lp_grad_kernel<T, true><<<(unsigned)grid, 256, 0, st>>>(P);
    return pqn_check_launch("pqn_action_logprobs_grad");
  }
  lp_grad_kernel<T, false><<<(unsigned)grid, 256, 0, st>>>(P);
  const int rc = pqn_check_launch("pqn_action_logprobs_grad");
  if (rc != PQN_OK) return rc;
  lp_grad_far_kernel<T><<<(unsigned)(A.n < 2048 ? A.n : 2048), 256, 0, st>>>(P);
  return pqn_check_launch("pqn_action_logprobs_grad");
}

extern "C" int64_t pqn_action_logprobs_workspace_bytes(int32_t n, int32_t a) {
  if (n <= 0 || a <= 0 || a > (1 << 30)) return 0;
  const int s = lp_splits(n, a, 4);      // of f32, the most
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
    return lp_launch_grad<decltype(t)>({lp_fill(a), a->dlogp, a->dentropy, a->dlse, a->dlogits, 0, 0}, (hipStream_t)stream);
  });
}
