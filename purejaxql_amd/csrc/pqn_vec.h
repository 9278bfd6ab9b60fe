// pqn_vec.h -- typed loads and stores and wave reductions shared by the operators on f32 / bf16 / f16 tensors
// (pqn_attn.hip, pqn_resnorm.hip, pqn_logprob.hip).  Arithmetic is f32; a 16-bit value is rounded once, to nearest even, when stored.
#pragma once
#include "pqn_common.h"

typedef __bf16 pqn_bf16;
typedef _Float16 pqn_f16;

PQN_D float pqn_to_f32(float x) { return x; }
PQN_D float pqn_to_f32(pqn_bf16 x) { return (float)x; }
PQN_D float pqn_to_f32(pqn_f16 x) { return (float)x; }

// W consecutive elements in one access (the caller has checked the alignment of W * sizeof(T) bytes); pqn_loose: of any element's
// alignment, which global memory takes in one access too
template <typename T, int W>
struct pqn_pack {
  T v[W];
} __attribute__((aligned(W * sizeof(T) > 16 ? 16 : W * sizeof(T))));

template <typename T, int W>
struct pqn_loose {
  T v[W];
};

template <typename T, int W>
PQN_D void pqn_load(float *dst, const T *src) {
  const pqn_pack<T, W> p = *(const pqn_pack<T, W> *)src;
#pragma unroll
  for (int i = 0; i < W; ++i) dst[i] = pqn_to_f32(p.v[i]);
}
template <typename T, int W>
PQN_D void pqn_store(T *dst, const float *src) {
  pqn_pack<T, W> p;
#pragma unroll
  for (int i = 0; i < W; ++i) p.v[i] = (T)src[i];
  *(pqn_pack<T, W> *)dst = p;
}

// reductions over the wave, the same in every lane: four DPP steps within the rows of 16 lanes (zeros come in from their ends, neutral
// for the sum and the maximum of unsigned values), two broadcasts across them, lane 63 read back
#define PQN_WAVE_STEPS(OP)                                                                          \
  OP(0x111, 0xf, true) OP(0x112, 0xf, true) OP(0x114, 0xf, true) OP(0x118, 0xf, true) OP(0x142, 0xa, false) OP(0x143, 0xc, false)
PQN_D uint32_t pqn_wave_max(uint32_t x) {
#define PQN_STEP(ctrl, rows, zero) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, zero));
  PQN_WAVE_STEPS(PQN_STEP)
#undef PQN_STEP
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}
PQN_D float pqn_wave_sum(float x) {
#define PQN_STEP(ctrl, rows, zero) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), ctrl, rows, 0xf, zero));
  PQN_WAVE_STEPS(PQN_STEP)
#undef PQN_STEP
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
PQN_D uint32_t pqn_wave_min(uint32_t x) { return ~pqn_wave_max(~x); }

// the same over aligned groups of G lanes (G = 4, 8, 16, 32, 64), in every lane of the group: exchanges within 4, 8 and 16 lanes by DPP (a
// mirrored row of equal halves is the other half), across them by a shuffle
template <int G, typename OP>
PQN_D uint32_t pqn_group_fold(uint32_t x, OP op) {
#define PQN_STEP(ctrl) x = op(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xf, 0xf, true));
  PQN_STEP(0xb1)                         // quad_perm [1, 0, 3, 2]
  PQN_STEP(0x4e)                         // quad_perm [2, 3, 0, 1]
  if constexpr (G >= 8) { PQN_STEP(0x141) }    // row_half_mirror
  if constexpr (G >= 16) { PQN_STEP(0x140) }   // row_mirror
#undef PQN_STEP
#pragma unroll
  for (int d = 16; d < G; d <<= 1) x = op(x, (uint32_t)__shfl_xor((int)x, d, 64));
  return x;
}
template <int G>
PQN_D float pqn_group_sum(float x) {
  return __uint_as_float(pqn_group_fold<G>(__float_as_uint(x), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
template <int G>
PQN_D float pqn_group_fmax(float x) {
  return __uint_as_float(pqn_group_fold<G>(__float_as_uint(x), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int G>
PQN_D uint32_t pqn_group_max(uint32_t x) {
  return pqn_group_fold<G>(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// a launch covers fewer than 2^32 threads along its first axis
inline bool pqn_one_launch(long long blocks, int threads) { return blocks * threads < (1ll << 32); }
inline int pqn_dtype_size(int dtype) { return dtype == PQN_DTYPE_F32 ? 4 : 2; }
inline bool pqn_dtype_known(int dtype) { return dtype == PQN_DTYPE_F32 || dtype == PQN_DTYPE_BF16 || dtype == PQN_DTYPE_F16; }
// f(T{}) with the element type of `dtype` (checked before)
template <typename F>
inline auto pqn_with_dtype(int dtype, F f) {
  return dtype == PQN_DTYPE_F32 ? f(float{}) : dtype == PQN_DTYPE_BF16 ? f(pqn_bf16{}) : f(pqn_f16{});
}
