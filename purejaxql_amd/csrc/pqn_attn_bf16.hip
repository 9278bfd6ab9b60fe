// pqn_attn_bf16.hip -- the chunked scan of pqn_attn.hip on bf16 tensors.  Chunks of 32 steps: 27 KB of LDS at the widest heads, two waves
// a SIMD by registers.
#include "pqn_attn_chunk.h"

int da_launch_chunk_bf16(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st) {
  return da_launch_chunk<pqn_bf16, 32>(A, X, passes, state, st);
}
