// pqn_attn_f32.hip -- the chunked scan of pqn_attn.hip on f32 tensors.  Chunks of 32 steps: three tiles of 32 x 128 floats and the
// weights between their steps are 55 KB of LDS at the widest heads; registers (two waves a SIMD) allow two workgroups to a CU.
#include "pqn_attn_chunk.h"

int da_launch_chunk_f32(const da_args &A, const da_split &X, int passes, bool state, hipStream_t st) {
  return da_launch_chunk<float, 32>(A, X, passes, state, st);
}
