// seq_tiles.hpp for bf16, softcapped scores.
#include "seq_tiles.hpp"

hipError_t rk_launch_seq_tiles_bf16_cap(const SeqAttnArgs &a, bool paged, hipStream_t st) {
  return paged ? launch_seq_tiles_d<RK_DTYPE_BF16, true, true>(a, st)
               : launch_seq_tiles_d<RK_DTYPE_BF16, false, true>(a, st);
}
