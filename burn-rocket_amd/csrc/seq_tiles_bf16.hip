// seq_tiles.hpp for bf16.
#include "seq_tiles.hpp"

hipError_t rk_launch_seq_tiles_bf16(const SeqAttnArgs &a, bool paged, hipStream_t st) {
  return paged ? launch_seq_tiles_d<RK_DTYPE_BF16, true, false>(a, st)
               : launch_seq_tiles_d<RK_DTYPE_BF16, false, false>(a, st);
}
