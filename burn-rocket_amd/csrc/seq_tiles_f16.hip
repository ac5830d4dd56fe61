// seq_tiles.hpp for fp16.
#include "seq_tiles.hpp"

hipError_t rk_launch_seq_tiles_f16(const SeqAttnArgs &a, bool paged, hipStream_t st) {
  return paged ? launch_seq_tiles_d<RK_DTYPE_F16, true, false>(a, st)
               : launch_seq_tiles_d<RK_DTYPE_F16, false, false>(a, st);
}
