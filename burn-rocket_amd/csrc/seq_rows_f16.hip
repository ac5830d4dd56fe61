// seq_rows.hpp for fp16.
#include "seq_rows.hpp"

hipError_t rk_launch_seq_rows_f16(const SeqAttnArgs &a, bool brief, bool paged, hipStream_t st) {
  return paged ? launch_seq_rows_d<RK_DTYPE_F16, true>(a, brief, st)
               : launch_seq_rows_d<RK_DTYPE_F16, false>(a, brief, st);
}
