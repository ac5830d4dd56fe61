// seq_rows.hpp for bf16.
#include "seq_rows.hpp"

hipError_t rk_launch_seq_rows_bf16(const SeqAttnArgs &a, bool brief, bool paged, hipStream_t st) {
  return paged ? launch_seq_rows_d<RK_DTYPE_BF16, true>(a, brief, st)
               : launch_seq_rows_d<RK_DTYPE_BF16, false>(a, brief, st);
}
