// Attention of a batch of sequences: which kernel takes a list of items.
#include "../../include/burn_rocket_amd.h"
#include "kernels.hpp"

size_t rk_seq_slot_bytes(int head_dim, SeqKind kind) {
  const size_t ndb = (head_dim + 15) / 16, qb = head_dim <= 128 ? 2 : 1;
  return kind == SEQ_ROWS ? ndb * 1024 + 128 : 4 * (1 + ndb * qb) * 1024;
}

hipError_t rk_launch_attention_seqs(const SeqAttnArgs &a, int n_items, SeqKind kind, int longest, bool paged, int dtype,
                                    hipStream_t st) {
  const bool f16 = dtype == RK_DTYPE_F16;
  if (!f16 && dtype != RK_DTYPE_BF16) return hipErrorInvalidValue;
  if (kind == SEQ_ROWS) {
    const bool brief = longest <= 4 * SEQ_ROWS_CHUNK;
    return f16 ? rk_launch_seq_rows_f16(a, n_items, brief, paged, st) : rk_launch_seq_rows_bf16(a, n_items, brief, paged, st);
  }
  if (a.softcap != 0.f)
    return f16 ? rk_launch_seq_tiles_f16_cap(a, n_items, paged, st) : rk_launch_seq_tiles_bf16_cap(a, n_items, paged, st);
  return f16 ? rk_launch_seq_tiles_f16(a, n_items, paged, st) : rk_launch_seq_tiles_bf16(a, n_items, paged, st);
}
