// Attention of a batch of sequences: which kernel takes a list of items.
#include "../../include/burn_rocket_amd.h"
#include "kernels.hpp"

size_t rk_seq_slot_bytes(int head_dim, SeqKind kind) {
  const size_t ndb = (head_dim + 15) / 16, qb = head_dim <= 128 ? 2 : 1;
  return kind == SEQ_ROWS ? ndb * 1024 + 128 : 4 * (1 + ndb * qb) * 1024;
}

hipError_t rk_launch_attention_seqs(const SeqAttnArgs &a, int longest_row, bool paged, int dtype, hipStream_t st) {
  const bool f16 = dtype == RK_DTYPE_F16;
  if (!f16 && dtype != RK_DTYPE_BF16) return hipErrorInvalidValue;
  if (a.rows.n && (!a.tiles.n || !seq_one_launch(a.head_dim))) {
    const bool brief = longest_row <= 4 * SEQ_ROWS_CHUNK;
    const hipError_t e = f16 ? rk_launch_seq_rows_f16(a, brief, paged, st) : rk_launch_seq_rows_bf16(a, brief, paged, st);
    if (e != hipSuccess) return e;
  }
  if (!a.tiles.n) return hipSuccess;
  SeqAttnArgs t = a;
  if (!seq_one_launch(a.head_dim)) t.rows.n = 0;
  if (a.softcap != 0.f) return f16 ? rk_launch_seq_tiles_f16_cap(t, paged, st) : rk_launch_seq_tiles_bf16_cap(t, paged, st);
  return f16 ? rk_launch_seq_tiles_f16(t, paged, st) : rk_launch_seq_tiles_bf16(t, paged, st);
}
