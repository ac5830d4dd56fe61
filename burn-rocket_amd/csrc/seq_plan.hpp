// Batches of sequences: the lists that the kernels on packed sequences and on a
// paged KV cache read, made and checked on the host.
//
// A sequence of a batch has q_len new tokens, the last of its kv_len keys (packed
// sequences: all of them). Its query rows are the pairs r = q·G + g of new token
// q and head g of a kv head's group of G: consecutive rows are the heads that
// read the same keys, so any group size fills a tile of rows without gaps. An
// item is a tile of rows of one sequence with a range of its keys; each runs once
// for every kv head. A tile whose keys are split between several items has as
// many partial softmax states, which a merge joins in ascending key order.
#pragma once

#include <stdint.h>

#include <string>
#include <vector>

struct SeqItem {
  int32_t tok0;     // row of the sequence's first new token in q and out (packed: in k and v too)
  int32_t pos0;     // key index of that token
  int32_t rows;     // query rows of the sequence, q_len·G; 0: the item is empty
  int32_t row0;     // first row of the tile
  int32_t kv_len;   // keys of the sequence
  int32_t k_begin;  // the item's keys [k_begin, k_end); k_begin is a multiple of the list's step
  int32_t k_end;
  int32_t k_lo;     // lowest key that a row of the tile sees: blocks of 16 keys below it are not read
  int32_t table;    // paged: where the sequence's page ids start in the table list
  int32_t n_parts;  // items of this tile
  int32_t sp;       // which of them, in key order
  int32_t part0;    // n_parts > 1: slot of the first one's state (of kv head g: part0·n_kv_heads + g)
};

// Where a new token goes: its page and its key index.
struct SeqTok {
  int32_t page, pos;
};

// Kinds of items: tiles of 16 rows with their keys over the waves of a workgroup
// (seq_rows.hpp) for sequences of at most SEQ_FEW_ROWS query rows, or for all of a small
// batch; for the others tiles of seq_tile_rows rows (seq_tiles.hpp).
enum SeqKind { SEQ_ROWS, SEQ_TILES };
constexpr int SEQ_FEW_ROWS = 16;
constexpr int SEQ_ROWS_CHUNK = 32;  // keys of a step of the first, ranges start at multiples
constexpr int SEQ_KEY_TILE = 64;    // and of the second
constexpr int seq_tile_rows(int head_dim) { return head_dim <= 128 ? 128 : 64; }
// Whether one launch takes both kinds of items: where the row items' buffers leave two
// workgroups a CU.
constexpr bool seq_one_launch(int head_dim) { return head_dim <= 128; }
constexpr int64_t SEQ_MAX_ROWS = INT32_MAX - 128;  // query rows of a sequence: a tile's last row stays inside 32 bits
constexpr int64_t SEQ_MAX_STRIDE = (int64_t)1 << 26;  // values between packed tokens: 16 of them stay below 2 GiB

struct SeqGeom {
  bool paged = false;
  int n_head = 0, n_kv_heads = 0, head_dim = 0;
  int mask_mode = 0;
  int64_t window = -1;
  int64_t n_pages = 0;
  int page_size = 0;
  bool uniform = false;  // no row sees a key (a causal window of 0): every row averages V
};

struct SeqBatch {
  const int32_t *q_lens = nullptr, *kv_lens = nullptr;
  const int32_t *page_table = nullptr;
  int64_t table_stride = 0, n_seqs = 0;
};

struct SeqList {
  std::vector<SeqItem> items;  // longest first
  int n_parts = 0;             // partial states (per kv head)
  int longest = 0;             // keys of the longest item
};
struct SeqLists {
  int64_t n_tokens = 0;
  int64_t max_q = 0;      // longest q_len
  int64_t max_pos = -1;   // largest key index of a new token
  bool clash = false;     // two new tokens go to one slot of a page
  SeqList rows, tiles;
  std::vector<SeqTok> toks;
  std::vector<int32_t> table;
};

// Checks without a device: "" or what is wrong. seq_check_geom also resolves
// negative windows (mask_mode) and `uniform`; *unsupported: the head dim is one
// that the kernels do not have.
std::string seq_check_geom(SeqGeom &g, bool *unsupported);
std::string seq_check_batch(const SeqGeom &g, const SeqBatch &b);
// The lists of a checked batch for a GPU of num_cus CUs.
void seq_build(const SeqGeom &g, const SeqBatch &b, int num_cus, SeqLists *out);
// The most items and partial states that seq_build lists for any batch of at most
// n_seqs sequences and n_tokens new tokens, none longer than max_q.
struct SeqBound {
  int64_t items = 0, parts = 0;
};
void seq_bound(const SeqGeom &g, int64_t n_seqs, int64_t n_tokens, int64_t max_q, int num_cus, SeqBound *rows,
               SeqBound *tiles);
