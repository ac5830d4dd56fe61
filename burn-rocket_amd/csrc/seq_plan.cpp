// Host side of the batches of sequences (seq_plan.hpp): checks and schedules.
#include "seq_plan.hpp"

#include <algorithm>

#include "../../include/burn_rocket_amd.h"

namespace {
constexpr int64_t MAX_KEYS = (int64_t)1 << 30;  // positions and windows stay inside 32 bits

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// First and last key that the query at position t sees, clipped to the sequence.
void visible(const SeqGeom &g, int64_t t, int64_t kv_len, int64_t *lo, int64_t *hi) {
  *lo = 0;
  *hi = kv_len - 1;
  if (g.uniform) return;
  if (g.mask_mode == RK_MASK_CAUSAL || g.mask_mode == RK_MASK_CAUSAL_WINDOW) *hi = std::min(*hi, t);
  if (g.mask_mode == RK_MASK_WINDOW) *hi = std::min(*hi, t + g.window);
  if (g.mask_mode == RK_MASK_WINDOW) *lo = std::max<int64_t>(0, t - g.window);
  if (g.mask_mode == RK_MASK_CAUSAL_WINDOW) *lo = std::max<int64_t>(0, t - g.window + 1);
}

int64_t kv_of(const SeqBatch &b, int64_t i) { return b.kv_lens ? b.kv_lens[i] : b.q_lens[i]; }
}  // namespace

std::string seq_check_geom(SeqGeom &g, bool *unsupported) {
  *unsupported = false;
  if (g.n_head <= 0 || g.n_kv_heads <= 0 || g.n_head % g.n_kv_heads != 0)
    return "n_head must be a positive multiple of n_kv_heads";
  if (g.n_head / g.n_kv_heads > 128) return "GQA group above 128";
  switch (g.head_dim) {
    case 32: case 48: case 64: case 72: case 80: case 96: case 112: case 128: case 256: break;
    default:
      *unsupported = true;
      return "head_dim " + std::to_string(g.head_dim) + " (supported: 32, 48, 64, 72, 80, 96, 112, 128, 256)";
  }
  if (g.mask_mode < RK_MASK_NONE || g.mask_mode > RK_MASK_CAUSAL_WINDOW) return "unknown mask mode";
  // window < 0 disables the window (ext.rs:99-126).
  if (g.mask_mode == RK_MASK_WINDOW && g.window < 0) g.mask_mode = RK_MASK_NONE;
  if (g.mask_mode == RK_MASK_CAUSAL_WINDOW && g.window < 0) g.mask_mode = RK_MASK_CAUSAL;
  g.window = std::min(g.window, MAX_KEYS);
  g.uniform = g.mask_mode == RK_MASK_CAUSAL_WINDOW && g.window == 0;
  if (g.paged) {
    if (g.page_size < 16 || g.page_size > 256 || (g.page_size & (g.page_size - 1)))
      return "page_size must be 16, 32, 64, 128 or 256";
    if (g.n_pages <= 0 || g.n_pages > INT32_MAX) return "n_pages must be in [1, 2^31)";
  }
  return "";
}

std::string seq_check_batch(const SeqGeom &g, const SeqBatch &b) {
  if (b.n_seqs < 0 || b.n_seqs > INT32_MAX) return "n_seqs must be in [0, 2^31)";
  if (b.n_seqs == 0) return "";
  if (!b.q_lens || (g.paged && (!b.kv_lens || !b.page_table))) return "null list";
  const int64_t G = g.n_head / g.n_kv_heads;
  int64_t toks = 0, ids = 0;
  for (int64_t i = 0; i < b.n_seqs; ++i) {
    const auto at = [&](const std::string &what) { return "sequence " + std::to_string(i) + ": " + what; };
    const int64_t q = b.q_lens[i], kv = kv_of(b, i);
    if (q < 0 || kv < q) return at("needs 0 <= q_len <= kv_len");
    if (kv > MAX_KEYS) return at("more than 2^30 keys");
    if (q * G > SEQ_MAX_ROWS) return at("q_len·(n_head/n_kv_heads) above 2^31 - 129");
    toks += q;
    if (toks > INT32_MAX) return "2^31 or more new tokens";
    if (!g.paged || q == 0) continue;
    const int64_t pages = ceil_div(kv, g.page_size);
    if (pages > b.table_stride) return at("its keys need more pages than a table row holds");
    ids += pages;
    if (ids > INT32_MAX) return "2^31 or more page ids";
    int64_t lo, hi;
    visible(g, kv - q, kv, &lo, &hi);
    for (int64_t p = lo / g.page_size; p < pages; ++p) {
      const int32_t id = b.page_table[i * b.table_stride + p];
      if (id < 0 || id >= g.n_pages)
        return at("page " + std::to_string(p) + " has id " + std::to_string(id) + " of " + std::to_string(g.n_pages));
    }
  }
  // items and merges are counted with 32 bits, a launch's workgroups too
  if ((toks * G / 16 + b.n_seqs + 4096) * g.n_kv_heads > INT32_MAX) return "2^31 or more row tiles";
  return "";
}

namespace {
// Workgroups that the GPU holds at once, per kv head (at least one): registers and LDS
// leave two per CU, one of those that take row items alone with heads above 64.
int64_t slots_per_head(const SeqGeom &g, int num_cus, bool one) {
  const int64_t slots = (int64_t)std::max(1, num_cus) * (one && g.head_dim > 64 ? 1 : 2);
  return std::max<int64_t>(1, slots / g.n_kv_heads);
}

constexpr int64_t PARTS = 32, PARTS_LONG = 1024;

// Splits the keys of the longest tiles where that shortens the launch, then sorts
// longest first: the short ones fill the last round. Fewer tiles than the GPU holds at
// once: items of equal length, as many as it holds (one more than that is another
// round: 512 query rows against 16901 keys, 128 tiles, took 152 us in 512 items and
// 206 in 516 on MI355X). More: only tiles longer than 5/4 of an even share. None where
// the longest would shrink by less than `cost` steps, which is what states to
// store and merge take (about 20 us for tiles of 128 rows). A tile has 16 parts at most up
// to `merged` steps, then PARTS, from PARTS_LONG steps on `most`.
void split(std::vector<SeqItem> &tiles, int step, int64_t slots, int64_t least, int64_t cost, int64_t merged, int64_t most,
           SeqList *out) {
  const auto steps = [&](const SeqItem &t) { return ceil_div(t.k_end - t.k_begin, step); };
  int64_t total = 0, longest = 0;
  for (const SeqItem &t : tiles) {
    total += steps(t);
    longest = std::max(longest, steps(t));
  }
  const int64_t max_parts = longest <= merged ? 16 : longest <= PARTS_LONG ? PARTS : most;
  int64_t quota = std::max(least, ceil_div(total, slots));
  if ((int64_t)tiles.size() < slots) {
    const auto items = [&](int64_t q) {
      int64_t n = 0;
      for (const SeqItem &t : tiles) n += std::min(ceil_div(steps(t), q), max_parts);
      return n;
    };
    while (items(quota) > slots) quota += 1 + quota / 64;
  } else {
    quota = std::max(least, ceil_div(5 * total, 4 * slots));
  }
  if (longest - quota < cost) quota = std::max<int64_t>(longest, 1);
  for (SeqItem &t : tiles) {
    const int64_t n = steps(t), parts = std::min(ceil_div(n, quota), max_parts);
    t.n_parts = (int32_t)parts;
    t.part0 = out->n_parts;
    if (parts > 1) out->n_parts += (int)parts;
    const int32_t k0 = t.k_begin, k1 = t.k_end;
    for (int64_t i = 0; i < parts; ++i) {
      t.sp = (int32_t)i;
      t.k_begin = (int32_t)(k0 + n * i / parts * step);
      t.k_end = i + 1 == parts ? k1 : (int32_t)(k0 + n * (i + 1) / parts * step);
      out->items.push_back(t);
    }
  }
  for (const SeqItem &t : out->items) out->longest = std::max(out->longest, t.k_end - t.k_begin);
  std::stable_sort(out->items.begin(), out->items.end(),
                   [&](const SeqItem &x, const SeqItem &y) { return steps(x) > steps(y); });
}
// Steps of an item at least, and steps that a split costs. (Row items of 4 chunks leave
// half the waves idle, but none with a second: one token on 500 keys, 4 kv heads of 128,
// 8.9 us, with 8 chunks 10.0.)
constexpr int64_t ROWS_LEAST = 4, ROWS_COST = 8, TILES_LEAST = 4, TILES_COST = 12;
}  // namespace

void seq_bound(const SeqGeom &g, int64_t n_seqs, int64_t n_tokens, int64_t max_q, int num_cus, SeqBound *rows,
               SeqBound *tiles) {
  // A tile of n steps has at most n / quota + 1 items, and quota is at least an even
  // share of the steps: splits add at most `slots` items. A split tile's states are at
  // most twice what its split added.
  const int64_t G = g.n_head / g.n_kv_heads, tr = seq_tile_rows(g.head_dim);
  const int64_t slots = slots_per_head(g, num_cus, false);
  n_seqs = std::min(n_seqs, n_tokens);  // those with new tokens
  // (a small batch has at most four tiles of 16 rows per CU and all heads)
  const int64_t few = std::min(n_tokens * G / 16 + n_seqs, ceil_div(4 * (int64_t)num_cus, g.n_kv_heads));
  *rows = SeqBound{(max_q * G > SEQ_FEW_ROWS ? std::max(n_seqs, few) : n_seqs) + slots, 2 * slots};
  *tiles = SeqBound{};
  if (max_q * G > SEQ_FEW_ROWS)
    *tiles = SeqBound{n_tokens * G / tr + std::min(n_seqs, n_tokens * G / (SEQ_FEW_ROWS + 1)) + slots, 2 * slots};
}

void seq_build(const SeqGeom &g, const SeqBatch &b, int num_cus, SeqLists *out) {
  *out = SeqLists{};
  const int64_t G = g.n_head / g.n_kv_heads;
  std::vector<SeqItem> rows, tiles;
  struct Piece {
    int32_t page, off, end;
  };
  std::vector<Piece> pieces;  // where new tokens go: slots [off, end) of a page
  // A small batch goes to the kernel of few rows whole: at most four tiles of 16 rows per
  // CU whose products (each tile reads its K and V itself) take less than the other
  // kernel's walk over the longest sequence, both over the keys that its new tokens see.
  // The constants fit 497 batches on MI355X, of which 29 take more than 1.05 times the faster
  // kernel. Rows -> tiles in us: 256 rows on 4096 keys, 32/4 heads of 128, 18.8, 27.3; 128 rows on
  // 30000 41.6, 68; 256 rows on 30000 73, 68; 16 times 64 on 2000 25, 30; 256 rows of 8/2 heads of 256 on 8000
  // 48.7, 38.3. One prompt, causal: 300 tokens of 16/8 heads of 128 9.8, 13.0; 400 12.5, 16.3; 500 15.0, 18.2 (tiles
  // by the rule); 800 of 14/2 heads of 80 17.1, 22.4; 800 of 12/12 heads of 64 11.5, 18.8; 1000 15.8, 14.2 (rows by
  // the rule); 200 of 32/4 heads of 128 10.2, 11.2; 300 15.9, 13.3. 64 tokens of 16/4 heads of 64, window 512, behind
  // 2000 to 100000 keys 8.0, 15-17.
  int64_t n16 = 0, n16_keys = 0, longest = 0;
  for (int64_t i = 0; i < b.n_seqs; ++i) {
    if (b.q_lens[i] == 0) continue;
    const int64_t t = ceil_div(b.q_lens[i] * G, 16) * g.n_kv_heads, kv = kv_of(b, i);
    int64_t lo, hi, skip;
    visible(g, kv - b.q_lens[i], kv, &lo, &skip);
    visible(g, kv - 1, kv, &skip, &hi);
    n16 += t;
    n16_keys += t * (hi + 1 - lo);
    longest = std::max(longest, hi + 1 - lo);
  }
  const bool small = n16 <= 4 * num_cus && n16_keys * g.head_dim <= num_cus * std::min(8000 + 220 * longest, (int64_t)393216);
  for (int64_t i = 0; i < b.n_seqs; ++i) {
    const int64_t q = b.q_lens[i], kv = kv_of(b, i), pos0 = kv - q;
    if (q == 0) continue;
    SeqItem it{};
    it.tok0 = (int32_t)out->n_tokens;
    it.pos0 = (int32_t)pos0;
    it.rows = (int32_t)(q * G);
    it.kv_len = (int32_t)kv;
    it.table = (int32_t)out->table.size();
    const bool few = small || q * G <= SEQ_FEW_ROWS;
    const int64_t tr = few ? 16 : seq_tile_rows(g.head_dim), step = few ? SEQ_ROWS_CHUNK : SEQ_KEY_TILE;
    for (int64_t r = 0; r < q * G; r += tr) {
      int64_t lo, hi, lo2, hi2;
      visible(g, pos0 + r / G, kv, &lo, &hi);
      visible(g, pos0 + (std::min(r + tr, q * G) - 1) / G, kv, &lo2, &hi2);
      it.row0 = (int32_t)r;
      it.k_lo = (int32_t)lo;
      it.k_begin = (int32_t)(lo / step * step);
      it.k_end = (int32_t)(hi2 + 1);
      (few ? rows : tiles).push_back(it);
    }
    out->n_tokens += q;
    out->max_q = std::max(out->max_q, q);
    out->max_pos = std::max(out->max_pos, kv - 1);
    if (!g.paged) continue;
    int64_t lo, hi;
    visible(g, pos0, kv, &lo, &hi);
    const int32_t *row = b.page_table + i * b.table_stride;
    const int64_t ps = g.page_size;
    for (int64_t p = 0; p < ceil_div(kv, ps); ++p) out->table.push_back(p < lo / ps ? 0 : row[p]);
    for (int64_t t = pos0; t < kv; ++t) out->toks.push_back(SeqTok{row[t / ps], (int32_t)t});
    for (int64_t t = pos0; t < kv;) {
      const int64_t e = std::min(kv, (t / ps + 1) * ps);
      pieces.push_back(Piece{row[t / ps], (int32_t)(t % ps), (int32_t)((e - 1) % ps + 1)});
      t = e;
    }
  }
  // Row items merge 16 states in one pass, which pays up to 13000 keys, or 16000 where
  // those parts give half the CUs work. MI355X, one token, heads of 128, 16 parts -> 32: one kv
  // head, 12000 keys 14.7 us, 14.0, 14000 16.0, 14.9, 20000 19.1, 16.4; four, 12000 14.9, 15.0, 14000 16.5,
  // 15.8, 20000 20.0, 17.5; eight, 14000 17.5, 19.5, 20000 20.9, 22.0.
  const int64_t row_heads = (int64_t)rows.size() * g.n_kv_heads;
  const int64_t row_merged = 64 * row_heads <= num_cus ? 416 : 512;
  // Tiles merge one state at a time, beside much more work: 128 rows on 8000 keys 31.7, 36.9; 16000
  // 44.7, 43.2; 24000 57.8, 49.2; heads of 64 on 16000 34.1, 37.4; 24000 43.2, 43.5; of 256 on 12000 44.5,
  // 42.6; 24000 70.7, 56.4.
  const int64_t tile_merged = g.head_dim <= 64 ? 384 : 256;
  // Twice the parts where those leave three quarters of the CUs idle: one token on 60000
  // keys, one kv head of 128, 27 us, 24.6 (on 20000 16.4, 18.4); of 256 51, 45; with four heads of 128 29.0, 31.8.
  const int64_t most = 4 * PARTS * row_heads <= num_cus ? 2 * PARTS : PARTS;
  split(rows, SEQ_ROWS_CHUNK, slots_per_head(g, num_cus, tiles.empty() || !seq_one_launch(g.head_dim)), ROWS_LEAST, ROWS_COST,
        row_merged, most, &out->rows);
  split(tiles, SEQ_KEY_TILE, slots_per_head(g, num_cus, false), TILES_LEAST, TILES_COST, tile_merged, PARTS, &out->tiles);
  std::sort(pieces.begin(), pieces.end(),
            [](const Piece &x, const Piece &y) { return x.page != y.page ? x.page < y.page : x.off < y.off; });
  for (size_t i = 1; i < pieces.size(); ++i)
    out->clash |= pieces[i].page == pieces[i - 1].page && pieces[i].off < pieces[i - 1].end;
}
