// The planner of batches of sequences behind a C interface, for tests without a device.
#include "../burn-rocket_amd/csrc/seq_plan.cpp"

extern "C" {
struct Geom {
  int32_t paged, n_head, n_kv_heads, head_dim, mask_mode, page_size;
  int64_t window, n_pages;
};
static SeqGeom geom_of(const Geom *a) {
  SeqGeom g;
  g.paged = a->paged;
  g.n_head = a->n_head;
  g.n_kv_heads = a->n_kv_heads;
  g.head_dim = a->head_dim;
  g.mask_mode = a->mask_mode;
  g.page_size = a->page_size;
  g.window = a->window;
  g.n_pages = a->n_pages;
  bool unsupported;
  return seq_check_geom(g, &unsupported).empty() ? g : SeqGeom{};
}

// counts: row items, tile items, row parts, tile parts, tokens, page ids, longest row item, clash; 1: refused.
int plan(const Geom *a, const int32_t *q_lens, const int32_t *kv_lens, const int32_t *table, int64_t stride, int64_t n,
         int num_cus, int64_t *counts, int32_t *items, int64_t room) {
  const SeqGeom g = geom_of(a);
  const SeqBatch b{q_lens, kv_lens, table, stride, n};
  if (g.n_head == 0 || !seq_check_batch(g, b).empty()) return 1;
  SeqLists l;
  seq_build(g, b, num_cus, &l);
  const int64_t c[8] = {(int64_t)l.rows.items.size(), (int64_t)l.tiles.items.size(), l.rows.n_parts, l.tiles.n_parts,
                        l.n_tokens, (int64_t)l.table.size(), l.rows.longest, l.clash};
  std::copy(c, c + 8, counts);
  if (c[0] + c[1] > room) return 2;
  const auto put = [&](const std::vector<SeqItem> &v) {
    const int32_t *from = (const int32_t *)v.data();
    items = std::copy(from, from + v.size() * (sizeof(SeqItem) / 4), items);
  };
  put(l.rows.items);
  put(l.tiles.items);
  return 0;
}

// bound: row items, row parts, tile items, tile parts.
void bound(const Geom *a, int64_t n_seqs, int64_t n_tokens, int64_t max_q, int num_cus, int64_t *out) {
  SeqBound r, t;
  seq_bound(geom_of(a), n_seqs, n_tokens, max_q, num_cus, &r, &t);
  out[0] = r.items;
  out[1] = r.parts;
  out[2] = t.items;
  out[3] = t.parts;
}
int item_words() { return sizeof(SeqItem) / 4; }
}
