// The order of expert tiles behind a C interface, for tests without a device.
#include "../burn-rocket_amd/csrc/moe_tiles.hpp"

// The tiles of n_experts experts of rows[e] rows each, as (expert, first row of the expert's, rows), in expert order and in
// the order of lengths; -1 where none was put. Returns their number, or -1 when one is put outside `room` tiles.
extern "C" int tile_lists(const int *rows, int n_experts, int T, int room, int *by_expert, int *by_length) {
  uint64_t total = 0, before = 0;
  for (int e = 0; e < n_experts; ++e) total += moe_tile_counts(rows[e], T);
  for (int i = 0; i < room * 3; ++i) by_expert[i] = by_length[i] = -1;
  bool inside = true;
  for (int e = 0; e < n_experts; ++e) {
    moe_tile_places(rows[e], T, before, total, [&](int at, int at_length, int r, int n) {
      if (at < 0 || at >= room || at_length < 0 || at_length >= room) {
        inside = false;
        return;
      }
      const int tile[3] = {e, r, n};
      for (int i = 0; i < 3; ++i) {
        by_expert[at * 3 + i] = tile[i];
        by_length[at_length * 3 + i] = tile[i];
      }
    });
    before += moe_tile_counts(rows[e], T);
  }
  return inside ? moe_tile_sum(total) : -1;
}
