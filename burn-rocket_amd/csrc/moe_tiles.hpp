// The order of a batch's expert tiles, as moe_lists_kernel makes it (plain C++: the host's tests compile it too).
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define RK_TILES_FN __host__ __device__ inline
#else
#define RK_TILES_FN inline
#endif

// A tile's length in quarters of the longest possible, from 4 (field 0) to 1 (field 3). A whole tile is field 0 for every T,
// those of fewer than four rows among them (very wide stacks have tiles of two).
RK_TILES_FN int moe_tile_field(int rows, int T) { return 4 - (4 * rows + T - 1) / T; }

// The tiles that an expert's `all` rows make, counted by field: four 16-bit counts in a word, so that one sum over experts
// adds them all. (At most 2^20 rows on tiles of 64 or more, or 24 576 on shorter ones, of up to 1024 experts: no field carries.)
RK_TILES_FN uint64_t moe_tile_counts(int all, int T) {
  const int tail = all % T;
  uint64_t k = (uint64_t)(all / T);
  if (tail) k += (uint64_t)1 << (16 * moe_tile_field(tail, T));
  return k;
}
RK_TILES_FN int moe_tile_count(uint64_t counts, int field) { return (int)(counts >> (16 * field) & 0xffff); }
RK_TILES_FN int moe_tile_sum(uint64_t counts) {
  return moe_tile_count(counts, 0) + moe_tile_count(counts, 1) + moe_tile_count(counts, 2) + moe_tile_count(counts, 3);
}

// An expert's tiles, as put(place in expert order, place in the order of lengths, first row, rows). before: the counts of the
// experts in front of it; total: of all. Longest first by fields, in expert order within one; an expert has any number of
// whole tiles and one shorter one at most, behind the whole ones of its field.
template <typename Put>
RK_TILES_FN void moe_tile_places(int all, int T, uint64_t before, uint64_t total, Put put) {
  int at = moe_tile_sum(before), whole = moe_tile_count(before, 0), r = 0;
  for (; r + T <= all; r += T) put(at++, whole++, r, T);
  if (r == all) return;
  const int f = moe_tile_field(all - r, T);
  int place = f == 0 ? whole : moe_tile_count(before, f);
  for (int longer = 0; longer < f; ++longer) place += moe_tile_count(total, longer);
  put(at, place, r, all - r);
}
