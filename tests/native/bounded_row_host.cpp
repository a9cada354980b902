// A bounded decode's line of tiles (csrc/bounded_row.h) on the host: for every
// length, window, sink count and table width of a range, each attended token
// lies in one tile of the line, no tile comes twice or without an attended
// token, and the line is no longer than the host's bound.  Exit status 1 and a
// line on stderr at the first rule broken.
#include <cstdint>
#include <cstdio>
#include <set>

#define __host__
#define __device__
#define __forceinline__ inline
#include "bounded_row.h"

static int check(int seq_len, int cap, int window, int sinks) {
  const fd::BoundedRow r = fd::bounded_row(seq_len, cap, window, sinks);
  const int len = seq_len < 0 ? 0 : (seq_len < cap ? seq_len : cap);
  auto bad = [&](const char* what) {
    std::fprintf(stderr, "bounded_row: %s (len %d, cap %d, window %d, sinks %d)\n", what, seq_len, cap, window, sinks);
    return 1;
  };
  if (r.tiles < 0 || r.tiles > fd::bounded_max_tiles(cap, window, sinks)) return bad("more tiles than the bound");
  std::set<int> tiles;
  for (int i = 0; i < r.tiles; ++i) {
    if (!tiles.insert(r.tile(i)).second) return bad("a tile twice");
    if (i > 0 && r.tile(i) <= r.tile(i - 1)) return bad("tiles out of order");
    if (r.tile(i) < 0 || 32 * r.tile(i) >= len) return bad("a tile behind the row");
  }
  std::set<int> wanted;
  for (int t = 0; t < len + 64; ++t) {
    const bool sees = t < len && (t < sinks || static_cast<int64_t>(t) >= static_cast<int64_t>(len) - window);
    if (r.attends(t) != sees) return bad("another token attended");
    if (sees) wanted.insert(t / 32);
  }
  if (tiles != wanted) return bad("not the tiles of the attended tokens");
  return 0;
}

int main() {
  const int caps[] = {8, 32, 96, 104, 320, 2048};
  const int windows[] = {1, 2, 31, 32, 33, 63, 64, 65, 100, 319, 320, 1000, 2147483647};
  const int sinks[] = {0, 1, 4, 31, 32, 33, 64, 100, 333, 2147483647};
  for (int cap : caps)
    for (int w : windows)
      for (int s : sinks) {
        for (int len = -1; len <= 400; ++len)
          if (check(len, cap, w, s)) return 1;
        for (int len : {2047, 2048, 2049, 2147483647, -2147483647 - 1})
          if (check(len, cap, w, s)) return 1;
      }
  return 0;
}
