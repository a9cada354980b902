// Which tokens of a row a bounded decode call attends, as a line of 32-token
// tiles.  Integer logic over the row's length only.
#pragma once

#include <stdint.h>

namespace fd {

// Row of `len` tokens of which t < sinks or t >= start are attended (all of them
// where start <= sinks).  The line holds the tiles with sinks, then the ones from
// the window's first to the row's last, each once, on the cache's own 32-token
// boundaries: a tile never spans more blocks than in the plain decode.
struct BoundedRow {
  int len, sinks, start;
  int sink_tiles, first_tile;  // line tile i is tile i below sink_tiles, else i - sink_tiles + first_tile
  int tiles;

  __host__ __device__ __forceinline__ int tile(int i) const {
    return i < sink_tiles ? i : i - sink_tiles + first_tile;
  }
  __host__ __device__ __forceinline__ bool attends(int t) const { return t < len && (t < sinks || t >= start); }
};

// seq_len: as given (negative: empty); cap: tokens that the block-table row
// holds; window > 0, sinks >= 0.
__host__ __device__ __forceinline__ BoundedRow bounded_row(int seq_len, int cap, int window, int sinks) {
  BoundedRow r;
  r.len = seq_len < 0 ? 0 : (seq_len < cap ? seq_len : cap);
  r.sinks = sinks < r.len ? sinks : r.len;
  r.start = r.len - window > r.sinks ? r.len - window : r.sinks;
  const int last = (r.len + 31) >> 5;
  r.first_tile = r.start >> 5;
  r.sink_tiles = (r.sinks + 31) >> 5;
  if (r.sink_tiles > r.first_tile) r.sink_tiles = r.first_tile;
  r.tiles = r.sink_tiles + last - r.first_tile;
  return r;
}

// Most tiles a row's line can have.
__host__ __forceinline__ int64_t bounded_max_tiles(int64_t cap, int64_t window, int64_t sinks) {
  const int64_t all = (cap + 31) / 32;
  // a window of w tokens touches at most (w + 62) / 32 tiles
  const int64_t some = (sinks + 31) / 32 + (window + 62) / 32;
  return all < some ? all : some;
}

}  // namespace fd
