// How a call of an operator with shaped scores or a shared prefix is cut into workgroups (host code, no device types:
// also compiled by the CPU tests).
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace ellm {

constexpr uint32_t kShapedRows = 128;   // query rows a workgroup of the tile kernel
constexpr uint32_t kShapedKeys = 64;    // keys a step

struct ShapedPlan {
  // own part: every K/V plane of a sequence, its rows (tokens x heads of the group) in tiles
  uint32_t rows_plane, tiles_plane, n_split;
  // prefix part (0 tiles: every workgroup of the own part walks the prefix ahead of its own keys):
  // the rows of all sequences of a K/V head, in tiles that read the prefix once for all of them
  uint32_t prefix_rows, prefix_tiles, prefix_split;
  uint32_t n_part;   // partial results a row; 1: rows are finished where they are computed
};

inline uint32_t shaped_ceil(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// Splits of a walk of `steps` steps when `walks` of them are there for `slots` workgroups: as many as find a place,
// none shorter than two steps.
inline uint32_t shaped_split(uint32_t steps, uint64_t walks, uint32_t slots) {
  uint32_t n = walks >= slots ? 1u : (uint32_t)(slots / walks);
  const uint32_t most = steps / 2 ? steps / 2 : 1;
  return n < most ? n : most;
}

// Rows of partial results a handle needs at most.
inline size_t shaped_part_rows(size_t interval, size_t batch, size_t q_heads, uint32_t n_cu) {
  const size_t most = (size_t)4 * n_cu * kShapedRows;   // 131072 rows, 68 MB, on 256 units
  size_t rows = 0;
  if (__builtin_mul_overflow(interval * batch, q_heads, &rows) || rows > most) return most;
  // (a row has at most as many partials as there are places for workgroups, in either part)
  return rows * 4 * n_cu < most ? rows * 4 * n_cu : most;
}

inline ShapedPlan shaped_plan(uint32_t interval, uint32_t batch, uint32_t n_kv_heads, uint32_t group, uint32_t own_keys,
                              uint32_t prefix, uint32_t n_cu, size_t part_rows) {
  ShapedPlan p{};
  const uint32_t slots = 2 * n_cu;
  p.rows_plane = interval * group;
  p.tiles_plane = shaped_ceil(p.rows_plane, kShapedRows);
  const uint64_t rows = (uint64_t)p.rows_plane * batch * n_kv_heads;
  const uint64_t walks = (uint64_t)p.tiles_plane * batch * n_kv_heads;
  const uint32_t own_steps = shaped_ceil(own_keys, kShapedKeys), prefix_steps = shaped_ceil(prefix, kShapedKeys);
  p.n_split = 1;
  p.n_part = 1;
  if (prefix && p.rows_plane <= kShapedRows / 2) {
    p.prefix_rows = p.rows_plane * batch;
    p.prefix_tiles = shaped_ceil(p.prefix_rows, kShapedRows);
    const uint64_t prefix_walks = (uint64_t)p.prefix_tiles * n_kv_heads;
    // places go to the two parts by their steps
    const uint64_t total = prefix_walks * prefix_steps + walks * own_steps;
    const uint32_t for_prefix = (uint32_t)(slots * (prefix_walks * prefix_steps) / total);
    p.prefix_split = shaped_split(prefix_steps, prefix_walks, for_prefix ? for_prefix : 1);
    p.n_split = shaped_split(own_steps, walks, slots > for_prefix ? slots - for_prefix : 1);
    while (rows * (p.prefix_split + p.n_split) > part_rows && p.prefix_split + p.n_split > 2) {
      if (p.prefix_split >= p.n_split) --p.prefix_split; else --p.n_split;
    }
    p.n_part = p.prefix_split + p.n_split;
    if (rows * p.n_part <= part_rows) return p;
    p.prefix_rows = p.prefix_tiles = p.prefix_split = 0;
    p.n_split = 1;
  }
  p.n_split = shaped_split(own_steps + prefix_steps, walks, slots);
  if (rows * p.n_split > part_rows) p.n_split = (uint32_t)(part_rows / rows);
  if (p.n_split == 0) p.n_split = 1;
  p.n_part = p.n_split;
  return p;
}

}  // namespace ellm
