// How a call of an operator with shaped scores or a shared prefix is cut into workgroups (host code, no device types:
// also compiled by the CPU tests).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "decode_shares.hpp"

namespace ellm {

// Division by a number that the host knows, for dividends below 2^31: a product and a shift on the device, where a division is
// some forty instructions.  With 2^(s-1) < d <= 2^s and m = floor(2^32 (2^s - d) / d) + 1 the quotient is
// floor((floor(m n / 2^32) + n) / 2^s) (Granlund and Montgomery, Division by invariant integers using multiplication, 1994).
struct Divisor {
  uint32_t d, m, s;
  ELLM_SHARES_FN uint32_t quotient(uint32_t n) const { return ((uint32_t)(((uint64_t)n * m) >> 32) + n) >> s; }
  ELLM_SHARES_FN uint32_t rest(uint32_t n, uint32_t q) const { return n - q * d; }
};
inline Divisor divisor(uint32_t d) {
  uint32_t s = 0;
  while (((uint64_t)1 << s) < d) ++s;
  return Divisor{d, (uint32_t)(((((uint64_t)1 << s) - d) << 32) / d + 1), s};
}
// Where split `split` of `n_split` begins in n steps (below 2^26; at most 2^12 splits): splits differ by a step at most.
ELLM_SHARES_FN uint32_t shaped_share(uint32_t n, uint32_t split, const Divisor& n_split) {
  const uint32_t whole = n_split.quotient(n);
  return split * whole + n_split.quotient(split * n_split.rest(n, whole));
}

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

// Splits of a walk of `steps` steps when `walks` of them, `rows` query rows in all, are there for `slots` workgroups: as many
// as find a place, none shorter than two steps, and no more than their partial results are worth.  A step is 1.7 us, a row's
// partial result 1 KB of traffic, 0.3 ns: n splits cost 1.7 steps / n + 0.0003 rows n, least at sqrt(5700 steps / rows); the
// launch that joins them adds some 4 us to the first split (241 tokens alone: 12.9 us whole, 16.9 in two).
inline uint32_t shaped_split(uint32_t steps, uint64_t walks, uint32_t slots, uint64_t rows, bool joined_anyway) {
  uint32_t n = walks >= slots ? 1u : (uint32_t)(slots / walks);
  const uint32_t most = steps / 2 ? steps / 2 : 1;
  if (n > most) n = most;
  while (n > 1 && (uint64_t)n * n * rows > 5700 * (uint64_t)steps) --n;
  if (!joined_anyway && 1700 * (uint64_t)(steps - shaped_ceil(steps, n)) < 4000 + 3 * n * rows / 10) return 1;
  return n;
}

// Places for workgroups of one kind: two a unit, or one where there are few steps for them, which halves the partial results
// (33 tokens of 5 sequences on 777, 3 steps a unit: 21.3 -> 19.4 us; the prefix of 2 sequences, 4 K/V heads, 32000 keys, 8
// steps a unit, ahead of the streaming kernels: 31.6 -> 26.2).
inline uint32_t shaped_slots(uint64_t steps, uint32_t n_cu) { return steps <= 16 * (uint64_t)n_cu ? n_cu : 2 * n_cu; }

// Rows of partial results a handle needs at most.
inline size_t shaped_part_rows(size_t interval, size_t batch, size_t q_heads, uint32_t n_cu) {
  const size_t most = (size_t)4 * n_cu * kShapedRows;   // 131072 rows, 68 MB, on 256 units
  size_t rows = 0;
  if (__builtin_mul_overflow(interval * batch, q_heads, &rows) || rows > most) return most;
  // (a row has at most as many partials as there are places for workgroups, in either part)
  return rows * 4 * n_cu < most ? rows * 4 * n_cu : most;
}

// Rows of a prefix that any query of a call sees: what the window leaves to the first of them, at own row `first`.
inline uint32_t shaped_prefix_seen(uint32_t prefix, uint32_t window, uint32_t first) {
  if (!window) return prefix;
  const uint32_t left = window - 1 > first ? window - 1 - first : 0u;
  return left < prefix ? left : prefix;
}

// Keys that the longest walks of a call read, as far as the host knows them (ranges of their own may shorten them): over a
// sequence's own rows, over the prefix (the rows that are seen of it) and own rows together.
struct ShapedWalks {
  uint32_t own, both;
};
inline ShapedWalks shaped_walks(uint32_t position, uint32_t interval, uint32_t group, uint32_t prefix, uint32_t window) {
  ShapedWalks w{position + interval, prefix + position + interval};
  if (window) {
    const uint32_t span = kShapedRows / group + 1;   // the positions that a workgroup's rows span
    const uint64_t reach = (uint64_t)window + (span < interval ? span : interval);
    if (reach < w.own) w.own = (uint32_t)reach;
    if (reach < w.both) w.both = (uint32_t)reach;
  }
  return w;
}

// (both_keys: ShapedWalks::both; 0: own_keys + prefix)
inline ShapedPlan shaped_plan(uint32_t interval, uint32_t batch, uint32_t n_kv_heads, uint32_t group, uint32_t own_keys,
                              uint32_t prefix, uint32_t n_cu, size_t part_rows, uint32_t both_keys = 0) {
  ShapedPlan p{};
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
    // two places a unit go to the two parts by their steps (one place each for few steps makes the longer of the two wait: 24
    // sequences, 8 K/V heads, behind 8000: 25.4 -> 49.6 us)
    const uint64_t total = prefix_walks * prefix_steps + walks * own_steps;
    const uint32_t slots = 2 * n_cu;
    uint32_t for_prefix = (uint32_t)(slots * (prefix_walks * prefix_steps) / total);
    if (for_prefix < prefix_walks) for_prefix = prefix_walks < slots ? (uint32_t)prefix_walks : slots;
    if (walks < slots && for_prefix > slots - walks) for_prefix = slots - (uint32_t)walks;   // (a place for each walk at least)
    p.prefix_split = shaped_split(prefix_steps, prefix_walks, for_prefix ? for_prefix : 1, rows, true);
    p.n_split = shaped_split(own_steps, walks, slots > for_prefix ? slots - for_prefix : 1, rows, true);
    while (rows * (p.prefix_split + p.n_split) > part_rows && p.prefix_split + p.n_split > 2) {
      if (p.prefix_split >= p.n_split) --p.prefix_split; else --p.n_split;
    }
    p.n_part = p.prefix_split + p.n_split;
    if (rows * p.n_part <= part_rows) return p;
    p.prefix_rows = p.prefix_tiles = p.prefix_split = 0;
    p.n_split = 1;
  }
  uint32_t steps = own_steps + prefix_steps;
  if (both_keys && shaped_ceil(both_keys, kShapedKeys) < steps) steps = shaped_ceil(both_keys, kShapedKeys);
  p.n_split = shaped_split(steps, walks, shaped_slots((uint64_t)walks * steps, n_cu), rows, false);
  if (rows * p.n_split > part_rows) p.n_split = (uint32_t)(part_rows / rows);
  if (p.n_split == 0) p.n_split = 1;
  p.n_part = p.n_split;
  return p;
}

// ---- chunks: the tile kernel or the one for short walks ----------------------------------------------
// Estimated times (us, launch included), fits to 565 back-to-back calls (binary16, capped; 32 / 4, 32 / 32 and 64 / 8 heads, 1
// to 24 sequences, 2 to 1600 tokens on up to 4000, with and without a shared prefix of 60 to 2500): the longest walk's chain of
// steps, the work there is, or K and V from memory, whichever is longest.  `longest` and `mean`: keys of the longest walk and
// of an average row.
struct ShapedShape {
  uint32_t rows_plane, planes, n_kv_heads, n_cu;
  double longest, mean, rows;   // (rows: of a sequence's own)
  double prefix;                // of those keys, as far as the window leaves them
  double own = 0.0;             // keys of the longest walk over own rows alone (0: longest - prefix)
  double steps(double walks, double seen, double keys) const { return walks * (seen / keys + 1); }
  double units() const { return 256.0 / n_cu; }
  double stream_us() const { return (planes * rows + n_kv_heads * prefix) * 512 / 6.5e6; }
};
inline double shaped_longest(double a, double b, double c) { return a > b ? (a > c ? a : c) : (b > c ? b : c); }
// Estimated (measured): 250 tokens, 32 / 4 heads, 12.4 (12.4); 1000 x 8 102 (104); 250 x 24 on 1000 146 (152); 8 on 4000, 31 splits,
// 14.8 (15.4); behind a prefix of 1000, 9 x 8, 64 / 8 heads, 17.3 (19.1); 9 x 24 on 100, 32 / 32 heads, 29.6 (33.3).
inline double shaped_tile_us(const ShapedShape& c, const ShapedPlan& p) {
  const double walks = c.planes * (double)p.tiles_plane, ahead = c.n_kv_heads * (double)p.prefix_tiles;
  const double apart = p.prefix_tiles ? c.prefix : 0.0;   // keys that packed rows of all sequences walk
  const double wgs = walks * p.n_split + ahead * p.prefix_split;
  const double work = (0.0083 * wgs + 0.0045 * (c.steps(walks, c.mean - apart, kShapedKeys) + c.steps(ahead, apart, kShapedKeys))) * c.units();
  const double own = p.prefix_tiles ? (c.own > 0.0 ? c.own : c.longest - apart) : c.longest;
  uint32_t longest = shaped_ceil(shaped_ceil((uint64_t)own, kShapedKeys), p.n_split);
  if (p.prefix_tiles) {
    const uint32_t other = shaped_ceil(shaped_ceil((uint64_t)apart, kShapedKeys), p.prefix_split);
    longest = other > longest ? other : longest;
  }
  const double partials = p.n_part > 1 ? 3.5 + 7.4e-5 * c.planes * (double)c.rows_plane * p.n_part : 0.0;
  return (5.0 + shaped_longest(0.8 + 1.65 * longest, work, c.stream_us()) + partials) * (p.prefix_tiles ? 0.914 : 1.0);
}
// wr = 1: 500 tokens, 32 / 4 heads, 12.9 (11.4); 33 x 5 on 800 15.2 (13.0); 250 x 24 on 1000 271 (255); 40 x 2 on 100 behind 300, 64 / 8
// heads, 11.3 (10.4); wr = 2: 500 tokens 18.2 (15.3); 1000 x 8 138 (132); 33 x 24 on 800 29.0 (28.7).
inline double shaped_short_us(const ShapedShape& c, uint32_t wr) {
  const double wgs = c.planes * (double)shaped_ceil(c.rows_plane, 32 * wr), tiles = c.steps(wgs * wr, c.mean, 32);
  const double work = (wr == 1 ? 0.0068 * wgs + 0.00103 * tiles : 0.0052 * wgs + 0.00084 * tiles) * c.units();
  const double chain = 1.2 + (wr == 1 ? 1.28 : 1.49) * shaped_ceil((uint64_t)c.longest, 128 / wr);
  return 5.0 + shaped_longest(chain, work, c.stream_us() * (wr == 1 ? 1.0 : 1.02)) + (wr == 1 ? 0.0 : 0.1);
}
// Blocks of 32 rows a workgroup of the short-walk kernel, 1 or 2; 0: the tile kernel, unless it is estimated 5 % slower.  Over
// those calls the choice was on average 0.6 % behind the best of the three; over 65 others and the kernels as they are now 1.4 %
// (capped), 2.4 % (scores as they are) and 1.9 % (slopes), at worst 28 %.  Against the tile kernel alone: 33 x 5 on 800 20.0 -> 13.0, 250 tokens 12.5 -> 7.5, 500 19.1 -> 11.8, 16 x 5 on 500, 32 / 32 heads, 19.9 -> 10.8, 40 x 2 on 100
// behind 300, 64 / 8 heads, 19.7 -> 10.3.
inline uint32_t shaped_short_rows(const ShapedShape& c, const ShapedPlan& plan) {
  const double tile = 1.047 * shaped_tile_us(c, plan), one = shaped_short_us(c, 1), two = shaped_short_us(c, 2);
  if (tile <= one && tile <= two) return 0;
  return one <= two ? 1 : 2;
}
// Whether its workgroups are dealt along a plane's tiles, one XCD to a plane: where planes overflow the XCDs' caches or do not
// come out even over them.
inline bool shaped_short_along(uint32_t planes, double rows) {
  return planes >= 32 && (planes % 8 || planes / 8.0 * rows * 512e-6 > 8.0);
}

// How a single-token step behind a shared prefix runs.  Walk: every sequence streams the prefix and its own rows as one
// plane (one launch; the prefix is small enough to be read again from the caches).  Mixed: prefix tiles and the sequences' own
// planes as tiles of one launch, joined by a second.  Apart: prefix tiles first, then the kernels that stream own rows, which
// join the two.  Own planes as tiles are the faster way while each has a unit and they are not the most of the work.  Us,
// walk / mixed / apart, binary16, query heads / K/V heads, sequences, prefix, longest own rows:
//   32 / 4,  2,  2000,    40:    9.4 /  11.8 /  14.4      64 / 8, 64,   300,    40:  13.2 /  22.2 /  16.6
//   32 / 4, 24,  2000,    40:   19.6 /  16.2 /  18.1      32 / 4, 64,  8000,  1000: 148.6 /  39.2 /  51.2
//   32 / 32, 8,  8000,    40:    154 /  31.2 /  31.4      64 / 8, 64,  8000,    40: 218.9 /  42.3 /  36.2
//   64 / 8, 24,  2000,  4000:      - /  64.5 /  66.5      64 / 8, 24,  2000, 24000:     - / 314.3 / 237.0
//   32 / 32, 24, 2000,    40:   95.8 /  28.1 /  18.7      64 / 8, 128, 32000, 4000:     - / 572.4 / 369.4
// A walk is cut into equal splits for the longest sequence.  Where lengths are uneven (positions on the device: the host knows
// the longest only), planes too few to even it out by their number and own rows long, that costs more than a launch over
// the prefix ahead of equal shares of the own rows (us, without a prefix / walk / apart; sequences, prefix, own rows):
//   32 / 4, 24,   100, 500-30000:   85 / 148 /  97        32 / 4,  8,  1000,   100-8000:  22.0 / 26.0 / 31.9
//   64 / 8, 20,  1000, 500-30000:  188 / 253 / 204         8 / 1,100,  1500,    50-4000:  24.4 / 35.4 / 39.7
//   32 / 4, 16,  2500, 500-16000:   47 /  83 /  64        32 /32,  8,   300,   100-1500:  29.0 / 33.6 / 42.7
//   32 / 4, 64,   600,  100-3000:   38 /  61 /  54        64 / 8, 64,   300,    64-2000:  46.9 / 52.0 / 62.4 (512 planes)
//   32 / 4, 32,   100,  100-4000:   27 /  41 /  39        32 / 4,  2,  2000, 1000-131072: 80.8 / 82.6 / 93.0 (nearly even)
enum class PrefixStep { kWalk, kMixed, kApart };
inline PrefixStep shaped_prefix_step(uint32_t batch, uint32_t n_kv_heads, uint32_t group, uint32_t own_keys, uint32_t prefix,
                                     uint32_t n_cu, bool uneven = false) {
  const uint64_t planes = (uint64_t)batch * n_kv_heads;
  if (planes * prefix <= 640 * (uint64_t)n_cu)
    return uneven && planes < 2 * (uint64_t)n_cu && planes * own_keys >= 1792 * (uint64_t)n_cu ? PrefixStep::kApart : PrefixStep::kWalk;
  const uint64_t own_steps = planes * shaped_ceil(own_keys, kShapedKeys);
  return group <= kShapedRows / 2 && planes <= n_cu && own_steps <= 48 * (uint64_t)n_cu ? PrefixStep::kMixed : PrefixStep::kApart;
}

// Single tokens behind a shared prefix: the prefix alone, rows of all sequences of a K/V head packed into tiles, every walk
// left as partial results for the launch that streams the sequences' own rows.
inline ShapedPlan shaped_prefix_plan(uint32_t batch, uint32_t n_kv_heads, uint32_t group, uint32_t prefix, uint32_t n_cu,
                                     size_t part_rows) {
  ShapedPlan p{};
  const uint64_t rows = (uint64_t)batch * n_kv_heads * group;
  p.rows_plane = group;
  p.prefix_rows = group * batch;
  p.prefix_tiles = shaped_ceil(p.prefix_rows, kShapedRows);
  const uint32_t steps = shaped_ceil(prefix, kShapedKeys);
  const uint64_t walks = (uint64_t)p.prefix_tiles * n_kv_heads;
  p.prefix_split = shaped_split(steps, walks, shaped_slots(walks * steps, n_cu), rows, true);
  if (rows * p.prefix_split > part_rows) p.prefix_split = (uint32_t)(part_rows / rows);
  p.n_part = p.prefix_split;   // (0: more rows than there is room for)
  return p;
}

}  // namespace ellm
