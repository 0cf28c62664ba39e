// Attention with shaped scores (a cap, a slope over the distance, a window, one key range for each query position) and
// over a prefix that a batch shares: what the host plans, the launches take and the kernels have in common.
//
// Keys are counted over both parts a query reads: 0 .. prefix - 1 are the shared prefix, prefix + r is row r of the
// query's own sequence.  For the query at position p (own row p - prefix) and the key at position j
//     x = scale q.k;   x <- cap tanh(x / cap)   (with a cap);   x <- x - slope[head] |p - j|   (with slopes)
// and the row sees begin <= j < end with p - j < window; begin = 0 and end = p + 1 without a range of their own.
// The kernels work in log2 units on an affine function of one value a score: y = a0 + a1 s - slope2 |p - j| with
//     s = q.k,                                  a1 = scale log2(e), a0 = 0                     without a cap,
//     s = 1 / (1 + 2^(q.k . 2 scale log2(e) / cap)),  a1 = -2 cap log2(e), a0 = cap log2(e)    with one
// (tanh z = 1 - 2 / (1 + e^2z)): two transcendental instructions more a score.  The cap's absolute error is a rounding
// or two of 2 cap log2(e), 2^-24 relative: 1e-5 of a binary order at a cap of 50, far below a 16-bit weight's 2^-9 or 2^-12.
#pragma once

#include "kernels.hpp"
#include "shaped_plan.hpp"

namespace ellm {

// What ellm_attn_set_scores / ellm_attn_set_shared_prefix leave in a handle, and the room both work in.
struct ShapedState {
  float cap;                   // 0: none
  const float* slopes;         // device, one a query head; null: none
  uint32_t window;             // 0: none
  const uint32_t* key_begin;   // device [sequence][bounds_pitch]; null: 0
  const uint32_t* key_end;     // null: position + 1
  size_t bounds_pitch;
  const void* prefix_k;        // device; null: no prefix
  const void* prefix_v;
  size_t prefix_stride_head, prefix_stride_pos;   // elements
  uint32_t prefix;             // rows of the prefix
  float* part_o;               // partial rows [part_rows][128] and [part_rows][2], from the first set call to destroy
  float* part_ml;
  size_t part_rows;
  // what a launch over the sequences' own rows joins to them: the prefix's partial results (0: none)
  uint32_t prefix_parts;
  bool walk_prefix;   // or it walks the prefix itself, ahead of every sequence's own rows
  bool scores() const { return cap != 0.0f || slopes || window || key_begin || key_end; }
  bool active() const { return scores() || prefix; }
};

// The state that a call sees: prefix rows that the window hides from every one of its queries are left off the front (positions
// count from the first row that stays: distances and windows are differences), and a prefix of which none stays is none.  With
// positions on the device the host knows no more than that they are at least 0.
inline ShapedState shaped_seen(ShapedState s, const AttnArgs& a) {
  const uint32_t seen = shaped_prefix_seen(s.prefix, s.window, a.positions ? 0u : a.position_index);
  const size_t hidden = (size_t)(s.prefix - seen) * s.prefix_stride_pos * sizeof(uint16_t);
  s.prefix = seen;
  s.prefix_k = seen ? (const char*)s.prefix_k + hidden : nullptr;
  s.prefix_v = seen ? (const char*)s.prefix_v + hidden : nullptr;
  return s;
}

// Scores in the kernels' terms: y = a0 + a1 s, s as above (c_in: what q.k is multiplied by under a cap).
struct ShapedScores {
  float c_in, a0, a1;
};
inline ShapedScores shaped_scores(const ShapedState& s, float scale) {
  constexpr float kLog2E = 1.4426950408889634f;
  ShapedScores f{0.0f, 0.0f, scale * kLog2E};
  if (s.cap != 0.0f) {
    f.c_in = 2.0f * scale * kLog2E / s.cap;
    f.a0 = s.cap * kLog2E;
    f.a1 = -2.0f * f.a0;
  } else if (!(f.a1 >= 1e-37f || f.a1 <= -1e-37f)) {
    // (a hidden score is an infinity times a1: a scale of zero is taken as one that no finite sum of products feels)
    f.a1 = 1e-37f;
  }
  return f;
}

struct ShapedArgs {
  AttnArgs a;   // description, tables and the run's own fields
  ShapedState s;
};

hipError_t launch_shaped(const ShapedArgs& args, hipStream_t stream);
// Chunks without a prefix and without positions of their own: 32 wr query rows a workgroup, wr 1 or 2.
hipError_t launch_shaped_short(const ShapedArgs& args, uint32_t wr, bool along, hipStream_t stream);
// Single tokens: the shared prefix alone, left as *parts partial results a row.
hipError_t launch_shaped_prefix(const ShapedArgs& args, uint32_t* parts, hipStream_t stream);

}  // namespace ellm
