// What the tile kernel and the short-walk kernel for shaped scores share on the device: their arguments, small helpers,
// the scan for values that are not finite.
#pragma once

#include "common.hpp"
#include "shaped.hpp"

namespace ellm {

struct ShapedKernelArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* prefix_k;
  const uint16_t* prefix_v;
  uint16_t* out;
  float* lse;
  const uint32_t* positions;
  const size_t* seq_offsets;
  const uint32_t* seq_caps;
  const float* slopes;
  const uint32_t* key_begin;
  const uint32_t* key_end;
  float* part_o;    // [row][n_part][128]
  float* part_ml;   // [row][n_part][2]: reference (log2 units), sum of weights
  size_t bounds_pitch;
  size_t q_token_stride;
  size_t kv_stride_seq, kv_stride_head, kv_stride_pos;
  size_t prefix_stride_head, prefix_stride_pos;
  uint32_t batch, batch_pitch, n_q_heads, n_kv_heads, group;
  uint32_t interval, position, capacity, prefix, window;
  uint32_t rows_plane, tiles_plane, n_split, own_wgs;
  uint32_t prefix_rows, prefix_tiles, prefix_split;
  uint32_t n_part;
  uint32_t whole;   // rows are finished here (one partial result, and nothing to join it to)
  Divisor by_planes, by_kv_heads, by_split, by_prefix_split, by_rows_plane, by_group, by_tiles;
  uint32_t along;   // short walks: an XCD takes the row tiles of a plane one after the other
  float c_in;     // with a cap: 2 scale log2(e) / cap
  float a0, a1;   // y = a0 + a1 s (shaped.hpp)
};

// The arguments of a call that its plan has no part in.
ShapedKernelArgs shaped_kernel_args(const ShapedArgs& args);

namespace {

constexpr uint32_t kNoKey = 0xffffffffu;

typedef __attribute__((address_space(3))) uint16_t LdsHalf;
typedef __attribute__((address_space(3))) u32x4 LdsU32x4;
typedef __attribute__((address_space(3))) u32x2 LdsU32x2;
typedef __attribute__((address_space(3))) f32x4 LdsF32x4;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 LdsI16x4;
constexpr int kBufferFlags = 0x00020000;  // raw buffer of 32-bit data, no swizzle (word 3 of the descriptor)

// The own row of a query: its sequence's position, `token` further on.
__device__ __forceinline__ uint32_t own_row(const ShapedKernelArgs& p, uint32_t seq, uint32_t token) {
  const uint32_t first = p.positions ? min(p.positions[seq], p.position) : p.position;
  return min(first + token, (p.seq_caps ? p.seq_caps[seq] : p.capacity) - 1);
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
  return ((uint64_t)uniform((uint32_t)(x >> 32)) << 32) | (uint64_t)uniform((uint32_t)x);
}
// The same value, of which the compiler knows nothing: sums with it are formed where they are needed instead of being
// kept in registers around a loop.
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}
// Packed pairs of 16-bit values: which are infinities or NaN, without compares (masks of lanes are scarce registers).
template <typename T>
struct Odd;
template <>
struct Odd<F16> {
  static constexpr uint32_t kInf = 0x7c00u, kOne = 0x3c00u, kLast = 0x0400u;   // infinity, one, the exponent's last bit
};
template <>
struct Odd<BF16> {
  static constexpr uint32_t kInf = 0x7f80u, kOne = 0x3f80u, kLast = 0x0080u;
};
constexpr uint32_t both(uint32_t half) { return half * 0x10001u; }
// the top bit of every half that is odd (an exponent of ones carries into it)
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t x) {
  return ((x & both(Odd<T>::kInf)) + both(Odd<T>::kLast)) & both(0x8000u);
}
__device__ __forceinline__ uint32_t whole_halves(uint32_t top) { return (top - (top >> 15)) | top; }
// The operand's finite values, zeros where it has others.
template <typename T>
__device__ __forceinline__ u32x4 finite_values(u32x4 a) {
#pragma unroll
  for (int w = 0; w < 4; ++w) a[w] &= ~whole_halves(odd_bits<T>(a[w]));
  return a;
}
// Ones where the operand has infinities or NaN other than `but` (in both halves).
template <typename T>
__device__ __forceinline__ u32x4 odd_values(u32x4 a, uint32_t but) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t d = a[w] ^ but, differs = ((d & both(0x7fffu)) + both(0x7fffu)) | d;   // (top bits)
    a[w] = whole_halves(odd_bits<T>(a[w]) & differs) & both(Odd<T>::kOne);
  }
  return a;
}

}  // namespace
}  // namespace ellm
