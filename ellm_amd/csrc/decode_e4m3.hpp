// The key stream of the single-token kernels over planes in 8 bits (e4m3.hpp): what stream_keys (decode_common.hpp) is for
// rows of 16 bits.
//
// A wave takes chunks of 32 keys and needs no LDS for them.  Scores S^T[key][head] = K.Q^T on 16x16x32: the A operand wants
// eight dims of key i in lane (i, g), and which eight of the 128 is free as long as Q's operand holds the same ones, so a lane
// loads 16 bytes of its key's row at a time and converts eight codes a step.  O^T[d][head] += V^T.P^T on 16x16x32 wants eight
// keys of one dim a lane, and which keys, and which dims the sixteen rows of a block are, is free again: lane (c, g) loads
// dims 8 c .. 8 c + 7 of the eight keys whose weights the scores' layout leaves in the lanes of group g (4 g .. 4 g + 3 and 16
// more), converts them and pairs keys with v_perm; block b then holds the dims 8 i + b.  Conversion is exact (a code times a power
// of two is a 16-bit value), so the result is that of the 16-bit kernel over the rows as they are read back.
//
// Vector instructions of a chunk (8 KB): 64 conversions, 32 permutes, some 90 for the soft-max; with the matrix instructions
// about 1100 cycles of a SIMD, a third of the time the chunk takes to arrive at the card's rate.
#pragma once

#include "decode_common.hpp"
#include "e4m3.hpp"

namespace ellm {
namespace dec {

constexpr int kChunk8 = 32;   // keys per wave step

// The scale of the scores in log2 units.  (A score that is hidden is an infinity times this: a scale of zero is taken as one that no
// finite product feels.)
inline float scale_log2_e4m3(float scale) {
  const float x = scale * kLog2e;
  return x >= 1e-37f || x <= -1e-37f || !(x == x) ? x : 1e-37f;
}

// Query heads of a group as the B operand that goes with the keys' own order of dims: lane (head c, group g) holds
// q[head][64 (s >> 1) + 16 g + 8 (s & 1) + 0..7] for s = 0..3; heads past the group's end are zero.
__device__ __forceinline__ void load_queries8(const uint16_t* q_rows, const Lane& t, uint32_t heads_here, u32x4 (&qreg)[4]) {
  const uint16_t* qrow = q_rows + (size_t)t.c * kHeadDim + 16 * t.g;
#pragma unroll
  for (int s = 0; s < 4; ++s)
    qreg[s] = (uint32_t)t.c < heads_here ? load16(qrow + 64 * (s >> 1) + 8 * (s & 1)) : u32x4{0, 0, 0, 0};
}

// A chunk on its way: codes of two blocks of sixteen keys (halves of a row), codes of eight value rows, and one row's scale:
// lanes 0..31 that of the chunk's keys, lanes 32..63 of its values.
struct Chunk8 {
  u32x4 k[2][2];
  u32x2 v[8];
  uint32_t scale;
};

__device__ __forceinline__ uint32_t scalar(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ __forceinline__ uint64_t scalar64(uint64_t x) {
  return ((uint64_t)scalar((uint32_t)(x >> 32)) << 32) | (uint64_t)scalar((uint32_t)x);
}
constexpr int kNonTemporal = 2;   // cache policy of a buffer load: streamed, not kept

// One wave's share of keys [k_begin, k_end) of a plane, as stream_keys; acc[b][r] of lane (head c, group g) is column
// 32 g + 8 r + b.  k_end is the plane's end (pos + 1) or a multiple of kChunk8 from k_begin on.
template <typename T>
__device__ __forceinline__ void stream_keys8(const DecodeKernelArgs& p, size_t plane, uint32_t k_begin, uint32_t k_end,
                                             uint32_t pos, const u32x4 (&qreg)[4], uint16_t* smem, const Lane& t,
                                             uint32_t rot_seed, float& m_out, float& l_out, f32x4 (&acc)[8]) {
  const int g = t.g, c = t.c;
  const uint32_t wave = scalar(t.wave);
  uint8_t* const scales = (uint8_t*)smem + wave * (2 * kChunk8);   // [keys' 32][values' 32]
  // Rows are fetched through buffer descriptors that begin with the chunk and end with the plane's last row (rows past it read as
  // zeros, and weigh nothing): scalar arithmetic, the lanes' own offsets never change.
  const uint64_t at_plane = scalar64(plane), kp = scalar64((uint64_t)p.k + at_plane), vp = scalar64((uint64_t)p.v + at_plane);
  const uint32_t pitch = (uint32_t)p.kv_stride_pos, scale_pitch = pitch / kHeadDim;
  const uint32_t k_off = c * pitch + 16 * g;
  uint32_t v_off[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v_off[e] = (16 * (e >> 2) + 4 * g + (e & 3)) * pitch + 8 * c;
  const uint8_t* const sp = (t.lane < kChunk8 ? p.k_scale : p.v_scale) + plane / kHeadDim;

  const uint32_t n_chunks = (k_end - k_begin + kChunk8 - 1) / kChunk8;
  const uint32_t my_chunks = n_chunks > wave ? (n_chunks - wave + kDecWaves - 1) / kDecWaves : 0;
  const uint32_t rot = scalar(rot_seed % max(my_chunks, 1u));
  auto first_key = [&](uint32_t it) {
    uint32_t r = it + rot;
    if (r >= my_chunks) r -= my_chunks;
    return scalar(k_begin + (wave + r * kDecWaves) * kChunk8);
  };
  auto fetch = [&](Chunk8& x, uint32_t it) __attribute__((always_inline)) {
    const uint32_t kb = first_key(it);
    const uint64_t off = (uint64_t)kb * pitch, left = (uint64_t)(pos - kb) * pitch + kHeadDim;
    const uint32_t bytes = scalar(left >> 32 ? 0xffffffffu : (uint32_t)left);
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(kp + off), 0, bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(vp + off), 0, bytes, 0x00020000);
    x.scale = sp[(size_t)min(kb + (t.lane & (kChunk8 - 1)), pos) * scale_pitch];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        x.k[b][h] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_off + 16 * b * pitch + 64 * h, 0, kNonTemporal);
#pragma unroll
    for (int e = 0; e < 8; ++e) x.v[e] = __builtin_amdgcn_raw_buffer_load_b64(vr, v_off[e], 0, kNonTemporal);
  };

  float m_run = -INFINITY, l_run = 0.0f;
  const float hidden = p.scale_log2 < 0.0f ? INFINITY : -INFINITY;   // (a product that comes out as -inf)
#pragma unroll
  for (int b = 0; b < 8; ++b) acc[b] = f32x4{0, 0, 0, 0};

  auto consume = [&](const Chunk8& x, uint32_t kb) __attribute__((always_inline)) {
    scales[t.lane] = (uint8_t)x.scale;
    __builtin_amdgcn_wave_barrier();
    f32x4 st[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const float scale = scale_of(scales[16 * b + c]);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const u32x2 lo = values4<T>(x.k[b][s >> 1][2 * (s & 1)], scale), hi = values4<T>(x.k[b][s >> 1][2 * (s & 1) + 1], scale);
        st[b] = Mfma<T>::m16x16x32(u32x4{lo[0], lo[1], hi[0], hi[1]}, qreg[s], s ? st[b] : f32x4{0, 0, 0, 0});
      }
    }
    if (kb + kChunk8 - 1 > pos) {   // (uniform: the plane's last chunk)
      const int32_t seen = (int32_t)(pos - kb) - 4 * g;
#pragma unroll
      for (int e = 0; e < 8; ++e) st[e >> 2][e & 3] = 16 * (e >> 2) + (e & 3) <= seen ? st[e >> 2][e & 3] : hidden;
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, st[e >> 2][e & 3] * p.scale_log2);
    top = max_with_partner_half(top);
    float a = top, b16 = top;
    swap_rows16(a, b16);
    const float m_new = fmaxf(m_run, fmaxf(a, b16));   // (key kb is always valid: finite, unless its row is NaN)
    if (__any(m_new != m_run)) {
      const float alpha = fast_exp2(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int b = 0; b < 8; ++b) acc[b] *= alpha;
      m_run = m_new;
    }
    float y[8], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = fast_exp2(__builtin_fmaf(st[e >> 2][e & 3], p.scale_log2, -m_new));
      sum += y[e];
    }
    l_run += sum;
    u32x4 pb;
#pragma unroll
    for (int w = 0; w < 4; ++w) pb[w] = Mfma<T>::pack2(y[2 * w], y[2 * w + 1]);
    const uint32_t s0 = *(const uint32_t*)(scales + kChunk8 + 4 * g), s1 = *(const uint32_t*)(scales + kChunk8 + 16 + 4 * g);
    u32x4 value[8];   // of key e: dims 8 c .. 8 c + 7
#pragma unroll
    for (int e = 0; e < 8; ++e) value[e] = values8<T>(x.v[e], ((e < 4 ? s0 : s1) >> (8 * (e & 3))) & 255u);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      u32x4 col;
#pragma unroll
      for (int w = 0; w < 4; ++w)
        col[w] = __builtin_amdgcn_perm(value[2 * w + 1][b >> 1], value[2 * w][b >> 1], (b & 1) ? 0x07060302u : 0x05040100u);
      acc[b] = Mfma<T>::m16x16x32(col, pb, acc[b]);
    }
    __builtin_amdgcn_wave_barrier();
  };

  Chunk8 even, odd;
  if (my_chunks) fetch(even, 0);
  for (uint32_t it = 0; it < my_chunks;) {
    if (it + 1 < my_chunks) fetch(odd, it + 1);
    consume(even, first_key(it));
    if (++it == my_chunks) break;
    if (it + 1 < my_chunks) fetch(even, it + 1);
    consume(odd, first_key(it));
    ++it;
  }

  l_run += xor_shuffle(l_run, 16);
  l_run += xor_shuffle(l_run, 32);
  m_out = m_run;
  l_out = l_run;
}

// acc of stream_keys8 in the order that merge_waves takes: quad b of lane (head, g) is columns 32 g + 4 b .. (kQuads8).
__device__ __forceinline__ void order_columns8(f32x4 (&acc)[8]) {
  f32x4 x[8];
#pragma unroll
  for (int b = 0; b < 8; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[b][e] = acc[4 * (b & 1) + e][b >> 1];
#pragma unroll
  for (int b = 0; b < 8; ++b) acc[b] = x[b];
}

}  // namespace dec
}  // namespace ellm
