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
// Vector instructions of a chunk (8 KB): 64 conversions, 32 permutes, some 110 for the soft-max and addresses; with the matrix
// instructions about 1100 cycles of a SIMD, a third of the time the chunk takes to arrive at the card's rate.  A wave has one chunk
// on its way while it computes on the one before, sent for when that one is converted and its registers are free; two or three
// ahead measured worse.  Measured (32 / 4 heads, bfloat16): 16 x 65536 keys 155 us, 6.97 TB/s; 24 of 1000-60000 131 us, 6.3 TB/s;
// 16 x 8192 24.5 us, 5.5 TB/s.
#pragma once

#include "decode_common.hpp"
#include "e4m3.hpp"

namespace ellm {
namespace dec {

constexpr int kChunk8 = 32;   // keys per wave step
// LDS of the stream lies behind what the waves are joined in: scales of a chunk, codes of a new row.
static_assert(kRedBytes + kDecWaves * (2 * kChunk8 + 2 * kHeadDim) <= kDecWaves * kWaveLdsHalves * 2, "LDS of the single-token kernels");

// The scale of the scores in log2 units.  (A score that is hidden is an infinity times this: a scale of zero is taken as 2^-149, which
// makes at most 2^-21 of any finite product.  Kernels keep values below 2^-126 as they are.)
inline float scale_log2_e4m3(float scale) {
  const float x = scale * kLog2e;
  return x == 0.0f ? 0x1p-149f : x;
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

// The row that a fused cache write adds to a plane (NewRow, decode_common.hpp): source rows, and where the row belongs.
struct NewRow8 {
  bool store;   // this workgroup is the one that writes it to the cache
  const uint16_t* k_row;
  const uint16_t* v_row;
  const uint16_t* rope_row;
  float eps;
  uint8_t* k_dst;
  uint8_t* v_dst;
  uint8_t* k_scale;
  uint8_t* v_scale;
};
// Of plane (sequence, kv head) at element `plane`, position pos (below its capacity).
__device__ __forceinline__ NewRow8 new_row8(const DecodeKernelArgs& p, size_t plane, uint32_t seq, uint32_t kvh, uint32_t pos,
                                            bool store) {
  const size_t src = ((size_t)seq * p.n_kv_heads + kvh) * kHeadDim, dst = plane + (size_t)pos * p.kv_stride_pos;
  const uint32_t turn = p.positions ? min(p.positions[seq], p.position) : p.position;   // (the cache write's rotary row)
  return NewRow8{store,
                 (const uint16_t*)p.pend.k_rows + src,
                 (const uint16_t*)p.pend.v_rows + src,
                 (const uint16_t*)p.pend.rope + (size_t)turn * p.pend.rope_pos_stride + (size_t)kvh * p.pend.rope_head_stride,
                 p.pend.eps,
                 (uint8_t*)p.k + dst,
                 (uint8_t*)p.v + dst,
                 (uint8_t*)p.k_scale + dst / kHeadDim,
                 (uint8_t*)p.v_scale + dst / kHeadDim};
}

// One wave's share of keys [k_begin, k_end) of a plane, as stream_keys: open() sends for the first of them, run() takes them.
// k_end is the plane's end (pos + 1) or a multiple of kChunk8 from k_begin on.  PENDING: the last key may be one that the cache
// does not hold yet (NewRow8); the wave with the fewest chunks makes its row, writes it and takes it as a chunk of one key.
// TURNS: two workgroups share a unit (run).
template <typename T, bool PENDING = false, bool TURNS = false>
struct Stream8 {
  uint64_t kp, vp;             // the plane's codes
  const uint8_t* sp;           // the lane's scales: keys' or values'
  uint32_t pitch, pos, k_begin, my_chunks, rot, wave;
  bool take_new;               // (PENDING) this wave takes the new row ...
  uint32_t new_pos;            // ... of this position
  u32x4 k_new, v_new, turn;    // ... and has its source rows
  Chunk8 first;

  __device__ __forceinline__ uint32_t first_key(uint32_t it) const {
    uint32_t r = it + rot;
    if (r >= my_chunks) r -= my_chunks;
    return scalar(k_begin + (wave + r * kDecWaves) * kChunk8);
  }
  // Rows are fetched through buffer descriptors that begin with the chunk and end with the plane's last row (rows past it read as
  // zeros, and weigh nothing): scalar arithmetic, the lanes' own offsets never change.
  __device__ __forceinline__ void fetch(Chunk8& x, uint32_t it, const Lane& t) const {
    const uint32_t kb = first_key(it), scale_pitch = pitch / kHeadDim;
    const uint64_t off = (uint64_t)kb * pitch, left = (uint64_t)(pos - kb) * pitch + kHeadDim;
    const uint32_t bytes = scalar(left >> 32 ? 0xffffffffu : (uint32_t)left);
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)(kp + off), 0, bytes, 0x00020000);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)(vp + off), 0, bytes, 0x00020000);
    x.scale = sp[(size_t)min(kb + (t.lane & (kChunk8 - 1)), pos) * scale_pitch];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        x.k[b][h] = __builtin_amdgcn_raw_buffer_load_b128(kr, (16 * b + t.c) * pitch + 16 * t.g + 64 * h, 0, kNonTemporal);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x.v[e] = __builtin_amdgcn_raw_buffer_load_b64(vr, (16 * (e >> 2) + 4 * t.g + (e & 3)) * pitch + 8 * t.c, 0, kNonTemporal);
  }

  __device__ __forceinline__ void open(const DecodeKernelArgs& p, size_t plane, uint32_t begin, uint32_t end, uint32_t last,
                                       const Lane& t, uint32_t rot_seed, const NewRow8& fresh) {
    wave = scalar(t.wave);
    const uint64_t at = scalar64(plane);
    kp = scalar64((uint64_t)p.k + at);
    vp = scalar64((uint64_t)p.v + at);
    sp = (t.lane < kChunk8 ? p.k_scale : p.v_scale) + plane / kHeadDim;
    pitch = (uint32_t)p.kv_stride_pos;
    k_begin = begin;
    pos = last;
    const bool with_new = PENDING && end == last + 1;
    if (with_new) {   // the stream ends ahead of the new key
      new_pos = last;
      end = last;
      pos = last ? last - 1 : 0;
    }
    const uint32_t n_chunks = (end - begin + kChunk8 - 1) / kChunk8;
    take_new = with_new && wave == n_chunks % kDecWaves;   // (uniform over the wave)
    my_chunks = n_chunks > wave ? (n_chunks - wave + kDecWaves - 1) / kDecWaves : 0;
    rot = scalar(rot_seed % max(my_chunks, 1u));
    if constexpr (PENDING) {   // ahead of the wave's first chunk, which arrives while the row is made
      if (take_new) {
        k_new = load16(fresh.k_row + 8 * t.c);
        v_new = load16(fresh.v_row + 8 * t.c);
        turn = load16(fresh.rope_row + 8 * t.c);
      }
    }
    if (my_chunks) fetch(first, 0, t);
  }

  // TURNS: of two workgroups on a unit the first one's waves are older and are served first: they end 8 us ahead of the second's on
  // shares of 85 us.  So the two (`second`) take turns, four chunks each, at the higher priority (us: 32 of 300-16000, 64 / 8 heads, 82.6 ->
  // 81.8; 100 of 100-4096 48.1 -> 47.4, 64 of 100-2000 21.8 -> 20.7, 10 of 1000-60000 64.6 -> 63.8; every chunk 81.7, 47.6, 21.2, 63.6).
  // Not where planes are cut alike (64 x 500 14.0 / 14.4).
  //
  // The wave's reference (log2 units), its sum, and its sums of values: acc[b][r] of lane (head c, group g) is column
  // 32 g + 8 r + b.
  __device__ __forceinline__ void run(const DecodeKernelArgs& p, const u32x4 (&qreg)[4], uint16_t* smem, const Lane& t, float& m_out,
                                      float& l_out, f32x4 (&acc)[8], const NewRow8& fresh, bool second = false) {
    const int g = t.g, c = t.c;
    uint8_t* const scales = (uint8_t*)smem + kRedBytes + wave * (2 * kChunk8);   // [keys' 32][values' 32]
    float m_run = -INFINITY, l_run = 0.0f;
    const float hidden = p.scale_log2 < 0.0f ? INFINITY : -INFINITY;   // (a product that comes out as -inf)
#pragma unroll
    for (int b = 0; b < 8; ++b) acc[b] = f32x4{0, 0, 0, 0};

    // keys kb .. kb + 31, of which those up to `last` count
    auto consume = [&](Chunk8& x, uint32_t kb, uint32_t last, uint32_t next) __attribute__((always_inline)) {
      scales[t.lane] = (uint8_t)x.scale;
      __builtin_amdgcn_wave_barrier();
      u32x4 kv[2][4], value[8];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint32_t scale = key_scale(scales[16 * b + c], scales[kChunk8 + 16 * b + c]);
#pragma unroll
        for (int s = 0; s < 4; ++s) kv[b][s] = values8<T>(u32x2{x.k[b][s >> 1][2 * (s & 1)], x.k[b][s >> 1][2 * (s & 1) + 1]}, scale);
      }
      const uint32_t s0 = *(const uint32_t*)(scales + kChunk8 + 4 * g), s1 = *(const uint32_t*)(scales + kChunk8 + 16 + 4 * g);
#pragma unroll
      for (int e = 0; e < 8; ++e) value[e] = values8<T>(x.v[e], ((e < 4 ? s0 : s1) >> (8 * (e & 3))) & 255u);
      __builtin_amdgcn_sched_barrier(0);
      if (next) fetch(x, next, t);
      __builtin_amdgcn_sched_barrier(0);
      f32x4 st[2];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s) st[b] = Mfma<T>::m16x16x32(kv[b][s], qreg[s], s ? st[b] : f32x4{0, 0, 0, 0});
      if (kb + kChunk8 - 1 > last) {   // (uniform: the plane's last chunk)
        const int32_t seen = (int32_t)(last - kb) - 4 * g;
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

    if constexpr (PENDING) {
      if (take_new) {
        float x[8];
        unpack8<T>(k_new, x);
        norm_rope8<T>(x, turn, fresh.eps);
        uint32_t kb, vb;
        const u32x2 k = row_codes16<T>(x, kb);
        unpack8<T>(v_new, x);
        const u32x2 v = row_codes16<T>(x, vb);
        uint8_t* const rows = (uint8_t*)smem + kRedBytes + kDecWaves * 2 * kChunk8 + wave * 2 * kHeadDim;
        if (g == 0) {
          *(u32x2*)(rows + 8 * c) = k;
          *(u32x2*)(rows + kHeadDim + 8 * c) = v;
          if (fresh.store) {
            *(u32x2*)(fresh.k_dst + 8 * c) = k;
            *(u32x2*)(fresh.v_dst + 8 * c) = v;
            if (c == 0) {
              *fresh.k_scale = (uint8_t)kb;
              *fresh.v_scale = (uint8_t)vb;
            }
          }
        }
        __builtin_amdgcn_wave_barrier();
        Chunk8 one{};   // its other rows are zeros, and do not count
        if (c == 0) {
          one.k[0][0] = load16(rows + 16 * g);
          one.k[0][1] = load16(rows + 64 + 16 * g);
        }
        if (g == 0) one.v[0] = *(const u32x2*)(rows + kHeadDim + 8 * c);
        one.scale = t.lane == 0 ? kb : t.lane == kChunk8 ? vb : 0u;
        consume(one, new_pos, new_pos, 0);
      }
    }
    for (uint32_t it = 0; it < my_chunks; ++it) {
      if constexpr (TURNS) {
        if (((it >> 2) & 1) != (uint32_t)second)
          __builtin_amdgcn_s_setprio(1);
        else
          __builtin_amdgcn_s_setprio(0);
      }
      consume(first, first_key(it), pos, it + 1 < my_chunks ? it + 1 : 0);
    }
    if constexpr (TURNS) __builtin_amdgcn_s_setprio(0);

    l_run += xor_shuffle(l_run, 16);
    l_run += xor_shuffle(l_run, 32);
    m_out = m_run;
    l_out = l_run;
  }
};

// What run() leaves, put where join_waves finds it: four columns at a time, 32 g + 4 b .. of lane (head, g).
__device__ __forceinline__ void put_waves8(uint16_t* smem, const Lane& t, uint32_t heads_here, float m_run, float l_run,
                                           const f32x4 (&acc)[8]) {
  f32x4 x[8];
#pragma unroll
  for (int b = 0; b < 8; ++b)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[b][e] = acc[4 * (b & 1) + e][b >> 1];
  put_waves<4, 32>(smem, t, heads_here, m_run, l_run, x);
}
}  // namespace dec
}  // namespace ellm
