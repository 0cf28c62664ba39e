// The tile kernel for attention with shaped scores or a shared prefix (shaped.hpp has the formulas), and the launch that
// joins the partial results of split walks.
//
// A workgroup of four waves owns 128 query rows that read the same K/V plane, 32 rows a wave, and walks the plane in
// steps of 64 keys, everything transposed so that a lane owns whole query rows:
//   S^T[key][row] = K . Q^T    A = K tile from LDS, B = Q in registers
//   O^T[d][row]  += V^T . P^T  A = V^T from LDS (transposing read), B = P^T in registers
// on 32x32x16 instructions: the C layout of S^T is, up to an order of the keys that the V^T read follows, the B layout
// of the second product.  Rows are (token, query head of the group), heads fastest: a tile of a group of eight spans
// sixteen positions, which keeps the part of a walk where its rows see different keys short.  K and V tiles come
// straight into LDS, two of each, the next pair on its way while one is multiplied; two workgroups share a compute unit
// and fill each other's waits.
//
// Masks are one key range [lo, hi) a row: a step that all of a wave's rows see whole takes no mask, one that none of them
// sees is passed over, and in between the range is two compares a score.  Value rows that only some rows of a step see
// may hold infinities and NaN: such a step looks at its values first (values_odd) and multiplies odd ones apart.
#include "common.hpp"
#include "shaped.hpp"

namespace ellm {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kRows = (int)kShapedRows;
constexpr int kKeys = (int)kShapedKeys;
constexpr int kTileBytes = kKeys * kHeadDim * 2;
constexpr int kAhead = 4;   // LDS operand reads in flight ahead of their product
constexpr uint32_t kNoKey = 0xffffffffu;
static_assert(kRows == 32 * kWaves, "32 rows a wave");

typedef __attribute__((address_space(3))) uint16_t LdsHalf;
typedef __attribute__((address_space(3))) u32x4 LdsU32x4;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 LdsI16x4;
constexpr int kBufferFlags = 0x00020000;  // raw buffer of 32-bit data, no swizzle (word 3 of the descriptor)

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
  uint32_t rows_plane, tiles_plane, n_split, planes, own_wgs;
  uint32_t prefix_rows, prefix_tiles, prefix_split;
  uint32_t n_part;
  float c_in;     // with a cap: 2 scale log2(e) / cap
  float a0, a1;   // y = a0 + a1 s (shaped.hpp)
};

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
// 16 bytes a lane from memory straight to LDS address lds_at + 16 x lane.  Written as asm: the compiler's own form of
// this load makes it wait for every outstanding one before each later LDS read.  (M0 is a register the compiler
// reserves and never uses itself in these kernels; one wait state between its write and the load.)
__device__ __forceinline__ void load_to_lds(const u32x4& rsrc, uint32_t voff, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds_at), "v"(voff), "s"(rsrc) : "memory");
}

// Where a query row is: sequence, position of its own row, query head.
struct Row {
  uint32_t seq, token, head;
};

template <typename T>
struct Odd;   // bits of infinities and NaN
template <>
struct Odd<F16> {
  static constexpr uint32_t kInf = 0x7c00u, kOne = 0x3c00u;
};
template <>
struct Odd<BF16> {
  static constexpr uint32_t kInf = 0x7f80u, kOne = 0x3f80u;
};

// The operand's finite values, zeros where it has others.
template <typename T>
__device__ __forceinline__ u32x4 finite_values(u32x4 a) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t lo = (a[w] & 0x7fffu) < Odd<T>::kInf ? 0xffffu : 0u, hi = ((a[w] >> 16) & 0x7fffu) < Odd<T>::kInf ? 0xffff0000u : 0u;
    a[w] &= lo | hi;
  }
  return a;
}
// Ones where the operand has infinities or NaN other than `but`.
template <typename T>
__device__ __forceinline__ u32x4 odd_values(u32x4 a, uint32_t but) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t x = a[w] & 0xffffu, y = a[w] >> 16;
    const uint32_t lo = ((x & 0x7fffu) >= Odd<T>::kInf) & (x != but) ? Odd<T>::kOne : 0u;
    const uint32_t hi = ((y & 0x7fffu) >= Odd<T>::kInf) & (y != but) ? Odd<T>::kOne << 16 : 0u;
    a[w] = lo | hi;
  }
  return a;
}

template <typename T, bool CAP, bool SLOPES>
__global__ __launch_bounds__(kThreads, 2) void shaped_tile_kernel(ShapedKernelArgs p) {
  // K tiles [2][64][128] then V tiles [2][64][128]; of the sixteen 16-byte pieces of a row, piece x of K row r sits at
  // x ^ (r & 15), of V row r at x ^ 2 (r & 7): reads meet few banks twice
  __shared__ __attribute__((aligned(256))) uint16_t smem[4 * kKeys * kHeadDim];
  __shared__ uint32_t s_lo[kWaves], s_hi[kWaves];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = (int)uniform((uint32_t)tid >> 6);
  const int j = lane & 31, g = lane >> 5;

  // ---- which rows, which part of the keys -------------------------------------------------------
  const bool on_prefix = blockIdx.x >= p.own_wgs;   // packed rows of all sequences against the prefix alone
  uint32_t id = on_prefix ? blockIdx.x - p.own_wgs : blockIdx.x;
  uint32_t seq0 = 0, kvh, split, n_split, tile;
  if (on_prefix) {
    kvh = id % p.n_kv_heads;
    id /= p.n_kv_heads;
    n_split = p.prefix_split;
    split = id % n_split;
    tile = id / n_split;
  } else {   // planes fastest: those that share an XCD's cache stay on it; the longest walks of causal prompts first
    const uint32_t plane = id % p.planes;
    id /= p.planes;
    seq0 = plane / p.n_kv_heads;
    kvh = plane % p.n_kv_heads;
    n_split = p.n_split;
    split = id % n_split;
    tile = p.tiles_plane - 1 - id / n_split;
  }
  const uint32_t n_rows = on_prefix ? p.prefix_rows : p.rows_plane;
  const uint32_t at_row = tile * kRows + 32 * wave + j;
  const bool valid = at_row < n_rows;
  Row row;
  {
    const uint32_t r = min(at_row, n_rows - 1);
    row.seq = on_prefix ? r / p.rows_plane : seq0;
    const uint32_t in_plane = on_prefix ? r % p.rows_plane : r;
    row.token = in_plane / p.group;
    row.head = kvh * p.group + in_plane % p.group;
  }
  uint32_t own = p.position;   // the query's own row
  if (p.positions) own = min(p.positions[row.seq], own);
  const uint32_t cap_seq = p.seq_caps ? p.seq_caps[row.seq] : p.capacity;
  own = min(own + row.token, cap_seq - 1);
  const uint32_t pos = p.prefix + own;
  uint32_t lo = 0, hi = pos + 1;
  if (p.key_begin) lo = p.key_begin[row.seq * p.bounds_pitch + own];
  if (p.key_end) hi = min(p.key_end[row.seq * p.bounds_pitch + own], cap_seq);
  if (p.window && pos + 1 > p.window) lo = max(lo, pos + 1 - p.window);
  // this workgroup's part of the keys: all, the prefix, or the sequence's own rows
  if (on_prefix) hi = min(hi, p.prefix);
  if (!on_prefix && p.prefix_tiles) lo = max(lo, p.prefix);
  if (lo >= hi) lo = hi = 0;   // sees nothing
  const bool live = valid && lo < hi;

  // ---- the steps from the first to the last key that any row sees, this split's share of them -----
  uint32_t wlo = live ? lo : kNoKey, whi = live ? hi : 0u;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    wlo = min(wlo, (uint32_t)__shfl_xor((int)wlo, x));
    whi = max(whi, (uint32_t)__shfl_xor((int)whi, x));
  }
  if (lane == 0) {
    s_lo[wave] = wlo;
    s_hi[wave] = whi;
  }
  __syncthreads();
  uint32_t hull_lo = kNoKey, hull_hi = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    hull_lo = min(hull_lo, uniform(s_lo[w]));
    hull_hi = max(hull_hi, uniform(s_hi[w]));
  }
  wlo = uniform(wlo);
  whi = uniform(whi);
  const uint32_t prefix_steps = (p.prefix + kKeys - 1) / kKeys;
  auto step_of = [&](uint32_t key) { return key < p.prefix ? key / kKeys : prefix_steps + (key - p.prefix) / kKeys; };
  uint32_t step = 0, end = 0;
  if (hull_lo < hull_hi) {
    const uint32_t first = step_of(hull_lo), n = step_of(hull_hi - 1) + 1 - first;
    step = first + (uint32_t)((uint64_t)n * split / n_split);
    end = first + (uint32_t)((uint64_t)n * (split + 1) / n_split);
  }

  u32x4 qreg[8];
  {
    const uint16_t* qrow = p.q + row.token * p.q_token_stride + ((size_t)row.seq * p.n_q_heads + row.head) * kHeadDim;
#pragma unroll
    for (int s = 0; s < 8; ++s) qreg[s] = load16(qrow + 16 * s + 8 * g);
  }
  float slope2 = 0.0f;
  if constexpr (SLOPES) slope2 = p.slopes[row.head] * kLog2e;

  // rows that are not stored see what the wave's others see, so that they never ask for a mask
  const uint32_t mlo = valid ? lo : 0u, mhi = valid ? hi : kNoKey;
  uint32_t all_lo = mlo, all_hi = mhi;   // the keys that every row of the wave sees
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    all_lo = max(all_lo, (uint32_t)__shfl_xor((int)all_lo, x));
    all_hi = min(all_hi, (uint32_t)__shfl_xor((int)all_hi, x));
  }
  all_lo = uniform(all_lo);
  all_hi = uniform(all_hi);

  // ---- staging ------------------------------------------------------------------------------------
  const size_t plane_at = seq_plane_offset(p.seq_offsets, p.kv_stride_seq, seq0) + kvh * p.kv_stride_head;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LdsHalf*)smem;
  const int ld_r = 16 * wave + (lane >> 4), ld_x = lane & 15;   // this lane's piece of each of the wave's four loads: row ld_r + 4 i
  const uint32_t wave_lds = lds0 + (uint32_t)wave * 16 * kHeadDim * 2;
  auto stage = [&](uint32_t s, uint32_t buf) __attribute__((always_inline)) {
    const bool ahead = s < prefix_steps;   // (uniform)
    const uint32_t first = (ahead ? s : s - prefix_steps) * kKeys, rows = ahead ? p.prefix : hull_hi - p.prefix;
    const size_t stride = ahead ? p.prefix_stride_pos : p.kv_stride_pos;
    const size_t at = (size_t)first * stride + (ahead ? kvh * p.prefix_stride_head : plane_at);
    // rows past the last one read as zeros
    const uint64_t span = ((uint64_t)(rows - 1 - first) * stride + kHeadDim) * 2;
    const uint32_t left = uniform(span > 0xffffffffull ? 0xffffffffu : (uint32_t)span);
    const uint64_t kat = uniform64((uint64_t)((ahead ? p.prefix_k : p.k) + at)),
                   vat = uniform64((uint64_t)((ahead ? p.prefix_v : p.v) + at));
    const u32x4 krsrc = {(uint32_t)kat, (uint32_t)(kat >> 32) & 0xffffu, left, (uint32_t)kBufferFlags};
    const u32x4 vrsrc = {(uint32_t)vat, (uint32_t)(vat >> 32) & 0xffffu, left, (uint32_t)kBufferFlags};
    const uint32_t to = uniform(wave_lds + buf * kTileBytes);
    const uint32_t pitch = 2 * (uint32_t)stride;
    // a scalar register that the vector unit wrote (readfirstlane) is a load's to read five wait states later
    asm volatile("s_nop 4" :: "s"(krsrc), "s"(vrsrc), "s"(to));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = ld_r + 4 * i;
      load_to_lds(krsrc, r * pitch + 16 * (ld_x ^ (r & 15)), to + 4 * i * kHeadDim * 2);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = ld_r + 4 * i;
      load_to_lds(vrsrc, r * pitch + 16 * (ld_x ^ (2 * (r & 7))), to + 2 * kTileBytes + 4 * i * kHeadDim * 2);
    }
  };

  // A operand of Q.K: keys 32 mb + j, dims 16 s + 8 g ..
  const uint32_t k_read = lds0 + j * kHeadDim * 2 + 16 * (g ^ (j & 15));
  auto k_operand = [&](uint32_t base, int mb, int s) {   // base: k_read in the step's buffer
    return *(const LdsU32x4*)((base ^ (32 * s)) + 32 * mb * kHeadDim * 2);
  };
  // A operand of P.V (rows = 32 dims, 16 keys): lane (dim j, key half g) holds keys {4g..4g+3, 8+4g..8+4g+3} of the 16,
  // in two transposing reads (keys +0 and +8).  A 16-lane block of such a read hands lane t element t & 3 of what its lanes
  // 4 e + (t >> 2), e = 0..3, address: lane s of a block points at key s >> 2, dims 4 (s & 3) .. of the block's sixteen.
  const int v_row = 4 * g + ((lane & 15) >> 2), v_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_read = lds0 + 2 * kTileBytes + v_row * kHeadDim * 2 + 16 * (v_piece ^ (2 * (v_row & 7))) + 8 * (lane & 1);
  auto v_operand = [&](uint32_t base, int cc, int db) {   // base: v_read in the step's buffer
    u32x4 a;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t at = (base ^ (64 * db)) + (16 * cc + 8 * half) * kHeadDim * 2;
      const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)at));
      a[2 * half] = x[0];
      a[2 * half + 1] = x[1];
    }
    return a;
  };

  // ---- walk ---------------------------------------------------------------------------------------
  float m_run = -INFINITY, l_run = 0.0f;   // reference of the row (log2 units), this lane's share of the sum
  f32x16 oacc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[db][r] = 0.0f;
  const float hidden = p.a1 < 0.0f ? INFINITY : -INFINITY;   // a score that comes out as y = -inf

  if (step < end) stage(step, 0);
  for (uint32_t buf = 0; step < end; ++step, buf ^= 1) {
    // this wave's loads have arrived and its reads of the other buffers are done; behind the barrier so have all
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + 1 < end) stage(step + 1, buf ^ 1);
    const bool ahead = step < prefix_steps;
    const uint32_t kb = ahead ? step * kKeys : p.prefix + (step - prefix_steps) * kKeys;
    const uint32_t keys_end = ahead ? min(p.prefix, kb + kKeys) : kb + kKeys;
    if (whi <= kb || wlo >= keys_end) continue;   // no row of this wave sees any of them
    const bool partly = all_lo > kb || all_hi < kb + kKeys || keys_end < kb + kKeys;

    // operands are read kAhead instructions ahead of the product that takes them; the scheduling barriers keep it so
    u32x4 ring[kAhead];
    const uint32_t ks = opaque(k_read + buf * kTileBytes), vs = opaque(v_read + buf * kTileBytes);
    f32x16 st[2];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) st[mb][r] = 0.0f;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = k_operand(ks, n & 1, n >> 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      st[n & 1] = Mfma<T>::m32x32x16(ring[n % kAhead], qreg[n >> 1], st[n & 1]);
      if (n + kAhead < 16) ring[n % kAhead] = k_operand(ks, (n + kAhead) & 1, (n + kAhead) >> 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (CAP) {
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[mb][r] = __builtin_amdgcn_rcpf(fast_exp2(st[mb][r] * p.c_in) + 1.0f);
    }
    // keys of the lane: kb + 4 g + off, off = 32 mb + 8 (r >> 2) + (r & 3)
    const int32_t from = (int32_t)(mlo - kb) - 4 * g, until = (int32_t)(min(mhi, keys_end) - kb) - 4 * g;
    if (partly) {
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t off = 32 * mb + 8 * (r >> 2) + (r & 3);
          st[mb][r] = off >= from && off < until ? st[mb][r] : hidden;
        }
    }
    // y of the step's scores, with `shift` added
    const float dist = (float)((int32_t)(pos - kb) - 4 * g);
    auto y_of = [&](int mb, int r, float shift) __attribute__((always_inline)) {
      if constexpr (SLOPES) shift = __builtin_fmaf(-slope2, fabsf(dist - (float)(32 * mb + 8 * (r >> 2) + (r & 3))), shift);
      return __builtin_fmaf(st[mb][r], p.a1, shift);
    };
    float top = -INFINITY;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, y_of(mb, r, p.a0));
    top = max_with_partner_half(top);
    if (__any(top > m_run)) {
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_new == -INFINITY ? 1.0f : fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db) oacc[db] *= alpha;
    }
    const float shift = p.a0 - (m_run == -INFINITY ? 0.0f : m_run);
    u32x4 pk[4];
    float sum = 0.0f;
#pragma unroll
    for (int cc = 0; cc < 4; ++cc)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int mb = cc >> 1, r = 8 * (cc & 1) + 2 * w;
        const float p0 = fast_exp2(y_of(mb, r, shift)), p1 = fast_exp2(y_of(mb, r + 1, shift));
        pk[cc][w] = Mfma<T>::pack2(p0, p1);
        sum += p0 + p1;
      }
    l_run += sum;

    bool odd = false;
    if (partly) {   // infinities or NaN among the step's values?
      uint32_t most = 0;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll 4
      for (int i = 0; i < 16; ++i) {
        const u32x4 x = *(const LdsU32x4*)(lds0 + (2 + buf) * kTileBytes + i * 1024 + 16 * lane);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          most = max(most, x[w] & 0x7fff0000u);
          most = max(most, (x[w] & 0x7fffu) << 16);
        }
      }
      odd = __any((most >> 16) >= Odd<T>::kInf);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!odd) {
#pragma unroll
      for (int n = 0; n < kAhead; ++n) ring[n] = v_operand(vs, n >> 2, n & 3);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        oacc[n & 3] = Mfma<T>::m32x32x16(ring[n % kAhead], pk[n >> 2], oacc[n & 3]);
        if (n + kAhead < 16) ring[n % kAhead] = v_operand(vs, (n + kAhead) >> 2, (n + kAhead) & 3);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      // finite values as ever; then how many a row sees of those that lead to +inf and to -inf (a NaN is one of each)
#pragma unroll
      for (int n = 0; n < 16; ++n) {
        oacc[n & 3] = Mfma<T>::m32x32x16(finite_values<T>(v_operand(vs, n >> 2, n & 3)), pk[n >> 2], oacc[n & 3]);
        __builtin_amdgcn_sched_barrier(0);
      }
      const int32_t from2 = (int32_t)opaque((uint32_t)from), until2 = (int32_t)opaque((uint32_t)until);
#pragma unroll
      for (int cc = 0; cc < 4; ++cc)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          pk[cc][w] = 0;   // ones for the keys a row sees
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 8 * (cc & 1) + 2 * w + h;
            const int32_t off = 32 * (cc >> 1) + 8 * (r >> 2) + (r & 3);
            pk[cc][w] |= (off >= from2) & (off < until2) ? Odd<T>::kOne << (16 * h) : 0u;
          }
        }
#pragma unroll 1
      for (int sign = 0; sign < 2; ++sign) {
        const uint32_t at = opaque(vs), but = Odd<T>::kInf | (sign ? 0u : 0x8000u);
        const float as = sign ? -INFINITY : INFINITY;
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          f32x16 n;
#pragma unroll
          for (int r = 0; r < 16; ++r) n[r] = 0.0f;
#pragma unroll
          for (int cc = 0; cc < 4; ++cc) {
            n = Mfma<T>::m32x32x16(odd_values<T>(v_operand(at, cc, db), but), pk[cc], n);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[db][r] += n[r] > 0.0f ? as : 0.0f;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  // ---- results ------------------------------------------------------------------------------------
  const float l = sum_with_partner_half(l_run);
  if (!valid) return;
  const size_t at = (size_t)row.token * p.batch_pitch + row.seq;
  if (p.n_part == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // (a row that sees no key is 0)
    uint16_t* orow = p.out + row.token * p.q_token_stride + ((size_t)row.seq * p.n_q_heads + row.head) * kHeadDim;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u32x2 w;
        w[0] = Mfma<T>::pack2(oacc[db][4 * b] * inv, oacc[db][4 * b + 1] * inv);
        w[1] = Mfma<T>::pack2(oacc[db][4 * b + 2] * inv, oacc[db][4 * b + 3] * inv);
        *(u32x2*)(orow + 32 * db + 8 * b + 4 * g) = w;
      }
    if (p.lse && g == 0) p.lse[at * p.n_q_heads + row.head] = (m_run + fast_log2(l)) * kLn2;
    return;
  }
  const size_t part = (((size_t)row.token * p.batch + row.seq) * p.n_q_heads + row.head) * p.n_part + split + (on_prefix ? p.n_split : 0);
  float* prow = p.part_o + part * kHeadDim;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *(f32x4*)(prow + 32 * db + 8 * b + 4 * g) = f32x4{oacc[db][4 * b], oacc[db][4 * b + 1], oacc[db][4 * b + 2], oacc[db][4 * b + 3]};
  if (g == 0) *(f32x2*)(p.part_ml + part * 2) = f32x2{m_run, l};
}

// Joins the partial results of a row: G lanes share its four columns (fold_splits).
template <typename T, int G>
__global__ __launch_bounds__(256) void shaped_merge_kernel(ShapedKernelArgs p) {
  constexpr uint32_t kQuads = kHeadDim / 4;
  const uint32_t sub = threadIdx.x % G;
  const size_t item = ((size_t)blockIdx.x * 256 + threadIdx.x) / G;
  const size_t r = item / kQuads;   // (token, sequence, head)
  const uint32_t dq = (uint32_t)(item % kQuads);
  if (r >= (size_t)p.interval * p.batch * p.n_q_heads) return;
  float l;
  f32x4 o;
  const float m = fold_splits<G, 4>(p.part_ml + r * p.n_part * 2, p.part_o + r * p.n_part * kHeadDim + 4 * dq, kHeadDim, sub,
                                    p.n_part, p.n_part, l, o);
  if (sub) return;
  const uint32_t head = (uint32_t)(r % p.n_q_heads), seq = (uint32_t)(r / p.n_q_heads % p.batch);
  const size_t token = r / p.n_q_heads / p.batch;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  u32x2 w;
  w[0] = Mfma<T>::pack2(o[0] * inv, o[1] * inv);
  w[1] = Mfma<T>::pack2(o[2] * inv, o[3] * inv);
  *(u32x2*)(p.out + token * p.q_token_stride + ((size_t)seq * p.n_q_heads + head) * kHeadDim + 4 * dq) = w;
  if (p.lse && dq == 0) p.lse[(token * p.batch_pitch + seq) * p.n_q_heads + head] = (m + fast_log2(l)) * kLn2;
}

template <typename T>
hipError_t launch(const ShapedKernelArgs& p, bool cap, bool slopes, hipStream_t stream) {
  const dim3 grid(p.own_wgs + p.prefix_tiles * p.prefix_split * p.n_kv_heads), block(kThreads);
  if (cap && slopes)
    hipLaunchKernelGGL((shaped_tile_kernel<T, true, true>), grid, block, 0, stream, p);
  else if (cap)
    hipLaunchKernelGGL((shaped_tile_kernel<T, true, false>), grid, block, 0, stream, p);
  else if (slopes)
    hipLaunchKernelGGL((shaped_tile_kernel<T, false, true>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((shaped_tile_kernel<T, false, false>), grid, block, 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.n_part == 1) return e;
  const size_t quads = (size_t)p.interval * p.batch * p.n_q_heads * (kHeadDim / 4);
  if (p.n_part > 8) {
    hipLaunchKernelGGL((shaped_merge_kernel<T, 8>), dim3((uint32_t)((quads * 8 + 255) / 256)), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((shaped_merge_kernel<T, 1>), dim3((uint32_t)((quads + 255) / 256)), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_shaped(const ShapedArgs& args, hipStream_t stream) {
  const AttnArgs& a = args.a;
  const ShapedState& s = args.s;
  // keys of a walk as far as the host knows them: the window bounds them, ranges of their own may shorten them
  uint32_t own_keys = a.position_index + a.position_interval;
  uint32_t prefix_keys = s.prefix;
  if (s.window) {
    const uint64_t reach = (uint64_t)s.window + a.position_interval;
    if (reach < own_keys) {
      own_keys = (uint32_t)reach;
    } else if (!a.positions) {   // (own rows of sequences that are shorter than the bound on the host leave more to the prefix)
      const uint64_t rest = reach - own_keys;
      if (rest < prefix_keys) prefix_keys = (uint32_t)rest;
    }
  }
  const ShapedPlan plan = shaped_plan(a.position_interval, a.batch, a.n_kv_heads, a.group, own_keys, prefix_keys, a.n_cu, s.part_rows);
  // (sizes of a launch are 32-bit; 128-row tiles of that many rows would be a chunk of 2^31 (token, head) rows)
  if ((uint64_t)a.position_interval * a.batch * a.n_q_heads > 0x7fffffffull) return hipErrorInvalidValue;
  ShapedKernelArgs p{};
  p.q = (const uint16_t*)a.q;
  p.k = (const uint16_t*)a.k;
  p.v = (const uint16_t*)a.v;
  p.prefix_k = (const uint16_t*)s.prefix_k;
  p.prefix_v = (const uint16_t*)s.prefix_v;
  p.out = (uint16_t*)a.out;
  p.lse = a.lse;
  p.positions = a.positions;
  p.seq_offsets = a.seq_offsets;
  p.seq_caps = a.seq_caps;
  p.slopes = s.slopes;
  p.key_begin = s.key_begin;
  p.key_end = s.key_end;
  p.part_o = s.part_o;
  p.part_ml = s.part_ml;
  p.bounds_pitch = s.bounds_pitch;
  p.q_token_stride = (size_t)a.batch_pitch * a.n_q_heads * kHeadDim;
  p.kv_stride_seq = a.kv_stride_seq;
  p.kv_stride_head = a.kv_stride_head;
  p.kv_stride_pos = a.kv_stride_pos;
  p.prefix_stride_head = s.prefix_stride_head;
  p.prefix_stride_pos = s.prefix_stride_pos;
  p.batch = a.batch;
  p.batch_pitch = a.batch_pitch;
  p.n_q_heads = a.n_q_heads;
  p.n_kv_heads = a.n_kv_heads;
  p.group = a.group;
  p.interval = a.position_interval;
  p.position = a.position_index;
  p.capacity = a.capacity;
  p.prefix = s.prefix;
  p.window = s.window;
  p.rows_plane = plan.rows_plane;
  p.tiles_plane = plan.tiles_plane;
  p.n_split = plan.n_split;
  p.planes = a.batch * a.n_kv_heads;
  p.own_wgs = p.planes * plan.tiles_plane * plan.n_split;
  p.prefix_rows = plan.prefix_rows;
  p.prefix_tiles = plan.prefix_tiles;
  p.prefix_split = plan.prefix_split;
  p.n_part = plan.n_part;
  if (s.cap != 0.0f) {
    p.c_in = 2.0f * a.scale * kLog2e / s.cap;
    p.a0 = s.cap * kLog2e;
    p.a1 = -2.0f * p.a0;
  } else {
    p.a0 = 0.0f;
    p.a1 = a.scale * kLog2e;
    // (a hidden score is an infinity times a1: a scale of zero is taken as one that no finite sum of products feels)
    if (!(fabsf(p.a1) >= 1e-37f)) p.a1 = 1e-37f;
  }
  return a.dtype == 0 ? launch<F16>(p, s.cap != 0.0f, s.slopes != nullptr, stream)
                      : launch<BF16>(p, s.cap != 0.0f, s.slopes != nullptr, stream);
}

}  // namespace ellm
