// Attention of a chunk of new tokens over planes in 8 bits (e4m3.hpp has the format): causal, every query sees the keys up to
// its own position.
//
// A workgroup of four waves owns 128 query rows that read the same K/V plane, 32 rows a wave, and walks the plane in steps of
// 64 keys, everything transposed so that a lane owns whole query rows:
//   S^T[key][row] = K . Q^T    A = K tile from LDS, B = Q in registers
//   O^T[d][row]  += V^T . P^T  A = V^T from LDS (transposing read), B = P^T in registers
// on 32x32x16 instructions: the C layout of S^T is, up to an order of the keys that the V^T read follows, the B layout of
// the second product.  Rows are (token, query head of the group), heads fastest.
//
// Rows arrive in 8 bits and are multiplied in 16: a tile goes from memory to registers, is converted once for the four waves
// (a code times a power of two is a 16-bit value, one instruction for two) and stored to LDS, two buffers of K and of V; the
// loads of a step are on their way while the one before is multiplied.
//
// A row whose scale is NaN reads as NaN.  A value row like that is taken as what its codes alone say (zeros, where the cache
// wrote them) and its key's scale as NaN instead: rows that see the key get weights, and so results, of NaN; rows that do not
// see it yet give it a weight of exactly 0, and 0 x NaN would be NaN.
#include <type_traits>

#include "e4m3.hpp"
#include "shaped_common.hpp"

namespace ellm {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kBuffers = 2;   // tiles of K, and of V, in LDS
constexpr int kRows = (int)kShapedRows;
static_assert(kRows == 32 * kWaves, "32 rows a wave");
constexpr int kAhead = 4;     // LDS operand reads in flight ahead of their products
constexpr int kKeys = (int)kShapedKeys;
constexpr int kTileBytes = kKeys * kHeadDim * 2;

struct E4m3Args {
  ShapedKernelArgs a;   // strides and planes of k and v: in codes
  const uint8_t* k_scale;
  const uint8_t* v_scale;
};

template <typename T>
__global__ __launch_bounds__(kThreads, 2) void e4m3_tile_kernel(E4m3Args args) {
  const ShapedKernelArgs& p = args.a;
  // K tiles [kBuffers][64][128] then V tiles [kBuffers][64][128]; of the sixteen 16-byte pieces of a row, piece x of K row r sits at
  // x ^ (r & 15), of V row r at x ^ 4 (r & 3): the lanes that a read serves at once (16 rows of a piece, 4 rows of 64
  // bytes) meet no bank twice
  __shared__ __attribute__((aligned(256))) uint16_t smem[2 * kBuffers * kKeys * kHeadDim];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = (int)uniform((uint32_t)tid >> 6);
  const int j = lane & 31, g = lane >> 5;

  // ---- which rows, which part of the keys -------------------------------------------------------
  // planes fastest: those that share an XCD's cache stay on it; the longest walks first
  uint32_t rest = p.by_planes.quotient(blockIdx.x);
  const uint32_t plane = p.by_planes.rest(blockIdx.x, rest);
  const uint32_t seq = p.by_kv_heads.quotient(plane), kvh = p.by_kv_heads.rest(plane, seq);
  uint32_t tile = p.by_split.quotient(rest);
  const uint32_t split = p.by_split.rest(rest, tile);
  tile = p.tiles_plane - 1 - tile;
  const uint32_t n_rows = p.rows_plane;
  const uint32_t wave_row = tile * kRows + 32 * wave;
  const uint32_t r_lane = min(wave_row + j, n_rows - 1);
  const bool valid = wave_row + j < n_rows;
  const uint32_t token = p.by_group.quotient(r_lane), head = kvh * p.group + p.by_group.rest(r_lane, token);
  u32x4 qreg[8];
  {
    const uint16_t* qrow = p.q + token * p.q_token_stride + ((size_t)seq * p.n_q_heads + head) * kHeadDim;
#pragma unroll
    for (int s = 0; s < 8; ++s) qreg[s] = load16(qrow + 16 * s + 8 * g);
  }
  const uint32_t row_end = p.position + token + 1;   // keys that the lane's row sees
  // of a range of rows: the keys that all of them see, and those that any does (0: there is none)
  auto seen_by_all = [&](uint32_t first) { return first < n_rows ? p.position + p.by_group.quotient(first) + 1 : 0u; };
  auto seen_by_any = [&](uint32_t first, uint32_t n) {
    return first < n_rows ? p.position + p.by_group.quotient(min(first + n, n_rows) - 1) + 1 : 0u;
  };
  const uint32_t w_all = uniform(seen_by_all(wave_row)), w_any = uniform(seen_by_any(wave_row, 32));
  const uint32_t keys = uniform(seen_by_any(tile * kRows, kRows));
  const uint32_t walk = (keys + kKeys - 1) / kKeys;
  const uint32_t step = uniform(shaped_share(walk, split, p.by_split)), end = uniform(shaped_share(walk, split + 1, p.by_split));
  const uint32_t w_end = uniform(min(end, (w_any + kKeys - 1) / kKeys));   // steps from here on show this wave nothing

  // ---- staging ------------------------------------------------------------------------------------
  const size_t plane_at = seq_plane_offset(p.seq_offsets, p.kv_stride_seq, seq) + kvh * p.kv_stride_head;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LdsHalf*)smem;
  // eight lanes move a row, sixteen codes each: rows ld_r and ld_r + 32 of a tile, codes 16 ld_x ..
  const uint32_t ld_r = tid >> 3, ld_x = tid & 7;
  struct Fetched {
    u32x4 codes[2];
    uint32_t scale[2];
  };
  Fetched kin, vin;
  uint32_t vin_keys[2];   // the scales of the value rows beside the key rows on their way
  auto fetch = [&](Fetched& x, const uint16_t* codes, const uint8_t* scales, uint32_t s) __attribute__((always_inline)) {
    const uint8_t* rows = (const uint8_t*)codes + plane_at;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const size_t at = (size_t)min(s * kKeys + ld_r + 32 * i, keys - 1) * p.kv_stride_pos;   // (rows past the last key: the last)
      x.codes[i] = load16(rows + at + 16 * ld_x);
      x.scale[i] = scales[(plane_at + at) / kHeadDim];
    }
  };
  auto fetch_k = [&](uint32_t s) __attribute__((always_inline)) {
    fetch(kin, p.k, args.k_scale, s);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      vin_keys[i] = args.v_scale[(plane_at + (size_t)min(s * kKeys + ld_r + 32 * i, keys - 1) * p.kv_stride_pos) / kHeadDim];
  };
  auto put = [&](const Fetched& x, int i, float scale, uint32_t at, uint32_t swizzle) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x2 lo = values4<T>(x.codes[i][2 * h], scale), hi = values4<T>(x.codes[i][2 * h + 1], scale);
      *(LdsU32x4*)(at + (ld_r + 32 * i) * kHeadDim * 2 + 16 * ((2 * ld_x + h) ^ swizzle)) = u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  };
  auto store_k = [&](uint32_t buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      put(kin, i, scale_of(vin_keys[i] == kScaleNan ? kScaleNan : kin.scale[i]), lds0 + buf * kTileBytes, ld_r & 15);
  };
  auto store_v = [&](uint32_t buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      put(vin, i, scale_of(vin.scale[i] == kScaleNan ? 127u : vin.scale[i]), lds0 + (kBuffers + buf) * kTileBytes, 4 * (ld_r & 3));
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
  const uint32_t v_read = lds0 + kBuffers * kTileBytes + v_row * kHeadDim * 2 + 16 * (v_piece ^ (4 * (v_row & 3))) + 8 * (lane & 1);
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
  // minus the row's reference (log2 units; +inf: no key seen yet), this lane's share of its sum
  float neg_m = valid ? INFINITY : 0.0f, l_run = 0.0f;
  f32x16 oacc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[db][r] = 0.0f;
  const float a1 = p.a1, hidden = a1 < 0.0f ? INFINITY : -INFINITY;

  // keys of the lane: first key + 4 g + off, off = 32 mb + 8 (r >> 2) + (r & 3) for register r of block mb
  auto off_of = [](int mb, int r) { return 32 * mb + 8 * (r >> 2) + (r & 3); };
  // st = q.k of step s; keys that the row does not see: an infinity that weighs nothing.  (ring: operands are read kAhead
  // ahead of the products that take them; the scheduling barriers keep the order as it is written.)
  auto scores = [&](f32x16 (&st)[2], u32x4 (&ring)[kAhead], uint32_t ks, uint32_t s) __attribute__((always_inline)) {
    f32x16 none;
#pragma unroll
    for (int r = 0; r < 16; ++r) none[r] = 0.0f;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = k_operand(ks, n >> 3, n & 7);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      st[n >> 3] = Mfma<T>::m32x32x16(ring[n % kAhead], qreg[n & 7], (n & 7) == 0 ? none : st[n >> 3]);
      if (n + kAhead < 16) ring[n % kAhead] = k_operand(ks, (n + kAhead) >> 3, (n + kAhead) & 7);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (uniform(w_all < (s + 1) * kKeys)) {
      const int32_t seen = (int32_t)((valid ? row_end : keys) - s * kKeys) - 4 * g;   // (rows that are not stored: any, of those there are)
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[mb][r] = off_of(mb, r) < seen ? st[mb][r] : hidden;
    }
  };
  // weights n of the sixteen pairs of st
  auto weights = [&](const f32x16 (&st)[2], u32x4 (&pk)[4], int n, float shift, float& sum) __attribute__((always_inline)) {
    const int cc = n >> 2, w = n & 3, mb = cc >> 1, r = 8 * (cc & 1) + 2 * w;
    const float p0 = fast_exp2(__builtin_fmaf(st[mb][r], a1, shift)), p1 = fast_exp2(__builtin_fmaf(st[mb][r + 1], a1, shift));
    pk[cc][w] = Mfma<T>::pack2(p0, p1);
    sum += p0 + p1;
  };
  // Where the weights of a step passed what they may add up to, rows move to their maximum and have them computed again.
  auto settle = [&](const f32x16 (&st)[2], u32x4 (&pk)[4], float sum) __attribute__((always_inline)) {
    const uint64_t over = __ballot(!(sum <= Mfma<T>::kMaxSum));
    if (over) {
      float top = -INFINITY;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, st[mb][r] * a1);
      top = max_with_partner_half(top);
      // (a row moves by what its own two lanes saw: its bits do not depend on its neighbours)
      const bool moves = (((over >> j) | (over >> (j + 32))) & 1) != 0;
      const float neg_new = moves ? fminf(neg_m, -top) : neg_m;   // (+inf while the row has seen no key)
      const float safe = neg_new == INFINITY ? 0.0f : neg_new;
      const float alpha = neg_m == INFINITY ? 1.0f : fast_exp2(safe - neg_m);   // (nothing to rescale ahead of a first reference)
      neg_m = neg_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db) oacc[db] *= alpha;
      sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 16; ++n) weights(st, pk, n, safe, sum);
    }
    l_run += sum;
  };

  // Turn t multiplies K of step t and V of step t - 1 (s + 1 and s, counted over the keys): P.V of a step runs beside the
  // weights of the next, whose vector instructions so find their place between the wave's own matrix instructions.
  // Weights swap registers from turn to turn; the first turn has no V, the last no K.  Meanwhile K of step t + 1 and V of
  // step t come from memory; they are converted and stored behind the scores.
  const uint32_t n_steps = end - step;
  auto turn = [&](u32x4 (&pk)[4], u32x4 (&next)[4], uint32_t t) __attribute__((always_inline)) {
    const uint32_t s = step + t - 1;
    // this wave's stores and reads of LDS are done; behind the barrier so are all
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (t + 1 < n_steps) fetch_k(step + t + 1);
    if (t < n_steps) fetch(vin, p.v, args.v_scale, step + t);
    const uint32_t kbuf = t % kBuffers, vbuf = (t + 1) % kBuffers;
    const bool has_k = uniform(s + 1 < w_end) != 0, has_v = uniform(t != 0 && s < w_end) != 0;
    const uint32_t vs = opaque(v_read + vbuf * kTileBytes);
    // Weights against the reference that each row already has: while no lane's sum of them passes kMaxSum the step's
    // maximum is not looked for.  A row without a reference (neg_m = +inf) makes its sums infinite or NaN and so asks for
    // one; so does a score that is not finite.
    float sum = 0.0f;
    const float shift = neg_m;
    f32x16 st[2];
    u32x4 ring[kAhead];
    __builtin_amdgcn_s_setprio(0);
    if (has_k) {
      scores(st, ring, opaque(k_read + kbuf * kTileBytes), s + 1);
    } else {
      asm volatile("" : "=v"(st[0]), "=v"(st[1]));   // (whatever the registers hold: nothing comes of it)
    }
    if (t + 1 < n_steps) store_k(vbuf);
    if (t < n_steps) store_v(kbuf);
    __builtin_amdgcn_s_setprio(1);   // (P.V and the weights ahead of the other workgroup's Q.K)
    if (has_v) {
#pragma unroll
      for (int n = 0; n < kAhead; ++n) ring[n] = v_operand(vs, n >> 2, n & 3);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 16; ++n) {   // (the last turn has no scores: its weights go nowhere)
        oacc[n & 3] = Mfma<T>::m32x32x16(ring[n % kAhead], pk[n >> 2], oacc[n & 3]);
        weights(st, next, n, shift, sum);
        if (n + kAhead < 16) ring[n % kAhead] = v_operand(vs, (n + kAhead) >> 2, (n + kAhead) & 3);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      sum = INFINITY;   // a wave's first step: no row has a reference yet
    }
    if (!has_k) return;
    settle(st, next, sum);
  };
  if (n_steps) {
    u32x4 even[4], odd[4];
    fetch_k(step);
    store_k(0);
    for (uint32_t t = 0;;) {
      turn(odd, even, t);
      if (t++ == n_steps) break;
      turn(even, odd, t);
      if (t++ == n_steps) break;
    }
  }

  // ---- results ------------------------------------------------------------------------------------
  // A lane holds pieces of 4 dims of its row, 16 bytes of a row an instruction: rows go through LDS (each wave its own
  // quarter, pieces permuted by the row so that no bank is met twice) and leave in whole lines.
  const float l = sum_with_partner_half(l_run);
  const float m = l == 0.0f ? -INFINITY : -neg_m;
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // (the others' last reads of the tiles)
  const uint32_t mine_lds = lds0 + (uint32_t)wave * (32 * kHeadDim * 4);
  if (p.whole) {
    const float inv = 1.0f / l;
    const uint32_t to = (uint32_t)(((size_t)token * p.batch_pitch + seq) * p.n_q_heads + head);   // (below 2^31: rows of the whole call)
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u32x2 w;
        w[0] = Mfma<T>::pack2(oacc[db][4 * b] * inv, oacc[db][4 * b + 1] * inv);
        w[1] = Mfma<T>::pack2(oacc[db][4 * b + 2] * inv, oacc[db][4 * b + 3] * inv);
        *(LdsU32x2*)(mine_lds + j * kHeadDim * 2 + 16 * ((4 * db + b) ^ (j & 15)) + 8 * g) = w;
      }
    if (p.lse && g == 0 && valid) p.lse[to] = (m + fast_log2(l)) * kLn2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 4);
      const u32x4 x = *(const LdsU32x4*)(mine_lds + r * kHeadDim * 2 + 16 * ((lane & 15) ^ (r & 15)));
      const size_t to_r = (uint32_t)__shfl((int)to, r);
      if (wave_row + r < n_rows) store16(p.out + to_r * kHeadDim + 8 * (lane & 15), x);
    }
    return;
  }
  const uint32_t part = ((token * p.batch + seq) * p.n_q_heads + head) * p.n_part + split;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *(LdsF32x4*)(mine_lds + j * kHeadDim * 4 + 16 * ((8 * db + 2 * b + g) ^ j)) =
          f32x4{oacc[db][4 * b], oacc[db][4 * b + 1], oacc[db][4 * b + 2], oacc[db][4 * b + 3]};
  if (g == 0 && valid) *(f32x2*)(p.part_ml + (size_t)part * 2) = f32x2{m, l};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 2 * i + g;
    const f32x4 x = *(const LdsF32x4*)(mine_lds + r * kHeadDim * 4 + 16 * (j ^ r));
    const size_t part_r = (uint32_t)__shfl((int)part, r);
    if (wave_row + r < n_rows) *(f32x4*)(p.part_o + part_r * kHeadDim + 4 * j) = x;
  }
}

}  // namespace

hipError_t launch_chunk_e4m3(const AttnArgs& a, hipStream_t stream) {
  ShapedState s{};
  s.part_o = a.prefill_part_o;
  s.part_ml = a.prefill_part_ml;
  s.part_rows = a.prefill_part_rows;
  const ShapedPlan plan = shaped_plan(a.position_interval, a.batch, a.n_kv_heads, a.group,
                                      a.position_index + a.position_interval, 0, a.n_cu, s.part_rows);
  E4m3Args p{shaped_kernel_args(ShapedArgs{a, s}), a.k_scale, a.v_scale};
  p.a.tiles_plane = plan.tiles_plane;
  p.a.n_split = plan.n_split;
  p.a.by_split = divisor(plan.n_split);
  p.a.n_part = plan.n_part;
  p.a.whole = plan.n_part == 1;
  const dim3 grid(p.a.by_planes.d * plan.tiles_plane * plan.n_split), block(kThreads);
  if (a.dtype == 0)
    hipLaunchKernelGGL(e4m3_tile_kernel<F16>, grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL(e4m3_tile_kernel<BF16>, grid, block, 0, stream, p);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || p.a.whole ? e : launch_shaped_merge(p.a, a.dtype, stream);
}

}  // namespace ellm
