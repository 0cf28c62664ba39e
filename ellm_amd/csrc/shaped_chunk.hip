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
// sees is passed over, and in between the range is one compare a score.  Value rows that only some rows of a step see
// may hold infinities and NaN: such a step looks at its values first (find_odd), multiplies odd ones apart and drops them.
//
// Weights are rounded to 16 bits for the second product (half a step each, relative: over random values that is as much as
// the rounding of the result), their sums are taken before it, in 32 bits; so are scores, references and results.
//
// What bounds it (8192 tokens, 32 / 4 heads, binary16, 550 GFLOP): the board's power and the vector unit, 350 us with
// constant operands and no weights, 555 without a cap, 645 with one (0.85 PFLOP/s; 69 us a plane's worth of transcendental
// instructions), 560 with slopes.  Against a plain loop (Q.K, soft-max with a maximum every step, P.V) 740: references
// that move only where a sum asks for it 8 %, addresses and descriptors in scalar registers that move on 5 %, priority 2 to
// 9 %, walks from the last step where scores fall with the distance 24 % of those.  Tried and dropped: eight waves of two
// groups half a step apart (256 rows; 5 % faster on long plain walks, 5 to 10 % slower on short ones), 64 rows a wave (scores land
// in accumulation registers: twice the time), operands read 3, 6 or 8 ahead (the same), three steps on their way instead of
// one where a workgroup has a unit to itself (1 to 8 % slower: the chain of a step, 1.7 us, bounds it, no trip to memory).
#include <type_traits>

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

// 16 bytes a lane from memory straight to LDS address lds_at + 16 x lane.  Written as asm: the compiler's own form of
// this load makes it wait for every outstanding one before each later LDS read.  (M0 is a register the compiler
// reserves and never uses itself in these kernels; one wait state between its write and the load.)
__device__ __forceinline__ void load_to_lds(const u32x4& rsrc, uint32_t voff, uint32_t lds_at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds_at), "v"(voff), "s"(rsrc) : "memory");
}

template <typename T, bool CAP, bool SLOPES>
__global__ __launch_bounds__(kThreads, 2) void shaped_tile_kernel(ShapedKernelArgs p) {
  // K tiles [kBuffers][64][128] then V tiles [kBuffers][64][128]; of the sixteen 16-byte pieces of a row, piece x of K row r sits at
  // x ^ (r & 15), of V row r at x ^ 4 (r & 3): the lanes that a read serves at once (16 rows of a piece, 4 rows of 64
  // bytes) meet no bank twice
  __shared__ __attribute__((aligned(256))) uint16_t smem[2 * kBuffers * kKeys * kHeadDim];
  __shared__ uint32_t s_lo[kWaves], s_hi[kWaves], s_all_lo[kWaves], s_all_hi[kWaves], s_odd[kBuffers];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = (int)uniform((uint32_t)tid >> 6);
  const int j = lane & 31, g = lane >> 5;

  // ---- which rows, which part of the keys -------------------------------------------------------
  const bool on_prefix = blockIdx.x >= p.own_wgs;   // packed rows of all sequences against the prefix alone
  uint32_t id = on_prefix ? blockIdx.x - p.own_wgs : blockIdx.x;
  uint32_t seq0 = 0, kvh, split, tile;
  if (on_prefix) {
    uint32_t rest = p.by_kv_heads.quotient(id);
    kvh = p.by_kv_heads.rest(id, rest);
    tile = p.by_prefix_split.quotient(rest);
    split = p.by_prefix_split.rest(rest, tile);
  } else {   // planes fastest: those that share an XCD's cache stay on it; the longest walks of causal prompts first
    uint32_t rest = p.by_planes.quotient(id);
    const uint32_t plane = p.by_planes.rest(id, rest);
    seq0 = p.by_kv_heads.quotient(plane);
    kvh = p.by_kv_heads.rest(plane, seq0);
    tile = p.by_split.quotient(rest);
    split = p.by_split.rest(rest, tile);
    tile = p.tiles_plane - 1 - tile;
  }
  const uint32_t n_rows = on_prefix ? p.prefix_rows : p.rows_plane;
  struct Row {   // this lane's query row: where it is, what it sees
    bool valid;
    uint32_t seq, token, head, pos;
    uint32_t lo, hi;   // (rows that are not stored see everything: they never ask for a mask)
  };
  Row row;
  const uint32_t wave_row = tile * kRows + 32 * wave;
  {
    const uint32_t at_row = wave_row + j, r = min(at_row, n_rows - 1);
    row.valid = at_row < n_rows;
    const uint32_t packed = on_prefix ? p.by_rows_plane.quotient(r) : 0u, in_plane = p.by_rows_plane.rest(r, packed);
    row.seq = seq0 + packed;
    row.token = p.by_group.quotient(in_plane);
    row.head = kvh * p.group + p.by_group.rest(in_plane, row.token);
  }
  u32x4 qreg[8];
  {
    const uint16_t* qrow = p.q + row.token * p.q_token_stride + ((size_t)row.seq * p.n_q_heads + row.head) * kHeadDim;
#pragma unroll
    for (int s = 0; s < 8; ++s) qreg[s] = load16(qrow + 16 * s + 8 * g);
  }
  const float slope2 = SLOPES ? p.slopes[row.head] * kLog2e : 0.0f;

  // ---- the keys that rows see, the steps from the first to the last of them, this split's share of those ---------------
  struct Reach {
    uint32_t lo, hi;           // the keys that any row sees (lo >= hi: none)
    uint32_t all_lo, all_hi;   // the keys that every row sees
  };
  Reach mine, all;   // the wave's, the workgroup's
  // this workgroup's part of what the query at `pos` sees: all, the prefix, or the sequence's own rows
  auto first_seen = [&](uint32_t pos) {
    const uint32_t lo = p.window && pos + 1 > p.window ? pos + 1 - p.window : 0u;
    return !on_prefix && p.prefix_tiles ? max(lo, p.prefix) : lo;
  };
  auto end_seen = [&](uint32_t pos) { return on_prefix ? min(pos + 1, p.prefix) : pos + 1; };
  if (uniform(!p.key_begin && !p.key_end && (on_prefix ? p.window == 0 : p.positions == nullptr))) {
    // ranges that move on with the rows: those of the first and the last row are all there is to know
    row.pos = p.prefix + p.position + row.token;
    if (SLOPES && p.positions) row.pos = p.prefix + own_row(p, row.seq, row.token);
    row.lo = on_prefix || !row.valid ? 0u : first_seen(row.pos);
    row.hi = !row.valid ? kNoKey : on_prefix ? p.prefix : end_seen(row.pos);
    auto reach = [&](uint32_t first, uint32_t last) {   // of rows first .. last
      if (first >= n_rows) return Reach{kNoKey, 0u, 0u, kNoKey};
      if (on_prefix) return Reach{0u, p.prefix, 0u, p.prefix};
      const uint32_t base = p.prefix + p.position, a = base + p.by_group.quotient(first),
                     b = base + p.by_group.quotient(min(last, n_rows - 1));
      return Reach{first_seen(a), end_seen(b), first_seen(b), end_seen(a)};
    };
    mine = reach(wave_row, wave_row + 31);
    all = reach(tile * kRows, tile * kRows + kRows - 1);
    if (tid < kBuffers) s_odd[tid] = 0;   // (behind the walk's first barrier)
  } else {
    const uint32_t own = own_row(p, row.seq, row.token);
    row.pos = p.prefix + own;
    uint32_t lo = first_seen(row.pos), hi = end_seen(row.pos);
    if (p.key_begin) lo = max(lo, p.key_begin[row.seq * p.bounds_pitch + own]);
    if (p.key_end) hi = min(p.key_end[row.seq * p.bounds_pitch + own], p.seq_caps ? p.seq_caps[row.seq] : p.capacity);
    if (lo >= hi) lo = hi = 0;   // sees nothing
    row.lo = row.valid ? lo : 0u;
    row.hi = row.valid ? hi : kNoKey;
    const bool live = row.valid && lo < hi;
    mine = Reach{live ? lo : kNoKey, live ? hi : 0u, row.lo, row.hi};
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      mine.lo = min(mine.lo, (uint32_t)__shfl_xor((int)mine.lo, x));
      mine.hi = max(mine.hi, (uint32_t)__shfl_xor((int)mine.hi, x));
      mine.all_lo = max(mine.all_lo, (uint32_t)__shfl_xor((int)mine.all_lo, x));
      mine.all_hi = min(mine.all_hi, (uint32_t)__shfl_xor((int)mine.all_hi, x));
    }
    if (lane == 0) {
      s_lo[wave] = mine.lo;
      s_hi[wave] = mine.hi;
      s_all_lo[wave] = mine.all_lo;
      s_all_hi[wave] = mine.all_hi;
    }
    if (tid < kBuffers) s_odd[tid] = 0;
    __syncthreads();
    all = Reach{kNoKey, 0u, 0u, kNoKey};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      all.lo = min(all.lo, s_lo[w]);
      all.hi = max(all.hi, s_hi[w]);
      all.all_lo = max(all.all_lo, s_all_lo[w]);
      all.all_hi = min(all.all_hi, s_all_hi[w]);
    }
  }
  const uint32_t wlo = uniform(mine.lo), whi = uniform(mine.hi), all_lo = uniform(mine.all_lo), all_hi = uniform(mine.all_hi);
  const uint32_t hull_lo = uniform(all.lo), hull_hi = uniform(all.hi), wg_lo = uniform(all.all_lo), wg_hi = uniform(all.all_hi);
  const uint32_t prefix_steps = (p.prefix + kKeys - 1) / kKeys;
  auto step_of = [&](uint32_t key) { return key < p.prefix ? key / kKeys : prefix_steps + (key - p.prefix) / kKeys; };
  uint32_t step = 0, end = 0;
  if (hull_lo < hull_hi) {
    const uint32_t first = step_of(hull_lo), n = step_of(hull_hi - 1) + 1 - first;
    const Divisor& by = on_prefix ? p.by_prefix_split : p.by_split;
    step = first + shaped_share(n, split, by);
    end = first + shaped_share(n, split + 1, by);
  }
  step = uniform(step);
  end = uniform(end);
  // Scores that fall with the distance are walked from the last step to the first: their references are then found in
  // the first step instead of moving in every one.  Step s of the walk is step place(s) of the keys.
  const uint32_t mirror = step + end - 1;
  auto place = [&](uint32_t s) { return SLOPES ? mirror - s : s; };
  auto first_key = [&](uint32_t s) {
    const uint32_t at = place(s);
    return at < prefix_steps ? at * kKeys : p.prefix + (at - prefix_steps) * kKeys;
  };
  auto keys_end = [&](uint32_t s) { return place(s) < prefix_steps ? min(p.prefix, first_key(s) + kKeys) : first_key(s) + kKeys; };
  // the walk's first step in the other of prefix and own rows than the one it starts in
  const uint32_t other_part = SLOPES ? mirror + 1 - prefix_steps : prefix_steps;
  // the steps in which any row of this wave sees keys
  uint32_t w_begin = end, w_end = end;
  if (wlo < whi) {
    const uint32_t from = max(step, step_of(wlo)), to = min(end, step_of(whi - 1) + 1);   // (places; from >= to: none of this split's)
    w_begin = SLOPES ? mirror + 1 - to : from;
    w_end = SLOPES ? mirror + 1 - from : to;
    if (from >= to) w_begin = w_end = end;
  }
  w_begin = uniform(w_begin);
  w_end = uniform(w_end);

  // ---- staging ------------------------------------------------------------------------------------
  const size_t plane_at = seq_plane_offset(p.seq_offsets, p.kv_stride_seq, seq0) + kvh * p.kv_stride_head;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LdsHalf*)smem;
  // four waves move a tile, four loads each; this lane's piece is piece ld_x of row ld_r + 4 i
  const int ld_r = 16 * wave + (lane >> 4), ld_x = lane & 15;
  const uint32_t wave_lds = lds0 + (uint32_t)wave * 16 * kHeadDim * 2;
  // byte offsets of this lane's pieces: row ld_r + 4 i, of K and of V; they change with the rows' distance only
  uint32_t off_k[4], off_v[4];
  auto aim = [&](uint32_t s) __attribute__((always_inline)) {
    const uint32_t pitch = 2 * (uint32_t)(place(s) < prefix_steps ? p.prefix_stride_pos : p.kv_stride_pos);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = ld_r + 4 * i;
      off_k[i] = r * pitch + 16 * (ld_x ^ (r & 15));
      off_v[i] = r * pitch + 16 * (ld_x ^ (4 * (r & 3)));
    }
  };
  // Where the next step of K and of V comes from: address, bytes up to the end of its last row that is read (rows past it
  // read as zeros), bytes from step to step; scalar registers that move on from call to call.
  struct Source {
    uint64_t at, left, pace;
  };
  auto source = [&](const uint16_t* own_rows, const uint16_t* prefix_rows, uint32_t s) __attribute__((always_inline)) {
    const bool ahead = place(s) < prefix_steps;   // (uniform)
    const uint32_t skip = (ahead ? place(s) : place(s) - prefix_steps) * kKeys, n = ahead ? p.prefix : hull_hi - p.prefix;
    const uint64_t pitch = 2 * (ahead ? p.prefix_stride_pos : p.kv_stride_pos);
    const uint16_t* plane = ahead ? prefix_rows + kvh * p.prefix_stride_head : own_rows + plane_at;
    return Source{uniform64((uint64_t)plane + skip * pitch), uniform64((n - 1 - skip) * pitch + 2 * kHeadDim),
                  uniform64(SLOPES ? 0 - kKeys * pitch : kKeys * pitch)};
  };
  // the source's next step on its way into buffer `buf`, pieces at `off`
  auto send = [&](Source& from, const uint32_t (&off)[4], uint32_t buf) __attribute__((always_inline)) {
    const uint64_t at = uniform64(from.at);
    const u32x4 rsrc = {(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu,
                        uniform(from.left >> 32 ? 0xffffffffu : (uint32_t)from.left), (uint32_t)kBufferFlags};
    const uint32_t to = uniform(wave_lds + buf * kTileBytes);
    // a scalar register that the vector unit wrote (readfirstlane) is a load's to read five wait states later
    asm volatile("s_nop 4" :: "s"(rsrc), "s"(to));
#pragma unroll
    for (int i = 0; i < 4; ++i) load_to_lds(rsrc, off[i], to + 4 * i * kHeadDim * 2);
    from.at += from.pace;
    from.left -= from.pace;
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

  Source ksrc = source(p.k, p.prefix_k, step), vsrc = source(p.v, p.prefix_v, step);

  aim(step);

  // ---- walk ---------------------------------------------------------------------------------------
  // minus the row's reference (log2 units; +inf: no key seen yet; rows that will see none need none), this lane's share of its sum
  float neg_m = row.lo < row.hi ? INFINITY : 0.0f, l_run = 0.0f;
  f32x16 oacc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[db][r] = 0.0f;
  // a score's value once it is finished: y = a1 s + a0 without slopes, y itself with them; one that comes out as -inf
  const float a0 = SLOPES ? 0.0f : p.a0, a1 = SLOPES ? 1.0f : p.a1;
  const float hidden = a1 < 0.0f ? INFINITY : -INFINITY;

  // keys of the lane: first key + 4 g + off, off = 32 mb + 8 (r >> 2) + (r & 3) for register r of block mb
  auto off_of = [](int mb, int r) { return 32 * mb + 8 * (r >> 2) + (r & 3); };
  // what the scores of a step become between the product and the weights, pair n of the eight of a block
  auto finish = [&](f32x16& st, int mb, int n, float dist) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 2 * n + h;
      float x = st[r];
      if constexpr (CAP) x = __builtin_amdgcn_rcpf(fast_exp2(x * p.c_in) + 1.0f);
      if constexpr (SLOPES) x = __builtin_fmaf(x, p.a1, __builtin_fmaf(-slope2, fabsf(dist - (float)off_of(mb, r)), p.a0));
      st[r] = x;
    }
  };
  struct Seen {   // which keys of a step a row sees: off - from < width, unsigned
    int32_t from;
    uint32_t width;
  };
  auto seen_of = [&](uint32_t s) {
    const uint32_t last = min(row.hi, keys_end(s));
    return Seen{(int32_t)(row.lo - first_key(s)) - 4 * g, last > row.lo ? last - row.lo : 0u};
  };
  auto partly = [&](uint32_t lo, uint32_t hi, uint32_t s) {   // not every one of the rows behind (lo, hi) sees all keys
    const uint32_t kb = first_key(s);
    return uniform(lo > kb || hi < kb + kKeys || keys_end(s) < kb + kKeys) != 0;
  };
  // st = the finished scores of step s.  (ring: operands are read kAhead ahead of the products that take them; the
  // scheduling barriers keep the order as it is written.)
  auto scores = [&](f32x16 (&st)[2], u32x4 (&ring)[kAhead], uint32_t ks, uint32_t s) __attribute__((always_inline)) {
    const float dist = SLOPES ? (float)((int32_t)(row.pos - first_key(s)) - 4 * g) : 0.0f;
    f32x16 none;
#pragma unroll
    for (int r = 0; r < 16; ++r) none[r] = 0.0f;
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = k_operand(ks, n >> 3, n & 7);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      st[n >> 3] = Mfma<T>::m32x32x16(ring[n % kAhead], qreg[n & 7], (n & 7) == 0 ? none : st[n >> 3]);
      if constexpr (CAP || SLOPES) {   // (the first half beside the products of the second)
        if (n >= 8) finish(st[0], 0, n - 8, dist);
      }
      if (n + kAhead < 16) ring[n % kAhead] = k_operand(ks, (n + kAhead) >> 3, (n + kAhead) & 7);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (CAP || SLOPES) {
#pragma unroll
      for (int n = 0; n < 8; ++n) finish(st[1], 1, n, dist);
    }
    if (partly(all_lo, all_hi, s)) {
      const Seen see = seen_of(s);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[mb][r] = (uint32_t)(off_of(mb, r) - see.from) < see.width ? st[mb][r] : hidden;
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
        for (int r = 0; r < 16; ++r) top = fmaxf(top, __builtin_fmaf(st[mb][r], a1, a0));
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
      for (int n = 0; n < 16; ++n) weights(st, pk, n, a0 + safe, sum);
    }
    l_run += sum;
  };
  // Value rows of which some rows of the workgroup see a part only: infinities and NaN among them (a wave looks at a quarter)
  const uint32_t v_quarter = lds0 + kBuffers * kTileBytes + wave * (kTileBytes / 4) + 16 * lane;
  auto find_odd = [&](uint32_t vbuf) __attribute__((always_inline)) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 x = *(const LdsU32x4*)(v_quarter + vbuf * kTileBytes + i * 1024);
#pragma unroll
      for (int w = 0; w < 4; ++w) found |= odd_bits<T>(x[w]);
    }
    if (__any(found != 0) && lane == 0) s_odd[vbuf] = 1;
  };
  // are multiplied apart: how many a row sees of those that lead to +inf and to -inf (a NaN is one of each) ...
  auto add_odd = [&](uint32_t vs, uint32_t s) __attribute__((always_inline)) {
    const Seen see = seen_of(s);
    const int32_t from = (int32_t)opaque((uint32_t)see.from);
    const uint32_t width = opaque(see.width);
    u32x4 ones[4];   // for the keys the row sees
#pragma unroll
    for (int cc = 0; cc < 4; ++cc)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        ones[cc][w] = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int32_t off = off_of(cc >> 1, 8 * (cc & 1) + 2 * w + h);
          ones[cc][w] |= (uint32_t)(off - from) < width ? Odd<T>::kOne << (16 * h) : 0u;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll 1
    for (int sign = 0; sign < 2; ++sign) {
      const uint32_t at = opaque(vs), but = both(Odd<T>::kInf | (sign ? 0u : 0x8000u));
      const float as = sign ? -INFINITY : INFINITY;
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        f32x16 n;
#pragma unroll
        for (int r = 0; r < 16; ++r) n[r] = 0.0f;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          n = Mfma<T>::m32x32x16(odd_values<T>(v_operand(at, cc, db), but), ones[cc], n);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[db][r] += n[r] > 0.0f ? as : 0.0f;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // ... and then taken out of the tile
  auto drop_odd = [&](uint32_t vbuf) __attribute__((always_inline)) {
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      LdsU32x4* at = (LdsU32x4*)(v_quarter + vbuf * kTileBytes + i * 1024);
      *at = finite_values<T>(*at);
    }
  };
  auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  // K of the walk's step i and V of the one before it on their way, into buffers i and i - 1 modulo kBuffers
  const uint32_t n_steps = end - step;
  auto send_pair = [&](uint32_t i) __attribute__((always_inline)) {
    // (V goes one step behind K: it is sent for first where K is to leave a part)
    if (i && i <= n_steps) {
      if (step + i - 1 == other_part) vsrc = source(p.v, p.prefix_v, other_part);
      send(vsrc, off_v, kBuffers + (i - 1) % kBuffers);
    }
    if (i < n_steps) {
      if (step + i == other_part) {
        aim(other_part);
        ksrc = source(p.k, p.prefix_k, other_part);
      }
      send(ksrc, off_k, i % kBuffers);
    }
  };
  // Turn t multiplies K of step t and V of step t - 1 (s + 1 and s, counted over the keys): P.V of a step runs beside the
  // weights of the next, whose vector instructions so find their place between the wave's own matrix instructions.
  // Weights swap registers from turn to turn; the first turn has no V, the last no K.
  auto turn = [&](u32x4 (&pk)[4], u32x4 (&next)[4], uint32_t t) __attribute__((always_inline)) {
    const uint32_t s = step + t - 1;
    // this wave's loads have arrived and its reads of the buffers to be filled are done; behind the barrier so have all
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    send_pair(t + 1);
    const uint32_t kbuf = t % kBuffers, vbuf = (t + 1) % kBuffers;
    const bool has_k = uniform(s + 1 >= w_begin && s + 1 < w_end) != 0, has_v = uniform(s + 1 > w_begin && s < w_end) != 0;
    const uint32_t vs = opaque(v_read + vbuf * kTileBytes);
    const bool look = t && partly(wg_lo, wg_hi, s);   // (the first turn has no V; the same for all waves)
    if (look) {
      find_odd(vbuf);
      meet();
      if (uniform(s_odd[vbuf])) {
        if (has_v) add_odd(vs, s);
        meet();
        drop_odd(vbuf);
        if (tid == 0) s_odd[vbuf] = 0;
        meet();
      }
    }
    // Weights against the reference that each row already has: while no lane's sum of them passes kMaxSum the step's
    // maximum is not looked for.  A row without a reference (neg_m = +inf) makes its sums infinite or NaN and so asks for
    // one; so does a score that is not finite.
    float sum = 0.0f;
    const float shift = a0 + neg_m;
    f32x16 st[2];
    u32x4 ring[kAhead];
    __builtin_amdgcn_s_setprio(0);
    if (has_k) {
      scores(st, ring, opaque(k_read + kbuf * kTileBytes), s + 1);
    } else {
      asm volatile("" : "=v"(st[0]), "=v"(st[1]));   // (whatever the registers hold: nothing comes of it)
    }
    __builtin_amdgcn_s_setprio(1);   // (P.V and the weights ahead of the other workgroup's Q.K: 1 to 9 %)
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
    send_pair(0);
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
  meet();   // (the others' last reads of the tiles)
  const uint32_t mine_lds = lds0 + (uint32_t)wave * (32 * kHeadDim * 4);
  const size_t at = (size_t)row.token * p.batch_pitch + row.seq;
  if (p.whole) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // (a row that sees no key is 0)
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u32x2 w;
        w[0] = Mfma<T>::pack2(oacc[db][4 * b] * inv, oacc[db][4 * b + 1] * inv);
        w[1] = Mfma<T>::pack2(oacc[db][4 * b + 2] * inv, oacc[db][4 * b + 3] * inv);
        *(LdsU32x2*)(mine_lds + j * kHeadDim * 2 + 16 * ((4 * db + b) ^ (j & 15)) + 8 * g) = w;
      }
    if (p.lse && g == 0 && row.valid) p.lse[at * p.n_q_heads + row.head] = (m + fast_log2(l)) * kLn2;
    const uint32_t to = (uint32_t)((at * p.n_q_heads + row.head));   // (below 2^31: rows of the whole call)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 4 * i + (lane >> 4);
      const u32x4 x = *(const LdsU32x4*)(mine_lds + r * kHeadDim * 2 + 16 * ((lane & 15) ^ (r & 15)));
      const size_t to_r = (uint32_t)__shfl((int)to, r);
      if (wave_row + r < n_rows) store16(p.out + to_r * kHeadDim + 8 * (lane & 15), x);
    }
    return;
  }
  const uint32_t part = ((row.token * p.batch + row.seq) * p.n_q_heads + row.head) * p.n_part + split + (on_prefix ? p.n_split : 0);
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *(LdsF32x4*)(mine_lds + j * kHeadDim * 4 + 16 * ((8 * db + 2 * b + g) ^ j)) =
          f32x4{oacc[db][4 * b], oacc[db][4 * b + 1], oacc[db][4 * b + 2], oacc[db][4 * b + 3]};
  if (g == 0 && row.valid) *(f32x2*)(p.part_ml + (size_t)part * 2) = f32x2{m, l};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 2 * i + g;
    const f32x4 x = *(const LdsF32x4*)(mine_lds + r * kHeadDim * 4 + 16 * (j ^ r));
    const size_t part_r = (uint32_t)__shfl((int)part, r);
    if (wave_row + r < n_rows) *(f32x4*)(p.part_o + part_r * kHeadDim + 4 * j) = x;
  }
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
hipError_t launch(const ShapedKernelArgs& p, bool cap, bool slopes, bool merge, hipStream_t stream) {
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
  if (e != hipSuccess || p.whole || !merge) return e;
  const size_t quads = (size_t)p.interval * p.batch * p.n_q_heads * (kHeadDim / 4);
  if (p.n_part > 8) {
    hipLaunchKernelGGL((shaped_merge_kernel<T, 8>), dim3((uint32_t)((quads * 8 + 255) / 256)), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((shaped_merge_kernel<T, 1>), dim3((uint32_t)((quads + 255) / 256)), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace

ShapedKernelArgs shaped_kernel_args(const ShapedArgs& args) {
  const AttnArgs& a = args.a;
  const ShapedState& s = args.s;
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
  p.rows_plane = a.position_interval * a.group;
  p.by_planes = divisor(a.batch * a.n_kv_heads);
  p.by_kv_heads = divisor(a.n_kv_heads);
  p.by_rows_plane = divisor(p.rows_plane);
  p.by_group = divisor(a.group);
  const ShapedScores f = shaped_scores(s, a.scale);
  p.c_in = f.c_in;
  p.a0 = f.a0;
  p.a1 = f.a1;
  return p;
}

namespace {

hipError_t launch_plan(const ShapedArgs& args, const ShapedPlan& plan, bool merge, hipStream_t stream) {
  const ShapedState& s = args.s;
  ShapedKernelArgs p = shaped_kernel_args(args);
  p.tiles_plane = plan.tiles_plane;
  p.n_split = plan.n_split;
  p.own_wgs = p.by_planes.d * plan.tiles_plane * plan.n_split;
  p.by_split = divisor(plan.n_split ? plan.n_split : 1);
  p.by_prefix_split = divisor(plan.prefix_split ? plan.prefix_split : 1);
  p.prefix_rows = plan.prefix_rows;
  p.prefix_tiles = plan.prefix_tiles;
  p.prefix_split = plan.prefix_split;
  p.n_part = plan.n_part;
  p.whole = merge && plan.n_part == 1;
  return args.a.dtype == 0 ? launch<F16>(p, s.cap != 0.0f, s.slopes != nullptr, merge, stream)
                           : launch<BF16>(p, s.cap != 0.0f, s.slopes != nullptr, merge, stream);
}

}  // namespace

hipError_t launch_shaped(const ShapedArgs& args, hipStream_t stream) {
  const AttnArgs& a = args.a;
  const ShapedState& s = args.s;
  const ShapedWalks keys = shaped_walks(a.position_index, a.position_interval, a.group, s.prefix, s.window);
  const ShapedPlan plan = shaped_plan(a.position_interval, a.batch, a.n_kv_heads, a.group, keys.own, s.prefix, a.n_cu, s.part_rows,
                                      s.window ? keys.both : 0);
  if (!a.positions && (!s.prefix || a.position_interval > 1)) {
    const double end = (double)s.prefix + a.position_index + a.position_interval;
    ShapedShape c{a.position_interval * a.group, a.batch * a.n_kv_heads, a.n_kv_heads, a.n_cu, (double)keys.both,
                  end - 0.5 * a.position_interval, (double)a.position_index + a.position_interval, (double)s.prefix, (double)keys.own};
    if (s.window) {
      if (s.window < c.mean) c.mean = s.window;
      if ((double)s.window + a.position_interval < c.rows) c.rows = (double)s.window + a.position_interval;
      if (c.prefix > c.mean) c.prefix = c.mean;
    }
    if (const uint32_t wr = shaped_short_rows(c, plan)) return launch_shaped_short(args, wr, shaped_short_along(c.planes, c.longest), stream);
  }
  return launch_plan(args, plan, true, stream);
}

hipError_t launch_shaped_prefix(const ShapedArgs& args, uint32_t* parts, hipStream_t stream) {
  const AttnArgs& a = args.a;
  const ShapedState& s = args.s;
  const ShapedPlan plan = shaped_prefix_plan(a.batch, a.n_kv_heads, a.group, s.prefix, a.n_cu, s.part_rows);
  if (plan.n_part == 0) return hipErrorInvalidValue;
  *parts = plan.n_part;
  return launch_plan(args, plan, false, stream);
}

}  // namespace ellm
