// Short walks with shaped scores (shaped.hpp has the formulas): chunks on a few hundred to a thousand or two keys.
//
// There the tile kernel's walk is a chain of a few steps between a start and an end that cost as much, and a split of it
// needs a second launch.  Here a workgroup of four waves owns 32 WR query rows of a K/V plane; its 4 / WR groups of WR waves
// take the keys in turns of 32, each group with tiles of its own in LDS, and meet once, in LDS: the longest walk is a
// quarter (WR = 1) or half (WR = 2) of a row's keys and nothing leaves the workgroup.  WR = 2 fetches every key row half as often.
// Products, masks and references are those of the tile kernel (shaped_chunk.hip): S^T = K . Q^T and O^T += V^T . P^T on
// 32x32x16 instructions, one key range [lo, hi) a row, references that move where a sum of weights asks for it, values that
// are not finite multiplied apart where only some rows see them, walks from the last key where scores fall with distance.
// What bounds it: the chain of turns, 1.05 us each (32 keys: fetch, eight products, scores and weights, eight products), and up
// to 6 us of launch, start and end.  Capped, binary16, us, tile kernel / this: 33 tokens x 5 on 777, 32 / 4 heads, 19.7 / 12.9; 241
// tokens 12.7 / 7.5; 16 x 5 on 500, 32 / 32 heads, 19.9 / 10.6; 8 x 5 on 1500 42.2 / 21.7; 618 tokens 24.0 / 16.8; 40 x 2 on 100
// behind a prefix of 300, 64 / 8 heads, 19.8 / 10.4 (shaped_plan.hpp chooses).  The two kernels of plain scores it stands beside
// take 11.2, 7.0 and 9.4 us for the first three; this one without a cap 11.6, 6.9 and 9.2.
#include "shaped_common.hpp"

namespace ellm {
namespace {

constexpr int kThreads = 4 * kWave;
constexpr int kKeys = 32;                                  // keys a turn of a group
constexpr int kTileBytes = kKeys * kHeadDim * 2;           // of K, and of V

// Waits for this wave's LDS accesses, then for the workgroup's waves (loads on their way to registers stay there).
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// PREFIX: there is a shared prefix, whose last tile may be a part of one (6 % of a walk without it).
template <typename T, bool CAP, bool SLOPES, bool PREFIX, int WR>
__global__ __launch_bounds__(kThreads, 2) void shaped_short_kernel(ShapedKernelArgs p) {
  constexpr int kGroups = 4 / WR;
  constexpr int kBufs = WR == 1 ? 1 : 2;     // (one wave: its LDS accesses are in order, no second buffer)
  constexpr int kPieces = 8 / WR;            // 16-byte pieces of K, and of V, that a lane moves a turn
  constexpr int kRows = 32 * WR;
  constexpr int kAhead = 4;                  // LDS operand reads ahead of their products
  // Tiles [group][buffer][K, V][32][128], pieces of a row permuted as in the tile kernel; then sums [group][row][128].
  constexpr int kBytes = kGroups * kBufs * 2 * kTileBytes;
  static_assert(kGroups * kRows * kHeadDim * 4 <= kBytes, "the groups' sums fit in the tiles' room");
  __shared__ __attribute__((aligned(256))) uint16_t smem[kBytes / 2];
  __shared__ f32x2 s_ml[kGroups * kRows];
  __shared__ uint32_t s_reach[WR][4], s_odd[kBufs];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = (int)uniform((uint32_t)tid >> 6);
  const int rw = wave % WR, kg = wave / WR;
  const int j = lane & 31, g = lane >> 5;

  // ---- which rows, which keys they see ------------------------------------------------------------
  // Longest walks of causal prompts first; planes fastest, or, where planes overflow the XCDs' caches or are dealt unevenly
  // to them, one XCD (workgroup id % 8) along a plane's tiles.
  uint32_t plane, order;
  if (p.along) {
    const uint32_t n = blockIdx.x >> 3, eight = p.by_tiles.quotient(n);
    plane = (blockIdx.x & 7) + 8 * eight;
    order = p.by_tiles.rest(n, eight);
  } else {
    order = p.by_planes.quotient(blockIdx.x);
    plane = p.by_planes.rest(blockIdx.x, order);
  }
  if (plane >= p.by_planes.d) return;
  const uint32_t row0 = kRows * (p.tiles_plane - 1 - order), n_rows = p.rows_plane;
  const uint32_t seq = p.by_kv_heads.quotient(plane), kvh = p.by_kv_heads.rest(plane, seq);
  const uint32_t wave_row = row0 + 32 * rw, r_here = min(wave_row + j, n_rows - 1);
  const bool valid = wave_row + j < n_rows;
  const uint32_t token = p.by_group.quotient(r_here), head = kvh * p.group + p.by_group.rest(r_here, token);
  u32x4 qreg[8];
  {
    const uint16_t* qrow = p.q + token * p.q_token_stride + ((size_t)seq * p.n_q_heads + head) * kHeadDim;
#pragma unroll
    for (int s = 0; s < 8; ++s) qreg[s] = load16(qrow + 16 * s + 8 * g);
  }
  const float slope2 = SLOPES ? p.slopes[head] * kLog2e : 0.0f;

  struct Reach {
    uint32_t lo, hi;           // the keys that any row sees (lo >= hi: none)
    uint32_t all_lo, all_hi;   // the keys that every row sees
  };
  Reach mine, all;   // the wave's, the workgroup's
  auto first_seen = [&](uint32_t pos) { return p.window && pos + 1 > p.window ? pos + 1 - p.window : 0u; };
  // (read again where it is needed: as a value kept around the loop it costs the walks of one wave 80 spilled registers)
  auto prefix = [&]() __attribute__((always_inline)) { return PREFIX ? p.prefix : 0u; };
  const uint32_t base = prefix() + p.position, pos = base + token;   // (key ranges do not go with a prefix)
  uint32_t lo = first_seen(pos), hi = pos + 1;
  if (uniform(!p.key_begin && !p.key_end)) {   // ranges that move on with the rows
    auto reach = [&](uint32_t first, uint32_t last) {
      if (first >= n_rows) return Reach{kNoKey, 0u, 0u, kNoKey};
      const uint32_t a = base + p.by_group.quotient(first), b = base + p.by_group.quotient(min(last, n_rows - 1));
      return Reach{first_seen(a), b + 1, first_seen(b), a + 1};
    };
    mine = reach(wave_row, wave_row + 31);
    all = reach(row0, row0 + kRows - 1);
  } else {
    if (p.key_begin) lo = max(lo, p.key_begin[seq * p.bounds_pitch + pos]);
    if (p.key_end) hi = min(p.key_end[seq * p.bounds_pitch + pos], p.seq_caps ? p.seq_caps[seq] : p.capacity);
    if (lo >= hi) lo = hi = 0;   // sees nothing
    const bool live = valid && lo < hi;
    mine = Reach{live ? lo : kNoKey, live ? hi : 0u, valid ? lo : 0u, valid ? hi : kNoKey};
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      mine.lo = min(mine.lo, (uint32_t)__shfl_xor((int)mine.lo, x));
      mine.hi = max(mine.hi, (uint32_t)__shfl_xor((int)mine.hi, x));
      mine.all_lo = max(mine.all_lo, (uint32_t)__shfl_xor((int)mine.all_lo, x));
      mine.all_hi = min(mine.all_hi, (uint32_t)__shfl_xor((int)mine.all_hi, x));
    }
    all = mine;
    if constexpr (WR > 1) {
      if (kg == 0 && lane == 0) {
        s_reach[rw][0] = mine.lo;
        s_reach[rw][1] = mine.hi;
        s_reach[rw][2] = mine.all_lo;
        s_reach[rw][3] = mine.all_hi;
      }
      meet();
#pragma unroll
      for (int w = 0; w < WR; ++w)
        all = Reach{min(all.lo, s_reach[w][0]), max(all.hi, s_reach[w][1]), max(all.all_lo, s_reach[w][2]), min(all.all_hi, s_reach[w][3])};
    }
  }
  if (!valid) lo = 0, hi = kNoKey;   // (rows that are not stored never ask for a mask)
  const uint32_t w_lo = uniform(mine.lo), w_hi = uniform(mine.hi), all_lo = uniform(mine.all_lo), all_hi = uniform(mine.all_hi);
  const uint32_t hull_lo = uniform(all.lo), hull_hi = uniform(all.hi), wg_lo = uniform(all.all_lo), wg_hi = uniform(all.all_hi);
  const uint32_t prefix_tiles = (prefix() + kKeys - 1) / kKeys;
  auto tile_of = [&](uint32_t key) { return key < prefix() ? key / kKeys : prefix_tiles + (key - prefix()) / kKeys; };
  const uint32_t first = tile_of(hull_lo), n_tiles = hull_lo < hull_hi ? tile_of(hull_hi - 1) + 1 - first : 0u;
  auto place = [&](uint32_t i) { return SLOPES ? first + n_tiles - 1 - i : first + i; };   // of the walk's tile i among the keys'
  auto key_of = [&](uint32_t i) {   // its first key
    const uint32_t at = place(i);
    return at < prefix_tiles ? at * kKeys : prefix() + (at - prefix_tiles) * kKeys;
  };
  auto keys_end = [&](uint32_t i) { return place(i) < prefix_tiles ? min(prefix(), key_of(i) + kKeys) : key_of(i) + kKeys; };

  // ---- staging: memory -> registers -> the group's tiles ------------------------------------------------
  const size_t plane_at = seq_plane_offset(p.seq_offsets, p.kv_stride_seq, seq) + kvh * p.kv_stride_head;
  const int ld_r = 4 * rw + (lane >> 4), ld_x = lane & 15;   // rows ld_r + 4 WR i
  u32x4 kst[kPieces], vst[kPieces];
  auto load = [&](uint32_t i) __attribute__((always_inline)) {
    const bool ahead = place(i) < prefix_tiles;   // (uniform)
    const uint32_t skip = ahead ? key_of(i) : key_of(i) - prefix(), n = ahead ? prefix() : hull_hi - prefix();
    const uint32_t pitch = 2 * (uint32_t)(ahead ? p.prefix_stride_pos : p.kv_stride_pos);   // bytes; 32 rows of it stay below 2^31
    const size_t plane = ahead ? kvh * p.prefix_stride_head : plane_at;
    // (bytes up to the end of the last row that is read: rows past it read as zeros)
    const uint64_t off = 2 * plane + (uint64_t)skip * pitch, left = (uint64_t)(n - 1 - skip) * pitch + 2 * kHeadDim;
    const uint32_t room = uniform(left >> 32 ? 0xffffffffu : (uint32_t)left);
    const uint64_t kat = uniform64((uint64_t)(ahead ? p.prefix_k : p.k) + off), vat = uniform64((uint64_t)(ahead ? p.prefix_v : p.v) + off);
    const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc((void*)kat, 0, room, kBufferFlags);
    const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc((void*)vat, 0, room, kBufferFlags);
    const uint32_t from = opaque(ld_r) * pitch + 16 * ld_x;   // (sums formed here, not kept around the loop)
#pragma unroll
    for (int n = 0; n < kPieces; ++n) kst[n] = __builtin_amdgcn_raw_buffer_load_b128(kr, from + 4 * WR * n * pitch, 0, 0);
#pragma unroll
    for (int n = 0; n < kPieces; ++n) vst[n] = __builtin_amdgcn_raw_buffer_load_b128(vr, from + 4 * WR * n * pitch, 0, 0);
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(LdsHalf*)smem + kg * kBufs * 2 * kTileBytes;
  // whether rows of the workgroup see a part of tile i only: its values may then hold anything where they are not seen
  auto look = [&](uint32_t i) {
    const uint32_t kb = key_of(i);
    return uniform(wg_lo > kb || wg_hi < kb + kKeys) != 0;
  };
  // (found in it: this wave's to know where the tile is its own, the workgroup's else)
  auto store = [&](uint32_t i, uint32_t buf) __attribute__((always_inline)) {
    const uint32_t x = opaque(ld_x);
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      const uint32_t r = ld_r + 4 * WR * n, at = lds0 + buf * 2 * kTileBytes + r * kHeadDim * 2;
      *(LdsU32x4*)(at + 16 * (x ^ (r & 15))) = kst[n];
      *(LdsU32x4*)(at + kTileBytes + 16 * (x ^ (4 * (r & 3)))) = vst[n];
    }
    if (look(i)) {
      uint32_t found = 0;
#pragma unroll
      for (int n = 0; n < kPieces; ++n)
#pragma unroll
        for (int w = 0; w < 4; ++w) found |= odd_bits<T>(vst[n][w]);
      const bool any = __any(found != 0) != 0;
      if (WR == 1) return any;
      if (any && lane == 0) s_odd[buf] = 1;
    }
    return false;
  };
  // operand addresses as in the tile kernel
  const uint32_t k_read = lds0 + j * kHeadDim * 2 + 16 * (g ^ (j & 15));
  const int v_row = 4 * g + ((lane & 15) >> 2), v_piece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_read = lds0 + kTileBytes + v_row * kHeadDim * 2 + 16 * (v_piece ^ (4 * (v_row & 3))) + 8 * (lane & 1);
  auto v_operand = [&](uint32_t base, int cc, int db) {
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

  // ---- a turn -------------------------------------------------------------------------------------
  // minus the row's reference (log2 units; +inf: no key seen yet; rows that see none need none), this lane's share of its sum
  float neg_m = lo < hi ? INFINITY : 0.0f, l_run = 0.0f;
  f32x16 oacc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[db][r] = 0.0f;
  const float a0 = SLOPES ? 0.0f : p.a0, a1 = SLOPES ? 1.0f : p.a1;
  const float hidden = a1 < 0.0f ? INFINITY : -INFINITY;
  auto off_of = [](int r) { return 8 * (r >> 2) + (r & 3); };   // keys of the lane: first key + 4 g + off
  bool started = false;
  struct Seen {   // which keys of a tile a row sees: off - from < width, unsigned
    int32_t from;
    uint32_t width;
  };
  auto seen_of = [&](uint32_t i) {
    const uint32_t last = min(hi, keys_end(i));
    return Seen{(int32_t)(lo - key_of(i)) - 4 * g, last > lo ? last - lo : 0u};
  };

  // Values that are not finite are multiplied apart, how many a row sees of those that lead to +inf and to -inf (a NaN is one
  // of each) ...
  auto add_odd = [&](uint32_t i, uint32_t buf) __attribute__((always_inline)) {
    const Seen see = seen_of(i);
    const uint32_t vs = v_read + buf * 2 * kTileBytes, width = opaque(see.width);
    const int32_t from = (int32_t)opaque((uint32_t)see.from);
    u32x4 ones[2];   // for the keys the row sees
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      ones[n >> 2][n & 3] = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        ones[n >> 2][n & 3] |= (uint32_t)(off_of(2 * n + h) - from) < width ? Odd<T>::kOne << (16 * h) : 0u;
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
        for (int cc = 0; cc < 2; ++cc) {
          n = Mfma<T>::m32x32x16(odd_values<T>(v_operand(at, cc, db), but), ones[cc], n);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[db][r] += n[r] > 0.0f ? as : 0.0f;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // ... and then taken out of the tile, each of the group's waves its share
  auto drop_odd = [&](uint32_t buf) __attribute__((always_inline)) {
    const uint32_t at = lds0 + (2 * buf + 1) * kTileBytes + 16 * opaque(kWave * rw + lane);
#pragma unroll 1
    for (int n = 0; n < kPieces; ++n) {
      LdsU32x4* x = (LdsU32x4*)(at + n * 16 * WR * kWave);
      *x = finite_values<T>(*x);
    }
  };

  auto compute = [&](uint32_t i, uint32_t buf) __attribute__((always_inline)) {
    const uint32_t kb = key_of(i), ke = keys_end(i);
    if (uniform(kb >= w_hi || ke <= w_lo)) return;
    const uint32_t ks = opaque(k_read + buf * 2 * kTileBytes), vs = opaque(v_read + buf * 2 * kTileBytes);
    f32x16 st;
#pragma unroll
    for (int r = 0; r < 16; ++r) st[r] = 0.0f;
    // operands are read kAhead ahead of the products that take them, those of V ahead of the weights (the scheduling
    // barriers keep the order as it is written: by itself the compiler reads one, waits, multiplies)
    u32x4 ring[kAhead];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) ring[n] = *(const LdsU32x4*)(ks ^ (32 * n));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      st = Mfma<T>::m32x32x16(ring[s % kAhead], qreg[s], st);
      if (s + kAhead < 8)
        ring[s % kAhead] = *(const LdsU32x4*)(ks ^ (32 * (s + kAhead)));
      else
        ring[s % kAhead] = v_operand(vs, (s + kAhead - 8) >> 2, (s + kAhead - 8) & 3);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (CAP || SLOPES) {
      const float dist = SLOPES ? (float)((int32_t)(pos - kb) - 4 * g) : 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float x = st[r];
        if constexpr (CAP) x = __builtin_amdgcn_rcpf(fast_exp2(x * p.c_in) + 1.0f);
        if constexpr (SLOPES) x = __builtin_fmaf(x, p.a1, __builtin_fmaf(-slope2, fabsf(dist - (float)off_of(r)), p.a0));
        st[r] = x;
      }
    }
    if (uniform(all_lo > kb || all_hi < kb + kKeys || ke < kb + kKeys)) {
      const Seen see = seen_of(i);
#pragma unroll
      for (int r = 0; r < 16; ++r) st[r] = (uint32_t)(off_of(r) - see.from) < see.width ? st[r] : hidden;
    }
    // Weights against the reference that each row already has; where their sum passes kMaxSum (or a row has none yet) rows
    // move to the turn's maximum and have them computed again.
    u32x4 pk[2];
    float sum = INFINITY;
    auto weights = [&](float shift) __attribute__((always_inline)) {
      sum = 0.0f;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const float p0 = fast_exp2(__builtin_fmaf(st[2 * n], a1, shift)), p1 = fast_exp2(__builtin_fmaf(st[2 * n + 1], a1, shift));
        pk[n >> 2][n & 3] = Mfma<T>::pack2(p0, p1);
        sum += p0 + p1;
      }
    };
    if (started) weights(a0 + neg_m);
    started = true;
    const uint64_t over = __ballot(!(sum <= Mfma<T>::kMaxSum));
    if (over) {
      float top = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, __builtin_fmaf(st[r], a1, a0));
      top = max_with_partner_half(top);
      const bool moves = (((over >> j) | (over >> (j + 32))) & 1) != 0;   // (by what the row's own two lanes saw)
      const float neg_new = moves ? fminf(neg_m, -top) : neg_m;           // (+inf while the row has seen no key)
      const float safe = neg_new == INFINITY ? 0.0f : neg_new;
      const float alpha = neg_m == INFINITY ? 1.0f : fast_exp2(safe - neg_m);
      neg_m = neg_new;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db) oacc[db] *= alpha;
      weights(a0 + safe);
    }
    l_run += sum;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      oacc[n & 3] = Mfma<T>::m32x32x16(ring[n % kAhead], pk[n >> 2], oacc[n & 3]);
      if (n + kAhead < 8) ring[n % kAhead] = v_operand(vs, (n + kAhead) >> 2, (n + kAhead) & 3);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // ---- walk ---------------------------------------------------------------------------------------
  if ((uint32_t)kg < n_tiles) load(kg);
  if constexpr (WR == 1) {
    for (uint32_t i = kg; i < n_tiles; i += kGroups) {
      const bool odd = store(i, 0);
      if (i + kGroups < n_tiles) load(i + kGroups);
      __builtin_amdgcn_wave_barrier();
      if (uniform(odd)) {
        add_odd(i, 0);
        __builtin_amdgcn_wave_barrier();
        drop_odd(0);
        __builtin_amdgcn_wave_barrier();
      }
      compute(i, 0);
      __builtin_amdgcn_wave_barrier();
    }
  } else {   // every group makes the same number of turns, so that all meet at the barriers
    const uint32_t n_turns = (n_tiles + kGroups - 1) / kGroups;
    if (tid < kBufs) s_odd[tid] = 0;
    meet();
    if ((uint32_t)kg < n_tiles) (void)store(kg, 0);
    if ((uint32_t)kg + kGroups < n_tiles) load(kg + kGroups);
    meet();
    for (uint32_t t = 0; t < n_turns; ++t) {
      const uint32_t i = kg + kGroups * t, buf = t & 1;
      if (uniform(s_odd[buf])) {
        if (i < n_tiles) add_odd(i, buf);
        meet();
        if (i < n_tiles) drop_odd(buf);
        if (tid == 0) s_odd[buf] = 0;
        meet();
      }
      if (i < n_tiles) compute(i, buf);
      if (i + kGroups < n_tiles) {
        (void)store(i + kGroups, buf ^ 1);
        if (i + 2 * kGroups < n_tiles) load(i + 2 * kGroups);
      }
      meet();
    }
  }

  // ---- the groups' rows meet in LDS; sixteen lanes finish a row ---------------------------------------------
  const float l_wave = sum_with_partner_half(l_run);
  const uint32_t red = (uint32_t)(uintptr_t)(LdsHalf*)smem;
  auto at_piece = [&](uint32_t group, uint32_t row, uint32_t piece) {   // four of a row's 128 sums
    return red + (group * kRows + row) * kHeadDim * 4 + 16 * (piece ^ (row & 31));
  };
  meet();   // (the others' last reads of the tiles)
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *(LdsF32x4*)at_piece(kg, 32 * rw + j, 8 * db + 2 * b + g) =
          f32x4{oacc[db][4 * b], oacc[db][4 * b + 1], oacc[db][4 * b + 2], oacc[db][4 * b + 3]};
  if (g == 0) s_ml[kg * kRows + 32 * rw + j] = f32x2{l_wave == 0.0f ? -INFINITY : -neg_m, l_wave};
  meet();
#pragma unroll
  for (int n = 0; n < kRows * 16 / kThreads; ++n) {
    const uint32_t rr = kThreads / 16 * n + (tid >> 4), d8 = tid & 15, r = row0 + rr;
    if (r >= n_rows) continue;
    float ms[kGroups], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < kGroups; ++w) {
      ms[w] = s_ml[w * kRows + rr][0];
      m = fmaxf(m, ms[w]);
    }
    f32x4 o[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int w = 0; w < kGroups; ++w) {
      const float weight = ms[w] == -INFINITY ? 0.0f : fast_exp2(ms[w] - m);
      l += weight * s_ml[w * kRows + rr][1];
      o[0] += weight * *(const LdsF32x4*)at_piece(w, rr, 2 * d8);
      o[1] += weight * *(const LdsF32x4*)at_piece(w, rr, 2 * d8 + 1);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;   // (a row that sees no key is 0)
    const uint32_t t = p.by_group.quotient(r), h = kvh * p.group + p.by_group.rest(r, t);
    u32x4 w4;
#pragma unroll
    for (int e = 0; e < 4; ++e) w4[e] = Mfma<T>::pack2(o[e >> 1][2 * (e & 1)] * inv, o[e >> 1][2 * (e & 1) + 1] * inv);
    store16(p.out + (size_t)t * p.q_token_stride + ((size_t)seq * p.n_q_heads + h) * kHeadDim + 8 * d8, w4);
    if (p.lse && d8 == 0) p.lse[((size_t)t * p.batch_pitch + seq) * p.n_q_heads + h] = (m + fast_log2(l)) * kLn2;
  }
}

template <typename T, bool PREFIX, int WR>
hipError_t launch(const ShapedKernelArgs& p, uint32_t wgs, bool cap, bool slopes, hipStream_t stream) {
  const dim3 grid(wgs), block(kThreads);
  if (cap && slopes)
    hipLaunchKernelGGL((shaped_short_kernel<T, true, true, PREFIX, WR>), grid, block, 0, stream, p);
  else if (cap)
    hipLaunchKernelGGL((shaped_short_kernel<T, true, false, PREFIX, WR>), grid, block, 0, stream, p);
  else if (slopes)
    hipLaunchKernelGGL((shaped_short_kernel<T, false, true, PREFIX, WR>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((shaped_short_kernel<T, false, false, PREFIX, WR>), grid, block, 0, stream, p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch(const ShapedKernelArgs& p, uint32_t wgs, uint32_t wr, bool cap, bool slopes, hipStream_t stream) {
  if (p.prefix) return wr == 1 ? launch<T, true, 1>(p, wgs, cap, slopes, stream) : launch<T, true, 2>(p, wgs, cap, slopes, stream);
  return wr == 1 ? launch<T, false, 1>(p, wgs, cap, slopes, stream) : launch<T, false, 2>(p, wgs, cap, slopes, stream);
}

}  // namespace

hipError_t launch_shaped_short(const ShapedArgs& args, uint32_t wr, bool along, hipStream_t stream) {
  const AttnArgs& a = args.a;
  ShapedKernelArgs p = shaped_kernel_args(args);
  const uint32_t planes = a.batch * a.n_kv_heads, rows = 32 * wr;
  p.tiles_plane = shaped_ceil(p.rows_plane, rows);
  p.by_tiles = divisor(p.tiles_plane);
  p.along = along;
  const uint32_t wgs = p.along ? (planes + 7) / 8 * 8 * p.tiles_plane : planes * p.tiles_plane;
  const bool cap = args.s.cap != 0.0f, slopes = args.s.slopes != nullptr;
  return a.dtype == 0 ? launch<F16>(p, wgs, wr, cap, slopes, stream) : launch<BF16>(p, wgs, wr, cap, slopes, stream);
}

}  // namespace ellm
