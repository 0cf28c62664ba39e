// Writes into a cache in 8 bits and reads from it (e4m3.hpp has the format): [token][sequence][kv_head][128] rows of 16 bits
// to their positions, the keys normalised and rotated on the way or as they are, and back.
//
// What bounds them is memory: a K and a V row are 512 bytes in 16 bits and 258 in 8, each touched once; for single tokens the
// launch.  Sixteen lanes own a row, eight elements each (16-byte loads, 8-byte stores, whole lines either way); the row's
// largest magnitude and the sum of its squares go round the sixteen by DPP, four steps each, and a row's place costs two
// multiplications (64-bit divisions and exchanges through LDS: 427 vector instructions a row against 259).
// Measured (bfloat16, four heads, key rows normalised and rotated / as they are / read): 2048 tokens 3.7 / 3.3 / 3.0 us, 16384
// 12.8 / 11.4 / 11.3 us (4.4 TB/s; a plain copy of the same bytes, 12.0 us), 131072 72.7 / 71.4 / 72.2 us (5.6 TB/s; a copy, 5.35).
// Two or four rows a lane on their way at once: 13.4 / 12.0 / 11.1 and 13.6 / 12.6 / 11.0 us at 16384, 4.6 and 6.6 us at 2048.
// Stores that may stay in the caches: 12.1 / 12.0 / 12.0 us at 16384, but 81.8 / 68.4 / 73.1 at 131072.
#include <algorithm>

#include "e4m3.hpp"
#include "kernels.hpp"

namespace ellm {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsWg = kThreads / 16;
constexpr size_t kMaxBlocks = 16384;
constexpr size_t kMaxRows = (size_t)1 << 31;   // (554 GB of rows)

// floor(n / d) for n < 2^31 as one multiplication, floor(n m / 2^(31 + s)) with s = ceil(log2 d) and m = ceil(2^(31 + s) / d), below
// 2^32: m d is 2^(31 + s) and less than d more, so n m / 2^(31 + s) is n / d and less than n / 2^(31 + s) <= 1 / d more.
struct Divisor {
  uint32_t d, m, s;
  explicit Divisor(uint32_t by) : d(by), m(0), s(0) {
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << 31 << s) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return __umulhi(2 * n, m) >> s; }
};

struct WriteArgs {
  uint8_t* k_dst;
  uint8_t* v_dst;
  uint8_t* k_scale;
  uint8_t* v_scale;
  const uint16_t* k_src;
  const uint16_t* v_src;
  const uint16_t* rope;
  const uint32_t* positions;
  KvLayout layout;
  Divisor heads, batch;
  size_t skip;   // source rows between the tokens' rows
  uint32_t rows, tokens, position_index, max_start;   // rows: tokens x batch x heads
  float eps;
};

template <typename T, bool NORM>
__global__ __launch_bounds__(kThreads) void kv_append_e4m3_kernel(WriteArgs p) {
  const uint32_t c = threadIdx.x & 15;
  // every lane of a wave runs the same number of trips: the loop holds lane exchanges
  for (uint32_t first = blockIdx.x * kRowsWg; first < p.rows; first += gridDim.x * kRowsWg) {
    uint32_t row = first + (threadIdx.x >> 4);
    bool live = row < p.rows;
    if (!live) row = 0;
    const uint32_t tb = p.heads.quotient(row), h = row - tb * p.heads.d, t = p.batch.quotient(tb), b = tb - t * p.batch.d;
    const size_t src = ((size_t)t * p.skip + row) * kHeadDim + 8 * c;
    const u32x4 kraw = load16_once(p.k_src + src), vraw = load16_once(p.v_src + src);
    const uint32_t pos = (p.positions ? min(p.positions[b], p.max_start) : p.position_index) + t;
    uint32_t pos_dst = pos;
    if (p.layout.seq_caps) {   // the sequence's capacity bounds its rows: of several tokens from its last row on, the last one stays
      const uint32_t last = p.layout.seq_caps[b] - 1;
      pos_dst = min(pos, last);
      live = live && (pos < last || t + 1 == p.tokens);
    }
    const size_t dst = seq_plane_offset(p.layout.seq_offsets, p.layout.stride_seq, b) + (size_t)h * p.layout.stride_head +
                       (size_t)pos_dst * kHeadDim;
    float x[8];
    unpack8<T>(kraw, x);
    if constexpr (NORM) norm_rope8<T>(x, load16(p.rope + (size_t)pos * kHeadDim + 8 * c), p.eps);
    uint32_t kb, vb;
    const u32x2 k = row_codes16<T>(x, kb);
    unpack8<T>(vraw, x);
    const u32x2 v = row_codes16<T>(x, vb);
    if (live) {
      __builtin_nontemporal_store(k, (u32x2*)(p.k_dst + dst + 8 * c));
      __builtin_nontemporal_store(v, (u32x2*)(p.v_dst + dst + 8 * c));
      if (c == 0) {
        p.k_scale[dst / kHeadDim] = (uint8_t)kb;
        p.v_scale[dst / kHeadDim] = (uint8_t)vb;
      }
    }
  }
}

struct ReadArgs {
  const uint8_t* k;
  const uint8_t* v;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  uint16_t* k_dst;
  uint16_t* v_dst;
  KvLayout layout;
  Divisor tokens, heads;
  size_t dst_token, dst_sequence, dst_head;
  uint32_t rows, position_index;   // rows: batch x heads x tokens, tokens fastest: the order of the cache
};

template <typename T>
__global__ __launch_bounds__(kThreads) void kv_read_e4m3_kernel(ReadArgs p) {
  const uint32_t c = threadIdx.x & 15;
  for (uint32_t row = blockIdx.x * kRowsWg + (threadIdx.x >> 4); row < p.rows; row += gridDim.x * kRowsWg) {
    const uint32_t bh = p.tokens.quotient(row), t = row - bh * p.tokens.d, b = p.heads.quotient(bh), h = bh - b * p.heads.d;
    const size_t src = seq_plane_offset(p.layout.seq_offsets, p.layout.stride_seq, b) + (size_t)h * p.layout.stride_head +
                       (size_t)(p.position_index + t) * kHeadDim;
    const u32x2 k = __builtin_nontemporal_load((const u32x2*)(p.k + src + 8 * c));
    const u32x2 v = __builtin_nontemporal_load((const u32x2*)(p.v + src + 8 * c));
    const uint32_t ks = p.k_scale[src / kHeadDim], vs = p.v_scale[src / kHeadDim];
    const size_t dst = t * p.dst_token + b * p.dst_sequence + h * p.dst_head + 8 * c;
    store16_once(p.k_dst + dst, values8<T>(k, ks));
    store16_once(p.v_dst + dst, values8<T>(v, vs));
  }
}

}  // namespace

hipError_t launch_kv_append_e4m3(const KvE4m3& cache, const void* k_src, const void* v_src, const void* rope,
                                 const uint32_t* positions, uint32_t n_tokens, uint32_t batch, uint32_t src_batch_pitch,
                                 uint32_t n_kv_heads, const KvLayout& layout, uint32_t position_index, uint32_t max_start,
                                 float eps, int dtype, hipStream_t stream) {
  const size_t rows = (size_t)n_tokens * batch * n_kv_heads;
  if (rows == 0) return hipSuccess;
  if (rows >= kMaxRows) return hipErrorInvalidValue;
  const WriteArgs p{cache.k, cache.v, cache.k_scale, cache.v_scale, (const uint16_t*)k_src, (const uint16_t*)v_src,
                    (const uint16_t*)rope, positions, layout, Divisor(n_kv_heads), Divisor(batch),
                    (size_t)(src_batch_pitch - batch) * n_kv_heads, (uint32_t)rows, n_tokens, position_index, max_start, eps};
  const size_t blocks = std::min((rows + kRowsWg - 1) / kRowsWg, kMaxBlocks);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, stream, p); };
  if (rope)
    dtype == 0 ? go(kv_append_e4m3_kernel<F16, true>) : go(kv_append_e4m3_kernel<BF16, true>);
  else
    dtype == 0 ? go(kv_append_e4m3_kernel<F16, false>) : go(kv_append_e4m3_kernel<BF16, false>);
  return hipGetLastError();
}

hipError_t launch_kv_read_e4m3(const KvE4m3& cache, void* k_dst, void* v_dst, size_t dst_token, size_t dst_sequence,
                               size_t dst_head, uint32_t n_tokens, uint32_t batch, uint32_t n_kv_heads,
                               const KvLayout& layout, uint32_t position_index, int dtype, hipStream_t stream) {
  const size_t rows = (size_t)n_tokens * batch * n_kv_heads;
  if (rows == 0) return hipSuccess;
  if (rows >= kMaxRows) return hipErrorInvalidValue;
  const ReadArgs p{cache.k, cache.v, cache.k_scale, cache.v_scale, (uint16_t*)k_dst, (uint16_t*)v_dst, layout,
                   Divisor(n_tokens), Divisor(n_kv_heads), dst_token, dst_sequence, dst_head, (uint32_t)rows, position_index};
  const size_t blocks = std::min((rows + kRowsWg - 1) / kRowsWg, kMaxBlocks);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, stream, p); };
  dtype == 0 ? go(kv_read_e4m3_kernel<F16>) : go(kv_read_e4m3_kernel<BF16>);
  return hipGetLastError();
}

}  // namespace ellm
