// Writes into a cache in 8 bits and reads from it (e4m3.hpp has the format): [token][sequence][kv_head][128] rows of 16 bits
// to their positions, the keys normalised and rotated on the way or as they are, and back.
//
// What bounds them is memory: a K and a V row are 512 bytes in 16 bits and 258 in 8, each touched once; for single tokens the
// launch.  Sixteen lanes own a row, eight elements each (16-byte loads, 8-byte stores, whole lines either way); the
// row's largest magnitude and the sum of its squares go round the sixteen by lane exchanges, four steps each.
#include "e4m3.hpp"
#include "kernels.hpp"

namespace ellm {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsWg = kThreads / 16;

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
  size_t rows;   // n_tokens x batch x n_kv_heads
  uint32_t batch, src_batch_pitch, n_kv_heads, position_index, max_start;
  float eps;
};

template <typename T, bool NORM>
__global__ __launch_bounds__(kThreads) void kv_append_e4m3_kernel(WriteArgs p) {
  const uint32_t c = threadIdx.x & 15;
  // every lane of a wave runs the same number of trips: the loop holds lane exchanges
  const size_t rows_per_pass = (size_t)gridDim.x * kRowsWg;
  const size_t passes = (p.rows + rows_per_pass - 1) / rows_per_pass;
  for (size_t pass = 0; pass < passes; ++pass) {
    const size_t row = pass * rows_per_pass + (size_t)blockIdx.x * kRowsWg + (threadIdx.x >> 4);
    const bool live = row < p.rows;
    size_t r = live ? row : 0;
    const uint32_t h = r % p.n_kv_heads;
    r /= p.n_kv_heads;
    const uint32_t b = r % p.batch, t = r / p.batch;
    const uint32_t pos = (p.positions ? min(p.positions[b], p.max_start) : p.position_index) + t;
    // (per-sequence capacities, where the cache has them, bound the row written)
    const uint32_t pos_dst = p.layout.seq_caps ? min(pos, p.layout.seq_caps[b] - 1) : pos;
    const size_t src = (((size_t)t * p.src_batch_pitch + b) * p.n_kv_heads + h) * kHeadDim + 8 * c;
    const size_t dst = seq_plane_offset(p.layout.seq_offsets, p.layout.stride_seq, b) + (size_t)h * p.layout.stride_head +
                       (size_t)pos_dst * kHeadDim;
    const u32x4 kraw = load16_once(p.k_src + src), vraw = load16_once(p.v_src + src);
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
  size_t rows;   // batch x n_kv_heads x n_tokens, tokens fastest: the order of the cache
  size_t dst_token, dst_sequence, dst_head;
  uint32_t n_tokens, n_kv_heads, position_index;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void kv_read_e4m3_kernel(ReadArgs p) {
  const uint32_t c = threadIdx.x & 15;
  for (size_t row = (size_t)blockIdx.x * kRowsWg + (threadIdx.x >> 4); row < p.rows; row += (size_t)gridDim.x * kRowsWg) {
    size_t r = row / p.n_tokens;
    const uint32_t t = (uint32_t)(row - r * p.n_tokens), h = r % p.n_kv_heads, b = r / p.n_kv_heads;
    const size_t src = seq_plane_offset(p.layout.seq_offsets, p.layout.stride_seq, b) + (size_t)h * p.layout.stride_head +
                       (size_t)(p.position_index + t) * kHeadDim;
    const size_t dst = t * p.dst_token + b * p.dst_sequence + h * p.dst_head + 8 * c;
    const u32x2 k = __builtin_nontemporal_load((const u32x2*)(p.k + src + 8 * c));
    const u32x2 v = __builtin_nontemporal_load((const u32x2*)(p.v + src + 8 * c));
    const float ks = scale_of(p.k_scale[src / kHeadDim]), vs = scale_of(p.v_scale[src / kHeadDim]);
    const u32x2 k0 = values4<T>(k[0], ks), k1 = values4<T>(k[1], ks), v0 = values4<T>(v[0], vs), v1 = values4<T>(v[1], vs);
    store16_once(p.k_dst + dst, u32x4{k0[0], k0[1], k1[0], k1[1]});
    store16_once(p.v_dst + dst, u32x4{v0[0], v0[1], v1[0], v1[1]});
  }
}

}  // namespace

hipError_t launch_kv_append_e4m3(const KvE4m3& cache, const void* k_src, const void* v_src, const void* rope,
                                 const uint32_t* positions, uint32_t n_tokens, uint32_t batch, uint32_t src_batch_pitch,
                                 uint32_t n_kv_heads, const KvLayout& layout, uint32_t position_index, uint32_t max_start,
                                 float eps, int dtype, hipStream_t stream) {
  const size_t rows = (size_t)n_tokens * batch * n_kv_heads;
  if (rows == 0) return hipSuccess;
  const WriteArgs p{cache.k, cache.v, cache.k_scale, cache.v_scale, (const uint16_t*)k_src, (const uint16_t*)v_src,
                    (const uint16_t*)rope, positions, layout, rows, batch, src_batch_pitch, n_kv_heads, position_index,
                    max_start, eps};
  size_t blocks = (rows + kRowsWg - 1) / kRowsWg;
  if (blocks > 16384) blocks = 16384;
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
  const ReadArgs p{cache.k, cache.v, cache.k_scale, cache.v_scale, (uint16_t*)k_dst, (uint16_t*)v_dst, layout, rows,
                   dst_token, dst_sequence, dst_head, n_tokens, n_kv_heads, position_index};
  size_t blocks = (rows + kRowsWg - 1) / kRowsWg;
  if (blocks > 16384) blocks = 16384;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(kThreads), 0, stream, p); };
  dtype == 0 ? go(kv_read_e4m3_kernel<F16>) : go(kv_read_e4m3_kernel<BF16>);
  return hipGetLastError();
}

}  // namespace ellm
