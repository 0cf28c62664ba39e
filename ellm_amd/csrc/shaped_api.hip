// C ABI of shaped scores and the shared prefix (declared in include/ellm_attn.h): checks of what is set, the room the
// kernels work in.
#include <hip/hip_runtime.h>

#include <cmath>

#include "handles.hpp"

namespace {

bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// What both set functions ask of a handle; the room for partial results, taken at the first that sets anything (`on`).
int prepare(ellm_attn* h, bool on) {
  if (!h) return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "null handle");
  if (int st = ellm::check_current_device(h->device)) return st;
  if (h->general)
    return ellm::set_error(ELLM_ERR_UNSUPPORTED, "shaped scores and shared prefixes take head_size 128 and 16-bit storage only");
  if (!std::isfinite(h->desc.inverse_sqrt_head * 4.0f))
    return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "inverse_sqrt_head %g is too large for shaped scores",
                           (double)h->desc.inverse_sqrt_head);
  ellm::ShapedState& s = h->shaped;
  if (!on || s.part_o) return ELLM_OK;
  const ellm_attn_desc& d = h->desc;
  const size_t rows = ellm::shaped_part_rows(d.max_position_interval, d.batch_size, d.attention_head_num, (uint32_t)h->n_cu);
  float *o = nullptr, *ml = nullptr;
  hipError_t e = hipMalloc((void**)&o, rows * 128 * sizeof(float));
  if (e == hipSuccess) e = hipMalloc((void**)&ml, rows * 2 * sizeof(float));
  if (e != hipSuccess) {
    (void)hipGetLastError();
    if (o) (void)hipFree(o);
    return ellm::set_error(ELLM_ERR_HIP, "hipMalloc(partial rows): %s", hipGetErrorString(e));
  }
  s.part_o = o;
  s.part_ml = ml;
  s.part_rows = rows;
  return ELLM_OK;
}

}  // namespace

int ellm::attn_run_shaped(ellm_attn* h, const ellm::AttnArgs& a, hipStream_t stream) {
  if ((uint64_t)a.position_interval * a.batch_pitch > 0x7fffffffull / a.n_q_heads)   // (2^39 bytes of queries)
    return ellm::set_error(ELLM_ERR_UNSUPPORTED, "shaped scores and shared prefixes take fewer than 2^31 query rows");
  const hipError_t e = ellm::launch_shaped(ellm::ShapedArgs{a, ellm::shaped_seen(h->shaped, a)}, stream);
  if (e != hipSuccess) return ellm::set_error(ELLM_ERR_HIP, "attention launch (shaped scores): %s", hipGetErrorString(e));
  return ELLM_OK;
}

extern "C" {

int ellm_attn_set_scores(ellm_attn* h, float score_cap, const float* distance_slopes, size_t window,
                         const uint32_t* key_begin, const uint32_t* key_end, size_t bounds_pitch) {
  if (!h) return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "null handle");
  if (score_cap != 0.0f && !(score_cap >= 0.0009765625f && score_cap <= 256.0f))
    return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "score_cap %g must be 0 (none) or in 2^-10..256", (double)score_cap);
  if (score_cap != 0.0f && !std::isfinite(h->desc.inverse_sqrt_head * 4.0f / score_cap))
    return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "inverse_sqrt_head %g is too large for a score_cap of %g",
                           (double)h->desc.inverse_sqrt_head, (double)score_cap);
  if (!aligned(distance_slopes, 4) || !aligned(key_begin, 4) || !aligned(key_end, 4))
    return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "slopes and key ranges must be 4-byte aligned device pointers");
  if ((key_begin || key_end) && bounds_pitch < h->desc.sequence_capacity)
    return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "bounds_pitch %zu is smaller than the sequence capacity %zu",
                           bounds_pitch, h->desc.sequence_capacity);
  if ((key_begin || key_end) && h->shaped.prefix)
    return ellm::set_error(ELLM_ERR_UNSUPPORTED, "key ranges do not go with a shared prefix");
  if (int st = prepare(h, score_cap != 0.0f || distance_slopes || window || key_begin || key_end)) return st;
  ellm::ShapedState& s = h->shaped;
  s.cap = score_cap;
  s.slopes = distance_slopes;
  s.window = window > 0xffffffffu ? 0xffffffffu : (uint32_t)window;   // (positions are below 2^31)
  s.key_begin = key_begin;
  s.key_end = key_end;
  s.bounds_pitch = key_begin || key_end ? bounds_pitch : 0;
  return ELLM_OK;
}

int ellm_attn_set_shared_prefix(ellm_attn* h, const void* k, const void* v, size_t head_stride, size_t position_stride,
                                size_t length) {
  if (!h) return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "null handle");
  if (length) {
    if (!k || !v) return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "k and v of the prefix must be non-null device pointers");
    if (!aligned(k, 16) || !aligned(v, 16))
      return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT, "k and v of the prefix must be 16-byte aligned");
    if (head_stride == 0 || head_stride % 8 || position_stride % 8 || position_stride < 128)
      return ellm::set_error(ELLM_ERR_INVALID_ARGUMENT,
                             "strides of the prefix must be non-zero multiples of 8 elements, rows 128 apart at least: "
                             "head_stride %zu, position_stride %zu", head_stride, position_stride);
    if (position_stride > ((size_t)1 << 24))
      return ellm::set_error(ELLM_ERR_UNSUPPORTED, "position_stride = %zu elements: rows may be at most 2^24 elements apart",
                             position_stride);
    if (length > 0x7fffffffu || h->desc.sequence_capacity > 0x7fffffffu - length)
      return ellm::set_error(ELLM_ERR_OUT_OF_RANGE, "a prefix of %zu positions ahead of %zu: more than 2^31 - 1", length,
                             h->desc.sequence_capacity);
    if (length > ((size_t)1 << 46) / position_stride)
      return ellm::set_error(ELLM_ERR_UNSUPPORTED, "a plane of the prefix spans more than 2^46 elements");
    if (h->shaped.key_begin || h->shaped.key_end)
      return ellm::set_error(ELLM_ERR_UNSUPPORTED, "key ranges do not go with a shared prefix");
  }
  if (int st = prepare(h, length != 0)) return st;
  ellm::ShapedState& s = h->shaped;
  s.prefix = (uint32_t)length;
  s.prefix_k = length ? k : nullptr;
  s.prefix_v = length ? v : nullptr;
  s.prefix_stride_head = length ? head_stride : 0;
  s.prefix_stride_pos = length ? position_stride : 0;
  return ELLM_OK;
}

}  // extern "C"
