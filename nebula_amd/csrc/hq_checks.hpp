// hq_checks.hpp — argument checks that the entry points of attention, rotary positions and state space layers share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hq_internal.hpp"

namespace hq::checks {

template <class... A>
hq_status fail(hq_status s, const char* fmt, A... a) {
  return hq_set_error(s, fmt, a...);
}
inline hq_status fail(hq_status s, const char* msg) { return hq_set_error(s, "%s", msg); }

inline hq_status from_hip(hipError_t e, const char* what) {
  if (e == hipSuccess) return hq_set_error(HQ_OK, "");
  return fail(HQ_ERR_DEVICE, "%s: %s", what, hipGetErrorString(e));
}

inline bool misaligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

// Elements an operand may span, and the largest stride: far inside int64 byte offsets.
constexpr int64_t kMaxSpan = (int64_t)1 << 46;

// Row and head strides of an operand of `heads` heads of `dim`, in either order.
inline hq_status check_strides(const char* name, int64_t row, int64_t head, uint32_t rows, uint32_t heads, uint32_t dim) {
  if (row < 0 || head < 0 || row > kMaxSpan || head > kMaxSpan)
    return fail(HQ_ERR_SHAPE, "%s: strides %lld, %lld out of range", name, (long long)row, (long long)head);
  if (row % 8 || head % 8)
    return fail(HQ_ERR_ALIGNMENT, "%s: strides %lld, %lld must be multiples of 8 elements", name, (long long)row,
                (long long)head);
  if ((rows > 1 && row < (int64_t)dim) || (heads > 1 && head < (int64_t)dim))
    return fail(HQ_ERR_SHAPE, "%s: strides %lld, %lld below head_dim=%u", name, (long long)row, (long long)head, dim);
  if ((double)row * rows + (double)head * heads > (double)kMaxSpan)
    return fail(HQ_ERR_SHAPE, "%s: the operand spans too much", name);
  return HQ_OK;
}

// Whether elements of different rows or heads share memory (strides as check_strides accepts them).
inline bool overlaps(int64_t row, int64_t head, uint32_t rows, uint32_t heads, uint32_t dim) {
  if (rows == 1 || heads == 1) return false;
  if (row >= (heads - 1) * head + dim || head >= (rows - 1) * row + dim) return false;
  for (uint32_t h = 1; h < heads; ++h) {  // head h of row 0 among head 0 of the rows on either side
    const int64_t at = h * head, t = at / row;
    if ((t < rows && at - t * row < dim) || (t + 1 < rows && (t + 1) * row - at < dim)) return true;
  }
  return false;
}

inline hq_status check_dtype(int d) {
  if (d != HQ_DTYPE_F16 && d != HQ_DTYPE_BF16) return fail(HQ_ERR_INVALID_ARG, "unknown dtype %d", d);
  return HQ_OK;
}

inline hq_status check_list(const char* name, const int32_t* p) {
  if (!p) return fail(HQ_ERR_INVALID_ARG, "%s is null", name);
  if (misaligned(p, 4)) return fail(HQ_ERR_ALIGNMENT, "%s must be 4-byte aligned", name);
  return HQ_OK;
}

// The caller's workspace after its checks, or the library's own, which grows to `need`; null where the call uses none.
inline hq_status workspace(void* ws, size_t bytes, size_t use, size_t need, hipStream_t s, void** out) {
  *out = nullptr;
  if (need == 0 || (ws && use == 0)) return HQ_OK;
  if (!ws) return hq_internal_workspace(s, use, need, out);
  if (bytes < use) return fail(HQ_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu this call needs", bytes, use);
  if (misaligned(ws, 256)) return fail(HQ_ERR_ALIGNMENT, "workspace must be 256-byte aligned");
  *out = ws;
  return HQ_OK;
}

}  // namespace hq::checks
