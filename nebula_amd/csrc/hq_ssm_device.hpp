// hq_ssm_device.hpp — what the state space kernels share: types, sequences, steps.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hq_device.hpp"
#include "hq_ssm.hpp"

namespace hq {

template <int DT>
__device__ __forceinline__ float to_f32(uint16_t v) {
  if constexpr (DT == HQ_DTYPE_F16) return f16_to_f32(v);
  else return __uint_as_float((uint32_t)v << 16);
}

// u / (1 + exp(-u)); the exponential overflows to infinity and its reciprocal to 0 where u is far below 0.
__device__ __forceinline__ float silu(float u) {
  return u * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -1.44269504f));
}

__device__ __forceinline__ uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ uint32_t clamp_to(int32_t v, uint32_t hi) { return v < 0 ? 0u : min((uint32_t)v, hi); }

// A sequence: its tokens [a, e), the row of its states, and whether they are read and kept.
struct Seq {
  uint32_t a, e, row;
  bool read, keep;
};

// Sequence b (uniform) of a call, by every wavefront for itself; `tell`: whether this one reports a bad row. A row that
// is named before it in the list is no row: its states would be read and written at once.
__device__ __forceinline__ Seq find_seq(const SeqArgs& s, uint32_t b, bool tell) {
  Seq q;
  q.a = s.cu ? clamp_to(s.cu[b], s.T) : b;
  q.e = s.cu ? clamp_to(s.cu[b + 1], s.T) : b + 1;
  const int32_t row = s.rows ? s.rows[b] : (int32_t)b;
  const bool begins = s.held && s.held[b] == 0;
  bool bad = row < 0 || row >= (int32_t)s.cache_rows;
  if (s.rows) {
    for (uint32_t i = 0; i < b; i += 64) {
      const uint32_t j = i + (threadIdx.x & 63u);
      if (__any(j < b && s.rows[min(j, b)] == row)) bad = true;
    }
  }
  q.row = bad ? 0u : (uint32_t)row;
  q.read = !bad && !begins;
  q.keep = !bad && !(s.refused && s.refused[q.row] != 0);
  if (bad && tell && (threadIdx.x & 63u) == 0) __hip_atomic_fetch_or(s.status, HQ_CACHE_BAD_ROW, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return q;
}

// The last sequence that begins at or before token t; t is its, or no sequence's. A wavefront counts offsets, 64 a load.
__device__ __forceinline__ uint32_t seq_of(const SeqArgs& s, uint32_t t) {
  if (!s.cu) return t;
  uint32_t count = 0;
  for (uint32_t i = 0; i < s.n; i += 64) {
    const uint32_t j = i + (threadIdx.x & 63u);
    count += __popcll(__ballot(j < s.n && clamp_to(s.cu[min(j, s.n)], s.T) <= t));
  }
  return count ? count - 1 : 0u;
}

// log(1 + exp(x)) = max(x, 0) + log(1 + u), u = exp(-|x|) in (0, 1], off by at most 8 units of 2^-24 of it, whose steps are
// counted here: the exponent's product with what it rounds away (1), the exponential (2); log(1 + u) = 2 z (1 + z^2 / 3 + ..),
// z = u / (2 + u) <= 1/3: the sum (1) and the corrected quotient (1), eight terms of the series (it ends at 3^-16 / 17; 2),
// the product (1).
__device__ __forceinline__ float softplus_of(float x) {
  constexpr float kLog2e = 1.44269504f, kRest = 1.92596303e-8f;
  const float v = fmaxf(-fabsf(x), -200.f), r = v * kLog2e, e = fmaf(v, kRest, fmaf(v, kLog2e, -r));
  const float p = __builtin_amdgcn_exp2f(r), u = fmaf(p, e * 0.69314718f, p);
  const float den = 2.f + u, q = __builtin_amdgcn_rcpf(den), z0 = u * q, z = fmaf(fmaf(-z0, den, u), q, z0), z2 = z * z;
  float s = 1.f / 15;
  s = fmaf(s, z2, 1.f / 13);
  s = fmaf(s, z2, 1.f / 11);
  s = fmaf(s, z2, 1.f / 9);
  s = fmaf(s, z2, 1.f / 7);
  s = fmaf(s, z2, 1.f / 5);
  s = fmaf(s, z2, 1.f / 3);
  const float l = fmaf(2.f * z * z2, s, 2.f * z);
  return x > 0.f ? x + l : x == x ? l : x;
}
__device__ __forceinline__ float step_of(float dt, bool softplus) { return softplus ? softplus_of(dt) : dt; }
__device__ __forceinline__ float load_dt(const ScanArgs& a, uint32_t t, uint32_t h, int dtype) {
  const int64_t at = t * a.dt_row + h;
  if (a.dt_f32) return static_cast<const float*>(a.dt)[at];
  const uint16_t v = static_cast<const uint16_t*>(a.dt)[at];
  return dtype == HQ_DTYPE_F16 ? to_f32<HQ_DTYPE_F16>(v) : to_f32<HQ_DTYPE_BF16>(v);
}

}  // namespace hq
