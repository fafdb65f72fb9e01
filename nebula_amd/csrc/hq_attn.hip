// hq_attn.hip — attention of packed prompts, over a paged cache and with shared prefixes
// (include/hq_attn.h).
//
// One wavefront per row (token, head): the head's dims lie over the lanes, a key's score is summed
// across them, and the row's maximum, sum and output run over the keys once.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>

#include "hq_attn.hpp"
#include "hq_device.hpp"
#include "hq_internal.hpp"

namespace hq {
namespace {

// Sequence of token t: its keys, the keys token t may see, and (paged) its table row.
struct Seq {
  uint32_t b;
  uint32_t limit;  // keys [0, limit)
  uint32_t k0;     // packed: first key
  const int32_t* table;
  bool ok;
};

__device__ __forceinline__ uint32_t clamp_u(int32_t v, uint32_t hi) { return v < 0 ? 0u : min((uint32_t)v, hi); }

__device__ Seq find_seq(const AttnArgs& a, uint32_t t) {
  Seq s{};
  uint32_t back = 1;
  s.b = t;
  if (a.cu_q) {
    uint32_t lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (a.cu_q[mid] <= (int32_t)t) lo = mid;
      else hi = mid;
    }
    s.b = lo;
    const int32_t b0 = a.cu_q[lo], b1 = min(a.cu_q[lo + 1], (int32_t)a.T);
    if ((int32_t)t < b0 || (int32_t)t >= b1) return s;
    back = (uint32_t)b1 - t;
  }
  uint32_t nk;
  if (a.k.table) {
    const int32_t row = a.k.rows ? a.k.rows[s.b] : (int32_t)s.b;
    if ((uint32_t)row >= a.k.cache_rows) {
      __hip_atomic_fetch_or(a.k.status, HQ_CACHE_BAD_ROW, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      nk = 0;
    } else {
      nk = clamp_u(a.k.lens[row], a.k.max_pages << a.k.page_shift);
      s.table = a.k.table + row * a.k.table_stride;
    }
  } else {
    s.k0 = clamp_u(a.k.cu_k[s.b], a.k.total_k);
    const uint32_t k1 = clamp_u(a.k.cu_k[s.b + 1], a.k.total_k);
    nk = k1 > s.k0 ? k1 - s.k0 : 0u;
  }
  s.limit = !a.causal ? nk : nk + 1 > back ? nk + 1 - back : 0u;
  s.ok = true;
  return s;
}

template <int DT>
__device__ __forceinline__ float in_f32(uint16_t v) {
  if constexpr (DT == HQ_DTYPE_F16) return f16_to_f32(v);
  else return __uint_as_float((uint32_t)v << 16);
}

template <int DT, int D>
__global__ __launch_bounds__(64) void hq_attn_simple_kernel(AttnArgs a) {
  constexpr int E = D / 64;
  const uint32_t t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, g = h / a.G;
  const Seq s = find_seq(a, t);
  if (!s.ok) return;
  const uint16_t* q = a.Q + t * a.q_row + h * a.q_head + lane * E;
  float x[E], o[E];
  for (int e = 0; e < E; ++e) {
    x[e] = in_f32<DT>(q[e]) * a.scale;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (uint32_t j = 0; j < s.limit; ++j) {
    int64_t ko, vo;
    if (a.k.table) {
      uint32_t page = (uint32_t)s.table[j >> a.k.page_shift];
      if (page >= a.k.pages) {
        __hip_atomic_fetch_or(a.k.status, HQ_CACHE_BAD_PAGE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        page = 0;
      }
      const int64_t in = page * a.k.page_stride + (j & ((1u << a.k.page_shift) - 1)) * a.k.k_row;
      ko = in + g * a.k.k_head;
      vo = in + g * a.k.v_head;
    } else {
      ko = (s.k0 + j) * a.k.k_row + g * a.k.k_head;
      vo = (s.k0 + j) * a.k.v_row + g * a.k.v_head;
    }
    float d = 0.f;
    for (int e = 0; e < E; ++e) d = fmaf(x[e], in_f32<DT>(a.k.K[ko + lane * E + e]), d);
#pragma unroll
    for (int w = 32; w; w >>= 1) d += __shfl_xor(d, w);
    const float n = fmaxf(m, d), safe = n == -INFINITY ? 0.f : n;
    const float al = expf(m - safe), p = expf(d - safe);
    l = l * al + p;
    for (int e = 0; e < E; ++e) o[e] = fmaf(p, in_f32<DT>(a.k.V[vo + lane * E + e]), o[e] * al);
    m = n;
  }
  uint16_t* out = a.O + t * a.o_row + h * a.o_head + lane * E;
  for (int e = 0; e < E; ++e) out[e] = f32_to_out<DT>(l == 0.f ? 0.f : o[e] / l);
  if (a.lse && lane == 0) a.lse[(size_t)t * a.H + h] = m + logf(l);
}

template <int DT>
hipError_t launch_dim(const AttnArgs& a, hipStream_t s) {
  const dim3 grid(a.T, a.H);
  if (a.D == 64) hipLaunchKernelGGL((hq_attn_simple_kernel<DT, 64>), grid, dim3(64), 0, s, a);
  else if (a.D == 128) hipLaunchKernelGGL((hq_attn_simple_kernel<DT, 128>), grid, dim3(64), 0, s, a);
  else if (a.D == 256) hipLaunchKernelGGL((hq_attn_simple_kernel<DT, 256>), grid, dim3(64), 0, s, a);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace

AttnPlan plan_attn(int, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return AttnPlan{}; }

void describe_attn(int, const AttnPlan&, char* buf, size_t len) { std::snprintf(buf, len, "hq_attn_simple_kernel, a wavefront a row"); }

hipError_t launch_attn(int dtype, const AttnArgs& a, const AttnPlan&, void*, hipStream_t s) {
  return dtype == HQ_DTYPE_F16 ? launch_dim<HQ_DTYPE_F16>(a, s) : launch_dim<HQ_DTYPE_BF16>(a, s);
}

}  // namespace hq
