// hq_rotary.hip — norms of query and key heads with their rotation, to tensors or into the cache's pages
// (include/hq_rotary.h).
//
// Bound by the bytes moved, each head read and written once: a lane holds 16 elements of a head as two 16-byte
// pieces, both members of its 8 pairs among them (pieces of the head R / 2 apart, or neighbours), so a rotation
// needs no exchange and a norm one sum over the D / 16 lanes of the head, by moves inside rows of 16 lanes. The
// angles of a token are the same for all its heads: a workgroup computes them once for its tokens and heads
// (64-bit turns, whole turns off, then fp32 sine and cosine) and keeps them in LDS. 4096 tokens of 24 + 4 heads of 256: 23.9 us
// for 117 MB, 4.9 TB/s; 16 tokens 3.3, 80 appended ones 4.4, 1008 of 48 + 8 heads of 128 8.2 (33 MB).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hq_device.hpp"
#include "hq_internal.hpp"
#include "hq_rotary.hpp"

namespace hq {
namespace {

constexpr uint32_t kThreads = 256;

// Sum over aligned groups of N lanes (4, 8 or 16), in every lane of the group.
template <int N>
__device__ __forceinline__ float group_sum(float x) {
#define HQ_ADD(CTRL) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true))
  HQ_ADD(0xB1);                          // the neighbour
  HQ_ADD(0x4E);                          // the other pair of four
  if constexpr (N >= 8) HQ_ADD(0x141);   // mirrored halves: the other four of eight
  if constexpr (N >= 16) HQ_ADD(0x140);  // mirrored rows: the other eight
#undef HQ_ADD
  return x;
}

// Place of a token in the cache: elements from the layer's beginning, or one of these.
constexpr int64_t kNoSequence = -2, kNoPlace = -1;

// Token t's place and position; off: cu in LDS.
__device__ int64_t find_place(const CacheArgs& c, const RotaryArgs& a, const int32_t* off, uint32_t t, int32_t& pos) {
  uint32_t i = t, back = 1;  // sequence, tokens from its end
  pos = 0;
  if (a.cu) {
    uint32_t lo = 0, hi = a.n;  // the last sequence that begins at or before t; it holds t if it does not end before it
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if ((uint32_t)off[mid] <= t) lo = mid;
      else hi = mid;
    }
    i = lo;
    if ((int32_t)t < off[i] || (int32_t)t >= off[i + 1]) return kNoSequence;
    back = (uint32_t)off[i + 1] - t;
  }
  const int32_t row = a.rows[i];
  uint32_t fault = HQ_CACHE_BAD_ROW;
  if (row >= 0 && row < (int32_t)c.rows) {
    const int64_t at = (int64_t)c.lens[row] - back;
    pos = (int32_t)at;
    if (!c.refused[row] && at >= 0 && at < (int64_t)c.max_pages << c.page_shift) {
      const uint32_t page = (uint32_t)c.table[row * c.table_stride + (at >> c.page_shift)];
      if (page < c.pages && c.refs[page] <= 1) return page * c.page_stride + (at & ((1 << c.page_shift) - 1)) * c.token_stride;
      fault = HQ_CACHE_BAD_PAGE;
    }
  }
  __hip_atomic_fetch_or(c.status, fault, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return kNoPlace;
}

// Workgroup (x, y): PASSES times `ts` tokens, the y-th 2^slots heads; a pass has a head of a token for each D / 16 lanes.
// Dynamic LDS: cosines and sines [tokens][R / 2], then, with a cache, places and positions of the tokens and cu.
template <int DT, int D, int LAYOUT, int PASSES, bool CACHE>
__global__ __launch_bounds__(kThreads) void hq_rotate_kernel(RotaryArgs a, CacheArgs c) {
  extern __shared__ __align__(16) unsigned char lds[];
  constexpr uint32_t kLanes = D / 16, kUnits = kThreads / kLanes;
  const uint32_t tid = threadIdx.x, lane = tid % kLanes, unit = tid / kLanes, half = a.R / 2;
  const uint32_t ts = kUnits >> a.slots, tokens = PASSES * ts, t0 = blockIdx.x * tokens;
  float2* cs = reinterpret_cast<float2*>(lds);
  int64_t* place = reinterpret_cast<int64_t*>(cs + tokens * half);
  int32_t* pos = reinterpret_cast<int32_t*>(place + tokens);
  int32_t* off = pos + tokens;

  // This lane's head and elements.
  uint32_t h = (blockIdx.y << a.slots) + (unit & ((1u << a.slots) - 1));
  const bool some = h < a.all, is_q = h < a.q.heads, is_v = h >= a.q.heads + a.k.heads;
  h -= is_q ? 0u : is_v ? a.q.heads + a.k.heads : a.q.heads;
  const RotaryHeads& head = is_q ? a.q : a.k;
  const uint16_t* in = is_v ? a.V : head.in;
  const int64_t in_row = is_v ? a.v_row : head.in_row, in_head = is_v ? a.v_head : head.in_head;
  const float* weight = is_v || !some ? nullptr : head.weight;
  const bool turned = lane < a.R / 16 && !is_v;
  const uint32_t e0 = LAYOUT == HQ_ROTARY_INTERLEAVED || lane >= a.R / 16 ? 16 * lane : 8 * lane;
  const uint32_t e1 = LAYOUT == HQ_ROTARY_INTERLEAVED || lane >= a.R / 16 ? e0 + 8 : e0 + half;

  u4 x[PASSES][2];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const uint32_t t = t0 + p * ts + (unit >> a.slots);
    x[p][0] = x[p][1] = u4{0, 0, 0, 0};
    if (some && t < a.T) {
      const uint16_t* s = in + t * in_row + h * in_head;
      x[p][0] = *reinterpret_cast<const u4*>(s + e0);
      x[p][1] = *reinterpret_cast<const u4*>(s + e1);
    }
  }
  f4 w[4];
  if (weight) {
    w[0] = *reinterpret_cast<const f4*>(weight + e0);
    w[1] = *reinterpret_cast<const f4*>(weight + e0 + 4);
    w[2] = *reinterpret_cast<const f4*>(weight + e1);
    w[3] = *reinterpret_cast<const f4*>(weight + e1 + 4);
  }
  if constexpr (CACHE) {
    if (a.cu) {
      for (uint32_t i = tid; i <= a.n; i += kThreads) off[i] = a.cu[i];
      __syncthreads();
    }
    for (uint32_t i = tid; i < tokens; i += kThreads) {
      int32_t p = 0;
      place[i] = t0 + i < a.T ? find_place(c, a, off, t0 + i, p) : kNoSequence;
      pos[i] = p;
    }
    __syncthreads();
  }
  for (uint32_t i = tid; i < tokens * half; i += kThreads) {
    const uint32_t tt = i / half, t = t0 + tt;
    double turn = 0;
    if (t < a.T) turn = (double)(CACHE ? pos[tt] : a.pos[t]) * a.turns[i - tt * half];
    float sin, cos;
    sincospif(2.f * (float)(turn - rint(turn)), &sin, &cos);
    cs[i] = make_float2(a.scale * cos, a.scale * sin);
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const uint32_t tt = p * ts + (unit >> a.slots), t = t0 + tt;
    float f[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) unpack_pair<DT>(x[p][i / 4][i % 4], f[2 * i], f[2 * i + 1]);
    float sum = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum = fmaf(f[i], f[i], sum);
    sum = group_sum<kLanes>(sum);  // (of every lane: those without a head have zeros)
    if (weight) {
      const float r = rsqrtf(sum * (1.f / D) + head.eps);
#pragma unroll
      for (int i = 0; i < 16; ++i) f[i] *= r * w[i / 4][i % 4];
    }
    if (turned) {
      const float4* angle = reinterpret_cast<const float4*>(cs + tt * half + 8 * lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        constexpr bool kNear = LAYOUT == HQ_ROTARY_INTERLEAVED;
        const float4 two = angle[i / 2];
        const float cos = i % 2 ? two.z : two.x, sin = i % 2 ? two.w : two.y;
        float& u = f[kNear ? 2 * i : i];
        float& v = f[kNear ? 2 * i + 1 : 8 + i];
        const float y = u * cos - v * sin;
        v = v * cos + u * sin;
        u = y;
      }
    }
    if (weight || turned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[p][i / 4][i % 4] = pack_pair<DT>(f[2 * i], f[2 * i + 1]);
    }
    uint16_t* to = nullptr;
    if (some && t < a.T) {
      if (!CACHE || is_q) {
        if (!CACHE || place[tt] != kNoSequence) to = head.out + t * head.out_row + h * head.out_head;
      } else if (place[tt] >= 0) {
        to = (is_v ? c.V : c.K) + place[tt] + h * c.head_stride;
      }
    }
    if (to) {
      *reinterpret_cast<u4*>(to + e0) = x[p][0];
      *reinterpret_cast<u4*>(to + e1) = x[p][1];
    }
  }
}

template <int DT, int D, int LAYOUT, int PASSES>
void launch(const RotaryArgs& a, const CacheArgs* cache, hipStream_t s) {
  const uint32_t ts = (kThreads * 16 / D) >> a.slots, tokens = PASSES * ts;
  const dim3 grid((a.T + tokens - 1) / tokens, (a.all + (1u << a.slots) - 1) >> a.slots);
  const uint32_t angles = tokens * a.R * 4, places = cache ? tokens * 12 + (a.cu ? (a.n + 1) * 4 : 0) : 0;
  if (cache) hipLaunchKernelGGL((hq_rotate_kernel<DT, D, LAYOUT, PASSES, true>), grid, dim3(kThreads), angles + places, s, a, *cache);
  else hipLaunchKernelGGL((hq_rotate_kernel<DT, D, LAYOUT, PASSES, false>), grid, dim3(kThreads), angles, s, a, CacheArgs{});
}

template <int DT, int D>
hipError_t launch_heads(int layout, RotaryArgs a, const CacheArgs* cache, hipStream_t s) {
  // Heads a workgroup takes: as many as a pass has room for, while a quarter at most of their places stay empty, since
  // they share angles; never below four, which keeps the angles' LDS within 16 KB.
  constexpr uint32_t kUnits = kThreads * 16 / D;
  a.slots = (uint32_t)__builtin_ctz(kUnits);
  while (a.slots > 2) {
    const uint32_t places = (a.all + (1u << a.slots) - 1) >> a.slots << a.slots;
    if (4 * places <= 5 * a.all) break;
    --a.slots;
  }
  // One pass while that makes at most four workgroups a CU: a short call's time is its chain of loads.
  const uint64_t one = (uint64_t)((a.T + (kUnits >> a.slots) - 1) / (kUnits >> a.slots)) * ((a.all + (1u << a.slots) - 1) >> a.slots);
  const bool small = one <= 4u * (uint32_t)cu_count();
  if (layout == HQ_ROTARY_HALF) small ? launch<DT, D, HQ_ROTARY_HALF, 1>(a, cache, s) : launch<DT, D, HQ_ROTARY_HALF, 4>(a, cache, s);
  else small ? launch<DT, D, HQ_ROTARY_INTERLEAVED, 1>(a, cache, s) : launch<DT, D, HQ_ROTARY_INTERLEAVED, 4>(a, cache, s);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_type(int layout, const RotaryArgs& a, const CacheArgs* cache, hipStream_t s) {
  switch (a.D) {
    case 64: return launch_heads<DT, 64>(layout, a, cache, s);
    case 128: return launch_heads<DT, 128>(layout, a, cache, s);
    default: return launch_heads<DT, 256>(layout, a, cache, s);
  }
}

}  // namespace

hipError_t launch_rotate(int dtype, int layout, RotaryArgs a, const CacheArgs* cache, hipStream_t s) {
  return dtype == HQ_DTYPE_F16 ? launch_type<HQ_DTYPE_F16>(layout, a, cache, s) : launch_type<HQ_DTYPE_BF16>(layout, a, cache, s);
}

}  // namespace hq
