// hq_attn.hip — attention of packed prompts, over a paged cache and with shared prefixes
// (include/hq_attn.h).
//
// Query heads of one key/value head see the same keys, so a row of the kernels' tiles is a (token,
// head of the group) pair, r = token * G + g: tiles fill up with G heads of few tokens as with one
// head of many. Scores are computed transposed, S^T = K Q^T, so that a lane holds one row's scores:
// its maximum and sum need one exchange between lane groups, and the weights P^T = exp2(c S^T - m)
// leave the registers that S^T came in as the second operand of O^T += V^T P^T. The keys of an MFMA
// step may come in any order as long as V^T has the same one, so P^T needs no exchange; V^T comes
// from LDS by transposing reads.
//
// hq_attn_tile_kernel: many rows. A workgroup's wavefronts hold 32 rows each and share tiles of 64
//   keys, copied into LDS one tile ahead.
// hq_attn_row_kernel: few rows (16) over many keys, as in decode steps: each wavefront takes tiles of
//   32 keys of its own, and the wavefronts' results are joined at the end.
// hq_attn_join_kernel: joins the parts of rows whose keys were split between workgroups.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdio>
#include <type_traits>

#include "hq_attn.hpp"
#include "hq_device.hpp"
#include "hq_internal.hpp"

namespace hq {

typedef __attribute__((address_space(1))) const void* global_ptr_t;
// 16 bytes per lane from any address straight into LDS: lane i writes lds + 16 i (lds wave-uniform). Not
// inside a template: clang's host pass does not know the builtin.
__device__ __forceinline__ void global_to_lds16(const void* p, void* lds) {
  __builtin_amdgcn_global_load_lds((global_ptr_t)p, (lds_ptr_t)lds, 16, 0, 0);
}

namespace {

typedef float f16x __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ f16x mfma32x32x16(u4 a, u4 b, f16x c) {
  if constexpr (DT == HQ_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// Four rows of 16 elements, 8 bytes from each lane of 16: lane i gets column i.
__device__ __forceinline__ u2 lds_read_tr(const unsigned char* p) {
  typedef __attribute__((address_space(3))) s4* lds_s4;
  return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p));
}

// Two weights, each rounded to nearest in the activation type (it is the type of V, and the MFMA has
// one for both operands).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == HQ_DTYPE_F16) return h2_bits(__builtin_convertvector((f2{a, b}), h2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
}

// The weights of fp16 are kept in their normal range: the running maximum's weight is 2^kLift, and the
// maximum may lag by kLag (powers of two) before the sums are rescaled. bf16 has fp32's range.
template <int DT>
struct Weights {
  static constexpr float kLift = DT == HQ_DTYPE_F16 ? 8.f : 0.f;
  static constexpr float kLag = DT == HQ_DTYPE_F16 ? 4.f : 8.f;
};

// Values of V at keys that some row may not see can be anything, and weight 0 times infinity is no 0. A
// fragment is split into its finite values (0 for the others) and a code for the others, whose
// products with 1 for the keys a row sees and 0 for the rest are counted by MFMA: up to 64 keys, so the
// counts are the digits to the base 128 of an fp32 sum below 2^21.
template <int DT>
__device__ __forceinline__ void split_odd(u4 f, u4& finite, u4& code) {
  constexpr uint32_t kExp = DT == HQ_DTYPE_F16 ? 0x7C00u : 0x7F80u, kMant = DT == HQ_DTYPE_F16 ? 0x03FFu : 0x007Fu;
  constexpr uint32_t kPos = DT == HQ_DTYPE_F16 ? 0x3C00u : 0x3F80u;  // 1
  constexpr uint32_t kNeg = DT == HQ_DTYPE_F16 ? 0x5800u : 0x4300u;  // 128
  constexpr uint32_t kNan = DT == HQ_DTYPE_F16 ? 0x7400u : 0x4680u;  // 16384
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t fin = 0, cod = 0;
#pragma unroll
    for (int e = 0; e < 32; e += 16) {
      const uint32_t x = f[w] >> e & 0xFFFFu;
      const bool odd = (x & kExp) == kExp;
      fin |= odd ? 0u : x << e;
      cod |= (odd ? (x & kMant) ? kNan : x & 0x8000u ? kNeg : kPos : 0u) << e;
    }
    finite[w] = fin;
    code[w] = cod;
  }
}
// What the counted values add to a sum.
__device__ __forceinline__ float odd_value(float count) {
  const uint32_t n = (uint32_t)count, pos = n & 127u, neg = n >> 7 & 127u;
  return n == 0 ? 0.f : n >> 14 || (pos && neg) ? NAN : pos ? INFINITY : -INFINITY;
}
// Two fragment elements: 1 where the key is below lim.
template <int DT>
__device__ __forceinline__ uint32_t seen2(uint32_t key, uint32_t lim) {
  constexpr uint32_t one = DT == HQ_DTYPE_F16 ? 0x3C00u : 0x3F80u;
  return (key < lim ? one : 0u) | (key + 1 < lim ? one << 16 : 0u);
}

constexpr float kNone = -FLT_MAX;  // the maximum of no score: finite, so that differences with it are no NaN

__device__ __forceinline__ void report(uint32_t* status, uint32_t what) {
  __hip_atomic_fetch_or(status, what, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t clamp_u(int32_t v, uint32_t hi) { return v < 0 ? 0u : min((uint32_t)v, hi); }
__device__ __forceinline__ uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// ---- sequences ----
// What a tile works on: rows [r0, R) of a sequence (or of a group, for its shared prefix) whose first
// token is q0, over keys [k0, k1) of n.
struct Work {
  uint32_t b, q0, R, r0;
  uint32_t nq, nk;       // new tokens, keys
  uint32_t key0;         // packed: row of key 0 in K and V
  int32_t row;           // paged: cache row
  bool ok;
};

// Cache row of sequence b and its length (0, reported, if there is no such row).
__device__ __forceinline__ uint32_t cached_len(const AttnKeys& k, uint32_t b, int32_t& row) {
  row = k.rows ? k.rows[b] : (int32_t)b;
  if ((uint32_t)row >= k.cache_rows) {
    report(k.status, HQ_CACHE_BAD_ROW);
    row = 0;
    return 0;
  }
  return clamp_u(k.lens[row], k.max_pages << k.page_shift);
}

// Tokens of entry b of a list of offsets (queries of a sequence, sequences of a group), held to [0, most].
__device__ __forceinline__ uint32_t span(const int32_t* cu, uint32_t b, uint32_t most, uint32_t& first) {
  first = clamp_u(cu[b], most);
  const uint32_t end = clamp_u(cu[b + 1], most);
  return end > first ? end - first : 0u;
}

// The idx-th tile of `rows` rows over all entries, by one wavefront: the entries' tiles are counted 64
// at a time. Inside an entry the last tile comes first: under the causal mask it has the most keys.
__device__ __forceinline__ bool find_tile(const int32_t* cu, uint32_t n, uint32_t most, uint32_t G, uint32_t rows, uint32_t idx,
                                          Work& w) {
  const uint32_t lane = threadIdx.x & 63u;
  if (!cu) {  // one token each
    const uint32_t per = (G + rows - 1) / rows;
    w.b = idx / per;
    if (w.b >= n) return false;
    w.q0 = w.b;
    w.nq = 1;
    w.R = G;
    w.r0 = (idx % per) * rows;
    return true;
  }
  uint32_t before = 0;
  for (uint32_t base = 0; base < n; base += 64) {
    const uint32_t b = base + lane;
    uint32_t first = 0, nq = 0;
    if (b < n) nq = span(cu, b, most, first);
    const uint32_t tiles = (nq * G + rows - 1) / rows;
    uint32_t x = tiles;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
      const uint32_t y = __shfl_up(x, d);
      if (lane >= d) x += y;
    }
    const uint64_t past = __ballot(before + x > idx);
    if (past) {
      const int at = __builtin_ctzll(past);
      w.b = base + at;
      w.q0 = uni(__shfl(first, at));
      w.nq = uni(__shfl(nq, at));
      w.R = w.nq * G;
      w.r0 = (uni(__shfl(before + x, at)) - 1 - idx) * rows;
      return true;
    }
    before += uni(__shfl(x, 63));
  }
  return false;
}

// The group of sequence b, and the tokens of its prefix that lie in whole pages.
__device__ __forceinline__ uint32_t shared_tokens(const AttnArgs& a, uint32_t g) {
  const uint32_t first = clamp_u(a.starts[g], a.B);
  if (first >= a.B) return 0;
  int32_t row;
  const uint32_t n = min(cached_len(a.k, first, row), clamp_u(a.prefix[g], 1u << 30));
  return n >> a.k.page_shift << a.k.page_shift;
}
__device__ __forceinline__ uint32_t group_of(const AttnArgs& a, uint32_t b) {
  uint32_t lo = 0, hi = a.groups;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (a.starts[mid] <= (int32_t)b) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t page_or_report(const AttnKeys& k, int32_t page) {
  if ((uint32_t)page < k.pages) return (uint32_t)page;
  report(k.status, HQ_CACHE_BAD_PAGE);
  return 0;
}

// ---- parts of rows whose keys are split ----
// Row (token t, head h) has `slots` places: fp32 O [D] (not divided by the sum), the maximum times c and
// the sum; a place without weight has sum 0 and no O.
struct Parts {
  float* o;
  f2* ml;
  uint32_t slots;
};

struct TilePlan {
  uint32_t splits, split_keys;  // workgroup s of a tile takes keys [s split_keys, (s + 1) split_keys), the last one all the rest
  uint32_t prefix;              // rows are the sequences of a group, keys its shared prefix
  uint32_t slot0;
  Parts parts;
};

// Keys of 16-byte chunk positions inside a row of LDS: chunk c of row r lies at c ^ f(r), so that the
// rows of one read do not meet in the same banks (64 of 4 bytes; a row is 2 D bytes). K is read 16 rows
// at the same chunk, V four rows of 64 bytes at a time (tile kernel).
template <int D>
__device__ __forceinline__ uint32_t swz_k(uint32_t r) {
  return D == 64 ? (r >> 1) & 7u : r & 15u;
}
template <int D>
__device__ __forceinline__ uint32_t swz_v(uint32_t r) {
  return D == 64 ? ((r >> 1) & 1u) << 2 : (r & 3u) << 2;
}

// ---- many rows ----
constexpr int kKeys = 64;  // keys of a tile

template <int D>
constexpr uint32_t tile_stage_bytes() {
  return 2u * kKeys * D * 2u;
}

template <int DT, int D, int NW, bool PAGED>
__global__ __launch_bounds__(NW * 64, D == 256 ? 1 : 2) void hq_attn_tile_kernel(AttnArgs a, TilePlan pl) {
  constexpr uint32_t BR = NW * 32;
  constexpr uint32_t kPitch = 2 * D, kStage = tile_stage_bytes<D>(), kVOff = kStage / 2;
  constexpr int kSteps = D / 16, kDims = D / 32;
  constexpr uint32_t kRowsPerLoad = 1024 / kPitch, kLoads = kKeys / kRowsPerLoad / NW;  // loads of a wavefront, K and V each
  extern __shared__ __align__(1024) unsigned char smem[];

  const uint32_t lane = threadIdx.x & 63u, wave = uni(threadIdx.x >> 6);
  const uint32_t l32 = lane & 31u, half = lane >> 5;

  // Heads run fastest: workgroups go to the XCDs in turn, so with eight key/value heads each XCD's L2
  // sees the keys of one.
  const uint32_t kvh = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv;
  const uint32_t split = rest % pl.splits, idx = rest / pl.splits;
  Work w{};
  if (!find_tile(pl.prefix ? a.starts : a.cu_q, pl.prefix ? a.groups : a.B, pl.prefix ? a.B : a.T, a.G, BR, idx, w)) return;
  const int32_t* table = nullptr;
  uint32_t nk;
  if constexpr (PAGED) {
    int32_t row;
    nk = cached_len(a.k, pl.prefix ? w.q0 : w.b, row);
    if (pl.prefix) nk = shared_tokens(a, w.b);
    table = a.k.table + row * a.k.table_stride;
  } else {
    nk = span(a.k.cu_k, w.b, a.k.total_k, w.key0);
  }
  nk = uni(nk);

  // This lane's row, and the keys it may see.
  const uint32_t r_mine = w.r0 + wave * 32 + l32;
  const bool live = r_mine < w.R;
  const uint32_t r = min(r_mine, w.R - 1), token = r / a.G, head = kvh * a.G + (r - token * a.G);
  uint32_t lim = nk;
  if (pl.prefix) {
    int32_t row;
    lim = min(nk, cached_len(a.k, w.q0 + token, row));
  } else if (a.causal) {
    const int64_t n = (int64_t)token + nk - w.nq + 1;
    lim = n < 0 ? 0u : (uint32_t)n;
  }
  uint32_t lim_min = lim, lim_max = lim;
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    lim_min = min(lim_min, (uint32_t)__shfl_xor((int)lim_min, d));
    lim_max = max(lim_max, (uint32_t)__shfl_xor((int)lim_max, d));
  }
  lim_min = uni(lim_min);
  lim_max = w.r0 + wave * 32 < w.R ? uni(lim_max) : 0u;

  // Keys of this workgroup: up to the last that any of its rows sees.
  uint32_t wg_lim = nk;
  if (!pl.prefix && a.causal) {
    const int64_t n = (int64_t)((min(w.r0 + BR, w.R) - 1) / a.G) + nk - w.nq + 1;
    wg_lim = n < 0 ? 0u : (uint32_t)n;
  }
  const uint32_t kbeg = split * pl.split_keys;
  const uint32_t kend = split + 1 == pl.splits ? wg_lim : min(wg_lim, kbeg + pl.split_keys);
  const uint32_t t0 = kbeg / kKeys, t1 = kend > kbeg ? (kend + kKeys - 1) / kKeys : t0;

  const uint16_t* const qp = a.Q + (int64_t)(w.q0 + token) * a.q_row + head * a.q_head + 8 * half;
  u4 q[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const u4*>(qp + 16 * s);

  const float c = a.scale * 1.44269504088896340736f;
  const uint16_t* const Kh = a.k.K + kvh * a.k.k_head;
  const uint16_t* const Vh = a.k.V + kvh * a.k.v_head;

  // Copies of tile t into a stage: load i of the wavefront brings rows kRowsPerLoad (i NW + wave) ...; a
  // lane's row and source chunk undo the swizzle. Keys past the last are copies of it (masked below).
  const uint32_t in_row = lane / (D / 8), in_chunk = lane % (D / 8);
  auto issue = [&](uint32_t t, uint32_t stage) {
    unsigned char* const base = smem + stage * kStage;
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t row = (i * NW + wave) * kRowsPerLoad + in_row;
      const uint32_t key = min(t * kKeys + row, nk - 1);
      int64_t ko, vo;
      if constexpr (PAGED) {
        const uint32_t page = page_or_report(a.k, table[key >> a.k.page_shift]);
        const int64_t in = page * a.k.page_stride + (key & ((1u << a.k.page_shift) - 1)) * a.k.k_row;
        ko = vo = in;
      } else {
        ko = (w.key0 + key) * a.k.k_row;
        vo = (w.key0 + key) * a.k.v_row;
      }
      unsigned char* const to = base + (i * NW + wave) * 1024;
      global_to_lds16(Kh + ko + (in_chunk ^ swz_k<D>(row)) * 8, to);
      global_to_lds16(Vh + vo + (in_chunk ^ swz_v<D>(row)) * 8, to + kVOff);
    }
  };

  // LDS places of this lane's fragments. K^T: row l32 (+ 32), dims 16 s + 8 half: chunk 2 s + half.
  uint32_t k_at[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) k_at[s] = l32 * kPitch + (((2 * s + half) ^ swz_k<D>(l32)) << 4);
  // V^T: keys 4 half + (lane % 16) / 4 (+ 8, + 16 steps), dims 32 dt + 16 (l32 / 16) + 4 (lane % 4).
  const uint32_t v_row = 4 * half + ((lane & 15u) >> 2);
  uint32_t v_at[kDims];
#pragma unroll
  for (int dt = 0; dt < kDims; ++dt)
    v_at[dt] = kVOff + v_row * kPitch + (((4 * dt + 2 * (l32 >> 4) + ((lane & 3u) >> 1)) ^ swz_v<D>(v_row)) << 4) + 8 * (lane & 1u);

  f16x o[kDims];
  float m, l;
  // Second pass (careful) only where a first one gave values that are not finite, or no weight at all:
  // values of V at keys a row may not see, times its weight 0, may have made them, or scores past 1e7.
  auto pass = [&](auto mode) {
    constexpr bool careful = decltype(mode)::value;
    m = kNone;
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt) o[dt] = f16x{};
    uint32_t ts = t0;
    asm volatile("" : "+s"(ts));  // what one pass computes is not held for the other
    if (t1 > ts) issue(ts, ts & 1u);
    for (uint32_t t = ts; t < t1; ++t) {
      __builtin_amdgcn_s_waitcnt(0);  // the wavefront's copies of tile t have landed, its reads of t - 1 are done
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if (t + 1 < t1) issue(t + 1, (t + 1) & 1u);
      if (t * kKeys >= lim_max) continue;
      const unsigned char* const st = smem + (t & 1u) * kStage;

      f16x s[2] = {f16x{}, f16x{}};
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
          s[kt] = mfma32x32x16<DT>(*reinterpret_cast<const u4*>(st + k_at[i] + kt * 32 * kPitch), q[i], s[kt]);

      const bool masked = t * kKeys + kKeys > lim_min;
      if (masked) {
        const uint32_t k0 = t * kKeys + 4 * half;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (k0 + 32 * kt + 8 * (v / 4) + v % 4 >= lim) s[kt][v] = -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(fmaxf(top, s[0][v]), s[1][v]);
      {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
      }
      if (__any((top - m) * c > Weights<DT>::kLag)) {
        const float n = (top - m) * c > Weights<DT>::kLag ? top : m, al = __builtin_amdgcn_exp2f((m - n) * c);
        m = n;  // each row by itself, so that its bits do not depend on its neighbours
        l *= al;
#pragma unroll
        for (int dt = 0; dt < kDims; ++dt) o[dt] *= al;
      }
      float mc = fmaxf(m * c, kNone) - Weights<DT>::kLift, cs = c;
      if constexpr (careful) {  // differences first: m c may be rounded by more than the exponential's range
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          s[0][v] = (s[0][v] - m) * c;
          s[1][v] = (s[1][v] - m) * c;
        }
        mc = -Weights<DT>::kLift;
        cs = 1.f;
      }
      u4 p[4];
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int v = 8 * (j & 1) + 2 * e;
          const float x = __builtin_amdgcn_exp2f(fmaf(s[j / 2][v], cs, -mc)), y = __builtin_amdgcn_exp2f(fmaf(s[j / 2][v + 1], cs, -mc));
          sum += x + y;
          p[j][e] = pack2<DT>(x, y);
        }
      l += sum;

      auto v_frag = [&](int dt, int j, uint32_t from = 0) {
        const u2 lo = lds_read_tr(st + from + v_at[dt] + 16 * j * kPitch), hi = lds_read_tr(st + from + v_at[dt] + (16 * j + 8) * kPitch);
        return u4{lo[0], lo[1], hi[0], hi[1]};
      };
      if (careful && masked) {
        uint32_t from = 0;
        asm volatile("" : "+s"(from));  // these reads are not the other branch's: not all taken before it
#pragma unroll
        for (int dt = 0; dt < kDims; ++dt) {
          f16x count = f16x{};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);  // one fragment at a time in registers
            const uint32_t key = t * kKeys + 16 * j + 4 * half;
            const u4 sees = {seen2<DT>(key, lim), seen2<DT>(key + 2, lim), seen2<DT>(key + 8, lim), seen2<DT>(key + 10, lim)};
            u4 finite, code;
            split_odd<DT>(v_frag(dt, j, from), finite, code);
            o[dt] = mfma32x32x16<DT>(finite, p[j], o[dt]);
            count = mfma32x32x16<DT>(code, sees, count);
          }
#pragma unroll
          for (int v = 0; v < 16; ++v) o[dt][v] += odd_value(count[v]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int dt = 0; dt < kDims; ++dt) o[dt] = mfma32x32x16<DT>(v_frag(dt, j), p[j], o[dt]);
      }
    }
    {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
      l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    }
    float bad = 0.f;
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
      for (int v = 0; v < 16; ++v) bad = fmaf(o[dt][v], 0.f, bad);
    return __syncthreads_or(!(bad == 0.f) || (l == 0.f && m != kNone)) != 0;
  };
  if (pass(std::false_type{})) pass(std::true_type{});
  if (!live) return;
  const uint32_t tok = w.q0 + token;
  const float mc = fmaxf(m * c, kNone) - Weights<DT>::kLift;
  if (pl.parts.slots) {
    const uint64_t at = ((uint64_t)tok * a.H + head) * pl.parts.slots + pl.slot0 + split;
    if (half == 0) pl.parts.ml[at] = f2{mc, l};
    if (l != 0.f)
#pragma unroll
      for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          *reinterpret_cast<f4*>(pl.parts.o + at * D + 32 * dt + 8 * v + 4 * half) =
              f4{o[dt][4 * v], o[dt][4 * v + 1], o[dt][4 * v + 2], o[dt][4 * v + 3]};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* const op = a.O + (int64_t)tok * a.o_row + head * a.o_head + 4 * half;
#pragma unroll
  for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = l == 0.f ? 0.f : o[dt][4 * v + e] * inv;
      *reinterpret_cast<u2*>(op + 32 * dt + 8 * v) = u2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
    }
  if (a.lse && half == 0) a.lse[(uint64_t)tok * a.H + head] = l == 0.f ? -INFINITY : (mc + __log2f(l)) * 0.69314718055994530942f;
}

// ---- few rows ----
constexpr int kRowKeys = 32;  // keys of a wavefront's tile

struct RowPlan {
  uint32_t splits, split_keys;
  uint32_t slot0;
  Parts parts;
};

// As swz_k / swz_v, for this kernel's reads: V 16 rows of 32 bytes.
template <int D>
__device__ __forceinline__ uint32_t swz_rv(uint32_t r) {
  return D == 64 ? ((r >> 1) & 3u) << 1 : (r & 7u) << 1;
}

template <int D>
constexpr uint32_t row_waves() {
  return D == 256 ? 2u : 4u;
}
template <int D>
constexpr uint32_t row_lds_bytes() {
  return row_waves<D>() * 2u * (2u * kRowKeys * D * 2u);
}

template <int DT, int D, bool PAGED>
__global__ __launch_bounds__(row_waves<D>() * 64) void hq_attn_row_kernel(AttnArgs a, RowPlan pl) {
  constexpr uint32_t NW = row_waves<D>();
  constexpr uint32_t kPitch = 2 * D, kStage = 2 * kRowKeys * kPitch, kVOff = kStage / 2;
  constexpr int kSteps = D / 32, kDims = D / 16;
  constexpr uint32_t kRowsPerLoad = 1024 / kPitch, kLoads = kRowKeys / kRowsPerLoad;
  extern __shared__ __align__(1024) unsigned char smem[];

  const uint32_t lane = threadIdx.x & 63u, wave = uni(threadIdx.x >> 6);
  const uint32_t l16 = lane & 15u, quad = lane >> 4;
  const uint32_t kvh = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv;
  const uint32_t split = rest % pl.splits, idx = rest / pl.splits;
  Work w{};
  if (!find_tile(a.cu_q, a.B, a.T, a.G, 16, idx, w)) return;
  const int32_t* table = nullptr;
  uint32_t nk, begin = 0;
  if constexpr (PAGED) {
    int32_t row;
    nk = cached_len(a.k, w.b, row);
    table = a.k.table + row * a.k.table_stride;
    if (a.groups) begin = min(nk, shared_tokens(a, group_of(a, w.b)));
  } else {
    nk = span(a.k.cu_k, w.b, a.k.total_k, w.key0);
  }
  nk = uni(nk);
  begin = uni(begin);

  const uint32_t r_mine = w.r0 + l16;
  const uint32_t r = min(r_mine, w.R - 1), token = r / a.G, head = kvh * a.G + (r - token * a.G);
  uint32_t lim = nk, wg_lim = nk;
  if (a.causal) {
    const int64_t n = (int64_t)token + nk - w.nq + 1, last = (int64_t)((min(w.r0 + 16, w.R) - 1) / a.G) + nk - w.nq + 1;
    lim = n < 0 ? 0u : (uint32_t)n;
    wg_lim = last < 0 ? 0u : (uint32_t)last;
  }
  const uint32_t kbeg = begin + split * pl.split_keys;
  const uint32_t kend = split + 1 == pl.splits ? wg_lim : min(wg_lim, kbeg + pl.split_keys);
  if (kend <= kbeg && split > 0) return;  // the join counts the parts by the lengths
  const uint32_t tiles = kend > kbeg ? (kend - kbeg + kRowKeys - 1) / kRowKeys : 0u;

  const uint16_t* const qp = a.Q + (int64_t)(w.q0 + token) * a.q_row + head * a.q_head + 8 * quad;
  u4 q[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const u4*>(qp + 32 * s);
  const float c = a.scale * 1.44269504088896340736f;
  const uint16_t* const Kh = a.k.K + kvh * a.k.k_head;
  const uint16_t* const Vh = a.k.V + kvh * a.k.v_head;
  unsigned char* const mine = smem + wave * 2 * kStage;

  const uint32_t in_row = lane / (D / 8), in_chunk = lane % (D / 8);
  auto page_of = [&](uint32_t t) -> int32_t {  // the page of key lane % 32 of tile t
    if constexpr (PAGED) return table[min(kbeg + t * kRowKeys + (lane & 31u), nk - 1) >> a.k.page_shift];
    else return 0;
  };
  auto issue = [&](uint32_t t, uint32_t stage, int32_t pages) {
    if constexpr (PAGED) pages = (int32_t)page_or_report(a.k, pages);
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t row = i * kRowsPerLoad + in_row, key = min(kbeg + t * kRowKeys + row, nk - 1);
      int64_t ko, vo;
      if constexpr (PAGED) {
        const uint32_t page = (uint32_t)__shfl(pages, row);
        ko = vo = page * a.k.page_stride + (key & ((1u << a.k.page_shift) - 1)) * a.k.k_row;
      } else {
        ko = (w.key0 + key) * a.k.k_row;
        vo = (w.key0 + key) * a.k.v_row;
      }
      unsigned char* const to = mine + stage * kStage + i * 1024;
      global_to_lds16(Kh + ko + (in_chunk ^ swz_k<D>(row)) * 8, to);
      global_to_lds16(Vh + vo + (in_chunk ^ swz_rv<D>(row)) * 8, to + kVOff);
    }
  };

  uint32_t k_at[kSteps], v_at[kDims];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) k_at[s] = l16 * kPitch + (((4 * s + quad) ^ swz_k<D>(l16)) << 4);
  const uint32_t v_row = 4 * quad + (l16 >> 2);
#pragma unroll
  for (int dt = 0; dt < kDims; ++dt)
    v_at[dt] = kVOff + v_row * kPitch + (((2 * dt + ((l16 & 3u) >> 1)) ^ swz_rv<D>(v_row)) << 4) + 8 * (l16 & 1u);

  f4 o[kDims];
  float m, l;
  // Twice only where the first pass gave values that are not finite, as in the tile kernel.
  auto pass = [&](auto mode) {
    constexpr bool careful = decltype(mode)::value;
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt) o[dt] = f4{};
    m = kNone;
    l = 0.f;
    int32_t next = 0;
    if (wave < tiles) {
      issue(wave, 0, page_of(wave));
      if (wave + NW < tiles) next = page_of(wave + NW);
    }
    uint32_t stage = 0;
    for (uint32_t t = wave; t < tiles; t += NW, stage ^= 1u) {
      if (t + NW < tiles) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the stage that is filled next
        issue(t + NW, stage ^ 1u, next);
        if (t + 2 * NW < tiles) {
          next = page_of(t + 2 * NW);
          __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * kLoads + (PAGED ? 1 : 0)));
        } else {
          __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * kLoads));
        }
      } else {
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
      }
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const unsigned char* const st = mine + stage * kStage;
      f4 s[2] = {f4{}, f4{}};
#pragma unroll
      for (int i = 0; i < kSteps; ++i)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
          s[kt] = mfma16x16x32<DT>(*reinterpret_cast<const u4*>(st + k_at[i] + kt * 16 * kPitch), q[i], s[kt]);
      const uint32_t k0 = kbeg + t * kRowKeys;
      const bool masked = k0 + kRowKeys > min(kend, uni(w.nq) == 1 ? kend : k0);
      const uint32_t stop = min(lim, kend);
      if (masked) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            if (k0 + 16 * kt + 4 * quad + v >= stop) s[kt][v] = -INFINITY;
      }
      float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (__any((top - m) * c > Weights<DT>::kLag)) {
        const float n = (top - m) * c > Weights<DT>::kLag ? top : m, al = __builtin_amdgcn_exp2f((m - n) * c);
        m = n;
        l *= al;
#pragma unroll
        for (int dt = 0; dt < kDims; ++dt) o[dt] *= al;
      }
      const float mc = fmaxf(m * c, kNone) - Weights<DT>::kLift;
      float p[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const float x = s[v / 4][v % 4];
        p[v] = __builtin_amdgcn_exp2f(careful ? fmaf(x - m, c, Weights<DT>::kLift) : fmaf(x, c, -mc));
        l += p[v];
      }
      const u4 pf = {pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7])};
      if (careful && masked) {
        uint32_t from = 0;
        asm volatile("" : "+s"(from));
        const u4 sees = {seen2<DT>(k0 + 4 * quad, stop), seen2<DT>(k0 + 4 * quad + 2, stop), seen2<DT>(k0 + 16 + 4 * quad, stop),
                         seen2<DT>(k0 + 16 + 4 * quad + 2, stop)};
#pragma unroll
        for (int dt = 0; dt < kDims; ++dt) {
          const u2 lo = lds_read_tr(st + from + v_at[dt]), hi = lds_read_tr(st + from + v_at[dt] + 16 * kPitch);
          u4 finite, code;
          split_odd<DT>(u4{lo[0], lo[1], hi[0], hi[1]}, finite, code);
          o[dt] = mfma16x16x32<DT>(finite, pf, o[dt]);
          const f4 count = mfma16x16x32<DT>(code, sees, f4{});
#pragma unroll
          for (int v = 0; v < 4; ++v) o[dt][v] += odd_value(count[v]);
        }
        continue;
      }
#pragma unroll
      for (int dt = 0; dt < kDims; ++dt) {
        const u2 lo = lds_read_tr(st + v_at[dt]), hi = lds_read_tr(st + v_at[dt] + 16 * kPitch);
        o[dt] = mfma16x16x32<DT>(u4{lo[0], lo[1], hi[0], hi[1]}, pf, o[dt]);
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float bad = 0.f;
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
      for (int v = 0; v < 4; ++v) bad = fmaf(o[dt][v], 0.f, bad);
    return __any(!(bad == 0.f) || (l == 0.f && m != kNone)) != 0;
  };
  if (pass(std::false_type{})) pass(std::true_type{});

  // Join the wavefronts: each brings its sums to the common maximum, [wavefront][row][dim].
  __syncthreads();
  float* const red = reinterpret_cast<float*>(smem);
  f2* const stat = reinterpret_cast<f2*>(smem + NW * 16 * (D + 4) * 4);
  if (quad == 0) stat[wave * 16 + l16] = f2{m, l};
  __syncthreads();
  float top = kNone;
#pragma unroll
  for (uint32_t i = 0; i < NW; ++i) top = fmaxf(top, stat[i * 16 + l16][0]);
  const float al = l == 0.f ? 0.f : __builtin_amdgcn_exp2f((m - top) * c);
#pragma unroll
  for (int dt = 0; dt < kDims; ++dt)
    *reinterpret_cast<f4*>(red + (wave * 16 + l16) * (D + 4) + 16 * dt + 4 * quad) = l == 0.f ? f4{} : o[dt] * al;
  __syncthreads();
  for (uint32_t u = threadIdx.x; u < 16 * (D / 4); u += NW * 64) {
    const uint32_t row = u / (D / 4), d = (u % (D / 4)) * 4;
    const uint32_t rr = w.r0 + row;
    if (rr >= w.R) continue;
    const uint32_t tk = w.q0 + rr / a.G, hd = kvh * a.G + rr % a.G;
    float mx = kNone, sum = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) mx = fmaxf(mx, stat[i * 16 + row][0]);
    f4 v = f4{};
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) {
      const f2 e = stat[i * 16 + row];
      if (e[1] != 0.f) sum += e[1] * __builtin_amdgcn_exp2f((e[0] - mx) * c);
      v += *reinterpret_cast<const f4*>(red + (i * 16 + row) * (D + 4) + d);
    }
    const float mc = fmaxf(mx * c, kNone) - Weights<DT>::kLift;
    if (pl.parts.slots) {
      const uint64_t at = ((uint64_t)tk * a.H + hd) * pl.parts.slots + pl.slot0 + split;
      if (d == 0) pl.parts.ml[at] = f2{mc, sum};
      if (sum != 0.f) *reinterpret_cast<f4*>(pl.parts.o + at * D + d) = v;
    } else {
      const float inv = 1.f / sum;
      if (sum == 0.f) v = f4{};
      else v *= inv;
      *reinterpret_cast<u2*>(a.O + (int64_t)tk * a.o_row + hd * a.o_head + d) = u2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
      if (a.lse && d == 0) a.lse[(uint64_t)tk * a.H + hd] = sum == 0.f ? -INFINITY : (mc + __log2f(sum)) * 0.69314718055994530942f;
    }
  }
}

// ---- joining parts ----
struct JoinPlan {
  Parts parts;
  uint32_t prefix_slots, prefix_keys;  // of a shared prefix, first
  uint32_t own_slots, own_keys;        // of the rows' own keys (tile kernel: all written; row kernel: those with keys)
  uint32_t all;                        // every place was written
};

template <int DT, int D>
__global__ __launch_bounds__(256) void hq_attn_join_kernel(AttnArgs a, JoinPlan pl) {
  constexpr int E = D / 64;
  const uint32_t lane = threadIdx.x & 63u;
  const uint64_t u = (uint64_t)blockIdx.x * 4 + uni(threadIdx.x >> 6);
  if (u >= (uint64_t)a.T * a.H) return;
  const uint32_t t = (uint32_t)(u / a.H), h = (uint32_t)(u % a.H);
  uint32_t b = t, nq = 1, q0 = t;
  if (a.cu_q) {
    uint32_t lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (a.cu_q[mid] <= (int32_t)t) lo = mid;
      else hi = mid;
    }
    b = lo;
    nq = span(a.cu_q, b, a.T, q0);
    if (t < q0 || t >= q0 + nq) return;  // of no sequence
  }
  uint32_t own = pl.own_slots;
  if (!pl.all) {
    uint32_t nk, begin = 0, k0;
    int32_t row;
    if (a.k.table) {
      nk = cached_len(a.k, b, row);
      if (a.groups) begin = min(nk, shared_tokens(a, group_of(a, b)));
    } else {
      nk = span(a.k.cu_k, b, a.k.total_k, k0);
    }
    // The rows of a tile share its workgroups: the last row's keys count.
    uint32_t last = nk;
    if (a.causal) {
      const uint32_t r = (t - q0) * a.G + h % a.G, end = min((r / 16 + 1) * 16, nq * a.G) - 1;
      const int64_t n = (int64_t)(end / a.G) + nk - nq + 1;
      last = n < 0 ? 0u : (uint32_t)n;
    }
    own = last > begin ? min(own, (last - begin + pl.own_keys - 1) / pl.own_keys) : 1u;
  }
  const uint64_t at = u * pl.parts.slots;
  const uint32_t n = pl.prefix_slots + own;
  float m = kNone;
  for (uint32_t i = lane; i < n; i += 64) {
    const f2 e = pl.parts.ml[at + i];
    if (e[1] != 0.f) m = fmaxf(m, e[0]);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  float l = 0.f, o[E] = {};
  for (uint32_t i = 0; i < n; ++i) {
    const f2 e = pl.parts.ml[at + i];
    if (e[1] == 0.f) continue;
    const float f = __builtin_amdgcn_exp2f(e[0] - m);
    l = fmaf(e[1], f, l);
    const float* p = pl.parts.o + (at + i) * D + lane * E;
#pragma unroll
    for (int k = 0; k < E; ++k) o[k] = fmaf(p[k], f, o[k]);
  }
  uint16_t* const out = a.O + (int64_t)t * a.o_row + h * a.o_head + lane * E;
#pragma unroll
  for (int k = 0; k < E; ++k) out[k] = f32_to_out<DT>(l == 0.f ? 0.f : o[k] / l);
  if (a.lse && lane == 0) a.lse[u] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994530942f;
}

template <int DT, int D, bool PAGED>
hipError_t launch_all(const AttnArgs& a, const AttnPlan& p, void* ws, hipStream_t s) {
  Parts parts{};
  if (p.slots) {
    parts.slots = p.slots;
    parts.ml = reinterpret_cast<f2*>(static_cast<unsigned char*>(ws) + kCounterBytes);
    parts.o = reinterpret_cast<float*>(static_cast<unsigned char*>(ws) + kCounterBytes + p.o_offset);
  }
  if (p.tile) {
    TilePlan t{p.tile_splits, p.tile_keys, p.prefix, 0, parts};
    auto k = hq_attn_tile_kernel<DT, D, 4, PAGED>;
    constexpr uint32_t lds = 2 * tile_stage_bytes<D>();
    static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (set != hipSuccess) return set;
    hipLaunchKernelGGL(k, dim3(p.tile_grid), dim3(256), lds, s, a, t);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.row) {
    RowPlan r{p.row_splits, p.row_keys, p.prefix ? p.tile_splits : 0u, parts};
    auto k = hq_attn_row_kernel<DT, D, PAGED>;
    constexpr uint32_t lds = row_lds_bytes<D>();
    static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (set != hipSuccess) return set;
    hipLaunchKernelGGL(k, dim3(p.row_grid), dim3(row_waves<D>() * 64), lds, s, a, r);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.slots) {
    JoinPlan j{};
    j.parts = parts;
    j.prefix_slots = p.prefix ? p.tile_splits : 0u;
    j.own_slots = p.prefix || p.row ? p.row_splits : p.tile_splits;
    j.own_keys = p.row_keys;
    j.all = !p.row;
    hipLaunchKernelGGL((hq_attn_join_kernel<DT, D>), dim3((uint32_t)(((uint64_t)a.T * a.H + 3) / 4)), dim3(256), 0, s, a, j);
    return hipGetLastError();
  }
  return hipSuccess;
}

template <int DT>
hipError_t launch_dim(const AttnArgs& a, const AttnPlan& p, void* ws, hipStream_t s) {
  const bool paged = a.k.table != nullptr;
  if (a.D == 64) return paged ? launch_all<DT, 64, true>(a, p, ws, s) : launch_all<DT, 64, false>(a, p, ws, s);
  if (a.D == 128) return paged ? launch_all<DT, 128, true>(a, p, ws, s) : launch_all<DT, 128, false>(a, p, ws, s);
  if (a.D == 256) return paged ? launch_all<DT, 256, true>(a, p, ws, s) : launch_all<DT, 256, false>(a, p, ws, s);
  return hipErrorInvalidValue;
}

uint32_t up(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

}  // namespace

AttnPlan plan_attn(int kind, uint32_t rows, uint32_t seqs, uint32_t groups, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                   uint32_t max_keys, uint32_t max_prefix) {
  AttnPlan p{};
  const uint32_t G = heads / kv_heads, cus = (uint32_t)cu_count();
  const uint64_t all_rows = (uint64_t)rows * G;
  p.prefix = kind == HQ_ATTN_SHARED;
  // Few rows a sequence: tiles of 16.
  p.row = p.prefix || all_rows <= 32ull * seqs;
  p.tile = p.prefix || !p.row;
  max_keys = std::max(max_keys, 1u);
  if (p.tile) {
    const uint32_t keys = p.prefix ? std::max(max_prefix, 1u) : max_keys;
    const uint32_t tiles = up(all_rows, 128) + (p.prefix ? groups : seqs);
    const uint32_t want = up(2 * cus, tiles * kv_heads);  // workgroups for two on each CU
    p.tile_keys = std::max(256u, up(up(keys, want), kKeys) * kKeys);
    p.tile_splits = std::max(1u, up(keys, p.tile_keys));
    p.tile_grid = tiles * kv_heads * p.tile_splits;
  }
  if (p.row) {
    const uint32_t waves = dim == 256 ? 2u : 4u, step = waves * kRowKeys;
    const uint32_t per = up(G, 16), tiles = rows == seqs ? seqs * per : up(all_rows, 16) + seqs;
    p.row_keys = std::max(step, up(up((uint64_t)tiles * kv_heads * max_keys, 8 * cus), step) * step);
    p.row_splits = up(max_keys, p.row_keys);
    p.row_grid = tiles * kv_heads * p.row_splits;
  }
  if (p.prefix || p.tile_splits > 1 || p.row_splits > 1) {
    p.slots = p.tile_splits + p.row_splits;
    const size_t places = (size_t)rows * heads * p.slots;
    p.o_offset = (places * sizeof(f2) + 255) / 256 * 256;
    p.ws = kCounterBytes + p.o_offset + places * dim * sizeof(float);
  }
  return p;
}

void describe_attn(int kind, const AttnPlan& p, char* buf, size_t len) {
  char t[160] = "", r[160] = "";
  if (p.tile) std::snprintf(t, sizeof t, "hq_attn_tile_kernel%s grid=%u splits=%u of %u keys", p.prefix ? "<prefix>" : "", p.tile_grid,
                            p.tile_splits, p.tile_keys);
  if (p.row) std::snprintf(r, sizeof r, "hq_attn_row_kernel grid=%u splits=%u of %u keys", p.row_grid, p.row_splits, p.row_keys);
  std::snprintf(buf, len, "%s%s%s%s ws=%zu", t, p.tile && p.row ? ", " : "", r, p.slots ? ", hq_attn_join_kernel" : "", p.ws);
  (void)kind;
}

hipError_t launch_attn(int dtype, const AttnArgs& a, const AttnPlan& p, void* ws, hipStream_t s) {
  return dtype == HQ_DTYPE_F16 ? launch_dim<HQ_DTYPE_F16>(a, p, ws, s) : launch_dim<HQ_DTYPE_BF16>(a, p, ws, s);
}

}  // namespace hq
