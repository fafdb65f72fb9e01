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
// hq_attn_prefix_kernel: both in one launch, for rows that share a prefix.
// hq_attn_join_kernel: joins the parts of rows whose keys were split between workgroups.
// Times in comments are an MI355X's, of calls replayed from a graph.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <type_traits>

#include "hq_attn.hpp"
#include "hq_device.hpp"
#include "hq_internal.hpp"

namespace hq {

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

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p;
}
// Transposing reads: four rows of 16 elements, 8 bytes from each lane of 16; lane i gets column i. A
// fragment is two of them.
template <int OFF, int NEXT>
__device__ __forceinline__ u4 lds_read_tr(uint32_t at) {
  typedef __attribute__((address_space(3))) s4* lds_s4;
  const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(at + OFF)));
  const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(at + OFF + NEXT)));
  return u4{a[0], a[1], b[0], b[1]};
}
// Several fragments, in asm and waited for there: the compiler holds the builtin back until every copy
// into LDS that it knows to be under way has landed.
template <int OFF, int NEXT>
__device__ __forceinline__ void lds_read_tr(const uint32_t (&at)[4], u4 (&f)[4]) {
  u2 a, b, c, d, e, g, h, i;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
      "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d), "=&v"(e), "=&v"(g), "=&v"(h), "=&v"(i)
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "i"(OFF), "i"(OFF + NEXT));
  f[0] = u4{a[0], a[1], b[0], b[1]};
  f[1] = u4{c[0], c[1], d[0], d[1]};
  f[2] = u4{e[0], e[1], g[0], g[1]};
  f[3] = u4{h[0], h[1], i[0], i[1]};
}
template <int I>
using Int = std::integral_constant<int, I>;
// f(Int<0>) .. f(Int<N - 1>).
template <int N, class F>
__device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(Int<N - 1>{});
  }
}

// Two weights, each rounded to nearest in the activation type (it is the type of V, and the MFMA has
// one for both operands): outputs are off by 1.1 to 1.4 times what they are with fp32 weights (relative to their
// norm, bf16 0.0019 to 0.0023 for 0.0015 to 0.0017, fp16 0.00019 to 0.00029 for 0.00017 to 0.00021).
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

// Weights are exp2(c s - fl(c m)): past 2^22 the product's rounding is more than 1/4 of a power of two, at 2^28 16
// powers and fp16's weights lose bits or vanish, at 2^31 fp32's do. Rows whose maximum is past it are computed
// again from c (s - m).
constexpr float kFar = 4194304.f;
constexpr float kNone = -FLT_MAX;  // the maximum of no score: finite, so that differences with it are no NaN

__device__ __forceinline__ void report(uint32_t* status, uint32_t what) {
  __hip_atomic_fetch_or(status, what, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t clamp_u(int32_t v, uint32_t hi) { return v < 0 ? 0u : min((uint32_t)v, hi); }
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

__device__ __forceinline__ uint32_t sum_lanes(uint32_t x) { return lane_value(scan_sum(x), 63); }
__device__ __forceinline__ uint32_t min_lanes(uint32_t x) {
  return lane_value(scan(x, ~0u, [](uint32_t a, uint32_t b) { return min(a, b); }), 63);
}
__device__ __forceinline__ uint32_t max_lanes(uint32_t x) {
  return lane_value(scan(x, 0, [](uint32_t a, uint32_t b) { return max(a, b); }), 63);
}
// f of the values of the lanes that are 16, 32 and 48 away.
template <class F>
__device__ __forceinline__ float over_quads(float x, F f) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// ---- sequences ----
// The loads that a workgroup starts with depend on each other (offsets, a row's number, its length, its
// pages, its keys), and short calls last little longer than they do: what does not depend on the last
// load's result is loaded beside it.

// What a tile works on: rows [r0, R) of a sequence, or of a group for its shared prefix, whose first token
// is q0 of nq.
struct Work {
  uint32_t b, q0, nq, R, r0;
  uint32_t key0;  // packed: row of key 0 in K and V
};

// Cache row of sequence b; a number out of range is reported where `ok` is asked, and stands for row 0.
__device__ __forceinline__ int32_t row_number(const AttnKeys& k, uint32_t b) { return k.rows ? k.rows[b] : (int32_t)b; }
__device__ __forceinline__ bool row_ok(const AttnKeys& k, int32_t row) { return (uint32_t)row < k.cache_rows; }
__device__ __forceinline__ int32_t row_length(const AttnKeys& k, int32_t row) { return k.lens[row_ok(k, row) ? row : 0]; }
__device__ __forceinline__ uint32_t length_or_report(const AttnKeys& k, int32_t row, int32_t len) {
  if (!row_ok(k, row)) {
    report(k.status, HQ_CACHE_BAD_ROW);
    return 0;
  }
  return clamp_u(len, k.max_pages << k.page_shift);
}
// The tokens of a group's shared prefix that lie in whole pages: no more than its first row holds.
__device__ __forceinline__ uint32_t whole_pages(const AttnKeys& k, int32_t first_row, int32_t first_len, int32_t prefix) {
  const uint32_t len = row_ok(k, first_row) ? clamp_u(first_len, k.max_pages << k.page_shift) : 0u;
  return min(len, clamp_u(prefix, 1u << 30)) >> k.page_shift << k.page_shift;
}

// Whether the groups hold each of B sequences once: starts from 0 to B, not falling. Where they don't, every workgroup finds
// so, none works on a prefix and all keys of a row are its own. Of entry b, and of entries base .. n - 1.
__device__ __forceinline__ bool entry_ok(int32_t first, int32_t end, uint32_t b, uint32_t n, uint32_t B) {
  return first <= end && (b > 0 || first == 0) && (b + 1 < n || end == (int32_t)B);
}
__device__ __forceinline__ bool entries_ok(const int32_t* starts, uint32_t base, uint32_t n, uint32_t B) {
  bool good = true;
  for (; base < n; base += 64) {
    const uint32_t b = min(base + (threadIdx.x & 63u), n - 1);
    good = good && entry_ok(starts[b], starts[b + 1], b, n, B);
  }
  return __ballot(!good) == 0;
}

// Tokens of entry b of a list of offsets (queries of a sequence, sequences of a group), held to [0, most].
__device__ __forceinline__ uint32_t span(const int32_t* cu, uint32_t b, uint32_t most, uint32_t& first) {
  first = clamp_u(cu[b], most);
  const uint32_t end = clamp_u(cu[b + 1], most);
  return end > first ? end - first : 0u;
}

// The idx-th tile of `rows` rows over all entries, by one wavefront: the entries' tiles are counted 64
// at a time. Inside an entry the last tile comes first: under the causal mask it has the most keys.
template <bool GROUPS>
__device__ __forceinline__ bool find_tile(const int32_t* cu, uint32_t n, uint32_t most, uint32_t G, uint32_t rows, uint32_t idx,
                                          Work& w) {
  const uint32_t lane = threadIdx.x & 63u;
  if (!cu) {  // one token each
    const uint32_t per = (G + rows - 1) / rows;
    w.b = uni(idx / per);
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
    if constexpr (GROUPS) {
      const uint32_t at = min(b, n - 1);
      const int32_t lo = cu[at], hi = cu[at + 1];
      if (__ballot(!entry_ok(lo, hi, at, n, most))) return false;
      first = (uint32_t)lo;
      nq = b < n ? (uint32_t)(hi - lo) : 0u;
    } else {
      if (b < n) nq = span(cu, b, most, first);
    }
    const uint32_t tiles = (nq * G + rows - 1) / rows;
    const uint32_t x = scan_sum(tiles);
    const uint64_t past = __ballot(before + x > idx);
    if (past) {
      const int at = __builtin_ctzll(past);
      w.b = base + at;
      w.q0 = lane_value(first, at);
      w.nq = lane_value(nq, at);
      w.R = w.nq * G;
      w.r0 = (before + lane_value(x, at) - 1 - idx) * rows;
      return !GROUPS || entries_ok(cu, base + 64, n, most);
    }
    before += lane_value(x, 63);
  }
  return false;
}

// Work of slot `slot` of `slots` where rows' keys are shared between workgroups (row kernel): the tiles of 16
// rows get slots by the keys they have, so that a batch of long and short rows ends together (32 rows of 30 to 8000
// tokens: 50 us, with equal shares 65; the search costs a uniform batch 0.5). A share is
// `unit` tiles of 32 keys, the least of three that the slots are enough for: sum / slots, where rounding up may
// cost more than there are; sum / (slots - tiles), where it can't; their mean. No tile has more shares than
// sqrt(its key tiles): the last workgroup reads the others' parts alone.
struct Share {
  uint32_t split, of;  // this workgroup's number among those of its tile
  int32_t row, len;    // paged: cache row of the sequence, and its length as read
};
template <uint32_t WAVES, bool PAGED, bool GROUPS>
__device__ __forceinline__ bool find_share(const AttnArgs& a, uint32_t slots, uint32_t like, uint32_t slot, Work& w, Share& sh) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t first, nq, tiles, keys;
  int32_t row, len;
  auto entry = [&](uint32_t b) __attribute__((always_inline)) {
    first = nq = keys = 0;
    row = len = 0;
    if (b < a.B) {
      if constexpr (PAGED) row = row_number(a.k, b);
      if (a.cu_q) {
        nq = span(a.cu_q, b, a.T, first);
      } else {
        first = b;
        nq = 1;
      }
      if constexpr (PAGED) {
        len = row_length(a.k, row);
        keys = GROUPS ? like : clamp_u(len, a.k.max_pages << a.k.page_shift);  // of a group: all alike
      } else if (a.k.cu_k == a.cu_q && a.k.total_k >= a.T) {
        keys = nq;
      } else {
        uint32_t k0;
        keys = span(a.k.cu_k, b, a.k.total_k, k0);
      }
    }
    tiles = (nq * a.G + 15) / 16;
    keys = min((keys + 31) / 32, 1u << 22);  // tiles of them
  };
  auto shares = [&](uint32_t unit) __attribute__((always_inline)) {
    const uint32_t most = (uint32_t)__builtin_ceilf(__builtin_amdgcn_sqrtf((float)keys));
    return max(1u, min(min((keys + unit - 1) / unit, most), 64u));
  };
  uint32_t all = 0, work = 0;
  for (uint32_t base = 0; base < a.B; base += 64) {
    entry(base + lane);
    all += sum_lanes(tiles);
    work += sum_lanes(tiles * keys);
  }
  uint32_t unit = 1u << 22;  // lists that are not offsets may name more tiles than there can be: one share each
  if (all < slots) {
    const uint32_t lo = max((work + slots - 1) / slots, WAVES), hi = max((work + slots - all - 1) / (slots - all), lo), mid = (lo + hi) / 2;
    uint32_t got = 0;
    for (uint32_t base = 0; base < a.B; base += 64) {
      if (a.B > 64) entry(base + lane);
      got += sum_lanes(tiles * shares(lo) << 16 | tiles * shares(mid));
    }
    unit = got >> 16 <= slots ? lo : (got & 0xFFFFu) <= slots ? mid : hi;
  }
  uint32_t before = 0;
  for (uint32_t base = 0; base < a.B; base += 64) {
    if (a.B > 64) entry(base + lane);
    const uint32_t each = shares(unit), mine = tiles * each;
    const uint32_t x = scan_sum(mine);
    const uint64_t past = __ballot(before + x > slot);
    if (past) {
      const int at = __builtin_ctzll(past);
      const uint32_t off = slot - before - lane_value(x - mine, at);
      w.b = base + at;
      w.q0 = lane_value(first, at);
      w.nq = lane_value(nq, at);
      w.R = w.nq * a.G;
      sh.of = lane_value(each, at);
      w.r0 = off / sh.of * 16;
      sh.split = off % sh.of;
      sh.row = (int32_t)lane_value((uint32_t)row, at);
      sh.len = (int32_t)lane_value((uint32_t)len, at);
      return true;
    }
    before += lane_value(x, 63);
  }
  return false;
}

// The group of sequence b, the last one that starts at or before it, where it starts, and whether all are sound (looked at
// here, with the entries at hand: in a pass of its own it took 0.4 us of 28).
__device__ __forceinline__ uint32_t group_of(const AttnArgs& a, uint32_t b, uint32_t& first, bool& ok) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t g = 0;
  bool good = true;
  first = 0;
  for (uint32_t base = 0; base < a.groups; base += 64) {
    const uint32_t i = min(base + lane, a.groups - 1);
    const int32_t at = a.starts[i], end = a.starts[i + 1];
    good = good && entry_ok(at, end, i, a.groups, a.B);
    const uint64_t before = __ballot(at <= (int32_t)b && base + lane < a.groups);
    if (before) {
      const int last = 63 - __builtin_clzll(before);
      g = base + last;
      first = clamp_u(__builtin_amdgcn_readlane(at, last), a.B - 1);
    }
  }
  ok = __ballot(!good) == 0;
  return g;
}

__device__ __forceinline__ uint32_t page_or_report(const AttnKeys& k, int32_t page) {
  if ((uint32_t)page < k.pages) return (uint32_t)page;
  report(k.status, HQ_CACHE_BAD_PAGE);
  return 0;
}

// Pages of tiles of KEYS keys, held in registers a batch of 64 blocks of 16 keys ahead: lane j of a batch
// holds block j, that is block j % (KEYS / 16) of the batch's tile j / (KEYS / 16); tile i of the wavefront
// begins at key first + i * step. Pages hold 16 tokens or more, so a block lies in one.
template <int KEYS>
struct Pages {
  static constexpr uint32_t kSub = KEYS / 16, kBatch = 64 / kSub;
  const int32_t* table;
  uint32_t first, step, nk;
  int32_t now, next;

  __device__ __forceinline__ int32_t load(const AttnKeys& k, uint32_t batch) const {
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t key = first + (uint64_t)(batch * kBatch + lane / kSub) * step + lane % kSub * 16;
    return table[min((uint32_t)min(key >> k.page_shift, (uint64_t)k.max_pages - 1), k.max_pages - 1)];
  }
  // Pages of batch `batch` as numbers that can be followed.
  __device__ __forceinline__ int32_t held(const AttnKeys& k, uint32_t batch, int32_t p) const {
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t key = first + (uint64_t)(batch * kBatch + lane / kSub) * step + lane % kSub * 16;
    return key < nk ? (int32_t)page_or_report(k, p) : 0;
  }
  __device__ __forceinline__ void start(const AttnKeys& k) {
    now = load(k, 0);
    next = load(k, 1);
    now = held(k, 0, now);
  }
  // Before tile i's first use of of(): every tile in turn.
  __device__ __forceinline__ void advance(const AttnKeys& k, uint32_t i) {
    if (i % kBatch || i == 0) return;
    now = held(k, i / kBatch, next);
    next = load(k, i / kBatch + 1);
  }
  // Page of block `sub` of tile i.
  __device__ __forceinline__ uint32_t page(uint32_t i, uint32_t sub) const {
    return (uint32_t)__builtin_amdgcn_readlane(now, i % kBatch * kSub + sub);
  }
};

// Keys from `base` (uniform) on, `rows` of them `step` bytes apart (at most 64 and 2^24): what lies past them
// reads as 0. A lane's offset is 32-bit; the descriptor is made anew for each tile, since a pool or an
// operand may span more than 4 GiB.
__device__ __forceinline__ u4 keys_words(const uint16_t* base, uint32_t rows, uint32_t step) {
  // All are uniform; said so, because the compiler multiplies 64-bit numbers in vector registers.
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  return u4{uni((uint32_t)p), uni((uint32_t)(p >> 32)) & 0xFFFFu, uni(rows * step), (uint32_t)kBufferFlags};
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t keys_rsrc(const uint16_t* base, uint32_t rows, uint32_t step) {
  const u4 d = keys_words(base, rows, step);
  return make_rsrc(reinterpret_cast<const void*>((uint64_t)d[1] << 32 | d[0]), d[2]);
}
// buffer_to_lds16 of such a descriptor, to LDS address `to` (uniform), unknown to the compiler's counts: it
// would hold every transposing read back until all copies under way have landed. Whoever uses it waits for
// its copies itself; the compiler's own waits for loads only become longer by it. It has no destination
// register.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // it warns that m0, its own, is not saved; named, it knows that what it put there is gone
__device__ __forceinline__ void copy_to_lds16(u4 d, uint32_t to, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(d) : "memory", "m0");
}
#pragma clang diagnostic pop

// ---- parts of rows whose keys are split ----
// Row (token t, head h) has `slots` places: fp32 O [D] (not divided by the sum), the maximum times c and
// the sum; a place without weight has sum 0 and no O.
struct Parts {
  float* o;
  f2* ml;
  uint32_t slots;
};

struct TilePlan {
  uint32_t splits;  // workgroups that share a tile's keys, in equal runs of them
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
// 4 operations a score and dim: bound by the matrix pipe, and as much by what feeds it. A fragment of K or
// V (1 KB from LDS) is one product of 32 rows, 32 cycles of LDS for the CU's four SIMDs and 32 of each
// one's matrix pipe; 32 scores a lane are about as many cycles of the vector pipe as their 16 + 16 products at
// 128 dims. So the three run side by side: the next tile's scores beside this one's exponentials, K fragments
// read a step and V fragments two products ahead. 8192 tokens on 48/8 heads of 128, bf16: 721 us in the trace of the
// counters, 1143 TFLOP/s, matrix pipe busy 67% (LDS as much, by its bytes) and vector pipe 61% at the 1.65 GHz that the card
// holds under it, no bank conflicts (718 to 760 us over boxes). Heads of 256 leave registers for one wavefront a SIMD (a workgroup
// a CU): 2048 + 1531 tokens on 24/4 heads 113 us, 711 TFLOP/s, matrix pipe 33%; tiles of 32 keys 10% slower there and
// everywhere, of 128 on heads of 64 slower too. Heads of 64 have twice the exponentials a product: 4096 tokens on 32/4 heads
// 84 us, 816 TFLOP/s, vector pipe 71%, matrix pipe 42%. A workgroup alone on its CU takes 1.1 us a tile, 0.9 without its copies: the rest is issue and
// latency, so short calls gain by sharing keys (tile_splits).
constexpr int kKeys = 64;  // keys of a tile

template <int D>
constexpr uint32_t tile_stage_bytes() {
  return 2u * kKeys * D * 2u;
}

template <int DT, int D, int NW, bool PAGED, bool PREFIX>
__device__ __forceinline__ void tile_body(const AttnArgs& a, const TilePlan& pl, uint32_t block) {
  constexpr uint32_t BR = NW * 32;
  constexpr uint32_t kPitch = 2 * D, kStage = tile_stage_bytes<D>(), kVOff = kStage / 2;
  constexpr int kSteps = D / 16, kDims = D / 32;
  constexpr uint32_t kRowsPerLoad = 1024 / kPitch, kLoads = kKeys / kRowsPerLoad / NW;  // loads of a wavefront, K and V each
  extern __shared__ __align__(1024) unsigned char smem[];

  const uint32_t lane = threadIdx.x & 63u, wave = uni(threadIdx.x >> 6);
  const uint32_t l32 = lane & 31u, half = lane >> 5;

  // Heads run fastest: workgroups go to the XCDs in turn, so with eight key/value heads each XCD's L2
  // sees the keys of one.
  const uint32_t kvh = block % a.Hkv, rest = block / a.Hkv;
  const uint32_t split = rest % pl.splits, idx = rest / pl.splits;
  Work w{};
  if (!find_tile<PREFIX>(PREFIX ? a.starts : a.cu_q, PREFIX ? a.groups : a.B, PREFIX ? a.B : a.T, a.G, BR, idx, w)) return;
  // This lane's row.
  const uint32_t r_mine = w.r0 + wave * 32 + l32;
  const bool live = r_mine < w.R;
  const uint32_t r = min(r_mine, w.R - 1), token = r / a.G, head = kvh * a.G + (r - token * a.G);

  const int32_t* table = nullptr;
  uint32_t nk, lim = 0;  // keys of the sequence, and those below lim this lane's row may see
  if constexpr (PAGED) {
    const int32_t row = row_number(a.k, PREFIX ? w.q0 : w.b);
    table = a.k.table + (row_ok(a.k, row) ? row : 0) * a.k.table_stride;
    if constexpr (PREFIX) {
      const int32_t own = row_number(a.k, w.q0 + token), prefix = a.prefix[w.b];
      const int32_t len = row_length(a.k, row), own_len = row_length(a.k, own);
      nk = uni(whole_pages(a.k, row, len, prefix));
      lim = min(nk, length_or_report(a.k, own, own_len));
    } else {
      nk = uni(length_or_report(a.k, row, row_length(a.k, row)));
    }
  } else if (a.k.cu_k == a.cu_q && a.k.total_k >= a.T) {
    nk = w.nq;
    w.key0 = w.q0;
  } else {
    nk = uni(span(a.k.cu_k, w.b, a.k.total_k, w.key0));
    w.key0 = uni(w.key0);
  }
  if constexpr (!PREFIX) {
    lim = nk;
    if (a.causal) {
      const int64_t n = (int64_t)token + nk - w.nq + 1;
      lim = n < 0 ? 0u : (uint32_t)n;
    }
  }
  const uint32_t lim_min = min_lanes(lim), lim_max = w.r0 + wave * 32 < w.R ? max_lanes(lim) : 0u;

  // Keys of this workgroup: up to the last that any of its rows sees.
  uint32_t wg_lim = nk;
  if (!PREFIX && a.causal) {
    const int64_t n = (int64_t)((min(w.r0 + BR, w.R) - 1) / a.G) + nk - w.nq + 1;
    wg_lim = n < 0 ? 0u : (uint32_t)n;
  }
  const uint32_t tiles = (wg_lim + kKeys - 1) / kKeys, per = (tiles + pl.splits - 1) / pl.splits;
  const uint32_t t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);

  const uint16_t* const qp = a.Q + (int64_t)(w.q0 + token) * a.q_row + head * a.q_head + 8 * half;
  u4 q[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const u4*>(qp + 16 * s);

  const float c = a.scale * 1.44269504088896340736f;
  const uint16_t* const Kh = a.k.K + kvh * a.k.k_head;
  const uint16_t* const Vh = a.k.V + kvh * a.k.v_head;

  // Copies of tile t into a stage: load i of the wavefront brings rows kRowsPerLoad (i NW + wave) ...; a
  // lane's row and source chunk undo the swizzle. Keys past the last are 0 (masked below).
  const uint32_t in_row = lane / (D / 8), in_chunk = lane % (D / 8);
  const uint32_t k_step = (uint32_t)a.k.k_row * 2, v_step = (uint32_t)a.k.v_row * 2, page_mask = (1u << a.k.page_shift) - 1;
  Pages<kKeys> pages{table, t0 * kKeys, kKeys, nk, 0, 0};
  const bool whole = !PAGED || a.k.page_shift >= 6;  // a tile lies in one page
  const uint32_t lds0 = uni(lds_address(smem)) + wave * 1024;
  // Offsets of load 0, and of load 1 less its rows: the swizzle of K goes with the row modulo 16, which later
  // loads have in common with one of them.
  uint32_t k_off[2], v_off[2];
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    const uint32_t row = (i * NW + wave) * kRowsPerLoad + in_row;
    k_off[i] = (wave * kRowsPerLoad + in_row) * k_step + ((in_chunk ^ swz_k<D>(row)) << 4);
    v_off[i] = (wave * kRowsPerLoad + in_row) * v_step + ((in_chunk ^ swz_v<D>(row)) << 4);
  }
  auto copy = [&](uint32_t t, const uint16_t* from, int64_t row_stride, uint32_t step, const uint32_t (&off)[2], uint32_t to)
                  __attribute__((always_inline)) {
    const uint32_t key = t * kKeys, left = min(nk - key, (uint32_t)kKeys);
    if (whole) {
      int64_t at;
      if constexpr (PAGED) at = pages.page(t - t0, 0) * a.k.page_stride + (key & page_mask) * row_stride;
      else at = (int64_t)(w.key0 + key) * row_stride;
      const u4 r = keys_words(from + at, left, step);
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) copy_to_lds16(r, to + i * NW * 1024, off[i & 1] + i * NW * kRowsPerLoad * step);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {  // a block of 16 rows each
        const uint32_t row0 = (i * NW + wave) * kRowsPerLoad, first = row0 & ~15u;
        const int64_t at = pages.page(t - t0, row0 / 16) * a.k.page_stride + ((key + first) & page_mask) * row_stride;
        copy_to_lds16(keys_words(from + at, left > first ? left - first : 0u, step), to + i * NW * 1024,
                      off[i & 1] + (row0 - first - wave * kRowsPerLoad) * step);
      }
    }
  };
  auto copy_k = [&](uint32_t t) __attribute__((always_inline)) {
    copy(t, Kh, a.k.k_row, k_step, k_off, lds0 + (t & 1u) * kStage);
  };
  auto copy_v = [&](uint32_t t) __attribute__((always_inline)) {
    copy(t, Vh, a.k.v_row, v_step, v_off, lds0 + (t & 1u) * kStage + kVOff);
  };

  // LDS places of this lane's fragments. K^T: row l32 (+ 32), dims 16 s + 8 half, chunk 2 s + half: the place of
  // step 0, s << 5 exclusive-or'ed. V^T: keys 4 half + (lane % 16) / 4 (+ 8, + 16 steps), dims 32 dt + 16
  // (l32 / 16) + 4 (lane % 4): dt << 6 likewise. (Held apart they are 14 registers that the kernel has not.)
  const uint32_t k_at = l32 * kPitch + ((half ^ swz_k<D>(l32)) << 4);
  const uint32_t v_row = 4 * half + ((lane & 15u) >> 2);
  const uint32_t v_at = lds_address(smem) + kVOff + v_row * kPitch + (((2 * (l32 >> 4) + ((lane & 3u) >> 1)) ^ swz_v<D>(v_row)) << 4) + 8 * (lane & 1u);

  f16x o[kDims];
  float m, l;

  auto opaque = [](uint32_t v) __attribute__((always_inline)) {  // what is computed from it stays in its tile
    asm volatile("" : "+v"(v));
    return v;
  };
  auto scores = [&](uint32_t at, f16x (&s)[2], int i) __attribute__((always_inline)) {  // step i of S^T = K Q^T
    const unsigned char* const p = smem + (at ^ (uint32_t)(i << 5));
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
      s[kt] = mfma32x32x16<DT>(*reinterpret_cast<const u4*>(p + kt * 32 * kPitch), q[i], i ? s[kt] : f16x{});
  };
  auto k_read = [&](uint32_t at, u4 (&f)[2], int i) __attribute__((always_inline)) {
    const unsigned char* const p = smem + (at ^ (uint32_t)(i << 5));
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) f[kt] = *reinterpret_cast<const u4*>(p + kt * 32 * kPitch);
  };
  auto mask = [&](uint32_t t, f16x (&s)[2]) __attribute__((always_inline)) {
    const uint32_t k0 = t * kKeys + 4 * half;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (k0 + 32 * kt + 8 * (v / 4) + v % 4 >= lim) s[kt][v] = -INFINITY;
  };
  auto both_halves = [&](float x, float y) {  // this lane's and the other half's
    const auto e = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    return f2{__uint_as_float(e[0]), __uint_as_float(e[1])};
  };
  // The maximum follows the scores only where it lags by more than kLag: each row by itself, so that its
  // bits do not depend on its neighbours, and the sums are rescaled only where some row's moves.
  auto follow = [&](float top) __attribute__((always_inline)) {
    const f2 e = both_halves(top, top);
    top = fmaxf(e[0], e[1]);
    if (__any((top - m) * c > Weights<DT>::kLag)) {
      const float n = (top - m) * c > Weights<DT>::kLag ? top : m, al = __builtin_amdgcn_exp2f((m - n) * c);
      m = n;
      l *= al;
#pragma unroll
      for (int dt = 0; dt < kDims; ++dt) o[dt] *= al;
    }
  };
  auto meet = [&]() __attribute__((always_inline)) {  // the wavefronts' copies have landed, their reads are done
    __builtin_amdgcn_s_waitcnt(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  auto reset = [&]() __attribute__((always_inline)) {
    m = kNone;
    l = 0.f;
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt) o[dt] = f16x{};
    if constexpr (PAGED)
      if (t1 > t0) pages.start(a.k);
  };

  // Tiles this wavefront computes: t0 .. tw - 1 (its rows see nothing of the others).
  const uint32_t tw = min(t1, (lim_max + kKeys - 1) / kKeys);
  reset();
  if (t1 > t0) {
    // The scores of a tile are computed while the weights of the one before are, and its maximum while that
    // one's second product runs: the matrix and the vector pipes each have the other's work beside theirs.
    f16x s0[2], s1[2];  // of a tile and of the next, in turn
    copy_k(t0);
    copy_v(t0);
    if (t0 + 1 < t1) {
      if constexpr (PAGED) pages.advance(a.k, 1);
      copy_k(t0 + 1);
    }
    meet();
    if (t0 < tw) {
      const uint32_t at = opaque(k_at + (t0 & 1u) * kStage);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) scores(at, s0, i);
      if (t0 * kKeys + kKeys > lim_min) mask(t0, s0);
      float top = s0[0][0];
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(fmaxf(top, s0[0][v]), s0[1][v]);
      follow(top);
    }
    auto tile = [&](uint32_t t, auto next, f16x (&s)[2], f16x (&ns)[2]) __attribute__((always_inline)) {
      constexpr bool more = decltype(next)::value;  // the next tile is this wavefront's too
      // With and without a next tile are two pieces of code: what they share is not taken out of them.
      if constexpr (more) asm volatile("" : "+v"(s[0]), "+v"(s[1]));
      const float mc = fmaxf(m * c, kNone) - Weights<DT>::kLift;
      u4 p[4];
      float sum = 0.f;
      const uint32_t at = opaque(k_at + ((t + 1) & 1u) * kStage);
      // The SIMD's other wavefront yields to scores and exponentials, which use both pipes: 8192 tokens on heads of
      // 128 752 -> 736 us, ragged prompts 38.4 -> 37.8. On heads of 64 it took 60.8 for 57.7 and 83.6 for
      // 86.4; on heads of 256 there is no other.
      if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);
      u4 kf[2][2];
      if constexpr (more) k_read(at, kf[0], 0);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        if constexpr (more) {
          if (i + 1 < kSteps) k_read(at, kf[(i + 1) & 1], i + 1);
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) ns[kt] = mfma32x32x16<DT>(kf[i & 1][kt], q[i], i ? ns[kt] : f16x{});
        }
#pragma unroll
        for (int u = 16 * i / kSteps; u < 16 * (i + 1) / kSteps; ++u) {  // weights 2 u, 2 u + 1 of 32
          const int v = 2 * (u & 7);
          const float x = __builtin_amdgcn_exp2f(fmaf(s[u / 8][v], c, -mc)), y = __builtin_amdgcn_exp2f(fmaf(s[u / 8][v + 1], c, -mc));
          sum += x + y;
          p[u / 4][u & 3] = pack2<DT>(x, y);
        }
        asm volatile("" : "+v"(sum));  // added here, not in a row afterwards
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
      l += sum;
      if constexpr (more) {
        // Both stay above, in turn.
        asm volatile("" : "+v"(ns[0]), "+v"(ns[1]), "+v"(p[0]), "+v"(p[1]), "+v"(p[2]), "+v"(p[3]));
      }
      // Products of a fragment of V each, read two of them ahead.
      constexpr int kAll = 4 * kDims, kAhead = 2;
      const uint32_t v0 = opaque(v_at + (t & 1u) * kStage);
      u4 vf[kAhead];
      auto v_read = [&](auto nc) __attribute__((always_inline)) {
        constexpr int n = decltype(nc)::value;
        vf[n % kAhead] = lds_read_tr<16 * (n / kDims) * (int)kPitch, 8 * (int)kPitch>(v0 ^ (uint32_t)(n % kDims << 6));
      };
      each<kAhead>(v_read);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (more)
        if ((t + 1) * kKeys + kKeys > lim_min) mask(t + 1, ns);
      float top = more ? ns[0][0] : 0.f;
      each<kAll>([&](auto nc) __attribute__((always_inline)) {
        constexpr int n = decltype(nc)::value;
        o[n % kDims] = mfma32x32x16<DT>(vf[n % kAhead], p[n / kDims], o[n % kDims]);
        if constexpr (n + kAhead < kAll) v_read(Int<n + kAhead>{});
        if constexpr (more)
#pragma unroll
          for (int v = 16 * n / kAll; v < 16 * (n + 1) / kAll; ++v) top = fmaxf(fmaxf(top, ns[0][v]), ns[1][v]);
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (more) follow(top);
    };
    auto ahead = [&](uint32_t t) __attribute__((always_inline)) {  // copies of the next tiles, before tile t
      meet();
      if (t + 1 < t1) copy_v(t + 1);
      if (t + 2 < t1) {
        if constexpr (PAGED) pages.advance(a.k, t + 2 - t0);
        copy_k(t + 2);
      }
    };
    uint32_t t = t0;
    for (; t + 2 < tw; t += 2) {
      ahead(t);
      tile(t, std::true_type{}, s0, s1);
      ahead(t + 1);
      tile(t + 1, std::true_type{}, s1, s0);
    }
    if (t + 1 < tw) {
      ahead(t);
      tile(t, std::true_type{}, s0, s1);
      ahead(++t);
      tile(t, std::false_type{}, s1, s0);
      ++t;
    } else if (t < tw) {
      ahead(t);
      tile(t, std::false_type{}, s0, s1);
      ++t;
    }
    for (; t < t1; ++t) ahead(t);  // the others' tiles
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (the last one asked for none)
  }
  // Again where values are not finite (V at keys a row may not see, times its weight 0, may have made them), or
  // scores are far (kFar). Tile by tile, differences of scores before the factor, and those values apart.
  auto odd = [&]() {
    const f2 e = both_halves(l, l);
    l = e[0] + e[1];
    float bad = 0.f;
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
      for (int v = 0; v < 16; ++v) bad = fmaf(o[dt][v], 0.f, bad);
    return !(bad == 0.f) || (m != kNone && fabsf(m * c) > kFar);
  };
  if (__syncthreads_or(odd())) {
    reset();
    for (uint32_t t = t0; t < t1; ++t) {
      meet();
      if constexpr (PAGED) pages.advance(a.k, t - t0);
      copy_k(t);
      copy_v(t);
      meet();
      if (t >= tw) continue;
      f16x s[2];
      const uint32_t k0 = opaque(k_at + (t & 1u) * kStage), v0 = opaque(v_at + (t & 1u) * kStage);
#pragma unroll
      for (int i = 0; i < kSteps; ++i) scores(k0, s, i);
      const bool masked = t * kKeys + kKeys > lim_min;
      if (masked) mask(t, s);
      float top = s[0][0];
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(fmaxf(top, s[0][v]), s[1][v]);
      follow(top);
      u4 p[4];
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        const int v = 2 * (u & 7);
        const float x = __builtin_amdgcn_exp2f(fmaf(s[u / 8][v] - m, c, Weights<DT>::kLift));
        const float y = __builtin_amdgcn_exp2f(fmaf(s[u / 8][v + 1] - m, c, Weights<DT>::kLift));
        l += x + y;
        p[u / 4][u & 3] = pack2<DT>(x, y);
      }
      each<4>([&](auto jc) __attribute__((always_inline)) {
        constexpr int j = decltype(jc)::value;
        const uint32_t key = t * kKeys + 16 * j + 4 * half;
        const u4 sees = {seen2<DT>(key, lim), seen2<DT>(key + 2, lim), seen2<DT>(key + 8, lim), seen2<DT>(key + 10, lim)};
#pragma unroll
        for (int d0 = 0; d0 < kDims; d0 += 2) {
          u4 f[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) f[i] = lds_read_tr<16 * j * (int)kPitch, 8 * (int)kPitch>(v0 ^ (uint32_t)((d0 + i) << 6));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            u4 finite, code;
            split_odd<DT>(f[i], finite, code);
            o[d0 + i] = mfma32x32x16<DT>(finite, p[j], o[d0 + i]);
            const f16x count = mfma32x32x16<DT>(code, sees, f16x{});
#pragma unroll
            for (int v = 0; v < 16; ++v) o[d0 + i][v] += odd_value(count[v]);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      });
    }
    odd();
  }
  if (!live) return;
  const uint32_t tok = w.q0 + token;
  const float mc = fmaxf(m * c, kNone) - Weights<DT>::kLift;
  if (pl.parts.slots) {
    const uint64_t at = ((uint64_t)tok * a.H + head) * pl.parts.slots + split;
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

template <int DT, int D, int NW, bool PAGED>
__global__ __launch_bounds__(NW * 64, D == 256 ? 1 : 2) void hq_attn_tile_kernel(AttnArgs a, TilePlan pl) {
  tile_body<DT, D, NW, PAGED, false>(a, pl, blockIdx.x);
}

// ---- few rows ----
constexpr int kRowKeys = 32;  // keys of a wavefront's tile

struct RowPlan {
  uint32_t slots;      // workgroups of a kv head where they share rows' keys (0: a workgroup for each 16 rows)
  uint32_t one;        // there is one tile, all slots are its shares
  uint32_t like;       // keys past the prefix that a group's rows are taken to have
  uint32_t* cnt;       // arrivals of a tile's workgroups, [kv head][its first slot], zero between launches
  float* o;            // their parts: [kv head][slot][16][D], and the maxima and sums [..][16]
  f2* ml;
  Parts to;            // where rows of a group leave their own keys' part, the last place (slots 0: rows are written out)
};

// As swz_v, for this kernel's reads: 16 rows of 32 bytes.
template <int D>
__device__ __forceinline__ uint32_t swz_rv(uint32_t r) {
  return D == 64 ? ((r >> 1) & 3u) << 1 : (r & 7u) << 1;
}

constexpr uint32_t kRowWaves = 4;
// Two stages of V per wavefront; the join of the wavefronts lies over them.
template <int D>
constexpr uint32_t row_lds_bytes() {
  const uint32_t stages = kRowWaves * 2u * (kRowKeys * D * 2u), join = kRowWaves * 16u * ((D + 4u) * 4u + 8u);
  return (stages > join ? stages : join) + 16u;
}
constexpr int kAgent = 16;  // cache policy of parts: seen by workgroups on other XCDs

// Tiles of 32 keys go to the shares' wavefronts in turn, (round * shares + share) * 4 + wavefront. A
// wavefront's K goes straight into the registers of its first product (a lane's 16 bytes of a row are 8
// consecutive dims, four lanes take 64 bytes), its V through LDS; both are a tile ahead, 32 KB a CU and more
// in flight. Bound by memory: 64 rows on 2048 tokens, 48/8 heads of 128, 91 us, 5.9 TB/s of keys and values (97 where
// pages hold tokens before heads); 16 rows on 37 to 8192, 24/4 heads of 256, 27 us, 4.0 TB/s (two wavefronts a workgroup, twice the parts to join
// by half the threads: 41). One row on 777: 8 us of launch, first loads, parts and join.
template <int DT, int D, bool PAGED, bool GROUPS>
__device__ __forceinline__ void row_body(const AttnArgs& a, const RowPlan& pl, uint32_t block) {
  constexpr uint32_t NW = kRowWaves;
  constexpr uint32_t kPitch = 2 * D, kStage = kRowKeys * kPitch;
  constexpr int kSteps = D / 32, kDims = D / 16;
  constexpr uint32_t kRowsPerLoad = 1024 / kPitch, kLoads = kRowKeys / kRowsPerLoad;
  extern __shared__ __align__(1024) unsigned char smem[];

  const uint32_t lane = threadIdx.x & 63u, wave = uni(threadIdx.x >> 6);
  const uint32_t l16 = lane & 15u, quad = lane >> 4;
  const uint32_t kvh = block % a.Hkv, slot = block / a.Hkv;
  Work w{};
  Share sh{0, 1, 0, 0};
  const bool find = pl.slots && !pl.one;
  if (find) {
    if (!find_share<NW, PAGED, GROUPS>(a, pl.slots, pl.like, slot, w, sh)) return;
  } else {
    if (!find_tile<false>(a.cu_q, a.B, a.T, a.G, 16, pl.one ? 0u : slot, w)) return;
    if (pl.one) {
      sh.split = slot;
      sh.of = pl.slots;
    }
    if constexpr (PAGED) sh.row = row_number(a.k, w.b);
  }
  const uint32_t split = sh.split;
  const uint32_t r_mine = w.r0 + l16;
  const uint32_t r = min(r_mine, w.R - 1), token = r / a.G, head = kvh * a.G + (r - token * a.G);
  const uint32_t t_first = split * NW + wave;

  const int32_t* table = nullptr;
  uint32_t nk, begin = 0;
  int32_t early = 0;  // pages of the first tile: lane j % 2 that of its block j
  bool grouped = true;
  if constexpr (PAGED) {
    uint32_t g = 0, first = 0;
    if constexpr (GROUPS) g = group_of(a, w.b, first, grouped);
    const int32_t row = sh.row;
    table = a.k.table + (row_ok(a.k, row) ? row : 0) * a.k.table_stride;
    if (!find) sh.len = row_length(a.k, row);
    if constexpr (GROUPS) {
      const int32_t first_row = row_number(a.k, first), prefix = a.prefix[g];
      const int32_t first_len = row_length(a.k, first_row);
      nk = uni(length_or_report(a.k, row, sh.len));
      begin = grouped ? min(nk, uni(whole_pages(a.k, first_row, first_len, prefix))) : 0u;
      if (!grouped) report(a.k.status, HQ_CACHE_BAD_ROW);
    }
    early = table[min((begin + t_first * kRowKeys + (lane & 1u) * 16) >> a.k.page_shift, a.k.max_pages - 1)];
    if constexpr (!GROUPS) nk = uni(length_or_report(a.k, row, sh.len));
  } else if (a.k.cu_k == a.cu_q && a.k.total_k >= a.T) {
    nk = w.nq;
    w.key0 = w.q0;
  } else {
    nk = uni(span(a.k.cu_k, w.b, a.k.total_k, w.key0));
    w.key0 = uni(w.key0);
  }

  uint32_t lim = nk, end = nk, full = nk;  // keys of this lane's row, of any row, of every row
  if (a.causal) {
    auto limit = [&](uint32_t t) {
      const int64_t n = (int64_t)t + nk - w.nq + 1;
      return n < 0 ? 0u : (uint32_t)n;
    };
    lim = limit(token);
    full = limit(w.r0 / a.G);
    end = limit((min(w.r0 + 16, w.R) - 1) / a.G);
  }
  const uint32_t tiles = end > begin ? (end - begin + kRowKeys - 1) / kRowKeys : 0u;
  const uint32_t active = max(1u, min(sh.of, (tiles + NW - 1) / NW));
  if (split >= active) return;

  const uint16_t* const qp = a.Q + (int64_t)(w.q0 + token) * a.q_row + head * a.q_head + 8 * quad;
  u4 q[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const u4*>(qp + 32 * s);
  const float c = a.scale * 1.44269504088896340736f;
  const uint16_t* const Kh = a.k.K + kvh * a.k.k_head;
  const uint16_t* const Vh = a.k.V + kvh * a.k.v_head;
  unsigned char* const mine = smem + wave * 2 * kStage;

  const uint32_t in_row = lane / (D / 8), in_chunk = lane % (D / 8);
  const uint32_t stride = active * NW;
  Pages<kRowKeys> pages{table, begin + (split * NW + wave) * kRowKeys, stride * kRowKeys, nk, 0, 0};
  const uint32_t k_step = (uint32_t)a.k.k_row * 2, v_step = (uint32_t)a.k.v_row * 2, page_mask = (1u << a.k.page_shift) - 1;
  const bool whole = !PAGED || (a.k.page_shift >= 5 && begin % kRowKeys == 0);  // a tile lies in one page
  // Offsets of the first loads of V, less their rows: the swizzle goes with the row modulo 8.
  uint32_t v_off[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) v_off[i] = in_row * v_step + ((in_chunk ^ swz_rv<D>(i * kRowsPerLoad + in_row)) << 4);
  const uint32_t k_off = l16 * k_step + 16 * quad;
  u4 kf[2][kSteps];
  // From here on: tile n of this wavefront, which begins at key k0. Keys past the last are 0 (masked below).
  auto rsrc_at = [&](uint32_t n, uint32_t k0, uint32_t row, const uint16_t* from, int64_t row_stride, uint32_t step) __attribute__((always_inline)) {
    int64_t at;
    if constexpr (PAGED) at = pages.page(n, row / 16) * a.k.page_stride + ((k0 + row) & page_mask) * row_stride;
    else at = (int64_t)(w.key0 + k0 + row) * row_stride;
    const uint32_t left = min(nk - k0, (uint32_t)kRowKeys);
    return keys_rsrc(from + at, left > row ? left - row : 0u, step);
  };
  auto load_k = [&](uint32_t n, uint32_t k0) __attribute__((always_inline)) {
    if (whole) {
      const __amdgpu_buffer_rsrc_t r = rsrc_at(n, k0, 0, Kh, a.k.k_row, k_step);
#pragma unroll
      for (uint32_t kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) kf[kt][s] = __builtin_amdgcn_raw_buffer_load_b128(r, k_off + 16 * kt * k_step + 64 * s, 0, 0);
    } else {
#pragma unroll
      for (uint32_t kt = 0; kt < 2; ++kt) {
        const __amdgpu_buffer_rsrc_t r = rsrc_at(n, k0, 16 * kt, Kh, a.k.k_row, k_step);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) kf[kt][s] = __builtin_amdgcn_raw_buffer_load_b128(r, k_off + 64 * s, 0, 0);
      }
    }
  };
  auto copy_v = [&](uint32_t n, uint32_t k0) __attribute__((always_inline)) {
    unsigned char* const to = mine + (n & 1u) * kStage;
    if (whole) {
      const __amdgpu_buffer_rsrc_t r = rsrc_at(n, k0, 0, Vh, a.k.v_row, v_step);
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) buffer_to_lds16(r, to + i * 1024, v_off[i & 3] + i * kRowsPerLoad * v_step);
    } else {
#pragma unroll
      for (uint32_t sub = 0; sub < 2; ++sub) {
        const __amdgpu_buffer_rsrc_t r = rsrc_at(n, k0, 16 * sub, Vh, a.k.v_row, v_step);
#pragma unroll
        for (uint32_t i = 0; i < kLoads / 2; ++i)
          buffer_to_lds16(r, to + (sub * (kLoads / 2) + i) * 1024, v_off[(sub * (kLoads / 2) + i) & 3] + i * kRowsPerLoad * v_step);
      }
    }
  };

  uint32_t v_at[kDims];
  const uint32_t v_row = 4 * quad + (l16 >> 2);
#pragma unroll
  for (int dt = 0; dt < kDims; ++dt)
    v_at[dt] = lds_address(mine) + v_row * kPitch + (((2 * dt + ((l16 & 3u) >> 1)) ^ swz_rv<D>(v_row)) << 4) + 8 * (l16 & 1u);

  f4 o[kDims];
  float m, l;
  // Tile n of this wavefront, from key k0; its V and K are under way. kMore: the next tile's are asked for,
  // V before and K after the first product (which frees the registers), so that every wait but the last
  // leaves a tile in flight. The counts need paths without branches around the copies.
  auto tile = [&](uint32_t n, uint32_t k0, auto mode, auto next) __attribute__((always_inline)) {
    constexpr bool careful = decltype(mode)::value, more = decltype(next)::value;
    if constexpr (more) {
      if constexpr (PAGED) pages.advance(a.k, n + 1);
      copy_v(n + 1, k0 + stride * kRowKeys);
    }
    f4 s[2] = {f4{}, f4{}};
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) s[kt] = mfma16x16x32<DT>(kf[kt][i], q[i], s[kt]);
    // V of this tile was asked for before its K; only the next tile's copies may be left.
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(more ? kLoads : 0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (more) load_k(n + 1, k0 + stride * kRowKeys);
    const bool masked = k0 + kRowKeys > full;
    if (masked) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          if (k0 + 16 * kt + 4 * quad + v >= lim) s[kt][v] = -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    top = over_quads(top, [](float x, float y) { return fmaxf(x, y); });
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
    const uint32_t stage_at = (n & 1u) * kStage;
#pragma unroll
    for (int d0 = 0; d0 < kDims; d0 += 4) {
      uint32_t at[4];
      u4 f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) at[i] = stage_at + v_at[d0 + i];
      lds_read_tr<0, 16 * (int)kPitch>(at, f);
      if constexpr (careful) {
        const u4 sees = {seen2<DT>(k0 + 4 * quad, lim), seen2<DT>(k0 + 4 * quad + 2, lim), seen2<DT>(k0 + 16 + 4 * quad, lim),
                         seen2<DT>(k0 + 16 + 4 * quad + 2, lim)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u4 finite, code;
          split_odd<DT>(f[i], finite, code);
          o[d0 + i] = mfma16x16x32<DT>(finite, pf, o[d0 + i]);
          const f4 count = mfma16x16x32<DT>(code, sees, f4{});
#pragma unroll
          for (int v = 0; v < 4; ++v) o[d0 + i][v] += odd_value(count[v]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d0 + i] = mfma16x16x32<DT>(f[i], pf, o[d0 + i]);
      }
    }
  };
  auto finish = [&]() {
    l = over_quads(l, [](float x, float y) { return x + y; });
    float bad = 0.f;
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt)
#pragma unroll
      for (int v = 0; v < 4; ++v) bad = fmaf(o[dt][v], 0.f, bad);
    return __any(!(bad == 0.f) || (m != kNone && fabsf(m * c) > kFar)) != 0;
  };
  auto start = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt) o[dt] = f4{};
    m = kNone;
    l = 0.f;
  };
  if (t_first < tiles) {
    uint32_t t = t_first, n = 0;
    start();
    int32_t now = 0;
    if constexpr (PAGED) {
      now = pages.load(a.k, 0);
      pages.next = pages.load(a.k, 1);
      const uint32_t key = begin + t * kRowKeys + (lane & 1u) * 16;
      pages.now = key < nk ? (int32_t)page_or_report(a.k, early) : 0;
    }
    copy_v(0, begin + t * kRowKeys);
    load_k(0, begin + t * kRowKeys);
    if constexpr (PAGED) pages.now = pages.held(a.k, 0, now);
    for (; t + stride < tiles; t += stride, ++n) tile(n, begin + t * kRowKeys, std::false_type{}, std::true_type{});
    tile(n, begin + t * kRowKeys, std::false_type{}, std::false_type{});
    // Again, tile by tile, where values are not finite or scores are far, as in the tile kernel.
    if (finish()) {
      start();
      if constexpr (PAGED) pages.start(a.k);
      for (t = t_first, n = 0; t < tiles; t += stride, ++n) {
        if constexpr (PAGED) pages.advance(a.k, n);
        copy_v(n, begin + t * kRowKeys);
        load_k(n, begin + t * kRowKeys);
        tile(n, begin + t * kRowKeys, std::true_type{}, std::false_type{});
      }
      finish();
    }
  } else {
#pragma unroll
    for (int dt = 0; dt < kDims; ++dt) o[dt] = f4{};
    m = kNone;
    l = 0.f;
  }

  // Join the wavefronts: each brings its sums to the common maximum, [wavefront][row][dim].
  __syncthreads();
  float* const red = reinterpret_cast<float*>(smem);
  f2* const stat = reinterpret_cast<f2*>(smem + NW * 16 * (D + 4) * 4);
  uint32_t* const flag = reinterpret_cast<uint32_t*>(smem + row_lds_bytes<D>() - 16);
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

  const uint32_t rows = min(16u, w.R - w.r0), units = rows * (D / 4);
  __amdgpu_buffer_rsrc_t po = make_rsrc(pl.o, 0), pm = po;
  auto joined = [&](uint32_t row, uint32_t d, f4& v, float& mc, float& sum) {
    float mx = kNone;
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) mx = fmaxf(mx, stat[i * 16 + row][0]);
    sum = 0.f;
    v = f4{};
#pragma unroll
    for (uint32_t i = 0; i < NW; ++i) {
      const f2 e = stat[i * 16 + row];
      if (e[1] != 0.f) sum += e[1] * __builtin_amdgcn_exp2f((e[0] - mx) * c);
      v += *reinterpret_cast<const f4*>(red + (i * 16 + row) * (D + 4) + d);
    }
    mc = fmaxf(mx * c, kNone) - Weights<DT>::kLift;
  };
  auto store = [&](uint32_t row, uint32_t d, f4 v, float mc, float sum) {
    const uint32_t rr = w.r0 + row, tk = w.q0 + rr / a.G, hd = kvh * a.G + rr % a.G;
    if (GROUPS) {
      const uint64_t at = ((uint64_t)tk * a.H + hd) * pl.to.slots + pl.to.slots - 1;
      if (d == 0) {
        pl.to.ml[at] = f2{mc, sum};
        if (!grouped)  // no workgroup has the other places
          for (uint32_t i = 1; i < pl.to.slots; ++i) pl.to.ml[at - i] = f2{kNone, 0.f};
      }
      *reinterpret_cast<f4*>(pl.to.o + at * D + d) = v;
      return;
    }
    if (sum == 0.f) v = f4{};
    else v *= 1.f / sum;
    *reinterpret_cast<u2*>(a.O + (int64_t)tk * a.o_row + hd * a.o_head + d) = u2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
    if (a.lse && d == 0) a.lse[(uint64_t)tk * a.H + hd] = sum == 0.f ? -INFINITY : (mc + __log2f(sum)) * 0.69314718055994530942f;
  };
  if (active > 1) {
    // Parts: the workgroup that arrives last joins them, in the order of their numbers.
    const uint64_t at = kvh * pl.slots + slot - split;
    po = make_rsrc(pl.o + at * 16 * D, sh.of * 16 * D * 4);
    pm = make_rsrc(pl.ml + at * 16, sh.of * 16 * 8);
    for (uint32_t u = threadIdx.x; u < units; u += NW * 64) {
      f4 v;
      float mc, sum;
      const uint32_t row = u / (D / 4), d = (u % (D / 4)) * 4;
      joined(row, d, v, mc, sum);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), po, ((split * 16 + row) * D + d) * 4, 0, kAgent);
      if (d == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, (f2{mc, sum})), pm, (split * 16 + row) * 8, 0, kAgent);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
      uint32_t* const cnt = pl.cnt + kvh * pl.slots + slot - split;
      const uint32_t last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == active - 1;
      if (last) __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *flag = last;
    }
    __syncthreads();
    if (!*flag) return;
  }
  for (uint32_t u = threadIdx.x; u < units; u += NW * 64) {
    const uint32_t row = u / (D / 4), d = (u % (D / 4)) * 4;
    float mx = kNone, sum = 0.f;
    f4 v = f4{};
    if (active == 1) joined(row, d, v, mx, sum);
    if (sum == 0.f) mx = kNone;
    // N parts from number p on, of n: what lies past the last is read again and left out.
    auto add = [&](auto batch, uint32_t p, uint32_t n, auto stat_of, auto o_of) __attribute__((always_inline)) {
      constexpr int N = decltype(batch)::value;
      f2 e[N];
      f4 x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t at = min(p + i, n - 1);
        e[i] = stat_of(at);
        x[i] = o_of(at);
      }
      float top = mx;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (p + i >= n) e[i][1] = 0.f;
        top = e[i][1] != 0.f ? fmaxf(top, e[i][0]) : top;
      }
      const float f = __builtin_amdgcn_exp2f(mx - top);
      mx = top;
      sum *= f;
      v *= f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float g = __builtin_amdgcn_exp2f(e[i][0] - top);
        if (e[i][1] != 0.f) {  // a part without weight left its O unwritten
          sum = fmaf(e[i][1], g, sum);
          v += x[i] * g;
        }
      }
    };
    if (active > 1) {
      auto own_stat = [&](uint32_t i) {
        return __builtin_bit_cast(f2, __builtin_amdgcn_raw_buffer_load_b64(pm, (i * 16 + row) * 8, 0, kAgent));
      };
      auto own_o = [&](uint32_t i) {
        return __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(po, ((i * 16 + row) * D + d) * 4, 0, kAgent));
      };
      if (active <= 8) add(Int<8>{}, 0, active, own_stat, own_o);
      else
        for (uint32_t p = 0; p < active; p += 16) add(Int<16>{}, p, active, own_stat, own_o);
    }
    store(row, d, v, mx, sum);
  }
}

template <int DT, int D, bool PAGED>
__global__ __launch_bounds__(kRowWaves * 64) void hq_attn_row_kernel(AttnArgs a, RowPlan pl) {
  row_body<DT, D, PAGED, false>(a, pl, blockIdx.x);
}

// ---- shared prefixes ----
// Groups' prefixes in tiles of many rows and what their sequences have past them in tiles of few are one
// launch: the first is bound by its products and the second by memory, and neither has workgroups enough. In
// two launches 64 rows after 4011 took 34.7 us for 31.6, 16 after 8192 28.8 for 22.7, 128 of 2 groups after 32768 165
// for 158.
template <int DT, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void hq_attn_prefix_kernel(AttnArgs a, TilePlan t, RowPlan r, uint32_t tile_blocks) {
  if (blockIdx.x < tile_blocks) tile_body<DT, D, 4, true, true>(a, t, blockIdx.x);
  else row_body<DT, D, true, true>(a, r, blockIdx.x - tile_blocks);
}

// ---- joining parts ----
// A wavefront a row and head, bound by the parts' way through memory: 15.7 MB in 5.6 us.
template <int DT, int D>
__global__ __launch_bounds__(256) void hq_attn_join_kernel(AttnArgs a, Parts parts) {
  constexpr int E = D / 64;
  typedef float fe __attribute__((ext_vector_type(E == 1 ? 2 : E)));  // E = 1 uses the first
  const uint32_t lane = threadIdx.x & 63u;
  const uint64_t u = (uint64_t)blockIdx.x * 4 + uni(threadIdx.x >> 6);
  if (u >= (uint64_t)a.T * a.H) return;
  const uint32_t t = (uint32_t)(u / a.H), h = (uint32_t)(u % a.H);
  if (a.cu_q) {
    uint32_t lo = 0, hi = a.B, q0;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (a.cu_q[mid] <= (int32_t)t) lo = mid;
      else hi = mid;
    }
    const uint32_t nq = span(a.cu_q, lo, a.T, q0);
    if (t < q0 || t >= q0 + nq) return;  // of no sequence
  }
  // Lane i weighs part i (at most 64).
  const uint64_t at = u * parts.slots;
  f2 e = {kNone, 0.f};
  if (lane < parts.slots) e = parts.ml[at + lane];
  float m = e[1] != 0.f ? e[0] : kNone;
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float f = e[1] != 0.f ? __builtin_amdgcn_exp2f(e[0] - m) : 0.f;
  float l = e[1] * f;
#pragma unroll
  for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
  float o[E] = {};
  const float* const src = parts.o + at * D + lane * E;
  constexpr uint32_t kBatch = 8;
  for (uint32_t p0 = 0; p0 < parts.slots; p0 += kBatch) {
    fe x[kBatch];
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i) {
      const float* const p = src + (uint64_t)min(p0 + i, parts.slots - 1) * D;
      if constexpr (E == 1) x[i][0] = *p;
      else x[i] = *reinterpret_cast<const fe*>(p);
    }
#pragma unroll
    for (uint32_t i = 0; i < kBatch; ++i) {
      const bool has = p0 + i < parts.slots && __builtin_amdgcn_readlane(__float_as_int(e[1]), (p0 + i) & 63u) << 1 != 0;
      const float g = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), (p0 + i) & 63u));
      if (has)  // a part without weight left its O unwritten
#pragma unroll
        for (int k = 0; k < E; ++k) o[k] = fmaf(x[i][k], g, o[k]);
    }
  }
  uint16_t* const out = a.O + (int64_t)t * a.o_row + h * a.o_head + lane * E;
#pragma unroll
  for (int k = 0; k < E; ++k) out[k] = f32_to_out<DT>(l == 0.f ? 0.f : o[k] / l);
  if (a.lse && lane == 0) a.lse[u] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994530942f;
}

uint32_t up(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

template <class K, class... Args>
hipError_t launch_lds(K k, uint32_t grid, uint32_t lds, hipStream_t s, Args... args) {
  hipLaunchKernelGGL(k, dim3(grid), dim3(256), lds, s, args...);
  return hipGetLastError();
}

template <int DT, int D, bool PAGED>
hipError_t launch_all(const AttnArgs& a, const AttnPlan& p, void* ws, hipStream_t s) {
  unsigned char* const w = static_cast<unsigned char*>(ws);
  Parts parts{};
  if (p.parts) {
    parts.slots = p.parts;
    parts.ml = reinterpret_cast<f2*>(w + p.part_ml);
    parts.o = reinterpret_cast<float*>(w + p.part_o);
  }
  const TilePlan t{p.tile_splits, parts};
  RowPlan r{};
  r.slots = p.row_slots;
  r.one = p.row_one;
  r.like = p.row_like;
  r.cnt = reinterpret_cast<uint32_t*>(w);
  r.o = reinterpret_cast<float*>(w + p.row_o);
  r.ml = reinterpret_cast<f2*>(w + p.row_ml);
  if (p.prefix) r.to = parts;
  constexpr uint32_t tile_lds = 2 * tile_stage_bytes<D>(), row_lds = row_lds_bytes<D>();
  auto allow = [](const void* k, uint32_t lds) { return hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, lds); };
  hipError_t e = hipSuccess;
  if (p.prefix) {
    if constexpr (PAGED) {
      auto k = hq_attn_prefix_kernel<DT, D>;
      constexpr uint32_t lds = std::max(tile_lds, row_lds);
      static const hipError_t set = allow(reinterpret_cast<const void*>(k), lds);
      e = set != hipSuccess ? set : launch_lds(k, p.tile_grid + p.row_grid, lds, s, a, t, r, p.tile_grid);
    }
  } else if (p.tile) {
    auto k = hq_attn_tile_kernel<DT, D, 4, PAGED>;
    static const hipError_t set = allow(reinterpret_cast<const void*>(k), tile_lds);
    e = set != hipSuccess ? set : launch_lds(k, p.tile_grid, tile_lds, s, a, t);
  } else {
    auto k = hq_attn_row_kernel<DT, D, PAGED>;
    static const hipError_t set = allow(reinterpret_cast<const void*>(k), row_lds);
    e = set != hipSuccess ? set : launch_lds(k, p.row_grid, row_lds, s, a, r);
  }
  if (e == hipSuccess && p.parts) e = launch_lds(hq_attn_join_kernel<DT, D>, up((uint64_t)a.T * a.H, 4), 0, s, a, parts);
  return e;
}

template <int DT>
hipError_t launch_dim(const AttnArgs& a, const AttnPlan& p, void* ws, hipStream_t s) {
  const bool paged = a.k.table != nullptr;
  if (a.D == 64) return paged ? launch_all<DT, 64, true>(a, p, ws, s) : launch_all<DT, 64, false>(a, p, ws, s);
  if (a.D == 128) return paged ? launch_all<DT, 128, true>(a, p, ws, s) : launch_all<DT, 128, false>(a, p, ws, s);
  if (a.D == 256) return paged ? launch_all<DT, 256, true>(a, p, ws, s) : launch_all<DT, 256, false>(a, p, ws, s);
  return hipErrorInvalidValue;
}

// Workgroups that share the keys of a tile of the tile kernel: the number of least time, in us of an MI355X.
// A tile of 64 keys and 128 dims takes a workgroup 1.2 where it has its CU to itself and two of them 1.9
// where they share one (heads of 256 never do). Parts are written and read at 1 us to 4.5 MB, to 1.3 MB beside the
// row workgroups of a shared prefix, and the join's launch is 6.5. On a chunk of 64 tokens after 6000, 24 tiles,
// 1 / 5 / 10 / 12 / 21 / 48 workgroups took 110 / 37 / 29 / 33 / 31 / 52 us (10 chosen); on 512 tokens after 7488, 192
// tiles, 1 / 2 / 4 / 8 / 16 took 195 / 146 / 139 / 142 / 184 (5); on a prompt of 512, 1 / 2 / 4 took 16 / 33 / 37 (1);
// on a prefix of 2000 under 5 groups of 20 rows, 1 / 2 / 4 / 6 / 12 took 66 / 40 / 29 / 34 / 39 (4).
//
// No more than `most`, which does not fall as the keys grow, so that a workspace for long keys holds what any shorter
// ones ask for: the best number for half as many keys again, in shares that need not be whole tiles. That
// one's times are lines over the keys, the more workgroups the flatter and the higher where they begin; the lowest of
// such lines is a flatter one the further out. Over 3000 shapes of 1 to 2000 tiles, each on up to 131,000 keys, the bound
// moves 1.7% of the choices, whose times by the same cost are 0.02% more over all of them and 14% more at the worst.
uint32_t tile_splits(uint64_t tiles, uint64_t rows, uint32_t dim, uint32_t keys, bool prefix, uint32_t& most) {
  const uint32_t steps = up(keys, kKeys), cus = (uint32_t)cu_count();
  struct Cost {
    double step, parts;  // us of a key tile in all workgroups, of their parts
  } cost[64];
  double least = 0;
  uint32_t n = 0;  // numbers whose parts alone do not cost more
  most = 1;
  for (uint32_t s = 1; s <= 63; ++s) {
    const uint64_t each = up(tiles * s, cus), pairs = dim == 256 ? 0 : each / 2;
    const double parts = prefix || s > 1 ? rows * s * dim * 4. / (prefix ? 1.3e6 : 4.5e6) + 6.5 : 0.;
    const double step = (dim / 128.) * (1.9 * pairs + 1.2 * (each - 2 * pairs)), t = 1.5 * steps / s * step + parts;
    if (s > 1 && parts >= least) break;
    cost[n++] = Cost{step, parts};
    if (s == 1 || t < least) {
      least = t;
      most = s;
    }
  }
  most = std::min(most, steps);
  uint32_t best = 1;
  for (uint32_t s = 1; s <= most; ++s) {
    const double t = up(steps, s) * cost[s - 1].step + cost[s - 1].parts;
    if (s == 1 || t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

// Workgroups of a kv head that share rows' keys in the row kernel: as many as LDS holds in one round, no
// more than pay for their parts (find_share). 0: a workgroup for each 16 rows.
uint32_t row_slots(uint32_t tiles, uint32_t kv_heads, uint32_t dim, uint32_t keys) {
  const uint64_t useful = (uint64_t)tiles * std::min(up(keys, kRowWaves * kRowKeys), (uint32_t)std::ceil(std::sqrt(up(keys, kRowKeys))));
  const uint32_t slots = (uint32_t)std::min<uint64_t>(useful, (dim == 256 ? 1 : 2) * (uint32_t)cu_count() / kv_heads);
  return slots > tiles && slots * kv_heads <= kMaxCounters ? slots : 0;
}

}  // namespace

AttnPlan plan_attn(int kind, uint32_t rows, uint32_t seqs, uint32_t groups, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                   uint32_t max_keys, uint32_t max_prefix) {
  AttnPlan p{};
  const uint32_t G = heads / kv_heads;
  const uint64_t all_rows = (uint64_t)rows * G;
  p.prefix = kind == HQ_ATTN_SHARED;
  // Few rows a sequence: tiles of 16. 16 sequences of 48 rows on up to 3000 keys took 34 us in tiles of 128 and 49
  // in tiles of 16, 8 of 24 rows 24 in both. It is the mean that counts, for the lengths are on the device: 16 single tokens on
  // 200 to 4096 keys and 64 tokens after 6000, 48/8 heads of 128, take 85 us in one call, in tiles of 16, and 52 in two
  // calls of a kind each, as a decoder's step makes them.
  p.row = p.prefix || all_rows <= 32ull * seqs;
  p.tile = p.prefix || !p.row;
  max_keys = std::max(max_keys, 1u);
  max_prefix = std::min(max_prefix, max_keys);
  // What the plan writes, and what it and every plan of fewer keys need at most.
  size_t ws = kCounterBytes, need = kCounterBytes;
  auto take = [&](size_t bytes, size_t most) {
    const size_t at = ws;
    ws += (bytes + 255) / 256 * 256;
    need += (most + 255) / 256 * 256;
    return at;
  };
  if (p.tile) {
    const uint32_t keys = p.prefix && max_prefix ? max_prefix : max_keys;
    const uint32_t tiles = up(all_rows, 128) + (p.prefix ? groups : seqs);
    // The sequences' lengths are not known here: as if all were alike.
    const uint32_t n = p.prefix ? groups : seqs, likely = n * up(up(all_rows, n), 128);
    uint32_t most;
    p.tile_splits = tile_splits((uint64_t)likely * kv_heads, (uint64_t)rows * heads, dim, keys, p.prefix, most);
    p.largest = (uint64_t)tiles * kv_heads * p.tile_splits;
    p.tile_grid = (uint32_t)p.largest;
    if (p.prefix || p.tile_splits > 1) p.parts = p.tile_splits + (p.prefix ? 1 : 0);
    const size_t all = (size_t)rows * heads, places = all * p.parts, held = p.prefix || most > 1 ? all * (most + (p.prefix ? 1 : 0)) : 0;
    p.part_ml = take(places * sizeof(f2), held * sizeof(f2));
    p.part_o = take(places * dim * sizeof(float), held * dim * sizeof(float));
  }
  if (p.row) {
    const uint32_t tiles = rows == seqs ? seqs * up(G, 16) : up(all_rows, 16) + seqs;
    // Where the prefixes are not known (0), all keys may lie in them, and all past them: 4 rows of 8192 keys of their own on
    // 48/8 heads of 128 took 94 us with one key taken to be past the prefix, and take 33.
    const uint32_t keys = p.prefix ? std::max(max_keys - max_prefix, 1u) : max_keys;
    p.row_slots = row_slots(tiles, kv_heads, dim, keys);
    p.row_one = p.row_slots && tiles == 1;
    p.row_like = keys;
    p.row_grid = (p.row_slots ? p.row_slots : tiles) * kv_heads;
    p.largest += (uint64_t)(p.row_slots ? p.row_slots : tiles) * kv_heads;
    // More keys have no fewer slots; those past a prefix are most where there is none.
    const uint32_t most = keys == max_keys ? p.row_slots : row_slots(tiles, kv_heads, dim, max_keys);
    const size_t place = (size_t)kv_heads * 16, places = p.row_slots * place, held = most * place;
    p.row_ml = take(places * sizeof(f2), held * sizeof(f2));
    p.row_o = take(places * dim * sizeof(float), held * dim * sizeof(float));
  }
  if (p.parts) p.largest = std::max(p.largest, ((uint64_t)rows * heads + 3) / 4);
  p.ws = ws > kCounterBytes ? ws : 0;
  p.need = need > kCounterBytes ? need : 0;
  return p;
}

void describe_attn(const AttnPlan& p, char* buf, size_t len) {
  const char* const shared = p.row_slots ? " shared" : "";
  char k[200];
  if (p.prefix)
    std::snprintf(k, sizeof k, "hq_attn_prefix_kernel grid=%u+%u splits=%u%s", p.tile_grid, p.row_grid, p.tile_splits, shared);
  else if (p.tile) std::snprintf(k, sizeof k, "hq_attn_tile_kernel grid=%u splits=%u", p.tile_grid, p.tile_splits);
  else std::snprintf(k, sizeof k, "hq_attn_row_kernel grid=%u%s", p.row_grid, shared);
  std::snprintf(buf, len, "%s%s ws=%zu", k, p.parts ? ", hq_attn_join_kernel" : "", p.ws);
}

hipError_t launch_attn(int dtype, const AttnArgs& a, const AttnPlan& p, void* ws, hipStream_t s) {
  return dtype == HQ_DTYPE_F16 ? launch_dim<HQ_DTYPE_F16>(a, p, ws, s) : launch_dim<HQ_DTYPE_BF16>(a, p, ws, s);
}

}  // namespace hq
