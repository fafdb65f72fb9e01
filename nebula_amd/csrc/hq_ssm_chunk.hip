// hq_ssm_chunk.hip — the selective scan of prompts in chunks of tokens, on matrix products (include/hq_ssm.h).
//
// Inside a chunk of L tokens with c_t = sum_{s <= t} A dt_s, a head's recursion is
//   y_t = exp(c_t) S_in C_t + sum_{s <= t} M_ts x_s + D x_t,   M_ts = exp(c_t - c_s) dt_s (B_s . C_t)
//   S_out = exp(c_end) S_in + sum_s w_s x_s B_s^T,             w_s = exp(c_end - c_s) dt_s
// so a token costs 4 N + 4 L operations a channel in place of 6 N on the vector units, and the state is touched once a
// chunk. A workgroup walks a run of chunks of one head (two heads of 64 of one group) with the state in the accumulators
// of four wavefronts, 32 channels each:
//   S^T [n][p] as products of 32 x 32: a lane holds one channel p and eight states n side by side, which is the next
//   product's operand as it stands (its rows, the columns of B in LDS, are taken in the order that makes them so);
//   y^T [p][t] = S C^T and x^T M^T, whose operand x^T is the one that the state's sum takes with its weights.
// B, C and x go through LDS, the next chunk's in registers meanwhile; M is computed once by the head's wavefronts and
// goes through LDS to all of them.
//
// Few sequences are dealt to several workgroups in runs of chunks: a launch of this kernel sums what each run adds to the state
// (kCarry), hq_ssm_join_kernel turns that into what enters each run, and a second launch computes the outputs from there.
//
// Bound by the vector pipe (parts of operands, decays, the gate) and the matrix pipe together: 59% and 32% busy at 8192 tokens of 48
// heads of 128x128, where a wavefront has 1350 vector instructions and 102 products a chunk and a SIMD two wavefronts: 191 us, of which
// carries, joins and outputs have 58, 11 and 122, for 373 MB of operands (78 us at a copy's rate). One workgroup a CU: 5 us a chunk,
// bound by its own chain.
//
// Sums are fp32, those of a chunk's exponents in 64 bits. What a matrix product's operands round away:
//   the state's terms w x (fp32 times 16 bits) are kept as three bf16 parts, or in fp16 as two parts of values scaled by a
//   power of two of their channel and chunk, because the state is fp32 and goes on for the whole sequence: 22 bits of them either
//   way (fp16: of those above 2^-17 of their channel's largest in the chunk, and 2^-39 of that of the others);
//   S as an operand, and M, are kept as two parts (16 bits, fp16: 22 of S, scaled as the terms are): with one, outputs would be
//   off by 1.4 times their own rounding.
//
// A product adds 0 x_s for tokens s behind t, which is no 0 for an infinite x_s or NaN. A chunk therefore ends before such an x and the
// next one begins with it; the exponents of a chunk's x are looked at on their way to LDS, so that a prompt without any pays a maximum.
// An infinite operand leaves NaN as the rest of its first part: its channel is lost either way, as an infinity or NaN.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>
#include <type_traits>

#include "hq_internal.hpp"
#include "hq_ssm_device.hpp"

namespace hq {
namespace {

typedef float f16x __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ f16x mfma32(u4 a, u4 b, f16x c) {
  if constexpr (DT == HQ_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

constexpr int BF = HQ_DTYPE_BF16;
constexpr uint32_t kChunkThreads = 256;
constexpr uint32_t kOwnBytes = 4096;  // of LDS for a wavefront: a chunk's x of 32 channels, then 32 tokens' fp32 outputs
constexpr uint32_t kColumns = 128;  // channels of a workgroup, four wavefronts of 32
constexpr uint32_t kScaleBytes = kColumns * 4;  // of LDS for their scales
constexpr uint32_t kLowBytes = 4 * 64 * 4;      // of LDS for the low parts of four wavefronts' sums

// Tokens of a chunk: the state of 256 leaves registers and LDS for 32.
template <int N>
constexpr int chunk_tokens() {
  return N == 256 ? 32 : 64;
}

// 16-byte pieces of a row of LDS: piece c of row r lies at c ^ swizzle(r), so that reads of one piece of 16 rows, and
// transposing reads of four pieces of four rows, meet in different banks (64 of 4 bytes).
template <int BYTES>
__device__ __forceinline__ uint32_t swizzle(uint32_t r) {
  if constexpr (BYTES >= 256) return (r & 3u) << 2 | (r >> 2 & 3u);
  else if constexpr (BYTES == 128) return (r >> 1 & 1u) << 2 | (r >> 2 & 3u);
  else return r >> 2 & 3u;  // rows of 64 bytes: four side by side
}
template <int BYTES>
__device__ __forceinline__ uint32_t piece_at(uint32_t r, uint32_t c) {
  return r * BYTES + ((c ^ swizzle<BYTES>(r)) << 4);
}

// A part of M in LDS, [token][earlier token]: 32 tokens with 32 earlier ones, then the 32 behind them with 64.
template <int L>
constexpr uint32_t m_bytes() {
  return L == 64 ? 32 * 64 + 32 * 128 : 32 * 64;
}
template <int L>
__device__ __forceinline__ uint32_t m_place(uint32_t block, uint32_t r, uint32_t c) {
  return L == 64 && block ? 32 * 64 + piece_at<128>(r, c) : piece_at<64>(r, c);
}

// The tiles of M, 16 tokens t with 16 earlier ones s, of a head's wavefront `part` of 4 or 2.
struct MTiles {
  int n, t[5], s[5];
};
constexpr MTiles m_tiles(int L, int waves, int part) {
  if (L == 32) {
    if (waves == 2) return part == 0 ? MTiles{2, {1, 1}, {0, 1}} : MTiles{1, {0}, {0}};
    return part == 0 ? MTiles{1, {1}, {0}} : part == 1 ? MTiles{1, {1}, {1}} : MTiles{1, {0}, {0}};
  }
  if (waves == 2) return part == 0 ? MTiles{5, {3, 3, 3, 3, 2}, {3, 0, 1, 2, 2}} : MTiles{5, {2, 2, 1, 1, 0}, {0, 1, 0, 1, 0}};
  if (part == 0) return {3, {3, 3, 3}, {0, 1, 2}};
  if (part == 1) return {3, {2, 2, 1}, {0, 1, 0}};
  return part == 2 ? MTiles{2, {0, 1}, {0, 1}} : MTiles{2, {2, 3}, {2, 3}};
}

// A fragment of the transposed tile [tokens][columns]: columns 32 c32 .., tokens 16 ks ..; lane: column (SWAP: the middle
// fours of 16 exchanged), eight tokens. `at`: what tr_place gives.
template <int BYTES, bool SWAP>
__device__ __forceinline__ void tr_place(uint32_t lane, uint32_t c32, uint32_t (&at)[2]) {
  const uint32_t j = lane & 3u, row = 8 * (lane >> 5) + (lane >> 2 & 3u);
  const uint32_t piece = 4 * c32 + 2 * (lane >> 4 & 1u) + (SWAP ? j & 1u : j >> 1), byte = 8 * (SWAP ? j >> 1 : j & 1u);
  at[0] = piece_at<BYTES>(row, piece) + byte;
  at[1] = piece_at<BYTES>(row + 4, piece) + byte;
}
__device__ __forceinline__ u4 tr_read(const unsigned char* p0, const unsigned char* p1) {
  typedef __attribute__((address_space(3))) s4* lds_s4;
  const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p0));
  const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p1));
  return u4{a[0], a[1], b[0], b[1]};
}

__device__ __forceinline__ float scan_add(float x) {
  return __uint_as_float(scan(__float_as_uint(x), 0, [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
// The same in 64 bits.
__device__ __forceinline__ double scan_add(double x) {
#define HQ_ADD(CTRL, ROWS)                                                                                                         \
  {                                                                                                                                \
    const uint64_t v = __builtin_bit_cast(uint64_t, x);                                                                            \
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);                        \
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);                \
    x += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);                                                                      \
  }
  HQ_ADD(0x111, 0xF)  // as in scan()
  HQ_ADD(0x112, 0xF)
  HQ_ADD(0x114, 0xF)
  HQ_ADD(0x118, 0xF)
  HQ_ADD(0x142, 0xA)
  HQ_ADD(0x143, 0xC)
#undef HQ_ADD
  return x;
}
// Of the two lanes that hold a channel.
__device__ __forceinline__ float max_of_halves(float x) {
  const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(v[0]), __uint_as_float(v[1]));
}

// 2^k that brings a maximum m to 2^14..2^15, and 2^-k: fp16 then holds 11 bits of a value and as many of the rest, down to
// 2^-39 of the maximum. No values, infinities or NaN: as they are.
__device__ __forceinline__ void range_scale(float m, float& up, float& down) {
  const uint32_t e = __float_as_uint(m) >> 23 & 255u;
  const uint32_t k = m == 0.f || e == 255u ? 127u : min(268u - e, 247u);  // 141 - e + 127
  up = __uint_as_float(k << 23);
  down = __uint_as_float((254u - k) << 23);
}

// The rest that one rounding of two values leaves, exactly, and the rounded ones. (For fp16 one instruction each, with a half
// of w as an operand. bf16 has such a one, a dot product of two, but its result is waited for: 8% slower.)
template <int DT>
__device__ __forceinline__ uint32_t take_part(float& a, float& b) {
  const uint32_t w = pack_pair<DT>(a, b);
  if constexpr (DT == HQ_DTYPE_F16) {
    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel_hi:[1,0,0]" : "+v"(a) : "v"(w));
    asm("v_fma_mix_f32 %0, %1, -1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(b) : "v"(w));
  } else {
    float x, y;
    unpack_pair<DT>(w, x, y);
    a -= x;
    b -= y;
  }
  return w;
}

// The largest exponents (of both halves) of 16-byte pieces of activations; an infinity or NaN has the type's largest.
template <int DT, int K>
__device__ __forceinline__ uint32_t exponents(const u4 (&x)[K]) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  constexpr uint32_t kMask = DT == HQ_DTYPE_F16 ? 0x7C007C00u : 0x7F807F80u;
  us2 m = {0, 0};
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, x[k][i] & kMask));
  return max((uint32_t)m[0], (uint32_t)m[1]);
}

// A place in LDS as the compiler has it: what is computed from it stays in its chunk. (Held from chunk to chunk, the places
// of all fragments are more registers than there are.)
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
  asm volatile("" : "+v"(v));
  return v;
}

// The order of a step: a product, then VALU other instructions and READS reads of LDS, N times.
template <int N, int VALU, int READS>
__device__ __forceinline__ void between() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    if constexpr (READS > 0) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    __builtin_amdgcn_sched_group_barrier(0x2, VALU, 0);
  }
}

// A uniform value that stays in its scalar registers.
template <class T>
__device__ __forceinline__ T held(T v) {
  asm volatile("" : "+s"(v));
  return v;
}

// Which run of chunks a workgroup works on.
struct Run {
  Seq q;
  uint32_t t0, t1;      // tokens
  uint32_t first, idx, last;  // runs of the whole call: the sequence's first, this one, the sequence's last
};

__device__ __forceinline__ bool find_run(const SeqArgs& s, uint32_t run_tokens, uint32_t idx, bool tell, Run& r) {
  uint32_t before = 0;
  for (uint32_t i = 0; i < s.n; i += 64) {
    const uint32_t b = i + (threadIdx.x & 63u);
    uint32_t runs = 0;
    if (b < s.n) {
      const uint32_t a = s.cu ? clamp_to(s.cu[b], s.T) : b, e = s.cu ? clamp_to(s.cu[b + 1], s.T) : b + 1;
      runs = e > a ? (e - a + run_tokens - 1) / run_tokens : 0u;
    }
    const uint32_t upto = scan_sum(runs) + before, all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    if (idx < all) {
      const uint64_t past = __ballot(upto > idx);  // some lane: the last one is
      const int lane = __builtin_ctzll(past);
      const uint32_t mine = (uint32_t)__builtin_amdgcn_readlane((int)runs, lane);
      r.last = (uint32_t)__builtin_amdgcn_readlane((int)upto, lane) - 1;
      r.first = r.last + 1 - mine;
      r.idx = idx;
      r.q = find_seq(s, i + lane, tell);
      r.t0 = r.q.a + (idx - r.first) * run_tokens;
      r.t1 = min(r.t0 + run_tokens, r.q.e);
      return true;
    }
    before = all;
  }
  return false;
}

struct ChunkArgs {
  uint32_t run_tokens, units, runs, blocks;  // tokens of a run; workgroups of a run; runs, workgroups of the launch less the padding
  float* states;                       // [runs][units][register quads][threads] f4: what a run adds to the state
  float* totals;                       // [runs][heads]: its whole decay's exponent
};

template <int N>
constexpr uint32_t vec_bytes() {
  return 4 * 2 * 3 * chunk_tokens<N>() * 4;
}
template <int N, bool CARRY>
constexpr uint32_t chunk_lds(uint32_t heads) {
  constexpr uint32_t L = chunk_tokens<N>();
  return (CARRY ? 1 : 2) * L * N * 2 + 4 * kOwnBytes + vec_bytes<N>() + (CARRY ? 0 : heads * 2 * m_bytes<L>() + kLowBytes + kScaleBytes) + 16;
}

// What a launch computes: outputs, outputs through a gate, or the state alone, of all runs but a sequence's last, for the runs
// behind them.
enum Kind : int { kPlain, kGated, kCarry };

template <int DT, int P, int N, int KIND>
__global__ __launch_bounds__(kChunkThreads, N == 256 ? 1 : 2) void hq_ssm_chunk_kernel(ScanArgs a, ChunkArgs pl) {
  constexpr bool CARRY = KIND == kCarry, GATED = KIND == kGated;
  constexpr int L = chunk_tokens<N>(), kHeads = kColumns / P, kWaves = P / 32;  // heads, wavefronts of a head
  constexpr int kTB = L / 32, kTS = L / 16, kNT = N / 32, kNS = N / 16;
  constexpr int kRow = 2 * N, kXRow = 64;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const sB = smem;
  unsigned char* const sX = sB + L * kRow;
  float* const vec = reinterpret_cast<float*>(sX + 4 * kOwnBytes);
  unsigned char* const sC = reinterpret_cast<unsigned char*>(vec) + vec_bytes<N>();
  unsigned char* const sM = sC + L * kRow;

  // Workgroups go to the eight XCDs in turn: a run of neighbouring ones, which share B and C, goes to one.
  const uint32_t block = (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (block >= pl.blocks) return;
  const uint32_t idx = block / pl.units, unit = block - idx * pl.units;
  const uint32_t of_group = a.H / a.G, per_group = (of_group + kHeads - 1) / kHeads;
  const uint32_t g = unit / per_group, head0 = (unit - g * per_group) * kHeads;  // the first head, in its group
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uni(tid >> 6), l32 = lane & 31u, half = lane >> 5;
  const uint32_t mine = wave / kWaves, part = wave % kWaves;  // this wavefront's head and 32 channels of it
  const bool live = head0 + mine < of_group;                  // (an odd group's last head is alone)
  const uint32_t h = g * of_group + min(head0 + mine, of_group - 1);

  Run run;
  if (!find_run(a.s, pl.run_tokens, idx, unit == 0 && tid < 64, run)) return;
  if (CARRY && run.idx == run.last) return;
  if (run.last >= pl.runs) {  // offsets that fall hold more tokens than there are: no room for the sequence's runs
    if (unit == 0 && tid == 0) __hip_atomic_fetch_or(a.s.status, HQ_CACHE_BAD_ROW, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return;
  }

  const float A = a.A[h] * 1.44269504f, D = !CARRY && a.D ? a.D[h] : 0.f, dt0 = a.dt_bias ? a.dt_bias[h] : 0.f;

  // ---- a chunk's inputs, on their way in registers ----
  constexpr int kPieces = N / 8, kRows = kChunkThreads / kPieces, kLoads = L / kRows, kXLoads = L / 16;
  u4 rb[kLoads], rc[CARRY ? 1 : kLoads], rx[kXLoads];
  uint32_t rdt = 0;  // as it is in memory: turned into a number here, it would be waited for
  // Addresses of the chunk that is loaded, and strides in bytes, kept in scalar registers (from the arguments anew, they
  // were 2 us of a chunk's loads). Lanes' offsets from them are 32-bit; a place past any operand reads as 0 without touching
  // memory: from the run's end on (`left` tokens), and for a chunk that there is none of, so that what is in flight is the
  // same on every way.
  const bool dt_f32 = a.dt_f32;
  const uint32_t b_step = held((uint32_t)a.b_row * 2), c_step = held((uint32_t)a.c_row * 2), x_step = held((uint32_t)a.x_row * 2);
  const uint32_t y_step = held((uint32_t)a.y_row * 2), z_step = held((uint32_t)a.z_row * 2), dt_size = dt_f32 ? 4 : 2;
  const uint32_t dt_step = held((uint32_t)a.dt_row * dt_size);
  uint64_t b_at = held(reinterpret_cast<uint64_t>(a.B + run.t0 * a.b_row + g * a.b_group));
  uint64_t c_at = held(reinterpret_cast<uint64_t>(a.C + run.t0 * a.c_row + g * a.c_group));
  uint64_t x_at = held(reinterpret_cast<uint64_t>(a.X + run.t0 * a.x_row + h * a.x_head + part * 32));
  uint64_t dt_at = held(reinterpret_cast<uint64_t>(a.dt) + (run.t0 * a.dt_row + h) * dt_size);
  uint64_t y_at = held(reinterpret_cast<uint64_t>(a.Y + run.t0 * a.y_row + h * a.y_head + part * 32));
  uint64_t z_at = held(reinterpret_cast<uint64_t>(a.Z + run.t0 * a.z_row + h * a.z_head + part * 32));
  auto rsrc = [](uint64_t at) __attribute__((always_inline)) { return make_rsrc(reinterpret_cast<const void*>(at), kOutOfRange - 1); };
  auto past = [](uint32_t off, bool there) __attribute__((always_inline)) { return there ? off : kOutOfRange; };
  auto load_x = [&](uint32_t left) __attribute__((always_inline)) {
    const uint32_t id = opaque(lane), xrow = id / 4, x_off = __umul24(xrow, x_step) + id % 4 * 16;  // the wavefront's channels
    const __amdgpu_buffer_rsrc_t bx = rsrc(x_at), bd = rsrc(dt_at);
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) rx[i] = __builtin_amdgcn_raw_buffer_load_b128(bx, past(x_off, xrow + i * 16 < left), i * 16 * x_step, 0);
    const uint32_t dt_off = past(id * dt_step, id < left);  // (up to 2^24 bytes: not in 24 bits)
    if (dt_f32) rdt = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(bd, dt_off, 0, 0);
    else rdt = __builtin_amdgcn_raw_buffer_load_b16(bd, dt_off, 0, 0);
  };
  // B and C in kBCLoads steps, so that they go out between other work.
  constexpr int kBCLoads = (CARRY ? 1 : 2) * kLoads;
  uint32_t b_off, c_off, bc_row;
  auto place_bc = [&]() __attribute__((always_inline)) {
    const uint32_t id = opaque(tid);
    bc_row = id / kPieces;
    b_off = __umul24(bc_row, b_step) + id % kPieces * 16;
    c_off = __umul24(bc_row, c_step) + id % kPieces * 16;
  };
  auto load_bc = [&](uint32_t left, int j) __attribute__((always_inline)) {
    const int i = CARRY ? j : j / 2;
    const bool is_c = !CARRY && j % 2, there = bc_row + i * kRows < left;
    if (is_c) rc[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc(c_at), past(c_off, there), i * kRows * c_step, 0);
    else rb[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc(b_at), past(b_off, there), i * kRows * b_step, 0);
  };
  auto put = [&]() __attribute__((always_inline)) {
    const uint32_t id = opaque(tid);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t at = piece_at<kRow>(id / kPieces + i * kRows, id % kPieces);
      *reinterpret_cast<u4*>(sB + at) = rb[i];
      if constexpr (!CARRY) *reinterpret_cast<u4*>(sC + at) = rc[i];
    }
  };
  // x goes through LDS for its order alone, to the wavefront that brought it.
  unsigned char* const own = sX + wave * kOwnBytes;
  constexpr uint32_t kOdd = DT == HQ_DTYPE_F16 ? 0x7C00u : 0x7F80u;  // the exponent of infinities and NaN
  uint32_t most = 0;
  auto look_x = [&]() __attribute__((always_inline)) { most = exponents<DT>(rx); };
  auto put_x = [&](uint32_t* odd) __attribute__((always_inline)) {
    const uint32_t id = opaque(lane), xrow = id / 4, at = piece_at<kXRow>(xrow, id % 4);
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) *reinterpret_cast<u4*>(own + at + i * 16 * kXRow) = rx[i];
    if (__builtin_expect(most == kOdd, 0)) {
#pragma unroll
      for (int i = kXLoads - 1; i >= 0; --i) {
        const u4 one[1] = {rx[i]};
        if (exponents<DT>(one) == kOdd) atomicMin(odd, xrow + i * 16);
      }
    }
  };
  load_x(run.t1 - run.t0);
  place_bc();
#pragma unroll
  for (int j = 0; j < kBCLoads; ++j) load_bc(run.t1 - run.t0, j);

  // ---- the state: s[nt][r] is channel l32, state 32 nt + 16 (r / 8) + 8 half + r % 8 ----
  f16x s[kNT];
  float* const kept = a.state + run.q.row * a.row_stride + ((size_t)h * P + part * 32 + l32) * N + 8 * half;
  auto place = [&](uint32_t i) { return pl.states + (((size_t)i * pl.units + unit) * (kNT * 4) * kChunkThreads + tid) * 4; };
#pragma unroll
  for (int i = 0; i < kNT; ++i) s[i] = f16x{};
  if (CARRY ? run.idx == run.first : run.first == run.last) {
    if (run.q.read) {
#pragma unroll
      for (int i = 0; i < kNT * 4; ++i) {
        const f4 v = *reinterpret_cast<const f4*>(kept + 16 * (i / 2) + 4 * (i & 1));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i / 4][(i & 3) * 4 + e] = v[e];
      }
    }
    // A sequence's first run reads its state here, for itself and, in the place of the last one, which has nothing to leave,
    // for the run of the outputs: by then the last of those may have replaced it.
    if constexpr (CARRY) {
      float* const p = place(run.last);
#pragma unroll
      for (int i = 0; i < kNT * 4; ++i)
        *reinterpret_cast<f4*>(p + i * 4 * kChunkThreads) = f4{s[i / 4][(i & 3) * 4], s[i / 4][(i & 3) * 4 + 1], s[i / 4][(i & 3) * 4 + 2], s[i / 4][(i & 3) * 4 + 3]};
    }
  } else if constexpr (!CARRY) {
    const float* const p = place(run.idx);
#pragma unroll
    for (int i = 0; i < kNT * 4; ++i) {
      const f4 v = *reinterpret_cast<const f4*>(p + i * 4 * kChunkThreads);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i / 4][(i & 3) * 4 + e] = v[e];
    }
  }

  // Of a chunk of n tokens, for this wavefront's head: steps and their sums, a token a lane, from the chunk's beginning and
  // from its end. Computed during the chunk before it, between products.
  float whole = 0;  // the whole chunk's exponent
  float* const lows = reinterpret_cast<float*>(smem + chunk_lds<N, CARRY>(kHeads) - 16 - kScaleBytes - kLowBytes) + wave * 64;
  auto sums = [&](uint32_t to, uint32_t n) __attribute__((always_inline)) {
    const float dt = lane < n ? step_of((dt_f32 ? __uint_as_float(rdt) : to_f32<DT>((uint16_t)rdt)) + dt0, a.softplus) : 0.f;
    // (2^-200 is 0 already: what one token forgets is no reason to lose the digits of the tokens behind it. Compared, not a maximum,
    // which would make a number of NaN.)
    const float forgets = dt * A, e = lane < n ? (forgets < -200.f ? -200.f : forgets) : 0.f;
    const float back = scan_add(__shfl(e, 63 - lane)), after = __shfl(back, (62 - lane) & 63);
    // The weights M take differences of two sums: what tokens before both of them forgot goes out again, and so must its
    // rounding. The sums are made in 64 bits and kept in two parts. (In fp32, steps of -115 in half a chunk took the digits of
    // fp16 outputs behind them.)
    float up;
    if constexpr (CARRY) {
      up = scan_add(e);
    } else {
      const double both = scan_add((double)e);
      up = (float)both;
      if (lane < L) lows[lane] = (float)(both - (double)up);
    }
    float* const cum = vec + (wave * 2 + to) * 3 * L;
    if (lane < L) {
      cum[lane] = up;
      cum[L + lane] = dt;
      cum[2 * L + lane] = __builtin_amdgcn_exp2f(lane == 63 ? 0.f : after) * dt;
    }
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(up), 63));
  };
  unsigned char* const m0 = sM + mine * 2 * m_bytes<L>();  // M's parts
  if constexpr (!CARRY) {
    // The tiles of 16 x 16 right of the diagonal that products of 32 tokens take in stay zero.
    for (uint32_t i = tid; i < kHeads * 2 * m_bytes<L>() / 16; i += kChunkThreads) *reinterpret_cast<u4*>(sM + i * 16) = u4{0, 0, 0, 0};
  }
  // Places of this lane's fragments; a step of products further is an exclusive or, 16 or 32 rows a sum.
  uint32_t tr_b[2], at_x[2];
  tr_place<kRow, true>(lane, 0, tr_b);
  tr_place<kXRow, false>(lane, 0, at_x);

  // odd[i]: the first token of a chunk (the i-th, modulo 2) with an x that is not finite.
  uint32_t* const odd = reinterpret_cast<uint32_t*>(smem + chunk_lds<N, CARRY>(kHeads) - 8);
  if (tid < 2) odd[tid] = L;
  __syncthreads();
  put();
  look_x();
  put_x(odd);
  float total = 0, next_whole = sums(0, min(run.t1 - run.t0, (uint32_t)L));
  uint32_t n, turn = 0;
  for (uint32_t t = run.t0; t < run.t1; t += n, turn ^= 1u) {
    __syncthreads();
    n = min(run.t1 - t, (uint32_t)L);
    // 0 times an infinity is no 0: the tokens before an x that is not finite, and it alone, are chunks of their own. What
    // lies past them in LDS is cleared.
    const uint32_t first = uni(odd[turn]);
    if (__builtin_expect(first < n, 0)) {
      n = max(first, 1u);
      next_whole = sums(turn, n);
      for (uint32_t i = tid; i < (L - n) * kPieces; i += kChunkThreads) *reinterpret_cast<u4*>(sB + n * kRow + i * 16) = u4{0, 0, 0, 0};
      for (uint32_t i = lane; i < (L - n) * 4; i += 64) *reinterpret_cast<u4*>(own + n * kXRow + i * 16) = u4{0, 0, 0, 0};
      __syncthreads();
    }
    if (tid == 0) odd[turn ^ 1u] = L;
    whole = next_whole;
    total += whole;
    // Of two wavefronts on a SIMD, the one that makes outputs goes first: its chain is the longer one, and the other's products of the
    // state's sums fill what it leaves (8 prompts of 512 tokens 82 -> 77 us, one of 8192 197 -> 192).
    if constexpr (!CARRY) __builtin_amdgcn_s_setprio(2);
    float* const cum = vec + (wave * 2 + turn) * 3 * L;  // of this chunk: exponents (of 2), steps, weights of the state's terms
    const float *const steps = cum + L, *const weights = steps + L;
    // Outputs leave as 16-byte pieces, four lanes a token: token lane / 4 + 16 i, channels 8 (lane % 4) ..
    u4 zr[kTB * 2];
    uint32_t out_at[kTB * 2];
    if constexpr (!CARRY) {
#pragma unroll
      for (int i = 0; i < kTB * 2; ++i) out_at[i] = 16 * i + lane / 4 < n && live ? 0u : kOutOfRange;
      if constexpr (GATED) {
        const uint32_t z_off = __umul24(lane / 4, z_step) + lane % 4 * 16;
#pragma unroll
        for (int i = 0; i < kTB * 2; ++i) zr[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc(z_at), out_at[i] | z_off, i * 16 * z_step, 0);
      }
    }
    const uint32_t left = run.t1 - t - n;  // (none: 0)
    b_at += (uint64_t)n * b_step;
    c_at += (uint64_t)n * c_step;
    x_at += (uint64_t)n * x_step;
    dt_at += (uint64_t)n * dt_step;
    load_x(left);
    __builtin_amdgcn_sched_barrier(0);

    u4 x[kTS];  // x^T: channel l32, tokens 16 i + 8 half ..
    auto read_x = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kTS; ++i) x[i] = tr_read(own + at_x[0] + i * 16 * kXRow, own + at_x[1] + i * 16 * kXRow);
    };
    if constexpr (CARRY) read_x();

    f16x y[kTB];
    if constexpr (!CARRY) {
      // M in tiles of 16 x 16, dealt to the head's wavefronts so that each has few rows of B and C to read: B_s . C_t, a lane one t
      // and four s.
      const uint32_t id = opaque(lane), l16 = id & 15u, quad = id >> 4, at = piece_at<kRow>(l16, quad);
      auto weights_of = [&](auto which) __attribute__((always_inline)) {
        constexpr MTiles kMine = m_tiles(L, kWaves, decltype(which)::value);
        f4 m[kMine.n];
#pragma unroll
        for (int k = 0; k < kMine.n; ++k) m[k] = f4{0, 0, 0, 0};
        f4 f[kMine.n];  // the decays and steps, while rows are on their way
#pragma unroll
        for (int k = 0; k < kMine.n; ++k) {
          const uint32_t tt = 16 * kMine.t[k] + l16, ss = 16 * kMine.s[k] + 4 * quad;
          const float ct = cum[tt], lt = lows[tt];
          const f4 cs = *reinterpret_cast<const f4*>(cum + ss), ls = *reinterpret_cast<const f4*>(lows + ss), ds = *reinterpret_cast<const f4*>(steps + ss);
#pragma unroll
          for (int v = 0; v < 4; ++v) f[k][v] = __builtin_amdgcn_exp2f((ct - cs[v]) + (lt - ls[v])) * ds[v];
        }
#pragma unroll
        for (int j = 0; j < N / 32; ++j)
#pragma unroll
          for (int k = 0; k < kMine.n; ++k) {
            const u4 fb = *reinterpret_cast<const u4*>(sB + 16 * kMine.s[k] * kRow + (at ^ (uint32_t)(j << 6)));
            const u4 fc = *reinterpret_cast<const u4*>(sC + 16 * kMine.t[k] * kRow + (at ^ (uint32_t)(j << 6)));
            m[k] = mfma16x16x32<DT>(fb, fc, m[k]);
          }
#pragma unroll
        for (int k = 0; k < kMine.n; ++k) {
          const uint32_t tt = 16 * kMine.t[k] + l16, ss = 16 * kMine.s[k] + 4 * quad;
          float w[4];
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            w[v] = f[k][v] * m[k][v];
            if (kMine.t[k] == kMine.s[k]) {
              const int32_t back = (int32_t)(tt - ss);  // tokens from the lane's first one to its own
              w[v] = v < back ? w[v] : v == back ? w[v] + D : 0.f;
            }
          }
          const uint32_t to = m_place<L>(kMine.t[k] / 2, tt & 31u, ss / 8) + (ss & 4u) * 2;
          u2 hi, lo;
          hi[0] = take_part<BF>(w[0], w[1]);
          hi[1] = take_part<BF>(w[2], w[3]);
          lo[0] = pack_pair<BF>(w[0], w[1]);
          lo[1] = pack_pair<BF>(w[2], w[3]);
          *reinterpret_cast<u2*>(m0 + to) = hi;
          *reinterpret_cast<u2*>(m0 + m_bytes<L>() + to) = lo;
        }
      };
      if (part == 0) weights_of(std::integral_constant<int, 0>{});
      else if (part == 1) weights_of(std::integral_constant<int, 1>{});
      else if constexpr (kWaves == 4) {
        if (part == 2) weights_of(std::integral_constant<int, 2>{});
        else if constexpr (L == 64) weights_of(std::integral_constant<int, 3>{});
      }
      __syncthreads();

      // y^T: what the state gives, decayed, and the chunk's own.
      // fp16: a channel's states have a scale of their own, so that what another channel holds, infinite or far larger, takes no
      // digits from them. Two lanes hold a channel as an operand, all of them as outputs: the way back goes through LDS.
      float up2 = 1.f;
      float* const downs = reinterpret_cast<float*>(smem + chunk_lds<N, CARRY>(kHeads) - 16 - kScaleBytes) + wave * 32;
      if constexpr (DT == HQ_DTYPE_F16) {
        float m = 0, down2;
#pragma unroll
        for (int i = 0; i < kNT; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(s[i][r]));
        range_scale(max_of_halves(m), up2, down2);
        if (lane < 32) downs[lane] = down2;
      }
      auto from_state = [&](float up) __attribute__((always_inline)) {
        const uint32_t id = opaque(lane), at_c = piece_at<kRow>(id & 31u, id >> 5);
        // A step's parts of the state are made, and C's fragments read, between the products of the step before it.
        u4 c[2][kTB], hi[2], lo[2];
        auto ready = [&](int k) __attribute__((always_inline)) {
#pragma unroll
          for (int b = 0; b < kTB; ++b) c[k & 1][b] = *reinterpret_cast<const u4*>(sC + (at_c ^ (uint32_t)(k << 5)) + 32 * b * kRow);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float u = s[k / 2][(k & 1) * 8 + 2 * i], v = s[k / 2][(k & 1) * 8 + 2 * i + 1];
            if constexpr (DT == HQ_DTYPE_F16) {
              u *= up;
              v *= up;
            }
            hi[k & 1][i] = take_part<DT>(u, v);
            lo[k & 1][i] = pack_pair<DT>(u, v);
          }
        };
        ready(0);
        place_bc();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < kNS; ++k) {
          if (k + 1 < kNS) ready(k + 1);
#pragma unroll
          for (int j = k * kBCLoads / kNS; j < (k + 1) * kBCLoads / kNS; ++j) load_bc(left, j);
#pragma unroll
          for (int b = 0; b < kTB; ++b) y[b] = mfma32<DT>(hi[k & 1], c[k & 1][b], k ? y[b] : f16x{});
#pragma unroll
          for (int b = 0; b < kTB; ++b) y[b] = mfma32<DT>(lo[k & 1], c[k & 1][b], y[b]);
          between<2 * kTB, 24 / (2 * kTB), 1>();
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int b = 0; b < kTB; ++b) {
          const float d = __builtin_amdgcn_exp2f(cum[32 * b + l32]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f4 down = {1.f, 1.f, 1.f, 1.f};
            if constexpr (DT == HQ_DTYPE_F16) down = *reinterpret_cast<const f4*>(downs + 8 * i + 4 * half);
#pragma unroll
            for (int v = 0; v < 4; ++v) y[b][4 * i + v] *= d * down[v];
          }
        }
      };
      from_state(up2);
      read_x();
      // M's fragments are read a step ahead; between the products, the next chunk's sums.
      look_x();
      next_whole = sums(turn ^ 1u, min(left, (uint32_t)L));
      const uint32_t idm = opaque(lane), at_m[2] = {m_place<L>(0, idm & 31u, idm >> 5), m_place<L>(1, idm & 31u, idm >> 5)};
      constexpr int kSteps = kTB == 2 ? 6 : 2;  // products of 16 earlier tokens: 2 for the first 32 tokens, 4 for the others
      u4 mf[2][2];
      auto read_m = [&](int j) __attribute__((always_inline)) {
        const int b = j < 2 ? 0 : 1, k = j < 2 ? j : j - 2;
        const unsigned char* const p = m0 + (at_m[b] ^ (uint32_t)(k << 5));
        mf[j & 1][0] = *reinterpret_cast<const u4*>(p);
        mf[j & 1][1] = *reinterpret_cast<const u4*>(p + m_bytes<L>());
      };
      read_m(0);
#pragma unroll
      for (int j = 0; j < kSteps; ++j) {
        const int b = j < 2 ? 0 : 1, k = j < 2 ? j : j - 2;
        if (j + 1 < kSteps) read_m(j + 1);
        u4 v = x[k], rest = u4{0, 0, 0, 0};
        if constexpr (DT == HQ_DTYPE_F16) {  // 11 bits are two bf16 parts, exactly
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float p, q;
            unpack_pair<DT>(v[i], p, q);
            v[i] = take_part<BF>(p, q);
            rest[i] = pack_pair<BF>(p, q);
          }
        }
        y[b] = mfma32<BF>(v, mf[j & 1][0], y[b]);
        y[b] = mfma32<BF>(v, mf[j & 1][1], y[b]);
        if constexpr (DT == HQ_DTYPE_F16) y[b] = mfma32<BF>(rest, mf[j & 1][0], y[b]);
      }
      __builtin_amdgcn_sched_barrier(0);

      // Through the wavefront's own LDS, whose x is in registers, 32 tokens at a time.
      const uint32_t idy = opaque(lane);
#pragma unroll
      for (int b = 0; b < kTB; ++b) {
        const uint32_t tt = idy & 31u, put_at = tt * 128 + ((idy >> 5 ^ (tt >> 1 & 7u)) << 4), get_t = idy / 4;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<f4*>(own + (put_at ^ (uint32_t)(i << 5))) = f4{y[b][4 * i], y[b][4 * i + 1], y[b][4 * i + 2], y[b][4 * i + 3]};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e2 = 0; e2 < 2; ++e2) {
            const uint32_t r = get_t + 16 * i;
            const f4 v = *reinterpret_cast<const f4*>(own + r * 128 + (((2 * (idy & 3u) + e2) ^ (r >> 1 & 7u)) << 4));
#pragma unroll
            for (int c = 0; c < 4; ++c) y[b][8 * i + 4 * e2 + c] = v[c];
          }
      }
    }

    if constexpr (!CARRY) put_x(odd + (turn ^ 1u));

    if constexpr (!CARRY) __builtin_amdgcn_s_setprio(0);
    // The state decayed, and the chunk's terms; between their products the outputs go out.
    const __amdgpu_buffer_rsrc_t by = rsrc(y_at);
    const uint32_t y_off = __umul24(lane / 4, y_step) + lane % 4 * 16;
    y_at += (uint64_t)n * y_step;
    z_at += (uint64_t)n * z_step;
    auto out = [&](int j) __attribute__((always_inline)) {
      if constexpr (!CARRY) {
        u4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float u = y[j / 2][8 * (j & 1) + 2 * i], v = y[j / 2][8 * (j & 1) + 2 * i + 1];
          if constexpr (GATED) {
            float z0, z1;
            unpack_pair<DT>(zr[j][i], z0, z1);
            u *= silu(z0);
            v *= silu(z1);
          }
          w[i] = pack_pair<DT>(u, v);
        }
        __builtin_amdgcn_raw_buffer_store_b128(w, by, out_at[j] | y_off, j * 16 * y_step, 0);
      }
    };
    constexpr int kOuts = kTB * 2;
    const float keep = __builtin_amdgcn_exp2f(whole);
    const uint32_t at_b[2] = {opaque(tr_b[0]), opaque(tr_b[1])};
    auto read_b = [&](int k, int i) __attribute__((always_inline)) {
      return tr_read(sB + (at_b[0] ^ (uint32_t)(i << 6)) + k * 16 * kRow, sB + (at_b[1] ^ (uint32_t)(i << 6)) + k * 16 * kRow);
    };
    auto weigh = [&](int k, float (&v)[8]) __attribute__((always_inline)) {
      const f4 w0 = *reinterpret_cast<const f4*>(weights + 16 * k + 8 * half), w1 = *reinterpret_cast<const f4*>(weights + 16 * k + 8 * half + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unpack_pair<DT>(x[k][i], v[2 * i], v[2 * i + 1]);
        v[2 * i] *= i < 2 ? w0[(2 * i) & 3] : w1[(2 * i) & 3];
        v[2 * i + 1] *= i < 2 ? w0[(2 * i + 1) & 3] : w1[(2 * i + 1) & 3];
      }
    };
    if constexpr (CARRY) {
      place_bc();
#pragma unroll
      for (int j = 0; j < kBCLoads; ++j) load_bc(left, j);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (DT == HQ_DTYPE_F16) {
      // Each channel's terms, two lanes', have a scale of their own.
      float v[kTS][8], up, scale_down, m = 0;
#pragma unroll
      for (int k = 0; k < kTS; ++k) {
        weigh(k, v[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[k][i]));
        __builtin_amdgcn_sched_barrier(0);
      }
      range_scale(max_of_halves(m), up, scale_down);
      u4 hi[kTS], lo[kTS];
#pragma unroll
      for (int k = 0; k < kTS; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float p = v[k][2 * i] * up, q = v[k][2 * i + 1] * up;
          hi[k][i] = take_part<DT>(p, q);
          lo[k][i] = pack_pair<DT>(p, q);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        f16x acc;
#pragma unroll
        for (int k = 0; k < kTS; ++k) {
          const u4 b = read_b(k, i);
          acc = mfma32<DT>(b, hi[k], k ? acc : f16x{});
          acc = mfma32<DT>(b, lo[k], acc);
        }
#pragma unroll
        for (int j = i * kOuts / kNT; j < (i + 1) * kOuts / kNT; ++j) out(j);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] = fmaf(s[i][r], keep, acc[r] * scale_down);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      u4 part3[2][3];
      auto ready = [&](int k) __attribute__((always_inline)) {
        float v[8];
        weigh(k, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          part3[k & 1][0][i] = take_part<DT>(v[2 * i], v[2 * i + 1]);
          part3[k & 1][1][i] = take_part<DT>(v[2 * i], v[2 * i + 1]);
          part3[k & 1][2][i] = pack_pair<DT>(v[2 * i], v[2 * i + 1]);
        }
      };
      ready(0);
#pragma unroll
      for (int i = 0; i < kNT; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] *= keep;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < kTS; ++k) {
        if (k + 1 < kTS) ready(k + 1);
#pragma unroll
        for (int j = k * kOuts / kTS; j < (k + 1) * kOuts / kTS; ++j) out(j);
#pragma unroll
        for (int i = 0; i < kNT; ++i) {
          const u4 b = read_b(k, i);
#pragma unroll
          for (int e2 = 0; e2 < 3; ++e2) s[i] = mfma32<DT>(b, part3[k & 1][e2], s[i]);
        }
        between<3 * kNT, CARRY ? 5 : 10, 0>();
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();
    if constexpr (CARRY) {
      look_x();
      next_whole = sums(turn ^ 1u, min(left, (uint32_t)L));
    }
    put();
    if constexpr (CARRY) put_x(odd + (turn ^ 1u));
  }

  if constexpr (CARRY) {
    float* const p = place(run.idx);
#pragma unroll
    for (int i = 0; i < kNT * 4; ++i)
      *reinterpret_cast<f4*>(p + i * 4 * kChunkThreads) = f4{s[i / 4][(i & 3) * 4], s[i / 4][(i & 3) * 4 + 1], s[i / 4][(i & 3) * 4 + 2], s[i / 4][(i & 3) * 4 + 3]};
    if (live && part == 0 && lane == 0) pl.totals[(size_t)run.idx * a.H + h] = total;
  } else if (run.idx == run.last && run.q.keep && live) {
#pragma unroll
    for (int i = 0; i < kNT * 4; ++i)
      *reinterpret_cast<f4*>(kept + 16 * (i / 2) + 4 * (i & 1)) =
          f4{s[i / 4][(i & 3) * 4], s[i / 4][(i & 3) * 4 + 1], s[i / 4][(i & 3) * 4 + 2], s[i / 4][(i & 3) * 4 + 3]};
  }
}

// Between the two launches: what enters each run of sequence blockIdx.y in place of what it leaves, the first one's own state,
// then S <- S times the run's decay + what the run adds. Workgroup x: 16 bytes a thread of a unit's state.
template <int P, int N>
__global__ __launch_bounds__(kChunkThreads) void hq_ssm_join_kernel(ScanArgs a, ChunkArgs pl) {
  constexpr uint32_t kQuads = N / 8, kHeads = kColumns / P, kWaves = P / 32;
  const uint32_t unit = blockIdx.x / kQuads, quad = blockIdx.x - unit * kQuads, b = blockIdx.y, lane = threadIdx.x & 63u;
  uint32_t first = 0, runs = 0;
  for (uint32_t i = 0; i <= b; i += 64) {
    const uint32_t j = min(i + lane, b), s0 = clamp_to(a.s.cu[j], a.s.T), s1 = clamp_to(a.s.cu[j + 1], a.s.T);
    const uint32_t mine = i + lane <= b && s1 > s0 ? (s1 - s0 + pl.run_tokens - 1) / pl.run_tokens : 0u, upto = scan_sum(mine);
    runs = (uint32_t)__builtin_amdgcn_readlane((int)mine, (int)(b & 63u));
    first += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
  }
  first -= runs;
  if (runs < 2 || first + runs > pl.runs) return;
  const uint32_t of_group = a.H / a.G, per_group = (of_group + kHeads - 1) / kHeads, g = unit / per_group;
  const uint32_t h = g * of_group + min((unit - g * per_group) * kHeads + uni(threadIdx.x >> 6) / kWaves, of_group - 1);
  const size_t step = (size_t)pl.units * kQuads * kChunkThreads;  // pieces of a run
  f4* const p = reinterpret_cast<f4*>(pl.states) + first * step + ((size_t)unit * kQuads + quad) * kChunkThreads + threadIdx.x;
  const float* const totals = pl.totals + (size_t)first * a.H + h;
  f4 s = p[(runs - 1) * step];
  constexpr uint32_t kAhead = 8;  // runs whose loads are in flight together
  for (uint32_t i0 = 0; i0 < runs; i0 += kAhead) {
    f4 v[kAhead];
    float d[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
      const uint32_t r = min(i0 + i, runs - 2);
      v[i] = p[r * step];
      d[i] = __builtin_amdgcn_exp2f(totals[(size_t)r * a.H]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) {
      if (i0 + i >= runs) break;
      p[(i0 + i) * step] = s;
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = i0 + i ? fmaf(s[e], d[i], v[i][e]) : v[i][e];  // (the first run has begun with its state)
    }
  }
}

template <int DT, int P, int N, int KIND>
hipError_t launch_one(const ScanArgs& a, const ChunkArgs& c, hipStream_t s) {
  auto k = hq_ssm_chunk_kernel<DT, P, N, KIND>;
  constexpr uint32_t lds = chunk_lds<N, KIND == kCarry>(kColumns / P);
  static const hipError_t set = hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (set != hipSuccess) return set;
  hipLaunchKernelGGL(k, dim3((c.blocks + 7) / 8 * 8), dim3(kChunkThreads), lds, s, a, c);
  return hipGetLastError();
}

template <int DT, int P, int N>
hipError_t launch(const ScanArgs& a, const ScanPlan& p, void* ws, hipStream_t s) {
  ChunkArgs c{p.run_tokens, p.units, p.runs, p.runs * p.units, nullptr, nullptr};
  if (p.split) {
    c.states = reinterpret_cast<float*>(static_cast<unsigned char*>(ws) + kCounterBytes);
    c.totals = c.states + (size_t)c.blocks * kColumns * N;
    hipError_t e = launch_one<DT, P, N, kCarry>(a, c, s);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((hq_ssm_join_kernel<P, N>), dim3(p.units * (N / 8), a.s.n), dim3(kChunkThreads), 0, s, a, c);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return a.Z ? launch_one<DT, P, N, kGated>(a, c, s) : launch_one<DT, P, N, kPlain>(a, c, s);
}

template <int DT>
hipError_t launch_type(const ScanArgs& a, const ScanPlan& p, void* ws, hipStream_t s) {
  switch (a.P * 1024 + a.N) {
    case 64 * 1024 + 64: return launch<DT, 64, 64>(a, p, ws, s);
    case 64 * 1024 + 128: return launch<DT, 64, 128>(a, p, ws, s);
    case 64 * 1024 + 256: return launch<DT, 64, 256>(a, p, ws, s);
    case 128 * 1024 + 64: return launch<DT, 128, 64>(a, p, ws, s);
    case 128 * 1024 + 128: return launch<DT, 128, 128>(a, p, ws, s);
    default: return launch<DT, 128, 256>(a, p, ws, s);
  }
}

}  // namespace

hipError_t launch_ssm_chunks(int dtype, const ScanArgs& a, const ScanPlan& p, void* ws, hipStream_t s) {
  return dtype == HQ_DTYPE_F16 ? launch_type<HQ_DTYPE_F16>(a, p, ws, s) : launch_type<HQ_DTYPE_BF16>(a, p, ws, s);
}

}  // namespace hq
