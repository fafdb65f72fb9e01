// hq_ssm.hip — the short causal convolution and the scan token by token (include/hq_ssm.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdio>

#include "hq_internal.hpp"
#include "hq_ssm_device.hpp"

namespace hq {
namespace {

// ---- the convolution ----
// Bound by the bytes moved, inputs and outputs once, and the arithmetic beside them (half the time alone: a product needs its
// exponential and reciprocal). A lane holds 8 channels of a run of TT tokens: the run's inputs and the W - 1 before it are
// loaded side by side, and each is W products' operand in registers. 2046 tokens of 10240 channels: 22 us, 3.8 TB/s of
// inputs and outputs; runs of 4, 6 and 16 tokens 23.9, 22.2 and 23.5.
//
// A sequence's first W - 1 tokens read the row's kept inputs, and its last ones replace them: whoever reads them
// writes them. So those first tokens are all the work of the run that the sequence begins in, up to W - 2 tokens past
// its end, and a run leaves out the first tokens of a sequence that begins before it.
constexpr uint32_t kRuns = 4;  // wavefronts, and runs, of a workgroup
constexpr uint32_t kRunTokens = 8;

template <int DT>
__device__ __forceinline__ void unpack8(u4 v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack_pair<DT>(v[i], f[2 * i], f[2 * i + 1]);
}

template <int DT>
__device__ __forceinline__ u4 pack8(const float (&y)[8]) {
  return u4{pack_pair<DT>(y[0], y[1]), pack_pair<DT>(y[2], y[3]), pack_pair<DT>(y[4], y[5]), pack_pair<DT>(y[6], y[7])};
}

// Weights, channel by channel, and biases of channels [c, c + 8).
template <int W>
__device__ __forceinline__ void load_weights(const ConvArgs& a, uint32_t c, float (&w)[8 * W], float (&bias)[8]) {
#pragma unroll
  for (int i = 0; i < 2 * W; ++i) {
    const f4 v = *reinterpret_cast<const f4*>(a.W + (size_t)c * W + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) bias[i] = a.bias ? a.bias[c + i] : 0.f;
}

// One token a sequence: bound by the wait for the row's number and then for its kept inputs, so everything else is loaded
// before them. 64 sequences of 10240 channels: 5.2 us (9.2 MB); 8.5 with the kernel below.
template <int DT, int W>
__global__ __launch_bounds__(64) void hq_ssm_conv_step_kernel(ConvArgs a) {
  const uint32_t c = (blockIdx.x * 64 + threadIdx.x) * 8, b = blockIdx.y;
  const bool some = c < a.C;
  const uint32_t cc = some ? c : 0u;
  const u4 x = *reinterpret_cast<const u4*>(a.X + b * a.ldx + cc);
  float w[8 * W], bias[8];
  load_weights<W>(a, cc, w, bias);
  const Seq q = find_seq(a.s, b, blockIdx.x == 0);
  uint16_t* kept = a.state + q.row * a.row_stride + cc;
  u4 in[W];
#pragma unroll
  for (int j = 0; j < W - 1; ++j) {
    in[j] = u4{0, 0, 0, 0};
    if (q.read) in[j] = *reinterpret_cast<const u4*>(kept + (size_t)j * a.C);
  }
  in[W - 1] = x;
  if (!some) return;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = bias[e];
#pragma unroll
  for (int j = 0; j < W; ++j) {
    float f[8];
    unpack8<DT>(in[j], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fmaf(w[e * W + j], f[e], y[e]);
  }
  if (a.silu) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = silu(y[e]);
  }
  *reinterpret_cast<u4*>(a.Y + b * a.ldy + c) = pack8<DT>(y);
  if (q.keep) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) *reinterpret_cast<u4*>(kept + (size_t)j * a.C) = in[j + 1];
  }
}

template <int DT, int W, int TT>
__global__ __launch_bounds__(64 * kRuns) void hq_ssm_conv_kernel(ConvArgs a) {
  constexpr int kLoads = TT + 2 * W - 3;  // tokens t0 - (W - 1) .. t0 + TT + W - 3
  // Channels go first in a grid of one axis (the second one's 2^16 would bound the tokens; tokens first: 23.5 for 22 us).
  const uint32_t across = (a.C / 8 + 63) / 64, by = blockIdx.x / across;
  const uint32_t c = ((blockIdx.x - by * across) * 64 + (threadIdx.x & 63u)) * 8;
  const uint32_t t0 = uni((by * kRuns + (threadIdx.x >> 6)) * TT);
  if (t0 >= a.s.T) return;  // (wavefronts share nothing)
  const bool some = c < a.C;
  const uint32_t cc = some ? c : 0u;
  u4 x[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int64_t t = (int64_t)t0 + i - (W - 1);
    x[i] = u4{0, 0, 0, 0};
    if (t >= 0 && t < a.s.T) x[i] = *reinterpret_cast<const u4*>(a.X + t * a.ldx + cc);
  }
  float w[8 * W], bias[8];
  load_weights<W>(a, cc, w, bias);

  uint32_t b = uni(seq_of(a.s, t0));
  uint32_t begin = a.s.cu ? clamp_to(a.s.cu[b], a.s.T) : b, end = a.s.cu ? clamp_to(a.s.cu[b + 1], a.s.T) : b + 1;
  // Most runs lie in one sequence, its first tokens not among them: every input is unpacked once.
  if (t0 >= (uint64_t)begin + (W - 1) && end >= (uint64_t)t0 + TT) {
    float in[W][8];  // token t's in place t % W
#pragma unroll
    for (int i = 0; i < W - 1; ++i) unpack8<DT>(x[i], in[i]);
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      unpack8<DT>(x[i + W - 1], in[(i + W - 1) % W]);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = bias[e];
#pragma unroll
        for (int j = 0; j < W; ++j) y[e] = fmaf(w[e * W + j], in[(i + j) % W][e], y[e]);
      }
      if (a.silu) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = silu(y[e]);
      }
      if (some) *reinterpret_cast<u4*>(a.Y + (int64_t)(t0 + i) * a.ldy + c) = pack8<DT>(y);
    }
    return;
  }
  u4 old[W - 1];  // the kept inputs of the sequence that begins in this run
#pragma unroll
  for (int i = 0; i < W - 1; ++i) old[i] = u4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < TT + W - 2; ++i) {
    const uint32_t t = t0 + i;
    // The sequence of token t: sequences that end at or before it are left behind.
    while (t >= end && b + 1 < a.s.n) {
      ++b;
      begin = a.s.cu ? clamp_to(a.s.cu[b], a.s.T) : b;
      end = a.s.cu ? clamp_to(a.s.cu[b + 1], a.s.T) : b + 1;
    }
    const bool mine = t >= begin && t < end &&
                      (i < TT ? begin >= t0 || t - begin >= W - 1u : begin >= t0 && begin < t0 + TT && t - begin < W - 1u);
    if (mine) {
      if (t == begin) {
        const Seq q = find_seq(a.s, b, c == 0);
        uint16_t* kept = a.state + q.row * a.row_stride + cc;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
          old[j] = u4{0, 0, 0, 0};
          if (q.read) old[j] = *reinterpret_cast<const u4*>(kept + (size_t)j * a.C);
        }
        // What is kept: inputs len - (W - 1) .. len - 1 of the sequence, those below 0 the old ones.
        const uint32_t len = end - begin;
        u4 now[W - 1];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
          if (len + j >= W - 1) now[j] = *reinterpret_cast<const u4*>(a.X + (int64_t)(begin + len + j - (W - 1)) * a.ldx + cc);
          else {
            now[j] = old[0];
#pragma unroll
            for (int k = 1; k < W - 1; ++k)
              if (len + j == (uint32_t)k) now[j] = old[k];
          }
        }
        if (q.keep && some) {
#pragma unroll
          for (int j = 0; j < W - 1; ++j) *reinterpret_cast<u4*>(kept + (size_t)j * a.C) = now[j];
        }
      }
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = bias[e];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        // Input t - (W - 1) + j: of the sequence, or one of the kept ones.
        u4 in = x[i + j];
        const uint32_t k = t - begin + j;  // its place, W - 1 added
        if (j < W - 1 && k < W - 1u) {
          in = old[j];
#pragma unroll
          for (int o = j + 1; o < W - 1; ++o)
            if (k == (uint32_t)o) in = old[o];
        }
        float f[8];
        unpack8<DT>(in, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(w[e * W + j], f[e], y[e]);
      }
      if (a.silu) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = silu(y[e]);
      }
      if (some) *reinterpret_cast<u4*>(a.Y + t * a.ldy + c) = pack8<DT>(y);
    }
  }
}

// Workgroups along the channels, and tokens of a wavefront: short sequences, whose runs would wait for one row of the states after
// the other, go one token a wavefront.
uint32_t conv_across(const ConvArgs& a) { return (a.C / 8 + 63) / 64; }
uint32_t conv_tile(const ConvArgs& a) { return a.s.T >= 32ull * a.s.n ? kRunTokens : 1; }

template <int DT, int W>
hipError_t launch_conv(const ConvArgs& a, hipStream_t s) {
  if (!a.s.cu) {
    hipLaunchKernelGGL((hq_ssm_conv_step_kernel<DT, W>), dim3(conv_across(a), a.s.n), dim3(64), 0, s, a);
    return hipGetLastError();
  }
  const dim3 grid((uint32_t)conv_workgroups(a));
  if (conv_tile(a) > 1) hipLaunchKernelGGL((hq_ssm_conv_kernel<DT, W, kRunTokens>), grid, dim3(64 * kRuns), 0, s, a);
  else hipLaunchKernelGGL((hq_ssm_conv_kernel<DT, W, 1>), grid, dim3(64 * kRuns), 0, s, a);
  return hipGetLastError();
}

template <int DT>
hipError_t launch_conv_type(const ConvArgs& a, hipStream_t s) {
  switch (a.width) {
    case 2: return launch_conv<DT, 2>(a, s);
    case 3: return launch_conv<DT, 3>(a, s);
    default: return launch_conv<DT, 4>(a, s);
  }
}

// ---- the scan, token by token ----
// Bound by the states' bytes, read and written once: a wavefront holds 8 rows of a head's state (32 a workgroup), every lane
// 4 elements of a row as one 16-byte piece, so that a load is 1 KB of memory in one piece. The sum over a row is
// one over the lanes that hold it, by moves between lanes. 64 sequences of 48 heads of 128x128: 89 us, 4.56 TB/s of states, inputs and
// outputs; one sequence 4.8, its launch and chain of loads.
constexpr uint32_t kColumnsOfRun = 128;  // channels of a workgroup of the chunk kernel
constexpr uint32_t kStepRows = 32;  // of a workgroup of four wavefronts

// Sum over aligned groups of NL lanes (16, 32 or 64), in every lane of the group.
template <int NL>
__device__ __forceinline__ float lanes_sum(float x) {
#define HQ_ADD(CTRL) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true))
  HQ_ADD(0xB1);   // the neighbour
  HQ_ADD(0x4E);   // the other pair of four
  HQ_ADD(0x141);  // the other four of eight
  HQ_ADD(0x140);  // the other eight of sixteen
#undef HQ_ADD
  if constexpr (NL >= 32) {
    const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(v[0]) + __uint_as_float(v[1]);
  }
  if constexpr (NL >= 64) {
    const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(v[0]) + __uint_as_float(v[1]);
  }
  return x;
}

template <int DT, int N>
__global__ __launch_bounds__(256) void hq_ssm_step_kernel(ScanArgs a) {
  constexpr uint32_t kLanes = N / 4, kAtOnce = 64 / kLanes, kLoads = 8 / kAtOnce;  // lanes of a row, rows of a load
  const uint32_t parts = a.P / kStepRows, h = blockIdx.x / parts, part = blockIdx.x - h * parts;
  const uint32_t lane = threadIdx.x & 63u, n = lane % kLanes * 4, g = h / (a.H / a.G);
  const uint32_t p0 = part * kStepRows + (threadIdx.x >> 6) * 8 + lane / kLanes;  // row of load i: p0 + i * kAtOnce
  const Seq q = find_seq(a.s, blockIdx.y, blockIdx.x == 0 && threadIdx.x < 64);
  if (q.a >= q.e) return;
  float* state = a.state + q.row * a.row_stride + (size_t)h * a.P * N + n;
  f4 s[kLoads];
#pragma unroll
  for (uint32_t i = 0; i < kLoads; ++i) {
    s[i] = f4{0, 0, 0, 0};
    if (q.read) s[i] = *reinterpret_cast<const f4*>(state + (size_t)(p0 + i * kAtOnce) * N);
  }
  const float A = a.A[h], D = a.D ? a.D[h] : 0.f, dt0 = a.dt_bias ? a.dt_bias[h] : 0.f;
  const uint32_t mine = min(lane % kLanes, kLoads - 1), p = p0 + mine * kAtOnce;  // the row whose output this lane writes
  for (uint32_t t = q.a; t < q.e; ++t) {
    const float dt = step_of(load_dt(a, t, h, DT) + dt0, a.softplus);
    const u2 bw = *reinterpret_cast<const u2*>(a.B + t * a.b_row + g * a.b_group + n);
    const u2 cw = *reinterpret_cast<const u2*>(a.C + t * a.c_row + g * a.c_group + n);
    const uint16_t* x = a.X + t * a.x_row + h * a.x_head;
    float z = 0;
    if (a.Z) z = to_f32<DT>(a.Z[t * a.z_row + h * a.z_head + p]);
    float b[4], c[4], xs[kLoads], y[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) xs[i] = to_f32<DT>(x[p0 + i * kAtOnce]);
    unpack_pair<DT>(bw[0], b[0], b[1]);
    unpack_pair<DT>(bw[1], b[2], b[3]);
    unpack_pair<DT>(cw[0], c[0], c[1]);
    unpack_pair<DT>(cw[1], c[2], c[3]);
    const float keep = expf(dt * A);
    float out = 0;
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const float dx = dt * xs[i];
      y[i] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = fmaf(s[i][e], keep, dx * b[e]);
        y[i] = fmaf(s[i][e], c[e], y[i]);
      }
      y[i] = lanes_sum<kLanes>(y[i]);
      if (mine == i) out = fmaf(D, xs[i], y[i]);
    }
    if (lane % kLanes < kLoads) {
      if (a.Z) out *= silu(z);
      a.Y[t * a.y_row + h * a.y_head + p] = f32_to_out<DT>(out);
    }
  }
  if (q.keep) {
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) *reinterpret_cast<f4*>(state + (size_t)(p0 + i * kAtOnce) * N) = s[i];
  }
}

template <int DT>
hipError_t launch_step(const ScanArgs& a, hipStream_t s) {
  const dim3 grid(a.H * (a.P / kStepRows), a.s.n);
  switch (a.N) {
    case 64: hipLaunchKernelGGL((hq_ssm_step_kernel<DT, 64>), grid, dim3(256), 0, s, a); break;
    case 128: hipLaunchKernelGGL((hq_ssm_step_kernel<DT, 128>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((hq_ssm_step_kernel<DT, 256>), grid, dim3(256), 0, s, a); break;
  }
  return hipGetLastError();
}

}  // namespace

uint64_t conv_workgroups(const ConvArgs& a) {
  if (!a.s.cu) return (uint64_t)conv_across(a) * a.s.n;
  const uint32_t per = conv_tile(a) * kRuns;
  return (uint64_t)((a.s.T + per - 1) / per) * conv_across(a);
}

hipError_t launch_ssm_conv(int dtype, const ConvArgs& a, hipStream_t s) {
  return dtype == HQ_DTYPE_F16 ? launch_conv_type<HQ_DTYPE_F16>(a, s) : launch_conv_type<HQ_DTYPE_BF16>(a, s);
}

// Which kernel, and how many tokens a run has, by a cost in time (us of an MI355X).
ScanPlan plan_scan(uint32_t tokens, uint32_t n, bool cu, uint32_t heads, uint32_t groups, uint32_t head_dim, uint32_t state_dim, uint32_t max_len) {
  ScanPlan p;
  p.largest = (uint64_t)heads * (head_dim / kStepRows) * n;
  // States of 256 are counted with one workgroup a CU, as fp16 has it (registers past 256); bf16 (at most 254) lets a second one in,
  // and is split as fp16 is.
  const uint32_t L = state_dim == 256 ? 32 : 64, two = 128 / head_dim, slots = (uint32_t)cu_count() * (state_dim == 256 ? 1 : 2);
  p.units = groups * ((heads / groups + two - 1) / two);
  // Few tokens a sequence go one by one. 48 heads of 128x128: 8 sequences of 6 and 8 tokens 18.3 and 23.9 us, in a chunk
  // 20.9; where there are more than workgroups at once, as 64 sequences are, of 4 and 6 tokens 93 and 116 us, in a chunk 96.
  if (!cu || tokens < ((uint64_t)n * p.units > slots ? 5ull : 8ull) * n) return p;
  p.chunk = true;
  const uint32_t longest = ((max_len && max_len < tokens ? max_len : tokens) + L - 1) / L;
  // Runs there may be: two rounds of workgroups and one a sequence.
  const uint32_t most = 2 * slots / p.units + n;
  uint32_t chunks = longest;
  if ((uint64_t)n * p.units < 2 * slots && longest > 1) {
    float best = 0;
    for (uint32_t k = 1; k <= std::min(longest, 64u); ++k) {
      const uint32_t even = (longest + k - 1) / k;  // the longest sequence in k even runs, and, for the others' sake, a chunk more
      if (k > 1 && tokens / ((even + 1) * L) + n > most) break;
      for (uint32_t c = even; c <= even + (k > 1); ++c) {
        const uint32_t runs = tokens / (c * L) + n;
        if (k > 1 && (runs > most || c >= longest)) continue;
        const uint64_t groups_of = (uint64_t)(k == 1 ? n : runs) * p.units, rounds = (groups_of + slots - 1) / slots;
        // In us, of states of 128, which stand for those of 64 and 256 too: a chunk of one workgroup a compute unit 5.15, of two at once 8.3; a carry is 0.45 of one; a launch about a chunk
        // before the first, and 3 or 18 apart. 48 heads of 128x128, 512 tokens: whole 45.6, runs of 2 chunks 42.8, of 1 47; 1024: whole
        // 83, of 4 55.2, of 2 57.7; 4096: of 13 119, of 7 110; 8192: of 26 215, of 13 191. 80 heads of 64x128, 1 to 1008 tokens: whole 90,
        // of 5 86 (fp16: 99, 88).
        const float one = state_dim != 256 && groups_of * 2 > slots ? 8.3f : 5.15f;
        const float cost = rounds * (c + 1) * one * (k > 1 ? 1.45f : 1.f) + (k > 1 ? 18.f : 3.f);
        if (k == 1 || cost < best) {
          best = cost;
          chunks = c;
        }
      }
    }
    const size_t run_bytes = (size_t)p.units * (kColumnsOfRun * state_dim + two) * 4;
    p.need = kCounterBytes + std::min((tokens + L - 1) / L + n, most) * run_bytes;
    p.split = chunks < longest;
    if (p.split) p.ws = kCounterBytes + (tokens / (chunks * L) + n) * run_bytes;
  }
  p.run_tokens = p.split ? chunks * L : (tokens + L - 1) / L * L;  // a whole sequence, whatever max_len says
  p.runs = p.split ? tokens / p.run_tokens + n : n;
  p.largest = (uint64_t)p.runs * p.units + 8;
  return p;
}

void describe_scan(const ScanPlan& p, char* buf, size_t len) {
  if (!p.chunk) snprintf(buf, len, "hq_ssm_step_kernel ws=%zu", p.ws);
  else snprintf(buf, len, "hq_ssm_chunk_kernel%s runs of %u tokens, grid=%u x %u ws=%zu", p.split ? " twice," : "", p.run_tokens, p.runs, p.units, p.ws);
}

hipError_t launch_ssm_scan(int dtype, const ScanArgs& a, const ScanPlan& p, void* ws, hipStream_t s) {
  if (p.chunk) return launch_ssm_chunks(dtype, a, p, ws, s);
  return dtype == HQ_DTYPE_F16 ? launch_step<HQ_DTYPE_F16>(a, s) : launch_step<HQ_DTYPE_BF16>(a, s);
}

}  // namespace hq
