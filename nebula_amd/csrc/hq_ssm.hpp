// hq_ssm.hpp — descriptors shared by the state space entry points and their kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hq_ssm.h"

namespace hq {

// The sequences of a call and the rows of the states that they are.
struct SeqArgs {
  const int32_t* rows;     // or null: row i
  const int32_t* held;     // or null: all continue
  const int32_t* cu;       // [n + 1], or null: token i is sequence i's
  uint32_t n, T;           // sequences, tokens
  uint32_t cache_rows;
  const int32_t* refused;  // or null
  uint32_t* status;
};

struct ConvArgs {
  SeqArgs s;
  const uint16_t* X;
  uint16_t* Y;
  int64_t ldx, ldy;
  const float* W;
  const float* bias;
  uint16_t* state;  // the layer's
  int64_t row_stride;
  uint32_t C, width;
  uint32_t silu;
};
uint64_t conv_workgroups(const ConvArgs& a);  // of its launch
hipError_t launch_ssm_conv(int dtype, const ConvArgs& a, hipStream_t s);

struct ScanArgs {
  SeqArgs s;
  const uint16_t* X;
  const uint16_t* B;
  const uint16_t* C;
  const void* dt;
  const uint16_t* Z;
  uint16_t* Y;
  const float* A;
  const float* D;
  const float* dt_bias;
  int64_t x_row, x_head, b_row, b_group, c_row, c_group, dt_row, z_row, z_head, y_row, y_head;
  float* state;  // the layer's
  int64_t row_stride;
  uint32_t H, G, P, N;  // heads, groups, head_dim, state_dim
  uint32_t dt_f32, softplus;
};

// How a scan is split, from host-side sizes alone (the lengths stay on the device).
struct ScanPlan {
  bool chunk = false;       // in chunks, else token by token
  bool split = false;       // sequences are cut into runs: a launch for what they add to the state comes first
  uint32_t run_tokens = 0, units = 0, runs = 0;  // tokens of a run, workgroups of one, runs of the call at most
  uint64_t largest = 0;     // workgroups of its largest launch
  size_t ws = 0, need = 0;  // workspace that is used, and that is asked for: it does not fall as sizes grow
};
ScanPlan plan_scan(uint32_t tokens, uint32_t n, bool cu, uint32_t heads, uint32_t groups, uint32_t head_dim, uint32_t state_dim, uint32_t max_len);
void describe_scan(const ScanPlan& p, char* buf, size_t len);
hipError_t launch_ssm_scan(int dtype, const ScanArgs& a, const ScanPlan& p, void* ws, hipStream_t s);
hipError_t launch_ssm_chunks(int dtype, const ScanArgs& a, const ScanPlan& p, void* ws, hipStream_t s);

}  // namespace hq
