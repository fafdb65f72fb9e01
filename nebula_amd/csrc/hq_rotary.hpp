// hq_rotary.hpp — descriptors shared by the rotary entry points and their kernel.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hq_attn.hpp"
#include "hq_rotary.h"

namespace hq {

struct RotaryHeads {
  const uint16_t* in;
  uint16_t* out;
  int64_t in_row, in_head, out_row, out_head;
  const float* weight;
  uint32_t heads;
  float eps;
};

struct RotaryArgs {
  RotaryHeads q, k;   // k's out is the cache where there is one
  const uint16_t* V;  // with a cache
  int64_t v_row, v_head;
  const double* turns;
  float scale;
  uint32_t R, T, D;
  uint32_t all;        // heads of a token: q, k and, with a cache, v
  uint32_t slots;      // log2 of the heads that a workgroup takes
  const int32_t* pos;  // without a cache
  const int32_t* rows;
  const int32_t* cu;
  uint32_t n;
};

hipError_t launch_rotate(int dtype, int layout, RotaryArgs a, const CacheArgs* cache, hipStream_t s);

}  // namespace hq
