// hq_ssm_api.cpp — the state space entry points of the C ABI (include/hq_ssm.h): argument validation, workspaces
// and launches. No exception crosses the ABI.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hq_attn.hpp"
#include "hq_checks.hpp"
#include "hq_internal.hpp"
#include "hq_ssm.hpp"

namespace {

using namespace hq::checks;

// Rows of a scan's operands at most 2^22 elements apart: the kernels multiply their bytes by a chunk's tokens in 24 bits.
constexpr int64_t kMaxRow = (int64_t)1 << 22;

hq_status check_sizes(uint32_t heads, uint32_t head_dim, uint32_t state_dim) {
  if (head_dim != 64 && head_dim != 128) return fail(HQ_ERR_UNSUPPORTED, "head_dim=%u must be 64 or 128", head_dim);
  if (state_dim != 64 && state_dim != 128 && state_dim != 256) return fail(HQ_ERR_UNSUPPORTED, "state_dim=%u must be 64, 128 or 256", state_dim);
  if (heads == 0 || heads > 1024) return fail(HQ_ERR_SHAPE, "heads=%u must be 1..1024", heads);
  return HQ_OK;
}

hq_status check_groups(uint32_t H, uint32_t G) {
  if (G == 0 || H % G) return fail(HQ_ERR_SHAPE, "heads=%u must be a positive multiple of groups=%u", H, G);
  return HQ_OK;
}

hq_status check_tokens(uint32_t tokens, uint32_t n, bool cu) {
  if (n == 0 || n > HQ_SSM_MAX_BATCH) return fail(HQ_ERR_SHAPE, "n=%u must be 1..%u", n, HQ_SSM_MAX_BATCH);
  if (tokens == 0 || tokens > (1u << 24)) return fail(HQ_ERR_SHAPE, "tokens=%u out of range", tokens);
  if (!cu && tokens != n) return fail(HQ_ERR_SHAPE, "tokens=%u: without cu there is one for each of the %u rows", tokens, n);
  return HQ_OK;
}

// What both calls need of the states, and the call's sequences.
hq_status check_states(const hq_state_cache* c, uint32_t layer, uint32_t tokens, const int32_t* rows, const int32_t* held, const int32_t* cu,
                       uint32_t n, hq::SeqArgs* s) {
  if (!c) return fail(HQ_ERR_INVALID_ARG, "cache is null");
  hq_status st;
  if ((st = check_dtype(c->dtype)) != HQ_OK) return st;
  if (!c->status) return fail(HQ_ERR_INVALID_ARG, "cache: status is null");
  if (misaligned(c->status, 4) || misaligned(c->refused, 4)) return fail(HQ_ERR_ALIGNMENT, "cache: status and refused must be 4-byte aligned");
  if (c->layers == 0 || c->layers > 4096 || c->rows == 0 || c->rows > (1u << 20))
    return fail(HQ_ERR_SHAPE, "cache: layers=%u, rows=%u out of range", c->layers, c->rows);
  if (layer >= c->layers) return fail(HQ_ERR_SHAPE, "layer=%u of %u", layer, c->layers);
  if ((st = check_tokens(tokens, n, cu != nullptr)) != HQ_OK) return st;
  if (misaligned(rows, 4) || misaligned(held, 4) || misaligned(cu, 4)) return fail(HQ_ERR_ALIGNMENT, "rows, held and cu must be 4-byte aligned");
  if (!rows && n > c->rows) return fail(HQ_ERR_SHAPE, "n=%u: the cache has %u rows", n, c->rows);
  *s = {rows, held, cu, n, tokens, c->rows, c->refused, c->status};
  return HQ_OK;
}

// Layer and row strides of `rows` pieces of `size` elements.
hq_status check_pool(const char* name, int64_t layer, int64_t row, uint32_t layers, uint32_t rows, int64_t size, int64_t unit) {
  if (row % unit || layer % unit) return fail(HQ_ERR_ALIGNMENT, "cache: %s strides %lld, %lld must be multiples of %lld", name, (long long)layer, (long long)row, (long long)unit);
  if (row < 0 || layer < 0 || row > kMaxSpan || layer > kMaxSpan || (rows > 1 && row < size) || (layers > 1 && layer < size) ||
      (double)row * rows + (double)layer * layers > (double)kMaxSpan)
    return fail(HQ_ERR_SHAPE, "cache: %s strides %lld, %lld out of range (a row has %lld elements)", name, (long long)layer, (long long)row, (long long)size);
  if (rows > 1 && layers > 1 && layer < (rows - 1) * row + size && row < (layers - 1) * layer + size)
    return fail(HQ_ERR_SHAPE, "cache: %s strides %lld, %lld make rows of different layers overlap", name, (long long)layer, (long long)row);
  return HQ_OK;
}

hq_status check_plan(const hq::ScanPlan& p) {
  if (p.largest > hq::kMaxGrid) return fail(HQ_ERR_SHAPE, "%llu workgroups: too many sequences and heads for one call", (unsigned long long)p.largest);
  return HQ_OK;
}

hq_status check_query(uint32_t tokens, uint32_t n, int cu, uint32_t heads, uint32_t groups, uint32_t head_dim, uint32_t state_dim) {
  hq_status st;
  if ((st = check_sizes(heads, head_dim, state_dim)) != HQ_OK || (st = check_groups(heads, groups)) != HQ_OK) return st;
  return check_tokens(tokens, n, cu != 0);
}

}  // namespace

extern "C" {

hq_status hq_ssm_conv(const hq_state_cache* cache, uint32_t layer, const void* X, int64_t ldx, void* Y, int64_t ldy, const float* W,
                      const float* bias, int silu, uint32_t tokens, const int32_t* rows, const int32_t* held, const int32_t* cu,
                      uint32_t n, hq_stream stream) {
  hq::ConvArgs a{};
  hq_status st = check_states(cache, layer, tokens, rows, held, cu, n, &a.s);
  if (st != HQ_OK) return st;
  const uint32_t C = cache->channels, w = cache->width;
  if (!cache->conv) return fail(HQ_ERR_INVALID_ARG, "cache: conv is null");
  if (misaligned(cache->conv, 16)) return fail(HQ_ERR_ALIGNMENT, "cache: conv must be 16-byte aligned");
  if (w < 2 || w > 4) return fail(HQ_ERR_UNSUPPORTED, "width=%u must be 2, 3 or 4", w);
  if (C == 0 || C % 8 || C > (1u << 20)) return fail(HQ_ERR_SHAPE, "channels=%u must be a positive multiple of 8, at most %u", C, 1u << 20);
  if ((uint64_t)tokens * C > (1ull << 37)) return fail(HQ_ERR_SHAPE, "tokens=%u of %u channels: too many for one call", tokens, C);
  if ((st = check_pool("conv", cache->conv_layer, cache->conv_row, cache->layers, cache->rows, (int64_t)(w - 1) * C, 8)) != HQ_OK) return st;
  if (!X || !Y || !W) return fail(HQ_ERR_INVALID_ARG, "X, Y or W is null");
  if (X == Y) return fail(HQ_ERR_INVALID_ARG, "Y is X: a convolution needs its inputs");
  if (misaligned(X, 16) || misaligned(Y, 16) || misaligned(W, 16) || misaligned(bias, 16))
    return fail(HQ_ERR_ALIGNMENT, "X, Y, W and bias must be 16-byte aligned");
  if ((st = check_strides("X", ldx, 0, tokens, 1, C)) != HQ_OK || (st = check_strides("Y", ldy, 0, tokens, 1, C)) != HQ_OK) return st;
  a.X = static_cast<const uint16_t*>(X);
  a.Y = static_cast<uint16_t*>(Y);
  a.ldx = ldx;
  a.ldy = ldy;
  a.W = W;
  a.bias = bias;
  a.state = static_cast<uint16_t*>(cache->conv) + layer * cache->conv_layer;
  a.row_stride = cache->conv_row;
  a.C = C;
  a.width = w;
  a.silu = silu != 0;
  if (hq::conv_workgroups(a) > hq::kMaxGrid)
    return fail(HQ_ERR_SHAPE, "%llu workgroups: too many tokens and channels for one call", (unsigned long long)hq::conv_workgroups(a));
  return from_hip(hq::launch_ssm_conv(cache->dtype, a, reinterpret_cast<hipStream_t>(stream)), "convolution launch");
}

hq_status hq_ssm_workspace_bytes(uint32_t tokens, uint32_t n, int cu, uint32_t heads, uint32_t groups, uint32_t head_dim, uint32_t state_dim,
                                 uint32_t max_len, size_t* bytes) {
  if (!bytes) return fail(HQ_ERR_INVALID_ARG, "bytes is null");
  hq_status st = check_query(tokens, n, cu, heads, groups, head_dim, state_dim);
  if (st != HQ_OK) return st;
  const hq::ScanPlan p = hq::plan_scan(tokens, n, cu != 0, heads, groups, head_dim, state_dim, max_len);
  if ((st = check_plan(p)) != HQ_OK) return st;
  *bytes = p.need;
  return hq_set_error(HQ_OK, "");
}

hq_status hq_describe_ssm(uint32_t tokens, uint32_t n, int cu, uint32_t heads, uint32_t groups, uint32_t head_dim, uint32_t state_dim, uint32_t max_len,
                          char* buf, size_t buf_len) {
  if (!buf || buf_len == 0) return fail(HQ_ERR_INVALID_ARG, "buf is null or empty");
  hq_status st = check_query(tokens, n, cu, heads, groups, head_dim, state_dim);
  if (st != HQ_OK) return st;
  const hq::ScanPlan p = hq::plan_scan(tokens, n, cu != 0, heads, groups, head_dim, state_dim, max_len);
  if ((st = check_plan(p)) != HQ_OK) return st;
  hq::describe_scan(p, buf, buf_len);
  return hq_set_error(HQ_OK, "");
}

hq_status hq_ssm_scan(const hq_state_cache* cache, uint32_t layer, const hq_ssm_io* io, const int32_t* rows, const int32_t* held,
                      const int32_t* cu, uint32_t n, uint32_t max_len, void* ws, size_t ws_bytes, hq_stream stream) {
  if (!io) return fail(HQ_ERR_INVALID_ARG, "io is null");
  hq::ScanArgs a{};
  const uint32_t T = io->tokens;
  hq_status st = check_states(cache, layer, T, rows, held, cu, n, &a.s);
  if (st != HQ_OK) return st;
  const uint32_t H = cache->heads, P = cache->head_dim, N = cache->state_dim, G = io->groups;
  if ((st = check_sizes(H, P, N)) != HQ_OK) return st;
  if (!cache->ssm) return fail(HQ_ERR_INVALID_ARG, "cache: ssm is null");
  if (misaligned(cache->ssm, 16)) return fail(HQ_ERR_ALIGNMENT, "cache: ssm must be 16-byte aligned");
  if ((st = check_pool("ssm", cache->ssm_layer, cache->ssm_row, cache->layers, cache->rows, (int64_t)H * P * N, 4)) != HQ_OK) return st;
  if ((st = check_groups(H, G)) != HQ_OK) return st;
  if ((uint64_t)T * H > (1u << 30)) return fail(HQ_ERR_SHAPE, "tokens=%u of %u heads: too many for one call", T, H);
  if (!io->X || !io->B || !io->C || !io->dt || !io->Y || !io->A) return fail(HQ_ERR_INVALID_ARG, "X, B, C, dt, Y or A is null");
  if (io->Y == io->X || io->Y == io->B || io->Y == io->C || io->Y == io->dt) return fail(HQ_ERR_INVALID_ARG, "Y is an input that others read");
  if (misaligned(io->X, 16) || misaligned(io->B, 16) || misaligned(io->C, 16) || misaligned(io->Y, 16) || misaligned(io->Z, 16))
    return fail(HQ_ERR_ALIGNMENT, "X, B, C, Z and Y must be 16-byte aligned");
  if (misaligned(io->dt, io->dt_f32 ? 4 : 2) || misaligned(io->A, 4) || misaligned(io->D, 4) || misaligned(io->dt_bias, 4))
    return fail(HQ_ERR_ALIGNMENT, "dt, A, D and dt_bias must be aligned to their elements");
  if ((st = check_strides("X", io->x_row, io->x_head, T, H, P)) != HQ_OK || (st = check_strides("B", io->b_row, io->b_group, T, G, N)) != HQ_OK ||
      (st = check_strides("C", io->c_row, io->c_group, T, G, N)) != HQ_OK || (st = check_strides("Y", io->y_row, io->y_head, T, H, P)) != HQ_OK ||
      (io->Z && (st = check_strides("Z", io->z_row, io->z_head, T, H, P)) != HQ_OK))
    return st;
  if (io->x_row > kMaxRow || io->b_row > kMaxRow || io->c_row > kMaxRow || io->y_row > kMaxRow || (io->Z && io->z_row > kMaxRow))
    return fail(HQ_ERR_SHAPE, "X, B, C, Y, Z: row strides %lld, %lld, %lld, %lld, %lld above %lld elements", (long long)io->x_row,
                (long long)io->b_row, (long long)io->c_row, (long long)io->y_row, (long long)io->z_row, (long long)kMaxRow);
  if (overlaps(io->y_row, io->y_head, T, H, P)) return fail(HQ_ERR_SHAPE, "Y: strides %lld, %lld make rows or heads overlap", (long long)io->y_row, (long long)io->y_head);
  if (io->Y == io->Z && ((T > 1 && io->y_row != io->z_row) || (H > 1 && io->y_head != io->z_head))) return fail(HQ_ERR_SHAPE, "Y is Z with other strides");
  if (io->dt_row < 0 || io->dt_row > kMaxRow || (T > 1 && io->dt_row < (int64_t)H))
    return fail(HQ_ERR_SHAPE, "dt: stride %lld out of range (heads=%u)", (long long)io->dt_row, H);
  a.X = static_cast<const uint16_t*>(io->X);
  a.B = static_cast<const uint16_t*>(io->B);
  a.C = static_cast<const uint16_t*>(io->C);
  a.dt = io->dt;
  a.Z = static_cast<const uint16_t*>(io->Z);
  a.Y = static_cast<uint16_t*>(io->Y);
  a.A = io->A;
  a.D = io->D;
  a.dt_bias = io->dt_bias;
  a.x_row = io->x_row;
  a.x_head = io->x_head;
  a.b_row = io->b_row;
  a.b_group = io->b_group;
  a.c_row = io->c_row;
  a.c_group = io->c_group;
  a.dt_row = io->dt_row;
  a.z_row = io->z_row;
  a.z_head = io->z_head;
  a.y_row = io->y_row;
  a.y_head = io->y_head;
  a.state = cache->ssm + layer * cache->ssm_layer;
  a.row_stride = cache->ssm_row;
  a.H = H;
  a.G = G;
  a.P = P;
  a.N = N;
  a.dt_f32 = io->dt_f32 != 0;
  a.softplus = io->softplus != 0;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hq::ScanPlan p = hq::plan_scan(T, n, cu != nullptr, H, G, P, N, max_len);
  void* w = nullptr;
  if ((st = check_plan(p)) != HQ_OK || (st = workspace(ws, ws_bytes, p.ws, p.need, s, &w)) != HQ_OK) return st;
  return from_hip(hq::launch_ssm_scan(cache->dtype, a, p, w, s), "scan launch");
}

}  // extern "C"
