// hq_attn_api.cpp — the attention, cache and rotary entry points of the C ABI (include/hq_attn.h,
// include/hq_rotary.h): argument validation, workspaces and launches. No exception crosses the ABI.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>

#include "hq_attn.hpp"
#include "hq_checks.hpp"
#include "hq_internal.hpp"
#include "hq_rotary.hpp"

namespace {

using namespace hq::checks;

// Rows of keys and values at most 2^23 elements apart: the kernels address 16 of them with 32-bit offsets.
constexpr int64_t kMaxRow = (int64_t)1 << 23;

hq_status check_dim(uint32_t D) {
  if (D != 64 && D != 128 && D != 256) return fail(HQ_ERR_UNSUPPORTED, "head_dim=%u must be 64, 128 or 256", D);
  return HQ_OK;
}
// Tokens and heads of a call: row numbers t * G + g and grid sizes are 32-bit.
hq_status check_counts(uint32_t rows, uint32_t seqs, uint32_t heads, uint32_t kv_heads) {
  if (rows == 0 || seqs == 0) return fail(HQ_ERR_SHAPE, "rows=%u and seqs=%u must be positive", rows, seqs);
  if (heads == 0 || kv_heads == 0 || heads % kv_heads)
    return fail(HQ_ERR_SHAPE, "heads=%u must be a positive multiple of kv_heads=%u", heads, kv_heads);
  if (heads > 1024 || rows > (1u << 24) || seqs > (1u << 20) || (uint64_t)rows * heads > (1u << 30))
    return fail(HQ_ERR_SHAPE, "rows=%u, seqs=%u, heads=%u: too many for one call", rows, seqs, heads);
  return HQ_OK;
}

hq_status check_io(const hq_attn_io* io, uint32_t seqs, uint32_t kv_heads, hq::AttnArgs* a) {
  if (!io) return fail(HQ_ERR_INVALID_ARG, "io is null");
  hq_status st;
  if (!io->Q || !io->O) return fail(HQ_ERR_INVALID_ARG, "Q or O is null");
  if ((st = check_dtype(io->dtype)) != HQ_OK || (st = check_dim(io->head_dim)) != HQ_OK ||
      (st = check_counts(io->rows, seqs, io->heads, kv_heads)) != HQ_OK)
    return st;
  if (!(io->scale > 0.f) || !std::isfinite(io->scale)) return fail(HQ_ERR_INVALID_ARG, "scale=%g must be positive and finite", (double)io->scale);
  if (misaligned(io->Q, 16) || misaligned(io->O, 16)) return fail(HQ_ERR_ALIGNMENT, "Q and O must be 16-byte aligned");
  if (misaligned(io->lse, 4)) return fail(HQ_ERR_ALIGNMENT, "lse must be 4-byte aligned");
  if ((st = check_strides("Q", io->q_row, io->q_head, io->rows, io->heads, io->head_dim)) != HQ_OK ||
      (st = check_strides("O", io->o_row, io->o_head, io->rows, io->heads, io->head_dim)) != HQ_OK)
    return st;
  if (overlaps(io->o_row, io->o_head, io->rows, io->heads, io->head_dim))
    return fail(HQ_ERR_SHAPE, "O: strides %lld, %lld make rows or heads overlap", (long long)io->o_row, (long long)io->o_head);
  *a = hq::AttnArgs{};
  a->Q = static_cast<const uint16_t*>(io->Q);
  a->O = static_cast<uint16_t*>(io->O);
  a->lse = io->lse;
  a->q_row = io->q_row;
  a->q_head = io->q_head;
  a->o_row = io->o_row;
  a->o_head = io->o_head;
  a->T = io->rows;
  a->H = io->heads;
  a->Hkv = kv_heads;
  a->G = io->heads / kv_heads;
  a->D = io->head_dim;
  a->scale = io->scale;
  a->B = seqs;
  return HQ_OK;
}

// A cache's own sizes, and the order of a page's heads and tokens.
hq_status check_cache(const hq_kv_cache* c, hq::CacheArgs* out) {
  if (!c) return fail(HQ_ERR_INVALID_ARG, "cache is null");
  if (!c->K || !c->V || !c->table || !c->lens || !c->refs || !c->status) return fail(HQ_ERR_INVALID_ARG, "cache: null pointer");
  hq_status st;
  if ((st = check_dtype(c->dtype)) != HQ_OK || (st = check_dim(c->head_dim)) != HQ_OK) return st;
  if (c->layers == 0 || c->pages == 0 || c->kv_heads == 0 || c->rows == 0 || c->max_pages == 0)
    return fail(HQ_ERR_SHAPE, "cache: layers=%u, pages=%u, kv_heads=%u, rows=%u and max_pages=%u must be positive",
                c->layers, c->pages, c->kv_heads, c->rows, c->max_pages);
  const uint32_t T = c->page_tokens;
  if (T < 16 || T > 65536 || (T & (T - 1))) return fail(HQ_ERR_SHAPE, "cache: page_tokens=%u must be a power of two, 16 to 65536", T);
  if ((uint64_t)c->kv_heads * c->head_dim > (uint64_t)kMaxRow)
    return fail(HQ_ERR_SHAPE, "cache: kv_heads=%u times head_dim=%u above %lld", c->kv_heads, c->head_dim, (long long)kMaxRow);
  if (c->pages > (1u << 21) || c->layers > 4096 || c->kv_heads > 1024 || c->rows > (1u << 20) ||
      (uint64_t)c->max_pages * T > (1u << 30))
    return fail(HQ_ERR_SHAPE, "cache: layers=%u, pages=%u, kv_heads=%u, rows=%u, max_pages=%u: too many", c->layers, c->pages, c->kv_heads,
                c->rows, c->max_pages);
  if (c->table_stride < (int64_t)c->max_pages || c->table_stride > (1 << 30))
    return fail(HQ_ERR_SHAPE, "cache: table_stride=%lld out of range (max_pages=%u)", (long long)c->table_stride, c->max_pages);
  const int64_t D = c->head_dim, dense = (int64_t)c->kv_heads * T * D;
  const bool heads_first = c->token_stride == D && c->head_stride == (int64_t)T * D;
  const bool tokens_first = c->head_stride == D && c->token_stride == (int64_t)c->kv_heads * D;
  if (!heads_first && !tokens_first)
    return fail(HQ_ERR_SHAPE, "cache: a page must be dense: head_stride=%lld, token_stride=%lld fit neither order",
                (long long)c->head_stride, (long long)c->token_stride);
  if (c->page_stride < dense || c->page_stride > kMaxSpan || c->page_stride % 8 || c->layer_stride % 8 ||
      (c->layers > 1 && c->layer_stride < dense) || c->layer_stride < 0 || c->layer_stride > kMaxSpan)
    return fail(HQ_ERR_SHAPE, "cache: page_stride=%lld, layer_stride=%lld must be multiples of 8 and at least a page (%lld)",
                (long long)c->page_stride, (long long)c->layer_stride, (long long)dense);
  // fork and copy_pages move it by one launch (16 KB a workgroup).
  if ((uint64_t)dense * c->layers * 4 > (1ull << 37))
    return fail(HQ_ERR_SHAPE, "cache: a page of %u layers has %lld bytes a layer: above 128 GiB", c->layers, (long long)dense * 4);
  if (misaligned(c->K, 16) || misaligned(c->V, 16)) return fail(HQ_ERR_ALIGNMENT, "cache: K and V must be 16-byte aligned");
  if (misaligned(c->table, 4) || misaligned(c->lens, 4) || misaligned(c->refs, 4) || misaligned(c->status, 4) || misaligned(c->refused, 4))
    return fail(HQ_ERR_ALIGNMENT, "cache: table, lens, refs, status and refused must be 4-byte aligned");
  hq::CacheArgs a{};
  a.K = static_cast<uint16_t*>(c->K);
  a.V = static_cast<uint16_t*>(c->V);
  a.layer_stride = c->layer_stride;
  a.page_stride = c->page_stride;
  a.head_stride = c->head_stride;
  a.token_stride = c->token_stride;
  a.layers = c->layers;
  a.pages = c->pages;
  a.kv_heads = c->kv_heads;
  a.page_shift = (uint32_t)__builtin_ctz(T);
  a.dim = c->head_dim;
  a.table = c->table;
  a.table_stride = c->table_stride;
  a.rows = c->rows;
  a.max_pages = c->max_pages;
  a.lens = c->lens;
  a.refs = c->refs;
  a.status = c->status;
  a.refused = c->refused;
  a.shape.runs = heads_first ? c->kv_heads : 1u;
  a.shape.per_token = heads_first ? c->head_dim : c->kv_heads * c->head_dim;
  a.shape.run_stride = heads_first ? c->head_stride : 0;
  *out = a;
  return HQ_OK;
}

hq_status check_batch(uint32_t n) {
  if (n == 0 || n > HQ_CACHE_MAX_BATCH) return fail(HQ_ERR_SHAPE, "n=%u must be 1..%u", n, HQ_CACHE_MAX_BATCH);
  return HQ_OK;
}

hq_status check_plan(const hq::AttnPlan& p) {
  if (p.largest > hq::kMaxGrid) return fail(HQ_ERR_SHAPE, "%llu workgroups: too many rows and heads for one call", (unsigned long long)p.largest);
  return HQ_OK;
}

hq_status run_attn(const hq::AttnArgs& a, int kind, int dtype, uint32_t max_keys, uint32_t max_prefix, void* ws, size_t bytes,
                   hq_stream stream) {
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const hq::AttnPlan p = hq::plan_attn(kind, a.T, a.B, a.groups, a.H, a.Hkv, a.D, max_keys, max_prefix);
  void* w = nullptr;
  hq_status st = check_plan(p);
  if (st != HQ_OK || (st = workspace(ws, bytes, p.ws, p.need, s, &w)) != HQ_OK) return st;
  return from_hip(hq::launch_attn(dtype, a, p, w, s), "attention launch");
}

// A layer of the cache as the keys of a call.
hq_status cache_keys(const hq_attn_io* io, const hq_kv_cache* cache, uint32_t layer, const int32_t* rows, uint32_t seqs,
                     hq::AttnArgs* a) {
  hq::CacheArgs c;
  hq_status st = check_cache(cache, &c);
  if (st != HQ_OK) return st;
  if ((st = check_io(io, seqs, c.kv_heads, a)) != HQ_OK) return st;
  if (io->dtype != cache->dtype || io->head_dim != c.dim)
    return fail(HQ_ERR_SHAPE, "the call's dtype %d and head_dim=%u differ from the cache's (%d, %u)", (int)io->dtype, io->head_dim,
                (int)cache->dtype, c.dim);
  if (layer >= c.layers) return fail(HQ_ERR_SHAPE, "layer=%u of %u", layer, c.layers);
  if (misaligned(rows, 4)) return fail(HQ_ERR_ALIGNMENT, "rows must be 4-byte aligned");
  if (!rows && seqs > c.rows) return fail(HQ_ERR_SHAPE, "seqs=%u: the cache has %u rows", seqs, c.rows);
  hq::AttnKeys& k = a->k;
  k.K = c.K + layer * c.layer_stride;
  k.V = c.V + layer * c.layer_stride;
  k.k_row = k.v_row = c.token_stride;
  k.k_head = k.v_head = c.head_stride;
  k.page_stride = c.page_stride;
  k.table = c.table;
  k.table_stride = c.table_stride;
  k.lens = c.lens;
  k.rows = rows;
  k.cache_rows = c.rows;
  k.max_pages = c.max_pages;
  k.pages = c.pages;
  k.page_shift = c.page_shift;
  k.status = c.status;
  return HQ_OK;
}

uint32_t capacity(const hq_kv_cache* c) { return c->max_pages * c->page_tokens; }

hq_status check_query(hq_attn_kind kind, uint32_t rows, uint32_t seqs, uint32_t groups, uint32_t heads, uint32_t kv_heads,
                      uint32_t dim, uint32_t max_keys) {
  if (kind < HQ_ATTN_PROMPT || kind > HQ_ATTN_SHARED) return fail(HQ_ERR_INVALID_ARG, "unknown kind %d", (int)kind);
  if (max_keys == 0) return fail(HQ_ERR_SHAPE, "max_keys=0: a query needs the bound that 0 stands for in a call (total_k, a row's capacity)");
  hq_status st;
  if ((st = check_dim(dim)) != HQ_OK || (st = check_counts(rows, seqs, heads, kv_heads)) != HQ_OK) return st;
  if (kind == HQ_ATTN_SHARED && (groups == 0 || groups > seqs || rows != seqs))
    return fail(HQ_ERR_SHAPE, "groups=%u, rows=%u: need 1..seqs=%u groups and a row for each sequence", groups, rows, seqs);
  return HQ_OK;
}

hq_status check_rotary(const hq_rotary* r, uint32_t head_dim, hq::RotaryArgs* a) {
  if (!r) return fail(HQ_ERR_INVALID_ARG, "rotary is null");
  if (!r->turns) return fail(HQ_ERR_INVALID_ARG, "rotary: turns is null");
  if (misaligned(r->turns, 8)) return fail(HQ_ERR_ALIGNMENT, "rotary: turns must be 8-byte aligned");
  if (r->layout != HQ_ROTARY_HALF && r->layout != HQ_ROTARY_INTERLEAVED) return fail(HQ_ERR_INVALID_ARG, "rotary: unknown layout %d", (int)r->layout);
  if (r->dim == 0 || r->dim % 16 || r->dim > head_dim)
    return fail(HQ_ERR_SHAPE, "rotary: dim=%u must be a multiple of 16, 16 to head_dim=%u", r->dim, head_dim);
  if (!(r->scale > 0.f) || !std::isfinite(r->scale)) return fail(HQ_ERR_INVALID_ARG, "rotary: scale=%g must be positive and finite", (double)r->scale);
  a->turns = r->turns;
  a->R = r->dim;
  a->scale = r->scale;
  return HQ_OK;
}

// One operand of a rotation; `out`: whether it is written to its Out.
hq_status check_heads(const char* name, const hq_rotary_heads* h, uint32_t tokens, uint32_t dim, bool out, hq::RotaryHeads* to) {
  if (!h->In || (out && !h->Out)) return fail(HQ_ERR_INVALID_ARG, "%s: In or Out is null", name);
  if (h->heads == 0 || h->heads > 1024) return fail(HQ_ERR_SHAPE, "%s: heads=%u must be 1..1024", name, h->heads);
  if (misaligned(h->In, 16) || (out && misaligned(h->Out, 16))) return fail(HQ_ERR_ALIGNMENT, "%s: In and Out must be 16-byte aligned", name);
  if (misaligned(h->weight, 16)) return fail(HQ_ERR_ALIGNMENT, "%s: weight must be 16-byte aligned", name);
  if (h->weight && (!(h->eps >= 0.f) || !std::isfinite(h->eps))) return fail(HQ_ERR_INVALID_ARG, "%s: eps=%g must not be negative, and finite", name, (double)h->eps);
  hq_status st;
  if ((st = check_strides(name, h->in_row, h->in_head, tokens, h->heads, dim)) != HQ_OK) return st;
  if (out) {
    if ((st = check_strides(name, h->out_row, h->out_head, tokens, h->heads, dim)) != HQ_OK) return st;
    if (overlaps(h->out_row, h->out_head, tokens, h->heads, dim))
      return fail(HQ_ERR_SHAPE, "%s: strides %lld, %lld make rows or heads of Out overlap", name, (long long)h->out_row, (long long)h->out_head);
    if (h->Out == h->In && ((tokens > 1 && h->out_row != h->in_row) || (h->heads > 1 && h->out_head != h->in_head)))
      return fail(HQ_ERR_SHAPE, "%s: Out is In with other strides", name);
  }
  *to = {static_cast<const uint16_t*>(h->In), static_cast<uint16_t*>(h->Out), h->in_row, h->in_head, h->out_row, h->out_head, h->weight, h->heads, h->eps};
  return HQ_OK;
}

hq_status check_rotated(uint32_t tokens, const hq::RotaryArgs& a) {
  if (tokens == 0 || tokens > (1u << 24) || (uint64_t)tokens * a.all > (1u << 30))
    return fail(HQ_ERR_SHAPE, "tokens=%u of %u heads: out of range for one call", tokens, a.all);
  return HQ_OK;
}

}  // namespace

extern "C" {

hq_status hq_attn_workspace_bytes(hq_attn_kind kind, uint32_t rows, uint32_t seqs, uint32_t groups, uint32_t heads,
                                  uint32_t kv_heads, uint32_t head_dim, uint32_t max_keys, uint32_t max_prefix, size_t* bytes) {
  if (!bytes) return fail(HQ_ERR_INVALID_ARG, "bytes is null");
  hq_status st = check_query(kind, rows, seqs, groups, heads, kv_heads, head_dim, max_keys);
  if (st != HQ_OK) return st;
  const hq::AttnPlan p = hq::plan_attn(kind, rows, seqs, groups, heads, kv_heads, head_dim, max_keys, max_prefix);
  if ((st = check_plan(p)) != HQ_OK) return st;
  *bytes = p.need;
  return hq_set_error(HQ_OK, "");
}

hq_status hq_describe_attn(hq_attn_kind kind, uint32_t rows, uint32_t seqs, uint32_t groups, uint32_t heads, uint32_t kv_heads,
                           uint32_t head_dim, uint32_t max_keys, uint32_t max_prefix, char* buf, size_t buf_len) {
  if (!buf || buf_len == 0) return fail(HQ_ERR_INVALID_ARG, "buf is null or empty");
  hq_status st = check_query(kind, rows, seqs, groups, heads, kv_heads, head_dim, max_keys);
  if (st != HQ_OK) return st;
  const hq::AttnPlan p = hq::plan_attn(kind, rows, seqs, groups, heads, kv_heads, head_dim, max_keys, max_prefix);
  if ((st = check_plan(p)) != HQ_OK) return st;
  hq::describe_attn(p, buf, buf_len);
  return hq_set_error(HQ_OK, "");
}

hq_status hq_attn_prompt(const hq_attn_io* io, const void* K, int64_t k_row, int64_t k_head, const void* V, int64_t v_row,
                         int64_t v_head, uint32_t kv_heads, uint32_t total_k, const int32_t* cu_q, const int32_t* cu_k,
                         uint32_t seqs, int causal, uint32_t max_k, void* ws, size_t ws_bytes, hq_stream stream) {
  hq::AttnArgs a;
  hq_status st = check_io(io, seqs, kv_heads, &a);
  if (st != HQ_OK) return st;
  if (total_k > 0 && (!K || !V)) return fail(HQ_ERR_INVALID_ARG, "K or V is null");
  if (misaligned(K, 16) || misaligned(V, 16)) return fail(HQ_ERR_ALIGNMENT, "K and V must be 16-byte aligned");
  if ((st = check_list("cu_q", cu_q)) != HQ_OK) return st;
  if (misaligned(cu_k, 4)) return fail(HQ_ERR_ALIGNMENT, "cu_k must be 4-byte aligned");
  if (total_k > (1u << 30)) return fail(HQ_ERR_SHAPE, "total_k=%u: too many keys", total_k);
  if (!cu_k && total_k < io->rows) return fail(HQ_ERR_SHAPE, "total_k=%u: without cu_k there is a key for each of the %u rows", total_k, io->rows);
  if ((st = check_strides("K", k_row, k_head, total_k, kv_heads, io->head_dim)) != HQ_OK ||
      (st = check_strides("V", v_row, v_head, total_k, kv_heads, io->head_dim)) != HQ_OK)
    return st;
  if (k_row > kMaxRow || v_row > kMaxRow)
    return fail(HQ_ERR_SHAPE, "K, V: row strides %lld, %lld above %lld elements", (long long)k_row, (long long)v_row, (long long)kMaxRow);
  a.cu_q = cu_q;
  a.causal = causal != 0;
  a.k.K = static_cast<const uint16_t*>(K);
  a.k.V = static_cast<const uint16_t*>(V);
  a.k.k_row = total_k > 1 ? k_row : std::max<int64_t>(k_row, io->head_dim);  // a row's bytes bound its reads
  a.k.k_head = k_head;
  a.k.v_row = total_k > 1 ? v_row : std::max<int64_t>(v_row, io->head_dim);
  a.k.v_head = v_head;
  a.k.cu_k = cu_k ? cu_k : cu_q;
  a.k.total_k = total_k;
  return run_attn(a, HQ_ATTN_PROMPT, io->dtype, max_k && max_k < total_k ? max_k : total_k, 0, ws, ws_bytes, stream);
}

hq_status hq_attn_paged(const hq_attn_io* io, const hq_kv_cache* cache, uint32_t layer, const int32_t* rows, const int32_t* cu_q,
                        uint32_t seqs, uint32_t max_len, void* ws, size_t ws_bytes, hq_stream stream) {
  hq::AttnArgs a;
  const hq_status st = cache_keys(io, cache, layer, rows, seqs, &a);
  if (st != HQ_OK) return st;
  if (misaligned(cu_q, 4)) return fail(HQ_ERR_ALIGNMENT, "cu_q must be 4-byte aligned");
  if (!cu_q && io->rows != seqs) return fail(HQ_ERR_SHAPE, "rows=%u: without cu_q there is one for each of the %u sequences", io->rows, seqs);
  a.cu_q = cu_q;
  a.causal = 1;
  const uint32_t cap = capacity(cache);
  return run_attn(a, HQ_ATTN_PAGED, io->dtype, max_len && max_len < cap ? max_len : cap, 0, ws, ws_bytes, stream);
}

hq_status hq_attn_shared_prefix(const hq_attn_io* io, const hq_kv_cache* cache, uint32_t layer, const int32_t* rows, uint32_t seqs,
                                const int32_t* starts, const int32_t* prefix_lens, uint32_t groups, uint32_t max_prefix,
                                uint32_t max_len, void* ws, size_t ws_bytes, hq_stream stream) {
  hq::AttnArgs a;
  hq_status st = cache_keys(io, cache, layer, rows, seqs, &a);
  if (st != HQ_OK) return st;
  if (io->rows != seqs) return fail(HQ_ERR_SHAPE, "rows=%u: one for each of the %u sequences", io->rows, seqs);
  if ((st = check_list("starts", starts)) != HQ_OK || (st = check_list("prefix_lens", prefix_lens)) != HQ_OK) return st;
  if (groups == 0 || groups > seqs) return fail(HQ_ERR_SHAPE, "groups=%u must be 1..%u", groups, seqs);
  a.causal = 1;
  a.starts = starts;
  a.prefix = prefix_lens;
  a.groups = groups;
  const uint32_t cap = capacity(cache), most = max_len && max_len < cap ? max_len : cap;
  return run_attn(a, HQ_ATTN_SHARED, io->dtype, most, max_prefix, ws, ws_bytes, stream);
}

hq_status hq_cache_workspace_bytes(const hq_kv_cache* cache, size_t* bytes) {
  if (!bytes) return fail(HQ_ERR_INVALID_ARG, "bytes is null");
  hq::CacheArgs c;
  const hq_status st = check_cache(cache, &c);
  if (st != HQ_OK) return st;
  *bytes = std::max(hq::cache_fork_bytes(), hq::cache_compact_bytes(c.pages));
  return hq_set_error(HQ_OK, "");
}

hq_status hq_cache_reserve(const hq_kv_cache* cache, const int32_t* rows, const int32_t* counts, uint32_t n, hq_stream stream) {
  hq::CacheArgs c;
  hq_status st;
  if ((st = check_cache(cache, &c)) != HQ_OK || (st = check_batch(n)) != HQ_OK || (st = check_list("rows", rows)) != HQ_OK ||
      (st = check_list("counts", counts)) != HQ_OK)
    return st;
  if (!c.refused) return fail(HQ_ERR_INVALID_ARG, "cache: refused is null");
  return from_hip(hq::launch_cache_reserve(c, rows, counts, n, reinterpret_cast<hipStream_t>(stream)), "reserve launch");
}

hq_status hq_cache_append(const hq_kv_cache* cache, uint32_t layer, const void* K, int64_t k_row, int64_t k_head, const void* V,
                          int64_t v_row, int64_t v_head, uint32_t tokens, const int32_t* rows, const int32_t* cu, uint32_t n,
                          hq_stream stream) {
  hq::CacheArgs c;
  hq_status st;
  if ((st = check_cache(cache, &c)) != HQ_OK || (st = check_batch(n)) != HQ_OK || (st = check_list("rows", rows)) != HQ_OK) return st;
  if (misaligned(cu, 4)) return fail(HQ_ERR_ALIGNMENT, "cu must be 4-byte aligned");
  if (!K || !V) return fail(HQ_ERR_INVALID_ARG, "K or V is null");
  if (misaligned(K, 16) || misaligned(V, 16)) return fail(HQ_ERR_ALIGNMENT, "K and V must be 16-byte aligned");
  if (layer >= c.layers) return fail(HQ_ERR_SHAPE, "layer=%u of %u", layer, c.layers);
  if (tokens == 0 || tokens > (1u << 24)) return fail(HQ_ERR_SHAPE, "tokens=%u out of range", tokens);
  if (!cu && tokens != n) return fail(HQ_ERR_SHAPE, "tokens=%u: without cu there is one for each of the %u rows", tokens, n);
  if ((st = check_strides("K", k_row, k_head, tokens, c.kv_heads, c.dim)) != HQ_OK ||
      (st = check_strides("V", v_row, v_head, tokens, c.kv_heads, c.dim)) != HQ_OK)
    return st;
  if ((uint64_t)tokens * c.kv_heads * (c.dim / 8) > 256 * hq::kMaxGrid)
    return fail(HQ_ERR_SHAPE, "tokens=%u of %u heads of %u: too many for one call", tokens, c.kv_heads, c.dim);
  if (!c.refused) return fail(HQ_ERR_INVALID_ARG, "cache: refused is null");
  return from_hip(hq::launch_cache_append(c, layer, static_cast<const uint16_t*>(K), k_row, k_head, static_cast<const uint16_t*>(V), v_row,
                                          v_head, tokens, rows, cu, n, reinterpret_cast<hipStream_t>(stream)),
                  "append launch");
}

hq_status hq_cache_fork(const hq_kv_cache* cache, const int32_t* parents, const int32_t* children, uint32_t n, void* ws,
                        size_t ws_bytes, hq_stream stream) {
  hq::CacheArgs c;
  hq_status st;
  if ((st = check_cache(cache, &c)) != HQ_OK || (st = check_batch(n)) != HQ_OK || (st = check_list("parents", parents)) != HQ_OK ||
      (st = check_list("children", children)) != HQ_OK)
    return st;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void* w = nullptr;
  if ((st = workspace(ws, ws_bytes, hq::cache_fork_bytes(), hq::cache_fork_bytes(), s, &w)) != HQ_OK) return st;
  return from_hip(hq::launch_cache_fork(c, parents, children, n, w, s), "fork launch");
}

hq_status hq_cache_free(const hq_kv_cache* cache, const int32_t* rows, uint32_t n, hq_stream stream) {
  hq::CacheArgs c;
  hq_status st;
  if ((st = check_cache(cache, &c)) != HQ_OK || (st = check_batch(n)) != HQ_OK || (st = check_list("rows", rows)) != HQ_OK) return st;
  return from_hip(hq::launch_cache_free(c, rows, n, reinterpret_cast<hipStream_t>(stream)), "free launch");
}

hq_status hq_cache_copy_pages(const hq_kv_cache* cache, const int32_t* src, const int32_t* dst, uint32_t n, hq_stream stream) {
  hq::CacheArgs c;
  hq_status st;
  if ((st = check_cache(cache, &c)) != HQ_OK || (st = check_batch(n)) != HQ_OK || (st = check_list("src", src)) != HQ_OK ||
      (st = check_list("dst", dst)) != HQ_OK)
    return st;
  return from_hip(hq::launch_cache_copy(c, src, dst, n, reinterpret_cast<hipStream_t>(stream)), "copy launch");
}

hq_status hq_cache_compact(const hq_kv_cache* cache, int32_t* out_table, int64_t out_stride, int32_t* out_refs, void* ws,
                           size_t ws_bytes, hq_stream stream) {
  hq::CacheArgs c;
  hq_status st;
  if ((st = check_cache(cache, &c)) != HQ_OK || (st = check_list("out_table", out_table)) != HQ_OK ||
      (st = check_list("out_refs", out_refs)) != HQ_OK)
    return st;
  if (out_stride < (int64_t)c.max_pages || out_stride > (1 << 30))
    return fail(HQ_ERR_SHAPE, "out_stride=%lld out of range (max_pages=%u)", (long long)out_stride, c.max_pages);
  if (out_table == c.table && out_stride != c.table_stride) return fail(HQ_ERR_SHAPE, "out_table is the cache's own with another stride");
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  void* w = nullptr;
  const size_t need = hq::cache_compact_bytes(c.pages);
  if ((st = workspace(ws, ws_bytes, need, need, s, &w)) != HQ_OK) return st;
  return from_hip(hq::launch_cache_compact(c, out_table, out_stride, out_refs, w, s), "compact launch");
}

hq_status hq_rotate(const hq_rotary* rotary, const hq_rotary_heads* q, const hq_rotary_heads* k, uint32_t tokens, uint32_t head_dim,
                    hq_dtype dtype, const int32_t* positions, hq_stream stream) {
  hq::RotaryArgs a{};
  hq_status st;
  if (!q) return fail(HQ_ERR_INVALID_ARG, "q is null");
  if ((st = check_dtype(dtype)) != HQ_OK || (st = check_dim(head_dim)) != HQ_OK || (st = check_rotary(rotary, head_dim, &a)) != HQ_OK ||
      (st = check_heads("q", q, tokens, head_dim, true, &a.q)) != HQ_OK ||
      (k && (st = check_heads("k", k, tokens, head_dim, true, &a.k)) != HQ_OK) || (st = check_list("positions", positions)) != HQ_OK)
    return st;
  a.T = tokens;
  a.D = head_dim;
  a.all = a.q.heads + a.k.heads;
  a.pos = positions;
  if ((st = check_rotated(tokens, a)) != HQ_OK) return st;
  if (k && (q->Out == k->Out || q->Out == k->In || k->Out == q->In))
    return fail(HQ_ERR_INVALID_ARG, "an Out of q or k is the other's: heads are written while others read them");
  return from_hip(hq::launch_rotate(dtype, rotary->layout, a, nullptr, reinterpret_cast<hipStream_t>(stream)), "rotation launch");
}

hq_status hq_cache_append_rotated(const hq_kv_cache* cache, uint32_t layer, const hq_rotary* rotary, const hq_rotary_heads* q,
                                  const hq_rotary_heads* k, const void* V, int64_t v_row, int64_t v_head, uint32_t tokens,
                                  const int32_t* rows, const int32_t* cu, uint32_t n, hq_stream stream) {
  hq::CacheArgs c;
  hq::RotaryArgs a{};
  hq_status st;
  if ((st = check_cache(cache, &c)) != HQ_OK || (st = check_batch(n)) != HQ_OK || (st = check_list("rows", rows)) != HQ_OK) return st;
  if (misaligned(cu, 4)) return fail(HQ_ERR_ALIGNMENT, "cu must be 4-byte aligned");
  if (!k || !V) return fail(HQ_ERR_INVALID_ARG, "k or V is null");
  if (misaligned(V, 16)) return fail(HQ_ERR_ALIGNMENT, "V must be 16-byte aligned");
  if (layer >= c.layers) return fail(HQ_ERR_SHAPE, "layer=%u of %u", layer, c.layers);
  if (!cu && tokens != n) return fail(HQ_ERR_SHAPE, "tokens=%u: without cu there is one for each of the %u rows", tokens, n);
  if (!c.refused) return fail(HQ_ERR_INVALID_ARG, "cache: refused is null");
  if ((st = check_rotary(rotary, c.dim, &a)) != HQ_OK || (q && (st = check_heads("q", q, tokens, c.dim, true, &a.q)) != HQ_OK) ||
      (st = check_heads("k", k, tokens, c.dim, false, &a.k)) != HQ_OK ||
      (st = check_strides("V", v_row, v_head, tokens, c.kv_heads, c.dim)) != HQ_OK)
    return st;
  if (k->heads != c.kv_heads) return fail(HQ_ERR_SHAPE, "k has %u heads, the cache %u", k->heads, c.kv_heads);
  a.V = static_cast<const uint16_t*>(V);
  a.v_row = v_row;
  a.v_head = v_head;
  a.T = tokens;
  a.D = c.dim;
  a.all = a.q.heads + 2 * a.k.heads;
  a.rows = rows;
  a.cu = cu;
  a.n = n;
  if ((st = check_rotated(tokens, a)) != HQ_OK) return st;
  if (q && (q->Out == k->In || q->Out == V)) return fail(HQ_ERR_INVALID_ARG, "q's Out is k or V: heads are written while others read them");
  c.K += layer * c.layer_stride;
  c.V += layer * c.layer_stride;
  return from_hip(hq::launch_rotate(cache->dtype, rotary->layout, a, &c, reinterpret_cast<hipStream_t>(stream)), "rotated append launch");
}

}  // extern "C"
