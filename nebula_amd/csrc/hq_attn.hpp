// hq_attn.hpp — descriptors shared by the attention and cache entry points and their kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hq_attn.h"

namespace hq {

// The keys of a call: rows of packed K and V (table == null), or pages.
struct AttnKeys {
  const uint16_t* K;
  const uint16_t* V;
  int64_t k_row, k_head, v_row, v_head;  // elements; paged: token and head strides inside a page
  int64_t page_stride;
  const int32_t* cu_k;   // packed: [B + 1]
  uint32_t total_k;
  const int32_t* table;  // paged: the cache's
  int64_t table_stride;
  const int32_t* lens;
  const int32_t* rows;   // cache row of sequence b, or null (row b)
  uint32_t cache_rows, max_pages, pages, page_shift;
  uint32_t* status;
};

struct AttnArgs {
  const uint16_t* Q;
  uint16_t* O;
  float* lse;
  int64_t q_row, q_head, o_row, o_head;
  uint32_t T, H, Hkv, G, D;  // tokens, query heads, key/value heads, H / Hkv, head_dim
  float scale;
  uint32_t B;
  const int32_t* cu_q;       // [B + 1], or null: token b is sequence b's
  uint32_t causal;
  AttnKeys k;
  // Shared prefixes: sequences [starts[g], starts[g + 1]) share prefix[g] tokens.
  const int32_t* starts;
  const int32_t* prefix;
  uint32_t groups;
};

// How a call is split, from host-side sizes alone (the lengths stay on the device).
struct AttnPlan {
  bool tile = false, row = false;  // the kernels that run
  bool prefix = false;             // both in one launch: tiles of many rows over shared prefixes, of few over the rest
  uint32_t tile_grid = 0, tile_splits = 0;
  uint32_t row_grid = 0;
  uint32_t row_slots = 0, row_one = 0, row_like = 0;  // workgroups of a kv head that share rows' keys (0: none share), keys of a row past its prefix
  uint32_t parts = 0;              // parts of a row that are joined by a launch of their own (0: rows are written out)
  size_t part_ml = 0, part_o = 0, row_ml = 0, row_o = 0, ws = 0;  // workspace offsets, and its size
  uint64_t largest = 0;            // workgroups of its largest launch
  size_t need = 0;                 // not falling in the keys: what calls of fewer keys need at most, and this one
};
// A launch has fewer than 2^32 threads in a grid's dimension; all here have 256 a workgroup.
constexpr uint64_t kMaxGrid = 0xFFFFFFFFu / 256u;
// max_prefix: 0, where it is not known.
AttnPlan plan_attn(int kind, uint32_t rows, uint32_t seqs, uint32_t groups, uint32_t heads, uint32_t kv_heads,
                   uint32_t dim, uint32_t max_keys, uint32_t max_prefix);
void describe_attn(const AttnPlan& p, char* buf, size_t len);
hipError_t launch_attn(int dtype, const AttnArgs& a, const AttnPlan& p, void* ws, hipStream_t stream);

// A page of one layer, K or V, as `runs` pieces of `run` consecutive elements per token count:
// heads before tokens: kv_heads pieces, head_stride apart, of tokens * head_dim; tokens before
// heads: one piece of tokens * kv_heads * head_dim.
struct PageShape {
  uint32_t runs;
  uint32_t per_token;   // elements of one token in a piece
  int64_t run_stride;
};

struct CacheArgs {
  uint16_t* K;
  uint16_t* V;
  int64_t layer_stride, page_stride, head_stride, token_stride;
  uint32_t layers, pages, kv_heads, page_shift, dim;
  int32_t* table;
  int64_t table_stride;
  uint32_t rows, max_pages;
  int32_t* lens;
  int32_t* refs;
  uint32_t* status;
  int32_t* refused;  // rows that the last reserve was refused for
  PageShape shape;
};

size_t cache_fork_bytes();
size_t cache_compact_bytes(uint32_t pages);
hipError_t launch_cache_reserve(const CacheArgs& c, const int32_t* rows, const int32_t* counts, uint32_t n, hipStream_t s);
hipError_t launch_cache_append(const CacheArgs& c, uint32_t layer, const uint16_t* K, int64_t k_row, int64_t k_head,
                               const uint16_t* V, int64_t v_row, int64_t v_head, uint32_t tokens, const int32_t* rows,
                               const int32_t* cu, uint32_t n, hipStream_t s);
hipError_t launch_cache_fork(const CacheArgs& c, const int32_t* parents, const int32_t* children, uint32_t n, void* ws,
                             hipStream_t s);
hipError_t launch_cache_free(const CacheArgs& c, const int32_t* rows, uint32_t n, hipStream_t s);
hipError_t launch_cache_copy(const CacheArgs& c, const int32_t* src, const int32_t* dst, uint32_t n, hipStream_t s);
hipError_t launch_cache_compact(const CacheArgs& c, int32_t* out_table, int64_t out_stride, int32_t* out_refs, void* ws,
                                hipStream_t s);

}  // namespace hq
