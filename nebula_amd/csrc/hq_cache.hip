// hq_cache.hip — page keeping of the key/value cache (include/hq_attn.h): reserve, append, fork,
// free, copy, compact.
//
// The state is the table, the lengths and a count per page; there is no list of free pages. A page is
// free when its count is zero, and new pages are the lowest free numbers, found by a scan over the
// counts, so what a call does follows from the state alone and not from the order in which
// workgroups or earlier calls ran. What has to be decided at one place (which pages a call takes,
// where compaction moves them) is one workgroup's work; pages are moved by a grid of their own.
//
// Bound by the bytes moved, read and written once. On an MI355X, replayed from a graph: append of 80 tokens to 8 heads of
// 128 2.8 us, reserve for 80 rows of a pool of 5000 pages 6.0; a fork of 32 children (88 MB of part-filled pages) 5 us of
// planning and 15 to 17 of copies; 128 pages of 16 layers copied (1.07 GB) 197, 5.4 TB/s; compaction of 1.03 GB 5 us of planning and
// 207 to 233 of copies, 4.4 to 5 TB/s, a large copy's rate.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "hq_attn.hpp"
#include "hq_device.hpp"
#include "hq_internal.hpp"

namespace hq {
namespace {

constexpr uint32_t kPlanThreads = 1024;  // of the one workgroup that decides
constexpr uint32_t kCopyThreads = 256;
constexpr uint32_t kUnitBytes = 16384;   // what one workgroup copies at a time: four 16-byte loads a thread in flight

__device__ __forceinline__ void report(uint32_t* status, uint32_t what) {
  __hip_atomic_fetch_or(status, what, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive sum over the workgroup's threads and their total; sh: 17 words. Barriers on both sides,
// so calls may follow each other.
__device__ uint32_t block_scan(uint32_t v, uint32_t* sh, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t x = scan_sum(v);
  __syncthreads();
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
    const uint32_t s = sh[w];
    before += w < wave ? s : 0u;
    all += s;
  }
  total = all;
  return before + x - v;
}

// Counts of pages 4 i .. 4 i + 3 (1, not free, past the pool's end).
__device__ __forceinline__ void four_refs(const int32_t* refs, uint32_t i, uint32_t pages, int32_t (&r)[4]) {
#pragma unroll
  for (uint32_t e = 0; e < 4; ++e) r[e] = 4 * i + e < pages ? refs[4 * i + e] : 1;
}

// The pool's free pages, the first 4096 pages' counts in registers: they are on their way while the call's
// lists are checked, and most calls need no others. A fork's plan takes 5.1 us so, and took 6.8 with each load
// after the last.
struct FreePages {
  int32_t r[4];
  uint32_t rank, total;  // free pages below this thread's four, and among all of them

  __device__ __forceinline__ void look(const CacheArgs& c) { four_refs(c.refs, threadIdx.x, c.pages, r); }
  __device__ __forceinline__ static uint32_t free_of(const int32_t (&r)[4]) {
    return (r[0] == 0) + (r[1] == 0) + (r[2] == 0) + (r[3] == 0);
  }
  // Whether there are `need`; stops as soon as there are.
  __device__ bool enough(const CacheArgs& c, uint32_t need, uint32_t* sh) {
    rank = block_scan(free_of(r), sh, total);
    uint32_t found = total;
    for (uint32_t base = 4 * kPlanThreads; base < c.pages && found < need; base += 4 * kPlanThreads) {
      int32_t q[4];
      four_refs(c.refs, base / 4 + threadIdx.x, c.pages, q);
      uint32_t more;
      block_scan(free_of(q), sh, more);
      found += more;
    }
    return found >= need;
  }
  // Calls give(rank, page) for the `need` lowest; after enough().
  template <class F>
  __device__ void take(const CacheArgs& c, uint32_t need, uint32_t* sh, F give) const {
    auto some = [&](const int32_t (&q)[4], uint32_t base, uint32_t at) {
      for (uint32_t e = 0; e < 4; ++e)
        if (q[e] == 0) {
          if (at < need) give(at, base + 4 * threadIdx.x + e);
          ++at;
        }
    };
    some(r, 0, rank);
    uint32_t found = total;
    for (uint32_t base = 4 * kPlanThreads; base < c.pages && found < need; base += 4 * kPlanThreads) {
      int32_t q[4];
      four_refs(c.refs, base / 4 + threadIdx.x, c.pages, q);
      uint32_t more;
      const uint32_t at = block_scan(free_of(q), sh, more);
      some(q, base, found + at);
      found += more;
    }
  }
};

// off[i] <= r < off[i + 1], off not falling over n + 1 entries.
__device__ __forceinline__ uint32_t owner(const uint32_t* off, uint32_t n, uint32_t r) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (off[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t pages_of(int32_t len, uint32_t shift) {
  return len > 0 ? (uint32_t)(((uint64_t)len + (1ull << shift) - 1) >> shift) : 0u;
}

// Whether list[i] appears before place i (a row named twice).
__device__ __forceinline__ bool repeated(const int32_t* list, uint32_t i) {
  const int32_t r = list[i];
  bool hit = false;
  for (uint32_t j = 0; j < i; ++j) hit |= list[j] == r;
  return hit;
}

__global__ __launch_bounds__(kPlanThreads) void hq_cache_reserve_kernel(CacheArgs c, const int32_t* rows, const int32_t* counts,
                                                                        uint32_t n) {
  __shared__ uint32_t sh[kPlanThreads / 64 + 1], off[HQ_CACHE_MAX_BATCH + 1], first[HQ_CACHE_MAX_BATCH], fault;
  __shared__ int32_t list[HQ_CACHE_MAX_BATCH];
  const uint32_t i = threadIdx.x;
  if (i == 0) fault = 0;
  list[i] = i < n ? rows[i] : -1;
  int32_t len = 0, more = i < n ? counts[i] : 0;
  FreePages pool;
  pool.look(c);
  __syncthreads();
  const int32_t row = list[i];
  uint32_t add = 0, bad = 0;
  if (i < n) {
    if (row < 0 || row >= (int32_t)c.rows || more < 0 || repeated(list, i)) {
      bad = HQ_CACHE_BAD_ROW;
    } else {
      len = c.lens[row];
      const uint64_t want = (uint64_t)(uint32_t)(len < 0 ? 0 : len) + (uint32_t)more;
      if (len < 0) bad = HQ_CACHE_BAD_ROW;
      else if (want > (uint64_t)c.max_pages << c.page_shift) bad = HQ_CACHE_ROW_FULL;
      else {
        first[i] = pages_of(len, c.page_shift);
        // More than the pool has is refused below; capped, the 1024 rows' sum stays inside 32 bits.
        add = min(pages_of((int32_t)want, c.page_shift) - first[i], c.pages + 1);
      }
    }
    if (bad) atomicOr(&fault, bad);
  }
  uint32_t need;
  const uint32_t at = block_scan(add, sh, need);
  if (i < n) off[i] = at;
  if (i == 0) off[n] = need;
  __syncthreads();
  bad = fault;
  if (!bad && !pool.enough(c, need, sh)) bad = HQ_CACHE_NO_PAGES;
  if (bad) {
    if (i == 0) report(c.status, bad);
    // What is appended to these rows before a reserve goes through would lie over their last tokens.
    if (i < n && row >= 0 && row < (int32_t)c.rows) c.refused[row] = 1;
    return;
  }
  pool.take(c, need, sh, [&](uint32_t r, uint32_t page) {
    const uint32_t j = owner(off, n, r);
    c.table[(int64_t)list[j] * c.table_stride + first[j] + (r - off[j])] = (int32_t)page;
    c.refs[page] = 1;
  });
  if (i < n) {
    c.lens[row] = len + more;
    c.refused[row] = 0;
  }
}

// One 16-byte piece per thread: (token, head, piece of the head).
__global__ __launch_bounds__(kCopyThreads) void hq_cache_append_kernel(CacheArgs c, const uint16_t* K, int64_t k_row, int64_t k_head,
                                                                       const uint16_t* V, int64_t v_row, int64_t v_head,
                                                                       uint32_t tokens, const int32_t* rows, const int32_t* cu,
                                                                       uint32_t n) {
  const uint32_t per_head = c.dim / 8, per_token = c.kv_heads * per_head;
  const uint64_t u = (uint64_t)blockIdx.x * kCopyThreads + threadIdx.x;
  const uint32_t t = (uint32_t)(u / per_token), p = (uint32_t)(u % per_token);
  if (t >= tokens) return;
  // The source is on its way beside the chain list - row - length - page - holders.
  const uint32_t h = p / per_head, e = (p % per_head) * 8;
  const u4 k = *reinterpret_cast<const u4*>(K + t * k_row + h * k_head + e), v = *reinterpret_cast<const u4*>(V + t * v_row + h * v_head + e);
  uint32_t i = t, back = 1;  // sequence, tokens from its end
  if (cu) {
    // The last sequence that begins at or before t; it holds t if it does not end before it.
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if ((uint32_t)cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    i = lo;
    const int32_t a = cu[i], b = cu[i + 1];
    if ((int32_t)t < a || (int32_t)t >= b) return;  // of no sequence
    back = (uint32_t)b - t;
  }
  const int32_t row = rows[i];
  if (row < 0 || row >= (int32_t)c.rows) {
    report(c.status, HQ_CACHE_BAD_ROW);
    return;
  }
  const int64_t at = (int64_t)c.lens[row] - back;
  if (c.refused[row] || at < 0 || at >= (int64_t)c.max_pages << c.page_shift) {
    report(c.status, HQ_CACHE_BAD_ROW);
    return;
  }
  const uint32_t page = (uint32_t)c.table[row * c.table_stride + (at >> c.page_shift)];
  if (page >= c.pages || c.refs[page] > 1) {
    report(c.status, HQ_CACHE_BAD_PAGE);
    return;
  }
  const int64_t to = page * c.page_stride + h * c.head_stride + (at & ((1 << c.page_shift) - 1)) * c.token_stride + e;
  *reinterpret_cast<u4*>(c.K + to) = k;
  *reinterpret_cast<u4*>(c.V + to) = v;
}

// Units of kUnitBytes that `tokens` tokens of a page hold.
__host__ __device__ inline uint32_t units_of(const PageShape& p, uint32_t tokens) {
  const uint64_t bytes = (uint64_t)p.runs * p.per_token * tokens * 2;
  return (uint32_t)((bytes + kUnitBytes - 1) / kUnitBytes);
}

// Unit u of the first `tokens` tokens of page src onto page dst, one pool and layer (base). Four loads
// of 16 bytes are in flight per thread before the stores.
__device__ __forceinline__ void copy_unit(uint16_t* base, const CacheArgs& c, uint32_t src, uint32_t dst, uint32_t tokens, uint32_t u) {
  const uint32_t run = c.shape.per_token / 8 * tokens, n = run * c.shape.runs;  // 16-byte pieces
  const uint16_t* s = base + src * c.page_stride;
  uint16_t* d = base + dst * c.page_stride;
  constexpr uint32_t kPieces = kUnitBytes / 16;
  u4 v[kPieces / kCopyThreads];
  int64_t o[kPieces / kCopyThreads];
#pragma unroll
  for (uint32_t k = 0; k < kPieces / kCopyThreads; ++k) {
    const uint32_t i = u * kPieces + k * kCopyThreads + threadIdx.x;
    const uint32_t r = c.shape.runs == 1 ? 0u : i / run;
    o[k] = i < n ? r * c.shape.run_stride + (int64_t)(i - r * run) * 8 : -1;
    if (o[k] >= 0) v[k] = *reinterpret_cast<const u4*>(s + o[k]);
  }
#pragma unroll
  for (uint32_t k = 0; k < kPieces / kCopyThreads; ++k)
    if (o[k] >= 0) *reinterpret_cast<u4*>(d + o[k]) = v[k];
}

// What fork decided, then per child the page of its part-filled end (or -1) and the parent's.
enum : uint32_t { kForkNone = 0, kForkAll = 1, kForkUndo = 2 };  // kForkUndo: some full page is bad, pages were taken
struct ForkPlan {
  uint32_t ok, pad[3];
  int2 tail[HQ_CACHE_MAX_BATCH];  // (from, to), (-1, -1): the parent ends with a full page
};

// Workgroup 0 plans; 1 + i looks over the full pages of parents[i] beside it (in the planning workgroup they took 3 us of 24
// at 32 children of 4 parents). cnt: their arrivals, 2^16 for each that met a bad number, 2^28 for a plan that
// refuses; the last one has the answer. Zero between calls.
__device__ __forceinline__ void fork_arrive(ForkPlan* plan, uint32_t* cnt, uint32_t add, uint32_t n) {
  const uint32_t sum = __hip_atomic_fetch_add(cnt, add + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + add + 1;
  if ((sum & 0xFFFFu) != n + 1) return;
  plan->ok = sum >> 28 ? kForkNone : sum >> 16 ? kForkUndo : kForkAll;
  __hip_atomic_store(cnt, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__global__ __launch_bounds__(kPlanThreads) void hq_cache_fork_plan_kernel(CacheArgs c, const int32_t* parents, const int32_t* children,
                                                                          uint32_t n, ForkPlan* plan, uint32_t* cnt) {
  if (blockIdx.x > 0) {
    const int32_t row = parents[blockIdx.x - 1];
    bool odd = false;
    if (row >= 0 && row < (int32_t)c.rows) {
      const int32_t len = c.lens[row];
      const uint32_t full = len > 0 ? min((uint32_t)len >> c.page_shift, c.max_pages) : 0u;
      for (uint32_t j = threadIdx.x; j < full; j += kPlanThreads) odd |= (uint32_t)c.table[row * c.table_stride + j] >= c.pages;
    }
    odd = __syncthreads_or(odd);
    if (threadIdx.x == 0) fork_arrive(plan, cnt, odd ? 1u << 16 : 0u, n);
    return;
  }
  __shared__ uint32_t sh[kPlanThreads / 64 + 1], fault;
  __shared__ int32_t list[HQ_CACHE_MAX_BATCH];
  __shared__ uint16_t who[HQ_CACHE_MAX_BATCH];
  const uint32_t i = threadIdx.x;
  if (i == 0) fault = 0;
  const int32_t k = i < n ? children[i] : -1, p = i < n ? parents[i] : -1;
  const bool rows = p >= 0 && p < (int32_t)c.rows && k >= 0 && k < (int32_t)c.rows;
  const int32_t len = rows ? c.lens[p] : 0, own = rows ? c.lens[k] : 0;
  FreePages pool;
  pool.look(c);
  list[i] = k;
  __syncthreads();
  uint32_t part = 0, bad = 0;
  int32_t from = -1;
  if (i < n) {
    bool both = false;  // the parent is some child: its row is not what it will be
    for (uint32_t j = 0; j < n; ++j) both |= list[j] == p;
    if (!rows || both || repeated(list, i) || own != 0 || len < 0) bad = HQ_CACHE_BAD_ROW;
    else {
      if (pages_of(len, c.page_shift) > c.max_pages) bad = HQ_CACHE_BAD_ROW;
      else if (len & ((1 << c.page_shift) - 1)) {
        part = 1;
        from = c.table[p * c.table_stride + (len >> c.page_shift)];
        if ((uint32_t)from >= c.pages) bad = HQ_CACHE_BAD_PAGE;
      }
    }
    if (bad) atomicOr(&fault, bad);
  }
  uint32_t need;
  const uint32_t at = block_scan(part, sh, need);
  if (part) who[at] = (uint16_t)i;
  if (i < n) plan->tail[i] = make_int2(from, -1);
  __syncthreads();
  bad = fault;
  if (!bad && !pool.enough(c, need, sh)) bad = HQ_CACHE_NO_PAGES;
  if (i == 0) fork_arrive(plan, cnt, bad ? 1u << 28 : 0u, n);
  if (bad) {
    if (i == 0) report(c.status, bad);
    return;
  }
  pool.take(c, need, sh, [&](uint32_t r, uint32_t page) {
    plan->tail[who[r]].y = (int32_t)page;
    c.refs[page] = 1;
  });
}

// Workgroup (x, child): x = 0 its row of the table, its length and the counts of the shared pages; the
// others the part-filled page, a unit of one layer of one pool each.
__global__ __launch_bounds__(kCopyThreads) void hq_cache_fork_kernel(CacheArgs c, const int32_t* parents, const int32_t* children,
                                                                     const ForkPlan* plan, uint32_t units) {
  const uint32_t i = blockIdx.y, ok = plan->ok;
  if (ok == kForkNone) return;
  const int32_t p = parents[i], k = children[i], len = c.lens[p];
  const int2 tail = plan->tail[i];
  if (blockIdx.x == 0) {
    if (ok == kForkUndo) {  // (here and not before the loads: stores ahead of them made the copies 1 us slower)
      if (threadIdx.x == 0) {
        if (tail.y >= 0) c.refs[tail.y] = 0;
        if (i == 0) report(c.status, HQ_CACHE_BAD_PAGE);
      }
      return;
    }
    const uint32_t full = (uint32_t)len >> c.page_shift;
    const int32_t* from = c.table + p * c.table_stride;
    int32_t* to = c.table + k * c.table_stride;
    for (uint32_t j = threadIdx.x; j < c.max_pages; j += kCopyThreads) {
      int32_t page = j < full ? from[j] : j == full ? tail.y : -1;
      if (j < full) atomicAdd(c.refs + page, 1);
      to[j] = page;
    }
    if (threadIdx.x == 0) c.lens[k] = len;
    return;
  }
  if (tail.x < 0 || ok == kForkUndo) return;
  const uint32_t tokens = (uint32_t)len & ((1u << c.page_shift) - 1);
  const uint32_t x = blockIdx.x - 1, u = x % units, l = x / units;  // l: layer, then pool
  if (u >= units_of(c.shape, tokens)) return;
  uint16_t* pool = l & 1 ? c.V : c.K;
  copy_unit(pool + (l >> 1) * c.layer_stride, c, (uint32_t)tail.x, (uint32_t)tail.y, tokens, u);
}

__global__ __launch_bounds__(kCopyThreads) void hq_cache_free_kernel(CacheArgs c, const int32_t* rows) {
  __shared__ uint32_t twice;
  const uint32_t i = blockIdx.x;
  const int32_t row = rows[i];
  if (threadIdx.x == 0) twice = 0;
  __syncthreads();
  for (uint32_t j = threadIdx.x; j < i; j += kCopyThreads)
    if (rows[j] == row) twice = 1;
  __syncthreads();
  if (twice || row < 0 || row >= (int32_t)c.rows) {
    if (threadIdx.x == 0) report(c.status, HQ_CACHE_BAD_ROW);
    return;
  }
  const uint32_t n = min(pages_of(c.lens[row], c.page_shift), c.max_pages);
  int32_t* t = c.table + row * c.table_stride;
  for (uint32_t j = threadIdx.x; j < n; j += kCopyThreads) {
    const uint32_t page = (uint32_t)t[j];
    if (page >= c.pages) report(c.status, HQ_CACHE_BAD_PAGE);
    else if (atomicSub(c.refs + page, 1) <= 0) {
      atomicAdd(c.refs + page, 1);
      report(c.status, HQ_CACHE_BAD_PAGE);
    }
    t[j] = -1;
  }
  __syncthreads();
  if (threadIdx.x == 0) c.lens[row] = 0;
}

// Workgroup (unit of a layer and pool, pair).
__global__ __launch_bounds__(kCopyThreads) void hq_cache_copy_kernel(CacheArgs c, const int32_t* src, const int32_t* dst, uint32_t units) {
  const uint32_t s = (uint32_t)src[blockIdx.y], d = (uint32_t)dst[blockIdx.y];
  if (s >= c.pages || d >= c.pages) {
    if (threadIdx.x == 0 && blockIdx.x == 0) report(c.status, HQ_CACHE_BAD_PAGE);
    return;
  }
  const uint32_t u = blockIdx.x % units, l = blockIdx.x / units;
  copy_unit((l & 1 ? c.V : c.K) + (l >> 1) * c.layer_stride, c, s, d, 1u << c.page_shift, u);
}

// Compaction's plan in the workspace: the number of moves, where every page goes, and the moves.
struct CompactPlan {
  uint32_t moves, pad[3];
  // int32 to[pages], src[pages], dst[pages] follow
};

__global__ __launch_bounds__(kPlanThreads) void hq_cache_compact_plan_kernel(CacheArgs c, int32_t* out_refs, CompactPlan* plan) {
  __shared__ uint32_t sh[kPlanThreads / 64 + 1];
  int32_t* to = reinterpret_cast<int32_t*>(plan + 1);
  int32_t *src = to + c.pages, *dst = src + c.pages;
  uint32_t live = 0;
  for (uint32_t base = 0; base < c.pages; base += 4 * kPlanThreads) {
    int32_t r[4];
    four_refs(c.refs, base / 4 + threadIdx.x, c.pages, r);
    uint32_t n = 0, total;
    for (uint32_t e = 0; e < 4; ++e) n += r[e] > 0 && base + 4 * threadIdx.x + e < c.pages;
    block_scan(n, sh, total);
    live += total;
  }
  // The k-th live page at or past `live` and the k-th free one below it: as many of either.
  uint32_t movers = 0, holes = 0;
  for (uint32_t base = 0; base < c.pages; base += 4 * kPlanThreads) {
    int32_t r[4];
    four_refs(c.refs, base / 4 + threadIdx.x, c.pages, r);
    const uint32_t p0 = base + 4 * threadIdx.x;
    uint32_t nm = 0, nh = 0, all;
    for (uint32_t e = 0; e < 4; ++e) {
      const uint32_t p = p0 + e;
      nm += p < c.pages && p >= live && r[e] > 0;
      nh += p < live && r[e] <= 0;
    }
    const uint32_t rm = block_scan(nm, sh, all);
    uint32_t m = movers + rm;
    movers += all;
    const uint32_t rh = block_scan(nh, sh, all);
    uint32_t h = holes + rh;
    holes += all;
    for (uint32_t e = 0; e < 4; ++e) {
      const uint32_t p = p0 + e;
      if (p >= c.pages) break;
      if (p >= live && r[e] > 0) src[m++] = (int32_t)p;
      else if (p < live && r[e] <= 0) dst[h++] = (int32_t)p;
      to[p] = (int32_t)p;
      out_refs[p] = r[e];
    }
  }
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < movers; k += kPlanThreads) {
    const int32_t s = src[k], d = dst[k], r = c.refs[s];
    to[s] = d;
    out_refs[d] = r;
    out_refs[s] = 0;
  }
  if (threadIdx.x == 0) plan->moves = movers;
}

// The table by the plan, then the moves: units of pages over the whole grid.
__global__ __launch_bounds__(kCopyThreads) void hq_cache_compact_kernel(CacheArgs c, int32_t* out_table, int64_t out_stride,
                                                                        const CompactPlan* plan, uint32_t units) {
  const int32_t* to = reinterpret_cast<const int32_t*>(plan + 1);
  const int32_t *src = to + c.pages, *dst = src + c.pages;
  const uint64_t cells = (uint64_t)c.rows * c.max_pages;
  for (uint64_t i = (uint64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < cells; i += (uint64_t)gridDim.x * kCopyThreads) {
    const uint32_t row = (uint32_t)(i / c.max_pages), j = (uint32_t)(i % c.max_pages);
    const int32_t p = c.table[row * c.table_stride + j];
    out_table[row * out_stride + j] = (uint32_t)p < c.pages ? to[p] : p;
  }
  const uint32_t per_page = units * 2 * c.layers;
  const uint64_t all = (uint64_t)plan->moves * per_page;
  for (uint64_t i = blockIdx.x; i < all; i += gridDim.x) {
    const uint32_t m = (uint32_t)(i / per_page), x = (uint32_t)(i % per_page), u = x % units, l = x / units;
    copy_unit((l & 1 ? c.V : c.K) + (l >> 1) * c.layer_stride, c, (uint32_t)src[m], (uint32_t)dst[m], 1u << c.page_shift, u);
  }
}

void* scratch(void* ws) { return static_cast<unsigned char*>(ws) + kCounterBytes; }

}  // namespace

size_t cache_fork_bytes() { return kCounterBytes + sizeof(ForkPlan); }
size_t cache_compact_bytes(uint32_t pages) { return kCounterBytes + sizeof(CompactPlan) + (size_t)pages * 12u; }

hipError_t launch_cache_reserve(const CacheArgs& c, const int32_t* rows, const int32_t* counts, uint32_t n, hipStream_t s) {
  hipLaunchKernelGGL(hq_cache_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, s, c, rows, counts, n);
  return hipGetLastError();
}

hipError_t launch_cache_append(const CacheArgs& c, uint32_t layer, const uint16_t* K, int64_t k_row, int64_t k_head,
                               const uint16_t* V, int64_t v_row, int64_t v_head, uint32_t tokens, const int32_t* rows,
                               const int32_t* cu, uint32_t n, hipStream_t s) {
  CacheArgs l = c;
  l.K += layer * c.layer_stride;
  l.V += layer * c.layer_stride;
  const uint64_t pieces = (uint64_t)tokens * c.kv_heads * (c.dim / 8);
  hipLaunchKernelGGL(hq_cache_append_kernel, dim3((uint32_t)((pieces + kCopyThreads - 1) / kCopyThreads)), dim3(kCopyThreads), 0, s, l, K,
                     k_row, k_head, V, v_row, v_head, tokens, rows, cu, n);
  return hipGetLastError();
}

hipError_t launch_cache_fork(const CacheArgs& c, const int32_t* parents, const int32_t* children, uint32_t n, void* ws, hipStream_t s) {
  ForkPlan* plan = static_cast<ForkPlan*>(scratch(ws));
  hipLaunchKernelGGL(hq_cache_fork_plan_kernel, dim3(1 + n), dim3(kPlanThreads), 0, s, c, parents, children, n, plan,
                     static_cast<uint32_t*>(ws));
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t units = units_of(c.shape, 1u << c.page_shift);
  hipLaunchKernelGGL(hq_cache_fork_kernel, dim3(1 + units * 2 * c.layers, n), dim3(kCopyThreads), 0, s, c, parents, children, plan, units);
  return hipGetLastError();
}

hipError_t launch_cache_free(const CacheArgs& c, const int32_t* rows, uint32_t n, hipStream_t s) {
  hipLaunchKernelGGL(hq_cache_free_kernel, dim3(n), dim3(kCopyThreads), 0, s, c, rows);
  return hipGetLastError();
}

hipError_t launch_cache_copy(const CacheArgs& c, const int32_t* src, const int32_t* dst, uint32_t n, hipStream_t s) {
  const uint32_t units = units_of(c.shape, 1u << c.page_shift);
  hipLaunchKernelGGL(hq_cache_copy_kernel, dim3(units * 2 * c.layers, n), dim3(kCopyThreads), 0, s, c, src, dst, units);
  return hipGetLastError();
}

hipError_t launch_cache_compact(const CacheArgs& c, int32_t* out_table, int64_t out_stride, int32_t* out_refs, void* ws, hipStream_t s) {
  CompactPlan* plan = static_cast<CompactPlan*>(scratch(ws));
  hipLaunchKernelGGL(hq_cache_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, c, out_refs, plan);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t units = units_of(c.shape, 1u << c.page_shift);
  hipLaunchKernelGGL(hq_cache_compact_kernel, dim3(8 * (uint32_t)cu_count()), dim3(kCopyThreads), 0, s, c, out_table, out_stride, plan,
                     units);
  return hipGetLastError();
}

}  // namespace hq
