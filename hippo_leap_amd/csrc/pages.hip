// Page copies (hl_kv_pages_copy) and the host's page bookkeeping
// (hl_page_pool_*).
//
// The copy is bound by memory: 2 * page_bytes per (pool, move).  The moves
// and the pools' addresses travel as kernel arguments, so that the call needs
// no device memory and may be captured.
#include <algorithm>
#include <cstring>
#include <new>
#include <vector>

#include "common.h"
#include "launch.h"

namespace hl {

constexpr int kCopyPools = 64, kCopyMoves = 256;
struct PagesCopyParams {
  uint64_t page16;  // 16-byte units of a page
  int n_moves;
  char* pool[kCopyPools];
  int32_t move[kCopyMoves][2];
};
static_assert(sizeof(PagesCopyParams) <= 4096, "kernel arguments");

// Workgroup (x, move, pool): 4 16-byte loads per thread in flight, 16 KB of
// the page per workgroup.  200 pages of 64 KB in 64 pools: 319 us, 5.26 TB/s; 3
// pages in 32 pools 5.5 us, the launch.
__global__ __launch_bounds__(256) void pages_copy_kernel(PagesCopyParams p) {
  const int m = blockIdx.y;
  char* pool = p.pool[blockIdx.z];
  const u32x4* src = (const u32x4*)pool + p.move[m][0] * p.page16;
  u32x4* dst = (u32x4*)pool + p.move[m][1] * p.page16;
  const uint64_t i0 = (uint64_t)blockIdx.x * 1024 + threadIdx.x;
  u32x4 x[4];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (i0 + 256 * u < p.page16) x[u] = src[i0 + 256 * u];
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (i0 + 256 * u < p.page16) dst[i0 + 256 * u] = x[u];
}

hipError_t pages_copy_launch(const hl_kv_pages* pages, const int32_t* moves, int n_moves, hipStream_t stream) {
  PagesCopyParams p;
  p.page16 = pages->page_bytes / 16;
  const unsigned per_page = (unsigned)((p.page16 + 1023) / 1024);
  for (int p0 = 0; p0 < pages->n_pools; p0 += kCopyPools) {
    const int np = std::min(kCopyPools, pages->n_pools - p0);
    for (int i = 0; i < np; ++i) p.pool[i] = (char*)pages->pools[p0 + i];
    for (int m0 = 0; m0 < n_moves; m0 += kCopyMoves) {
      p.n_moves = std::min(kCopyMoves, n_moves - m0);
      memcpy(p.move, moves + 2 * (size_t)m0, sizeof(int32_t) * 2 * p.n_moves);
      hipLaunchKernelGGL(pages_copy_kernel, dim3(per_page, p.n_moves, np), dim3(256), 0, stream, p);
      if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
  }
  return hipSuccess;
}

}  // namespace hl

using namespace hl;

// refs[p]: sequences that hold page p.  Free pages are handed out lowest
// first, so that a pool stays compact while it can: `low` is a bound below
// which none is free.
struct hl_page_pool {
  std::vector<int32_t> refs;
  int free_count = 0;
  int low = 0;
};

namespace {
bool table_ok(const hl_page_pool* pool, const int32_t* table, int bps, const char* who, int* rc) {
  if (!pool || !table || bps <= 0) {
    *rc = set_error(HL_EINVAL, "%s: null pool or table, or no blocks", who);
    return false;
  }
  return true;
}
bool held(const hl_page_pool* pool, int32_t page) {
  return page >= 0 && page < (int32_t)pool->refs.size() && pool->refs[page] > 0;
}
int take(hl_page_pool* pool) {  // a free page exists
  int p = pool->low;
  while (pool->refs[p]) ++p;
  pool->refs[p] = 1;
  pool->low = p + 1;
  --pool->free_count;
  return p;
}
void drop(hl_page_pool* pool, int32_t page) {
  if (--pool->refs[page] == 0) {
    ++pool->free_count;
    pool->low = std::min(pool->low, (int)page);
  }
}
}  // namespace

extern "C" {

int hl_page_pool_create(hl_page_pool** pool, int n_pages) {
  if (!pool || n_pages <= 0) return set_error(HL_EINVAL, "page pool: null result or no pages (n_pages=%d)", n_pages);
  *pool = nullptr;
  try {
    hl_page_pool* p = new hl_page_pool;
    try {
      p->refs.assign((size_t)n_pages, 0);
    } catch (...) {
      delete p;
      throw;
    }
    p->free_count = n_pages;
    *pool = p;
  } catch (const std::bad_alloc&) {
    return set_error(HL_ECAPACITY, "page pool: no host memory for %d pages", n_pages);
  }
  return HL_OK;
}

void hl_page_pool_destroy(hl_page_pool* pool) { delete pool; }

int hl_page_pool_free_count(const hl_page_pool* pool) {
  return pool ? pool->free_count : set_error(HL_EINVAL, "page pool: null");
}

int hl_page_pool_refs(const hl_page_pool* pool, int page) {
  if (!pool || page < 0 || page >= (int)pool->refs.size()) return set_error(HL_EINVAL, "page pool: no page %d", page);
  return pool->refs[page];
}

int hl_page_pool_extend(hl_page_pool* pool, int32_t* table, int bps, int old_len, int new_len, int32_t move[2]) {
  int rc;
  if (!table_ok(pool, table, bps, "page pool extend", &rc)) return rc;
  if (!move) return set_error(HL_EINVAL, "page pool extend: null move");
  if (old_len < 0 || new_len < old_len) return set_error(HL_EINVAL, "page pool extend: lengths %d -> %d", old_len, new_len);
  if (((int64_t)new_len + 31) / 32 > bps)
    return set_error(HL_ECAPACITY, "page pool extend: %d positions need more than %d blocks", new_len, bps);
  move[0] = move[1] = -1;
  if (new_len == old_len) return HL_OK;
  const int first = old_len / 32, last = (new_len - 1) / 32;
  // What is needed, before anything changes.
  int need = 0;
  bool copy = false;
  for (int t = first; t <= last; ++t) {
    if (table[t] == -1) {
      if (t == first && old_len % 32) return set_error(HL_EINVAL, "page pool extend: block %d is part-filled but has no page", t);
      ++need;
    } else if (!held(pool, table[t])) {
      return set_error(HL_EINVAL, "page pool extend: block %d names page %d, which is not held", t, table[t]);
    } else if (pool->refs[table[t]] > 1) {  // shared: this sequence gets one of its own
      if (t == first && old_len % 32) copy = true;
      ++need;
    }
  }
  if (need > pool->free_count)
    return set_error(HL_ECAPACITY, "page pool extend: %d pages needed, %d free", need, pool->free_count);
  for (int t = first; t <= last; ++t) {
    const int32_t old = table[t];
    if (old != -1 && pool->refs[old] == 1) continue;
    table[t] = take(pool);
    if (old != -1) drop(pool, old);
    if (t == first && copy) {
      move[0] = old;
      move[1] = table[t];
    }
  }
  return HL_OK;
}

int hl_page_pool_fork(hl_page_pool* pool, const int32_t* from, int32_t* to, int bps, int len) {
  int rc;
  if (!table_ok(pool, from, bps, "page pool fork", &rc) || !table_ok(pool, to, bps, "page pool fork", &rc)) return rc;
  if (from == to || overlaps(from, sizeof(int32_t) * bps, to, sizeof(int32_t) * bps))
    return set_error(HL_EINVAL, "page pool fork: the tables overlap");
  if (len < 0 || ((int64_t)len + 31) / 32 > bps) return set_error(HL_EINVAL, "page pool fork: length %d in %d blocks", len, bps);
  const int n = (int)(((int64_t)len + 31) / 32);
  for (int t = 0; t < bps; ++t)
    if (to[t] != -1) return set_error(HL_EINVAL, "page pool fork: the new table holds page %d at block %d", to[t], t);
  for (int t = 0; t < n; ++t)  // -1: a block that a window left behind
    if (from[t] != -1 && !held(pool, from[t]))
      return set_error(HL_EINVAL, "page pool fork: block %d names page %d, which is not held", t, from[t]);
  for (int t = 0; t < n; ++t) {
    to[t] = from[t];
    if (from[t] != -1) ++pool->refs[from[t]];
  }
  return HL_OK;
}

int hl_page_pool_release(hl_page_pool* pool, int32_t* table, int bps, int first, int count) {
  int rc;
  if (!table_ok(pool, table, bps, "page pool release", &rc)) return rc;
  if (first < 0 || count < 0 || (int64_t)first + count > bps)
    return set_error(HL_EINVAL, "page pool release: blocks %d .. + %d of %d", first, count, bps);
  // A table that names one page twice holds it twice (refs permitting).
  for (int t = first; t < first + count; ++t) {
    if (table[t] == -1) continue;
    if (!held(pool, table[t])) {
      rc = set_error(HL_EINVAL, "page pool release: block %d names page %d, which is not held", t, table[t]);
      for (int u = first; u < t; ++u)  // as it was
        if (table[u] != -1) {
          if (pool->refs[table[u]]++ == 0) --pool->free_count;
        }
      return rc;
    }
    if (--pool->refs[table[t]] == 0) ++pool->free_count;
  }
  for (int t = first; t < first + count; ++t) {
    if (table[t] != -1 && pool->refs[table[t]] == 0) pool->low = std::min(pool->low, (int)table[t]);
    table[t] = -1;
  }
  return HL_OK;
}

int hl_page_pool_compact(hl_page_pool* pool, int32_t* tables, int n_tables, int bps, int32_t* moves, int max_moves,
                         int* n_moves) {
  int rc;
  if (!table_ok(pool, tables, bps, "page pool compact", &rc)) return rc;
  if (n_tables <= 0 || (max_moves > 0 && !moves) || max_moves < 0 || !n_moves)
    return set_error(HL_EINVAL, "page pool compact: no tables, or a null result");
  *n_moves = 0;
  const size_t n = (size_t)n_tables * bps;
  const int np = (int)pool->refs.size();
  try {
    std::vector<int32_t> seen(np, 0), to(np, -1);
    for (size_t i = 0; i < n; ++i) {
      if (tables[i] == -1) continue;
      if (!held(pool, tables[i]))
        return set_error(HL_EINVAL, "page pool compact: table %zu names page %d, which is not held", i / bps, tables[i]);
      ++seen[tables[i]];
    }
    int lo = 0, moved = 0;
    for (int hi = np - 1; hi > lo && moved < max_moves; --hi) {
      if (pool->refs[hi] == 0 || seen[hi] != pool->refs[hi]) continue;  // free, or held elsewhere too
      while (lo < hi && pool->refs[lo]) ++lo;
      if (lo >= hi) break;
      moves[2 * moved] = hi;
      moves[2 * moved + 1] = lo;
      ++moved;
      to[hi] = lo;
      pool->refs[lo] = pool->refs[hi];
      pool->refs[hi] = 0;
    }
    for (size_t i = 0; i < n; ++i)
      if (tables[i] != -1 && to[tables[i]] != -1) tables[i] = to[tables[i]];
    pool->low = 0;
    *n_moves = moved;
  } catch (const std::bad_alloc&) {
    return set_error(HL_ECAPACITY, "page pool compact: no host memory");
  }
  return HL_OK;
}

}  // extern "C"
