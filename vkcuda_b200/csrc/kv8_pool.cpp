// kv8_pool.cpp - which pages of a paged K/V cache belong to which sequence.
//
// Host bookkeeping only: the pool hands out page numbers, counts how many
// sequences hold each, and says which pages have to be copied on the device
// (vc_kv8_copy_pages) for a fork that diverges or a compaction. Free pages
// are handed out lowest first, so that a run of the same calls gives the same
// pages. Every call either does all it was asked or changes nothing.
#include <cstdint>
#include <functional>
#include <map>
#include <mutex>
#include <new>
#include <queue>
#include <vector>

#include "../../include/vc_b200.h"

namespace {

struct Sequence {
  std::vector<int32_t> pages;
  int64_t tokens = 0;
};

struct Pool {
  std::mutex mu;
  int num_pages = 0, page_size = 0;
  std::vector<int32_t> held;  // sequences that hold each page
  std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>> free_pages;
  std::map<int64_t, Sequence> sequences;
  int64_t next_id = 1;

  int32_t take() {
    const int32_t p = free_pages.top();
    free_pages.pop();
    held[p] = 1;
    return p;
  }
  void drop(int32_t p) {
    if (--held[p] == 0) free_pages.push(p);
  }
};

// No C++ exception leaves a C entry: what the bookkeeping's own memory cannot
// hold is out of memory.
template <class F>
int guarded(void *pool, F &&f) {
  if (!pool) return VC_INVALID_VALUE;
  Pool &p = *static_cast<Pool *>(pool);
  try {
    std::lock_guard<std::mutex> lk(p.mu);
    return f(p);
  } catch (const std::bad_alloc &) {
    return VC_OUT_OF_MEMORY;
  } catch (...) {
    return VC_UNKNOWN;
  }
}

}  // namespace

extern "C" {

int vc_kv8_pool_create(void **pool, int num_pages, int page_size) {
  if (!pool || num_pages <= 0 || page_size <= 0) return VC_INVALID_VALUE;
  *pool = nullptr;
  Pool *p = nullptr;
  try {
    p = new Pool();
    p->num_pages = num_pages;
    p->page_size = page_size;
    p->held.assign(num_pages, 0);
    for (int i = 0; i < num_pages; ++i) p->free_pages.push(i);
  } catch (...) {
    delete p;
    return VC_OUT_OF_MEMORY;
  }
  *pool = p;
  return VC_SUCCESS;
}

int vc_kv8_pool_destroy(void *pool) {
  delete static_cast<Pool *>(pool);
  return VC_SUCCESS;
}

int vc_kv8_pool_new(void *pool, int64_t *seq) {
  if (!seq) return VC_INVALID_VALUE;
  return guarded(pool, [&](Pool &p) {
    p.sequences.emplace(p.next_id, Sequence());
    *seq = p.next_id++;
    return (int)VC_SUCCESS;
  });
}

int vc_kv8_pool_fork(void *pool, int64_t seq, int64_t *child) {
  if (!child) return VC_INVALID_VALUE;
  return guarded(pool, [&](Pool &p) {
    auto it = p.sequences.find(seq);
    if (it == p.sequences.end()) return (int)VC_INVALID_VALUE;
    p.sequences.emplace(p.next_id, it->second);
    for (int32_t page : it->second.pages) ++p.held[page];
    *child = p.next_id++;
    return (int)VC_SUCCESS;
  });
}

int vc_kv8_pool_extend(void *pool, int64_t seq, int64_t tokens, int32_t *copy_src,
                       int32_t *copy_dst) {
  if (!copy_src || !copy_dst || tokens < 0) return VC_INVALID_VALUE;
  return guarded(pool, [&](Pool &p) {
    auto it = p.sequences.find(seq);
    if (it == p.sequences.end()) return (int)VC_INVALID_VALUE;
    Sequence &s = it->second;
    if (tokens > (int64_t)p.num_pages * p.page_size) return (int)VC_OUT_OF_MEMORY;
    const int64_t end = s.tokens + tokens;
    const int64_t want = (end + p.page_size - 1) / p.page_size;
    const int64_t more = want - (int64_t)s.pages.size();
    // The last page takes new tokens only if it has room; a page that another
    // sequence holds too is copied first.
    const bool copy = tokens > 0 && s.tokens % p.page_size != 0 && p.held[s.pages.back()] > 1;
    if (more + (copy ? 1 : 0) > (int64_t)p.free_pages.size()) return (int)VC_OUT_OF_MEMORY;
    s.pages.reserve((size_t)want);
    *copy_src = *copy_dst = -1;
    if (copy) {
      *copy_src = s.pages.back();
      *copy_dst = p.take();
      p.drop(*copy_src);
      s.pages.back() = *copy_dst;
    }
    for (int64_t i = 0; i < more; ++i) s.pages.push_back(p.take());
    s.tokens = end;
    return (int)VC_SUCCESS;
  });
}

int vc_kv8_pool_free(void *pool, int64_t seq) {
  return guarded(pool, [&](Pool &p) {
    auto it = p.sequences.find(seq);
    if (it == p.sequences.end()) return (int)VC_INVALID_VALUE;
    for (int32_t page : it->second.pages) p.drop(page);
    p.sequences.erase(it);
    return (int)VC_SUCCESS;
  });
}

int vc_kv8_pool_pages(void *pool, int64_t seq, int32_t *pages, int capacity, int *n_pages,
                      int64_t *n_tokens) {
  if (!n_pages || capacity < 0 || (capacity > 0 && !pages)) return VC_INVALID_VALUE;
  return guarded(pool, [&](Pool &p) {
    auto it = p.sequences.find(seq);
    if (it == p.sequences.end()) return (int)VC_INVALID_VALUE;
    const Sequence &s = it->second;
    *n_pages = (int)s.pages.size();
    if (n_tokens) *n_tokens = s.tokens;
    if (!pages) return (int)VC_SUCCESS;  // asked for the counts alone
    if ((size_t)capacity < s.pages.size()) return (int)VC_INVALID_VALUE;
    for (int i = 0; i < capacity; ++i) pages[i] = i < *n_pages ? s.pages[i] : -1;
    return (int)VC_SUCCESS;
  });
}

int vc_kv8_pool_info(void *pool, int *free_pages, int *sequences) {
  return guarded(pool, [&](Pool &p) {
    if (free_pages) *free_pages = (int)p.free_pages.size();
    if (sequences) *sequences = (int)p.sequences.size();
    return (int)VC_SUCCESS;
  });
}

int vc_kv8_pool_compact(void *pool, int32_t *copy_src, int32_t *copy_dst, int capacity,
                        int *n_copies) {
  if (!n_copies || capacity < 0 || (capacity > 0 && (!copy_src || !copy_dst)))
    return VC_INVALID_VALUE;
  return guarded(pool, [&](Pool &p) {
    const int live = p.num_pages - (int)p.free_pages.size();
    int moves = 0;
    for (int i = live; i < p.num_pages; ++i) moves += p.held[i] > 0;
    *n_copies = moves;
    if (moves > capacity) return (int)VC_INVALID_VALUE;
    // Pages from `live` on move, in order, into the free ones below it: no
    // page is both read and written, so the copies need no order.
    std::vector<int32_t> to(p.num_pages);
    std::vector<int32_t> left;
    left.reserve(p.num_pages);
    for (int i = live; i < p.num_pages; ++i) left.push_back(i);
    std::priority_queue<int32_t, std::vector<int32_t>, std::greater<int32_t>> free_after(
        std::greater<int32_t>(), std::move(left));
    // Nothing below allocates.
    for (int i = 0; i < p.num_pages; ++i) to[i] = i;
    int at = 0, n = 0;
    for (int i = live; i < p.num_pages; ++i) {
      if (!p.held[i]) continue;
      while (p.held[at]) ++at;
      copy_src[n] = i;
      copy_dst[n++] = at;
      to[i] = at;
      p.held[at] = p.held[i];
      p.held[i] = 0;
    }
    for (auto &s : p.sequences)
      for (int32_t &page : s.second.pages) page = to[page];
    p.free_pages.swap(free_after);
    return (int)VC_SUCCESS;
  });
}

}  // extern "C"
