// Host side of the paged KV cache: which pages each sequence holds.  No GPU
// work happens here; calls return the page copies the caller has to launch.
//
// A page carries the number of sequences that hold it.  Free pages are handed
// out lowest id first (a min-heap), which keeps a pool dense by itself and
// compaction short.  Every call checks and reserves before it changes
// anything, so a failed call leaves the pool as it was, and no C++ exception
// leaves a C entry point.
#include <algorithm>
#include <functional>
#include <new>
#include <vector>

#include "rc_internal.cuh"

namespace {

struct Seq {
  std::vector<int32_t> pages;   // ceil(len / page_size) of them
  int len = 0;
  bool live = false;
};

}  // namespace

struct rc_pages {
  int n_pages, page_size;
  std::vector<int> refs;           // [n_pages] sequences that hold the page
  std::vector<int32_t> free_ids;   // min-heap of the pages with refs == 0; capacity n_pages
  std::vector<Seq> seqs;
  std::vector<int> free_seqs;      // capacity kept at seqs.size()
};

namespace {

using Greater = std::greater<int32_t>;

int32_t take_page(rc_pages *p) {
  std::pop_heap(p->free_ids.begin(), p->free_ids.end(), Greater());
  const int32_t id = p->free_ids.back();
  p->free_ids.pop_back();
  p->refs[id] = 1;
  return id;
}

void drop_page(rc_pages *p, int32_t id) {
  if (--p->refs[id] == 0) {
    p->free_ids.push_back(id);   // within the reserved capacity
    std::push_heap(p->free_ids.begin(), p->free_ids.end(), Greater());
  }
}

Seq *find(const rc_pages *p, int seq) {
  if (seq < 0 || seq >= (int)p->seqs.size() || !p->seqs[seq].live) return nullptr;
  return const_cast<Seq *>(&p->seqs[seq]);
}

int pages_for(const rc_pages *p, long long tokens) { return (int)((tokens + p->page_size - 1) / p->page_size); }

int new_seq(rc_pages *p) {
  if (!p->free_seqs.empty()) {
    const int s = p->free_seqs.back();
    p->free_seqs.pop_back();
    return s;
  }
  p->free_seqs.reserve(p->seqs.size() + 1);
  p->seqs.emplace_back();
  return (int)p->seqs.size() - 1;
}

}  // namespace

#define RC_PAGES_TRY(name, ...)                                   \
  try {                                                           \
    __VA_ARGS__                                                   \
  } catch (const std::exception &e) {                             \
    ::rc::set_error(name ": %s", e.what());                       \
    return RC_ERR_CUDA;                                           \
  }

#define RC_PAGES_SEQ(name, p, seq)                                \
  const auto s = find(p, seq);                                    \
  if (!s) {                                                       \
    ::rc::set_error(name ": unknown sequence %d", seq);           \
    return RC_ERR_NOT_FOUND;                                      \
  }

extern "C" {

int rc_pages_create(int pages, int page_size, rc_pages **out) {
  RC_CHECK_ARG(out, "rc_pages_create: out is NULL");
  *out = nullptr;
  RC_CHECK_ARG(pages >= 1 && page_size >= 1, "rc_pages_create: pages (%d) and page_size (%d) must be positive", pages,
               page_size);
  RC_PAGES_TRY("rc_pages_create", {
    rc_pages *p = new rc_pages{pages, page_size, {}, {}, {}, {}};
    try {
      p->refs.assign(pages, 0);
      p->free_ids.resize(pages);
    } catch (...) {
      delete p;
      throw;
    }
    for (int i = 0; i < pages; ++i) p->free_ids[i] = i;   // ascending: a min-heap
    *out = p;
  })
  return RC_OK;
}

int rc_pages_destroy(rc_pages *p) {
  delete p;
  return RC_OK;
}

int rc_pages_new(rc_pages *p, int *seq) {
  RC_CHECK_ARG(p && seq, "rc_pages_new: NULL argument");
  RC_PAGES_TRY("rc_pages_new", {
    const int id = new_seq(p);
    p->seqs[id].len = 0;
    p->seqs[id].live = true;
    *seq = id;
  })
  return RC_OK;
}

int rc_pages_extend(rc_pages *p, const int32_t *seqs, const int32_t *counts, int n, int32_t *src, int32_t *dst,
                    int *n_copies) {
  RC_CHECK_ARG(p && n_copies && n >= 0 && (n == 0 || (seqs && counts && src && dst)), "rc_pages_extend: bad argument");
  *n_copies = 0;
  RC_PAGES_TRY("rc_pages_extend", {
    // First count: every sequence's new pages, and a page for each tail that is
    // still shared once the sequences before it in the list took their own.
    std::vector<int> refs = p->refs;
    std::vector<char> seen(p->seqs.size(), 0);
    std::vector<char> own_tail(n, 0);
    long long need = 0;
    for (int i = 0; i < n; ++i) {
      RC_PAGES_SEQ("rc_pages_extend", p, seqs[i])
      RC_CHECK_ARG(!seen[seqs[i]], "rc_pages_extend: sequence %d is listed twice", seqs[i]);
      seen[seqs[i]] = 1;
      RC_CHECK_ARG(counts[i] >= 0, "rc_pages_extend: %d tokens for sequence %d", counts[i], seqs[i]);
      const long long len = (long long)s->len + counts[i];
      RC_CHECK_ARG(len <= 0x7fffffff - p->page_size, "rc_pages_extend: %lld tokens in one sequence", len);
      const int fresh = pages_for(p, len) - (int)s->pages.size();
      own_tail[i] = counts[i] > 0 && s->len % p->page_size != 0 && refs[s->pages.back()] > 1;
      if (own_tail[i]) --refs[s->pages.back()];
      need += fresh + own_tail[i];
    }
    if (need > (long long)p->free_ids.size()) {
      ::rc::set_error("rc_pages_extend: %lld pages needed, %d free", need, (int)p->free_ids.size());
      return RC_ERR_FULL;
    }
    for (int i = 0; i < n; ++i) {
      Seq &s = p->seqs[seqs[i]];
      s.pages.reserve(pages_for(p, (long long)s.len + counts[i]));
    }
    int k = 0;
    for (int i = 0; i < n; ++i) {
      Seq &s = p->seqs[seqs[i]];
      if (own_tail[i]) {
        src[k] = s.pages.back();
        dst[k] = take_page(p);
        --p->refs[src[k]];   // another sequence holds it still
        s.pages.back() = dst[k++];
      }
      s.len += counts[i];
      while ((int)s.pages.size() < pages_for(p, s.len)) s.pages.push_back(take_page(p));
    }
    *n_copies = k;
  })
  return RC_OK;
}

int rc_pages_fork(rc_pages *p, int seq, int *child) {
  RC_CHECK_ARG(p && child, "rc_pages_fork: NULL argument");
  RC_PAGES_SEQ("rc_pages_fork", p, seq)
  RC_PAGES_TRY("rc_pages_fork", {
    std::vector<int32_t> pages = s->pages;
    const int len = s->len;
    const int id = new_seq(p);   // may move p->seqs: s is not used past here
    for (int32_t pg : pages) ++p->refs[pg];
    p->seqs[id].pages.swap(pages);
    p->seqs[id].len = len;
    p->seqs[id].live = true;
    *child = id;
  })
  return RC_OK;
}

int rc_pages_trim(rc_pages *p, int seq, int n) {
  RC_CHECK_ARG(p, "rc_pages_trim: NULL argument");
  RC_PAGES_SEQ("rc_pages_trim", p, seq)
  RC_CHECK_ARG(n >= 0 && n <= s->len, "rc_pages_trim: %d tokens of a sequence of %d", n, s->len);
  const int keep = pages_for(p, n);
  while ((int)s->pages.size() > keep) {
    drop_page(p, s->pages.back());
    s->pages.pop_back();
  }
  s->len = n;
  return RC_OK;
}

int rc_pages_free(rc_pages *p, int seq) {
  RC_CHECK_ARG(p, "rc_pages_free: NULL argument");
  RC_PAGES_SEQ("rc_pages_free", p, seq)
  for (int32_t pg : s->pages) drop_page(p, pg);
  s->pages.clear();
  s->len = 0;
  s->live = false;
  p->free_seqs.push_back(seq);   // within the reserved capacity
  return RC_OK;
}

int rc_pages_compact(rc_pages *p, int32_t *src, int32_t *dst, int *n) {
  RC_CHECK_ARG(p && src && dst && n, "rc_pages_compact: NULL argument");
  *n = 0;
  RC_PAGES_TRY("rc_pages_compact", {
    const int used = p->n_pages - (int)p->free_ids.size();
    std::vector<int32_t> to(p->n_pages, -1);
    int lo = 0, k = 0;
    for (int pg = used; pg < p->n_pages; ++pg) {
      if (p->refs[pg] == 0) continue;
      while (p->refs[lo] != 0) ++lo;   // as many free ids below ``used`` as pages in use from it on
      to[pg] = lo++;
      src[k] = pg;
      dst[k++] = to[pg];
    }
    for (int i = 0; i < k; ++i) {
      p->refs[dst[i]] = p->refs[src[i]];
      p->refs[src[i]] = 0;
    }
    if (k)
      for (Seq &s : p->seqs)
        for (int32_t &pg : s.pages)
          if (to[pg] >= 0) pg = to[pg];
    for (int i = 0; i < p->n_pages - used; ++i) p->free_ids[i] = used + i;
    *n = k;
  })
  return RC_OK;
}

int rc_pages_info(const rc_pages *p, int *free_pages, int *high_water) {
  RC_CHECK_ARG(p && free_pages && high_water, "rc_pages_info: NULL argument");
  *free_pages = (int)p->free_ids.size();
  int top = p->n_pages;
  while (top > 0 && p->refs[top - 1] == 0) --top;
  *high_water = top;
  return RC_OK;
}

int rc_pages_len(const rc_pages *p, int seq, int *tokens) {
  RC_CHECK_ARG(p && tokens, "rc_pages_len: NULL argument");
  RC_PAGES_SEQ("rc_pages_len", p, seq)
  *tokens = s->len;
  return RC_OK;
}

int rc_pages_table(const rc_pages *p, const int32_t *seqs, int n, int32_t *table, int ld, int32_t *kv_len) {
  RC_CHECK_ARG(p && seqs && table && kv_len && n >= 0 && ld >= 0, "rc_pages_table: bad argument");
  for (int i = 0; i < n; ++i) {
    RC_PAGES_SEQ("rc_pages_table", p, seqs[i])
    RC_CHECK_ARG((int)s->pages.size() <= ld, "rc_pages_table: sequence %d has %d pages, the table %d columns", seqs[i],
                 (int)s->pages.size(), ld);
  }
  for (int i = 0; i < n; ++i) {
    const Seq *s = find(p, seqs[i]);
    std::copy(s->pages.begin(), s->pages.end(), table + (size_t)i * ld);
    std::fill(table + (size_t)i * ld + s->pages.size(), table + (size_t)(i + 1) * ld, -1);
    kv_len[i] = s->len;
  }
  return RC_OK;
}

}  // extern "C"
