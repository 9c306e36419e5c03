// Page-cache operators: the work of one workgroup of every kernel, apart from how a workgroup synchronises.
//
// State (three int32 arrays of the caller): table[S][B] page ids of every sequence, lengths[S] tokens, refs[P] how
// many sequences use a page.  A page is free exactly when refs is 0, and pages are always given out lowest id first in
// the order of the call's entries, so a call's result depends on its inputs alone and on no order of workgroups.
//
// Every operator is a plan and its application.  The plan checks all entries of the call before anything is changed
// (a call with a bad entry, or with too few free pages, changes nothing and leaves its reason in the status word),
// gives out the pages and writes a list of page moves; the application, in a launch of its own, writes the tables and
// carries the moves out in every pool.
//
// Finding the lowest free pages: workgroup i of a scan reads refs of the i-th segment of pages and writes the segment's
// free ids, in order, and their count; the plan, one workgroup, sums the counts and looks the k-th free page up by a
// binary search over them.  A pool of few segments is scanned by the plan itself.  (All in one launch, the plan being
// the part of the workgroup that arrives last, needs fences between the XCDs' caches, which cost more than a launch:
// extend over 98 segments 50 us, over two 16, where one segment takes 6.)
//
// X is the workgroup: the GPU's (page_kernels.hip) or, in the tests, a set of host threads.  It has kThreads, tid,
// block, blocks, sync(), scan(v, &total) (exclusive sum over the threads), any(flags) (bitwise or over the threads),
// atomic_add / atomic_exch / atomic_or.
#ifndef MMR_CSRC_PAGE_OPS_H_
#define MMR_CSRC_PAGE_OPS_H_

#include <cstdint>

#include "group_ops.h"
#include "mmreshard.h"

namespace mmr {

struct PageMove {
  int32_t src, dst;
};

struct PageState {
  int32_t* table;
  int32_t* lengths;
  int32_t* refs;
  int32_t S, B, P, T;
  int32_t capacity;  // tokens a row holds: B * T, at most 2^31 - 1
  FastDiv div_T;
};

enum PageHeader {
  kPageOk = 1,
  kPageMoves = 2,
  kPageStatus = 3,
  kPageLive = 4,
  kPageFree = 5,
  kPageRows = 6,
  kPageForkBad = 7,  // what page_fork_check found; zero between calls
  kPageHeaderInts = 64
};

struct PageWork {
  int32_t* header;
  int32_t* seg_free;    // free pages of every segment
  int32_t* seg_before;  // free pages before every segment, once a plan has summed them
  int32_t* free_ids;  // segment s's free ids at s * segment size, ascending
  int32_t* live_ids;
  int32_t* mark;  // max(S, P) zeros between calls
  int32_t* len;   // per entry: tokens before the call
  int32_t* rank;  // per entry: first fresh page, -1 none
  PageMove* moves;
  int32_t* map;  // which move of a compact takes a page, or brings one there
  int32_t n_segments;
};

constexpr int kPagesPerThread = 4;
constexpr int32_t kExtendFew = 4096;  // fresh pages up to which the plan of extend writes the tables itself
constexpr int32_t kMaxPageSegments = 4096;

// One buffer of a pool: the tile of one device.
struct PageBuffer {
  char* base;
  uint64_t page_bytes;
};

struct PageMover {
  const PageBuffer* buffers;
  uint32_t n_buffers;
  uint32_t chunks;  // chunks of kPageChunkBytes in the largest page
  FastDiv div_chunks;
  uint32_t lane_bits;  // page_lane_bits
};

constexpr uint32_t kPageChunkBytes = 8192;
constexpr int kPageThreads = 256;

MMR_HD int32_t page_blocks(const PageState& st, int32_t tokens) {
  const int32_t full = static_cast<int32_t>(fdiv(static_cast<uint32_t>(tokens), st.div_T));
  return full + (full * static_cast<int64_t>(st.T) != tokens);
}

// Free (and live) ids of a segment.
template <class X>
MMR_HD void page_scan_segment(X& x, const PageState& st, const PageWork& w, int32_t segment, bool live) {
  constexpr int32_t kSegment = kPagesPerThread * X::kThreads;
  const int32_t at = segment * kSegment + x.tid * kPagesPerThread;
  int32_t r[kPagesPerThread];
  x.load4(st.refs, at, st.P, r);  // ids beyond the pool read as in use
  int32_t n_free = 0;
  for (int i = 0; i < kPagesPerThread; ++i) n_free += r[i] == 0;
  int32_t total = 0;
  const int32_t before = x.scan(n_free, &total);
  int32_t f = segment * kSegment + before;
  int32_t l = at - before;  // the segment's ids before this thread's that are not free
  for (int i = 0; i < kPagesPerThread; ++i) {
    if (at + i >= st.P) break;
    if (r[i] == 0) w.free_ids[f++] = at + i;
    else if (live) w.live_ids[l++] = at + i;
  }
  if (x.tid == 0) w.seg_free[segment] = total;
}

// Up to so many segments a plan scans itself (compact of 8,192 pages, two segments: 16.2 us, with a launch for the scan
// 17.9; of 16,384, four: 21.9 and 19.9).
constexpr int32_t kPlanScans = 2;

template <class X>
MMR_HD void page_plan_scan(X& x, const PageState& st, const PageWork& w, bool live) {
  if (w.n_segments > kPlanScans) return;  // done by the launch before
  for (int32_t s = 0; s < w.n_segments; ++s) page_scan_segment(x, st, w, s, live);
  x.sync();
}

// The free pages of all segments, once every segment is scanned: summed by the plan, or taken from what the plan
// published (`counted`).
template <class X, int32_t kSegment = kPagesPerThread * X::kThreads>
struct FreePages {
  const PageWork* w;
  int32_t* prefix;  // shared: free pages before every segment
  int32_t total;

  MMR_HD FreePages(X& x, const PageWork& work, int32_t* shared, bool counted = false) : w(&work), prefix(shared), total(0) {
    if (counted) {
      for (int32_t s = x.tid; s < work.n_segments; s += X::kThreads) prefix[s] = work.seg_before[s];
      total = work.header[kPageFree];
      x.sync();
      return;
    }
    for (int32_t base = 0; base < work.n_segments; base += X::kThreads) {
      const int32_t s = base + x.tid;
      int32_t sum = 0;
      const int32_t before = x.scan(s < work.n_segments ? work.seg_free[s] : 0, &sum);
      if (s < work.n_segments) prefix[s] = total + before;
      total += sum;
    }
    x.sync();
  }
  // for the launches behind a plan
  MMR_HD void publish(X& x) const {
    for (int32_t s = x.tid; s < w->n_segments; s += X::kThreads) w->seg_before[s] = prefix[s];
  }
  // last segment whose count of earlier pages is at most k
  template <class Before>
  MMR_HD int32_t segment_of(int32_t k, Before before) const {
    int32_t lo = 0, hi = w->n_segments;
    while (hi - lo > 1) {
      const int32_t mid = (lo + hi) >> 1;
      if (before(mid) <= k) lo = mid;
      else hi = mid;
    }
    return lo;
  }
  MMR_HD int32_t kth_free(int32_t k) const {
    const int32_t s = segment_of(k, [this](int32_t i) { return prefix[i]; });
    return w->free_ids[s * kSegment + (k - prefix[s])];
  }
  MMR_HD int32_t live_before(int32_t s) const { return s * kSegment - prefix[s]; }
  MMR_HD int32_t kth_live(int32_t k) const {
    const int32_t s = segment_of(k, [this](int32_t i) { return live_before(i); });
    return w->live_ids[s * kSegment + (k - live_before(s))];
  }
  MMR_HD int32_t free_below(int32_t id) const {
    const int32_t s = id / kSegment;
    if (s >= w->n_segments) return total;
    const int32_t count = (s + 1 < w->n_segments ? prefix[s + 1] : total) - prefix[s];
    int32_t lo = 0, hi = count;  // free ids of the segment below id
    while (lo < hi) {
      const int32_t mid = (lo + hi) >> 1;
      if (w->free_ids[s * kSegment + mid] < id) lo = mid + 1;
      else hi = mid;
    }
    return prefix[s] + lo;
  }
};

template <class X>
MMR_HD void page_verdict(X& x, const PageWork& w, uint32_t bad, int32_t moves, int32_t live) {
  if (x.tid) return;
  w.header[kPageOk] = bad == 0;
  w.header[kPageMoves] = bad ? 0 : moves;
  if (live >= 0) w.header[kPageLive] = live;
  if (bad) x.atomic_or(&w.header[kPageStatus], static_cast<int32_t>(bad));
}

// A page that a sequence with tokens names: it is there, and somebody uses it.
MMR_HD uint32_t page_held(const PageState& st, int32_t page) {
  if (page < 0 || page >= st.P) return MMR_PAGES_BAD_PAGE;
  return st.refs[page] > 0 ? 0 : MMR_PAGES_BAD_COUNT;
}

// Full pages of entry e's parent; 0 where page_fork_entry finds the entry bad.
MMR_HD int32_t page_fork_full(const PageState& st, const int32_t* parents, const int32_t* children, int32_t e) {
  const int32_t parent = parents[e];
  if (children[e] == MMR_PAGES_NONE || parent < 0 || parent >= st.S) return 0;
  const int32_t l = st.lengths[parent];
  return l < 0 || l > st.capacity ? 0 : static_cast<int32_t>(fdiv(static_cast<uint32_t>(l), st.div_T));
}

// The pages a fork shares, checked before anything is written: one entry a workgroup, in the launch before the plan.
template <class X>
MMR_HD void page_fork_check(X& x, const PageState& st, const PageWork& w, const int32_t* parents, const int32_t* children,
                            int32_t n, uint32_t block, uint32_t blocks) {
  uint32_t bad = 0;
  for (int32_t e = static_cast<int32_t>(block); e < n; e += static_cast<int32_t>(blocks)) {
    const int32_t full = page_fork_full(st, parents, children, e);
    for (int32_t i = x.tid; i < full; i += X::kThreads) bad |= page_held(st, st.table[static_cast<int64_t>(parents[e]) * st.B + i]);
  }
  if (bad) x.atomic_or(&w.header[kPageForkBad], static_cast<int32_t>(bad));
}

// Entry e of fork: its flags; the parent's tokens and, where its last page is partly filled, that page.
template <class X>
MMR_HD uint32_t page_fork_entry(X& x, const PageState& st, const PageWork& w, int32_t parent, int32_t child, int32_t* len,
                                int32_t* src) {
  *len = 0;
  *src = -1;
  if (child == MMR_PAGES_NONE) return 0;
  if (parent < 0 || parent >= st.S || child < 0 || child >= st.S) return MMR_PAGES_BAD_SEQUENCE;
  uint32_t flags = 0;
  const int32_t l = st.lengths[parent];
  if (l < 0 || l > st.capacity) return MMR_PAGES_TOO_LONG;
  if (st.lengths[child] != 0) flags |= MMR_PAGES_NOT_EMPTY;
  if (x.atomic_exch(&w.mark[child], 1)) flags |= MMR_PAGES_REPEATED;
  *len = l;
  const int32_t full = static_cast<int32_t>(fdiv(static_cast<uint32_t>(l), st.div_T));
  if (full * static_cast<int64_t>(st.T) != l) {
    const int32_t page = st.table[static_cast<int64_t>(parent) * st.B + full];
    flags |= page_held(st, page);
    *src = page;
  }
  return flags;
}

// `prepared`: the launch before has scanned every segment and checked the shared pages; else the plan does it, place after
// place of the parents' rows (n * B under 2^31).
template <class X>
MMR_HD void page_fork_plan(X& x, const PageState& st, const PageWork& w, int32_t* shared, const int32_t* parents,
                           const int32_t* children, int32_t n, bool prepared = false) {
  if (!prepared) page_plan_scan(x, st, w, false);
  const FreePages<X> pages(x, w, shared);
  int32_t fresh = 0;
  uint32_t bad = 0;
  if (prepared) {
    if (x.tid == 0) bad = static_cast<uint32_t>(x.atomic_exch(&w.header[kPageForkBad], 0));
  } else {
    for (int32_t at = x.tid; at < n * st.B; at += X::kThreads) {
      const int32_t e = at / st.B, i = at - e * st.B;
      if (i < page_fork_full(st, parents, children, e)) bad |= page_held(st, st.table[static_cast<int64_t>(parents[e]) * st.B + i]);
    }
  }
  for (int32_t base = 0; base < n; base += X::kThreads) {
    const int32_t e = base + x.tid;
    int32_t src = -1, len = 0;
    if (e < n) bad |= page_fork_entry(x, st, w, parents[e], children[e], &len, &src);
    int32_t sum = 0;
    const int32_t rank = fresh + x.scan(static_cast<int32_t>(src >= 0), &sum);
    if (e < n) {
      w.len[e] = len;
      w.rank[e] = src >= 0 ? rank : -1;
      if (src >= 0) w.moves[rank].src = src;
    }
    fresh += sum;
  }
  bad = x.any(bad);  // every mark is set by now
  for (int32_t e = x.tid; e < n; e += X::kThreads)
    if (children[e] >= 0 && children[e] < st.S) x.atomic_exch(&w.mark[children[e]], 0);
  if (fresh > pages.total) bad |= MMR_PAGES_OUT_OF_PAGES;
  if (!bad)
    for (int32_t r = x.tid; r < fresh; r += X::kThreads) w.moves[r].dst = pages.kth_free(r);
  page_verdict(x, w, bad, fresh, -1);
}

// Tables of the forked sequences; `block` of `blocks` workgroups share the entries.  The plan has checked the pages; they are
// looked at again so that a table which is written while the call runs cannot lead out of refs.
template <class X>
MMR_HD void page_fork_rows(X& x, const PageState& st, const PageWork& w, const int32_t* parents, const int32_t* children,
                           int32_t n, uint32_t block, uint32_t blocks) {
  uint32_t bad = 0;
  for (int32_t e = static_cast<int32_t>(block); e < n; e += static_cast<int32_t>(blocks)) {
    const int32_t len = w.len[e], rank = w.rank[e], child = children[e];
    if (child == MMR_PAGES_NONE) continue;
    const int32_t full = static_cast<int32_t>(fdiv(static_cast<uint32_t>(len), st.div_T));
    const int32_t* from = st.table + static_cast<int64_t>(parents[e]) * st.B;
    int32_t* to = st.table + static_cast<int64_t>(child) * st.B;
    for (int32_t i = x.tid; i < full; i += X::kThreads) {
      const int32_t page = from[i];
      to[i] = page;
      if (page >= 0 && page < st.P) x.atomic_add(&st.refs[page], 1);
      else bad |= MMR_PAGES_BAD_PAGE;
    }
    if (x.tid == 0) {
      st.lengths[child] = len;
      if (rank >= 0) {
        const int32_t page = w.moves[rank].dst;
        to[full] = page;
        st.refs[page] = 1;
      }
    }
  }
  if (bad) x.atomic_or(&w.header[kPageStatus], static_cast<int32_t>(bad));
}

// The plan writes the tables itself if that takes few rounds, or `whole` says that no launch follows; else page_extend_rows
// does.
template <class X>
MMR_HD void page_extend_plan(X& x, const PageState& st, const PageWork& w, int32_t* shared, const int32_t* slots,
                             const int32_t* counts, int32_t n, bool whole) {
  page_plan_scan(x, st, w, false);
  const FreePages<X> pages(x, w, shared);
  int64_t fresh = 0;
  uint32_t bad = 0;
  for (int32_t base = 0; base < n; base += X::kThreads) {
    const int32_t e = base + x.tid;
    int32_t need = 0, old = 0;
    if (e < n) {
      const int32_t s = slots[e], c = counts[e];
      if (s == MMR_PAGES_NONE) {
        // no entry
      } else if (s < 0 || s >= st.S) {
        bad |= MMR_PAGES_BAD_SEQUENCE;
      } else {
        if (x.atomic_exch(&w.mark[s], 1)) bad |= MMR_PAGES_REPEATED;
        old = st.lengths[s];
        if (c < 0 || old < 0 || old > st.capacity || c > st.capacity - old) {
          bad |= MMR_PAGES_TOO_LONG;
          old = 0;
        } else {
          const int32_t have = page_blocks(st, old);
          need = page_blocks(st, old + c) - have;
          if (c > 0 && have * static_cast<int64_t>(st.T) != old) {  // new tokens go to a partly filled page
            const int32_t page = st.table[static_cast<int64_t>(s) * st.B + have - 1];
            if (page < 0 || page >= st.P) bad |= MMR_PAGES_BAD_PAGE;
            else if (st.refs[page] != 1) bad |= MMR_PAGES_SHARED_TAIL;
          }
        }
      }
    }
    int64_t sum = 0;  // the wishes of a call may add up to more than 2^31 pages
    const int64_t rank = fresh + x.scan(static_cast<int64_t>(need), &sum);
    if (e < n) {
      w.len[e] = old;
      w.rank[e] = static_cast<int32_t>(rank <= pages.total ? rank : pages.total);
    }
    fresh += sum;
  }
  if (fresh > pages.total) bad |= MMR_PAGES_OUT_OF_PAGES;
  bad = x.any(bad);  // every mark is set and every rank written by now
  for (int32_t e = x.tid; e < n; e += X::kThreads)
    if (slots[e] >= 0 && slots[e] < st.S) x.atomic_exch(&w.mark[slots[e]], 0);
  const bool rows = !bad && !whole && fresh > kExtendFew;
  if (!bad && !rows) {
    for (int32_t k = x.tid; k < static_cast<int32_t>(fresh); k += X::kThreads) {
      int32_t lo = 0, hi = n;  // the last entry whose fresh pages start at or before k takes page k
      while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if (w.rank[mid] <= k) lo = mid;
        else hi = mid;
      }
      const int32_t page = pages.kth_free(k);
      st.table[static_cast<int64_t>(slots[lo]) * st.B + page_blocks(st, w.len[lo]) + (k - w.rank[lo])] = page;
      st.refs[page] = 1;
    }
    for (int32_t e = x.tid; e < n; e += X::kThreads)
      if (slots[e] != MMR_PAGES_NONE) st.lengths[slots[e]] = w.len[e] + counts[e];
  }
  if (rows) pages.publish(x);
  if (x.tid == 0) {
    w.header[kPageFree] = pages.total;
    w.header[kPageRows] = rows;
  }
  page_verdict(x, w, bad, 0, -1);
}

template <class X, int32_t kSegment>
MMR_HD void page_extend_rows(X& x, const PageState& st, const PageWork& w, int32_t* shared, const int32_t* slots,
                             const int32_t* counts, int32_t n) {
  if (!w.header[kPageRows]) return;
  const FreePages<X, kSegment> pages(x, w, shared, true);
  for (int32_t e = static_cast<int32_t>(x.block); e < n; e += static_cast<int32_t>(x.blocks)) {
    if (slots[e] == MMR_PAGES_NONE) continue;
    const int32_t old = w.len[e], all = old + counts[e], rank = w.rank[e], have = page_blocks(st, old);
    int32_t* row = st.table + static_cast<int64_t>(slots[e]) * st.B + have;
    for (int32_t i = x.tid, need = page_blocks(st, all) - have; i < need; i += X::kThreads) {
      const int32_t page = pages.kth_free(rank + i);
      row[i] = page;
      st.refs[page] = 1;
    }
    if (x.tid == 0) st.lengths[slots[e]] = all;
  }
}

// One workgroup per entry.  The length is taken by an exchange, so of two entries that name a sequence one frees it and
// the other finds it empty.
template <class X>
MMR_HD void page_free(X& x, const PageState& st, const PageWork& w, int32_t* shared, const int32_t* slots) {
  const int32_t s = slots[x.block];
  uint32_t bad = 0;
  if (s < 0 || s >= st.S) {  // uniform over the workgroup
    if (x.tid == 0 && s != MMR_PAGES_NONE) x.atomic_or(&w.header[kPageStatus], MMR_PAGES_BAD_SEQUENCE);
    return;
  }
  if (x.tid == 0) shared[0] = x.atomic_exch(&st.lengths[s], 0);
  x.sync();
  int32_t len = shared[0];
  if (len < 0 || len > st.capacity) {
    bad |= MMR_PAGES_TOO_LONG;
    len = len < 0 ? 0 : st.capacity;
  }
  const int32_t blocks = page_blocks(st, len);
  const int32_t* row = st.table + static_cast<int64_t>(s) * st.B;
  for (int32_t i = x.tid; i < blocks; i += X::kThreads) {
    const int32_t page = row[i];
    if (page < 0 || page >= st.P) {
      bad |= MMR_PAGES_BAD_PAGE;
    } else if (x.atomic_add(&st.refs[page], -1) <= 0) {
      x.atomic_add(&st.refs[page], 1);  // nobody used it: stays as it was
      bad |= MMR_PAGES_BAD_COUNT;
    }
  }
  if (bad) x.atomic_or(&w.header[kPageStatus], static_cast<int32_t>(bad));
}

// Moves k = first, first + step, ... of a compact.
template <class Pages>
MMR_HD void page_compact_moves(const PageState& st, const PageWork& w, const Pages& pages, int32_t moves, int32_t live,
                               int32_t first, int32_t step) {
  for (int32_t k = first; k < moves; k += step) {
    const int32_t dst = pages.kth_free(k), src = pages.kth_live(live - moves + k);
    w.moves[k] = PageMove{src, dst};
    w.map[src] = w.map[dst] = k;
    st.refs[dst] = st.refs[src];
    st.refs[src] = 0;
  }
}

// `whole`: the plan lists the moves itself; else page_compact_list does, in a launch of its own.
template <class X>
MMR_HD void page_compact_plan(X& x, const PageState& st, const PageWork& w, int32_t* shared, bool whole) {
  page_plan_scan(x, st, w, true);
  const FreePages<X> pages(x, w, shared);
  const int32_t live = st.P - pages.total;
  const int32_t moves = pages.free_below(live);  // as many live pages stand at or after `live`
  if (whole) {
    page_compact_moves(st, w, pages, moves, live, x.tid, X::kThreads);
  } else {
    pages.publish(x);
    if (x.tid == 0) w.header[kPageFree] = pages.total;
  }
  page_verdict(x, w, 0, moves, live);
}

template <class X, int32_t kSegment>
MMR_HD void page_compact_list(X& x, const PageState& st, const PageWork& w, int32_t* shared) {
  const FreePages<X, kSegment> pages(x, w, shared, true);
  page_compact_moves(st, w, pages, w.header[kPageMoves], w.header[kPageLive], static_cast<int32_t>(x.block) * X::kThreads + x.tid,
                     static_cast<int32_t>(x.blocks) * X::kThreads);
}

template <class X>
MMR_HD void page_compact_rows(X& x, const PageState& st, const PageWork& w, uint32_t block, uint32_t blocks) {
  const int32_t live = w.header[kPageLive], moves = w.header[kPageMoves];
  uint32_t bad = 0;
  for (int32_t s = static_cast<int32_t>(block); s < st.S; s += static_cast<int32_t>(blocks)) {
    int32_t len = st.lengths[s];
    if (len < 0 || len > st.capacity) {
      bad |= MMR_PAGES_TOO_LONG;
      len = len < 0 ? 0 : st.capacity;
    }
    const int32_t n = page_blocks(st, len);
    int32_t* row = st.table + static_cast<int64_t>(s) * st.B;
    for (int32_t i = x.tid; i < n; i += X::kThreads) {
      const int32_t page = row[i];
      if (page < 0 || page >= st.P) {
        bad |= MMR_PAGES_BAD_PAGE;
        continue;
      }
      // A page at or after `live` that was in use has moved, and every page before it that was not has been filled: a row
      // that names one of these, or one behind `live` that did not move, is out of step with the counts.  What the map
      // holds for a page without a move is left from an earlier call.
      const int32_t k = w.map[page];
      const PageMove mv = k >= 0 && k < moves ? w.moves[k] : PageMove{-1, -1};
      if (mv.src == page) row[i] = mv.dst;
      else if (mv.dst == page || page >= live) bad |= MMR_PAGES_BAD_COUNT;
    }
  }
  if (bad) x.atomic_or(&w.header[kPageStatus], static_cast<int32_t>(bad));
}

// Pairs of a copy: every destination once, no destination that is also a source.  A page copied onto itself is no move.
// `sorted`: the moves are listed by destination, which the marks give without a sort: a pass over the pages in place of
// one over the pairs.
template <class X>
MMR_HD void page_copy_plan(X& x, const PageState& st, const PageWork& w, const int32_t* src, const int32_t* dst, int32_t n,
                           bool sorted) {
  uint32_t bad = 0;
  for (int32_t e = x.tid; e < n; e += X::kThreads) {
    const int32_t s = src[e], d = dst[e];
    if (d == MMR_PAGES_NONE) continue;
    if (s < 0 || s >= st.P || d < 0 || d >= st.P) bad |= MMR_PAGES_BAD_PAGE;
    else if (s != d && x.atomic_exch(&w.mark[d], e + 1)) bad |= MMR_PAGES_REPEATED;
  }
  x.sync();  // every mark is set
  int32_t moves = 0;
  for (int32_t base = 0; base < n; base += X::kThreads) {
    const int32_t e = base + x.tid;
    const int32_t s = e < n ? src[e] : 0, d = e < n ? dst[e] : 0;
    const bool inside = s >= 0 && s < st.P && d >= 0 && d < st.P;
    if (inside && s != d && w.mark[s]) bad |= MMR_PAGES_OVERLAP;
    if (sorted) continue;
    int32_t sum = 0;
    const int32_t at = moves + x.scan(static_cast<int32_t>(inside && s != d), &sum);
    if (inside && s != d) w.moves[at] = PageMove{s, d};
    moves += sum;
  }
  bad = x.any(bad);  // every mark is read
  for (int32_t base = 0; sorted && !bad && base < st.P; base += kPagesPerThread * X::kThreads) {
    const int32_t first = base + x.tid * kPagesPerThread;
    int32_t e[kPagesPerThread], here = 0, sum = 0;
    for (int i = 0; i < kPagesPerThread; ++i) {
      e[i] = first + i < st.P ? w.mark[first + i] : 0;
      here += e[i] != 0;
    }
    int32_t at = moves + x.scan(here, &sum);
    for (int i = 0; i < kPagesPerThread; ++i)
      if (e[i]) w.moves[at++] = PageMove{src[e[i] - 1], first + i};
    moves += sum;
  }
  x.sync();
  for (int32_t e = x.tid; e < n; e += X::kThreads) {
    const int32_t d = dst[e];
    if (d >= 0 && d < st.P) x.atomic_exch(&w.mark[d], 0);
  }
  page_verdict(x, w, bad, moves, -1);
}

constexpr int32_t kFewPairs = 64;

// The same checks for at most kFewPairs pairs, made by every workgroup of the copy for itself, so that a small copy is one
// launch: pair i is thread i's.  shared: 2 * kFewPairs words.  True if the pairs may be carried out.
template <class X>
MMR_HD bool page_copy_few(X& x, const PageState& st, const PageWork& w, int32_t* shared, const int32_t* src, const int32_t* dst,
                          int32_t n) {
  int32_t s = -1, d = -1;
  if (x.tid < n) {
    s = src[x.tid], d = dst[x.tid];
    if (d == MMR_PAGES_NONE) s = d;  // no pair, and no move, as for a page copied onto itself
    shared[x.tid] = s;
    shared[kFewPairs + x.tid] = d;
  }
  x.sync();
  uint32_t bad = 0;
  if (x.tid < n && d != MMR_PAGES_NONE) {
    if (s < 0 || s >= st.P || d < 0 || d >= st.P) {
      bad |= MMR_PAGES_BAD_PAGE;
    } else if (s != d) {
      for (int32_t i = 0; i < n; ++i) {
        if (i == x.tid || shared[i] == shared[kFewPairs + i]) continue;
        if (shared[i] < 0 || shared[i] >= st.P) continue;  // a bad pair, as told by its own thread
        if (shared[kFewPairs + i] == d) bad |= MMR_PAGES_REPEATED;
        if (shared[kFewPairs + i] == s) bad |= MMR_PAGES_OVERLAP;
      }
    }
  }
  bad = x.any(bad);
  if (bad && x.block == 0 && x.tid == 0) x.atomic_or(&w.header[kPageStatus], static_cast<int32_t>(bad));
  return bad == 0;
}

// Pages in use, into header[kPageLive].
template <class X>
MMR_HD void page_count(X& x, const PageState& st, const PageWork& w, int32_t* shared) {
  page_plan_scan(x, st, w, false);
  const FreePages<X> pages(x, w, shared);
  if (x.tid == 0) w.header[kPageLive] = st.P - pages.total;
}

// Lanes that share a page of at most a chunk, where a workgroup moves several: a power of two.
inline uint32_t page_lane_bits(uint64_t largest) {
  uint32_t bits = 0;
  const uint64_t lanes = (largest + 15) / 16;
  while ((1u << bits) < static_cast<uint32_t>(kPageThreads) && (1u << bits) < lanes) ++bits;
  return bits;
}

// Items of a launch: chunks of pages, or, PACKED, groups of pages that a workgroup moves together.
template <bool PACKED>
MMR_HD uint32_t page_items(const PageMover& m, uint32_t n_moves) {
  if (!PACKED) return n_moves * m.n_buffers * m.chunks;
  const uint32_t together = static_cast<uint32_t>(kPageThreads) >> m.lane_bits;
  return (n_moves + together - 1) / together * m.n_buffers;
}

// Item `item` of the moves, buffer after buffer, move after move: the pages of one buffer are worked off together, so
// that the workgroups in flight share their address translations.  move(i): move i.  M: memory policy of chunk_ops.h.
// Pages of a multiple of 16 bytes move as aligned 16-byte vectors.  Others move as 16-byte vectors at any alignment, the
// last one slid back to end with the page (it repeats bytes of its neighbour, with the same values), pages under 16 bytes
// byte by byte.  PACKED (no page longer than 16 bytes a lane): 2^lane_bits lanes a page.
template <class M, bool ALIGNED, bool PACKED, class Move>
MMR_HD void page_move_chunk(const PageMover& m, Move move, uint32_t n_moves, uint32_t item, uint32_t thread) {
  uint32_t bi, mi, chunk = 0, tid = thread;
  if (PACKED) {
    const uint32_t together = static_cast<uint32_t>(kPageThreads) >> m.lane_bits, groups = (n_moves + together - 1) / together;
    bi = item / groups;
    mi = (item - bi * groups) * together + (thread >> m.lane_bits);
    tid = thread & ((1u << m.lane_bits) - 1);
    if (mi >= n_moves) return;
  } else {
    const uint32_t rest = fdiv(item, m.div_chunks);
    chunk = item - rest * m.chunks;
    bi = rest / n_moves, mi = rest - bi * n_moves;
  }
  const PageBuffer b = m.buffers[bi];
  const PageMove mv = move(mi);
  if (mv.src == mv.dst) return;
  const uint64_t begin = static_cast<uint64_t>(chunk) * kPageChunkBytes;
  if (begin >= b.page_bytes) return;  // a smaller page than the largest
  const uint64_t left = b.page_bytes - begin;
  const uint32_t bytes = left < kPageChunkBytes ? static_cast<uint32_t>(left) : kPageChunkBytes;
  typename M::cptr s = M::cplace(b.base + static_cast<uint64_t>(mv.src) * b.page_bytes + begin);
  typename M::ptr d = M::place(b.base + static_cast<uint64_t>(mv.dst) * b.page_bytes + begin);
  constexpr uint32_t kUnroll = PACKED ? 1 : kPageChunkBytes / 16 / kPageThreads;
  if (ALIGNED) {
    V16 v[kUnroll];
#pragma unroll
    for (uint32_t u = 0; u < kUnroll; ++u) {
      const uint32_t at = (tid + u * kPageThreads) * 16;
      if (at < bytes) v[u] = M::load16(s + at);
    }
#pragma unroll
    for (uint32_t u = 0; u < kUnroll; ++u) {
      const uint32_t at = (tid + u * kPageThreads) * 16;
      if (at < bytes) M::store16(d + at, v[u]);
    }
    return;
  }
  if (b.page_bytes < 16) {
    // a larger page of another pool may have set few lanes
    for (uint32_t at = tid; at < bytes; at += PACKED ? 1u << m.lane_bits : static_cast<uint32_t>(kPageThreads))
      M::template storeu<uint8_t>(d + at, M::template loadu<uint8_t>(s + at));
    return;
  }
  // the last vector of a page may reach back into the chunk before: begin > 0 or the page holds 16 bytes here
  V16 v[kUnroll];
#pragma unroll
  for (uint32_t u = 0; u < kUnroll; ++u) {
    const uint32_t at = (tid + u * kPageThreads) * 16;
    const int64_t slid = at + 16 <= bytes ? static_cast<int64_t>(at) : static_cast<int64_t>(bytes) - 16;
    if (at < bytes) v[u] = M::load16u(s + slid);
  }
#pragma unroll
  for (uint32_t u = 0; u < kUnroll; ++u) {
    const uint32_t at = (tid + u * kPageThreads) * 16;
    const int64_t slid = at + 16 <= bytes ? static_cast<int64_t>(at) : static_cast<int64_t>(bytes) - 16;
    if (at < bytes) M::template storeu<V16>(d + slid, v[u]);
  }
}

}  // namespace mmr

#endif  // MMR_CSRC_PAGE_OPS_H_
