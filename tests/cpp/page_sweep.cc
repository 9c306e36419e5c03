// Host run of the page-cache and rotary kernels, for tests only: the same per-workgroup routines (page_ops.h,
// rotary_ops.h) with host threads as the lanes of a workgroup, on heap buffers of exactly the sizes the kernels may
// touch, under the address and undefined-behaviour sanitizers, or the thread sanitizer.  Random valid and invalid
// calls, every result compared with a plain model.  Never a fallback of the library.
#include <pthread.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <random>
#include <set>
#include <thread>
#include <vector>

#include "page_ops.h"
#include "rotary_ops.h"

using namespace mmr;

namespace {

[[noreturn]] void die(const char* what, int64_t a = 0, int64_t b = 0) {
  std::printf("FAILED: %s (%lld, %lld)\n", what, (long long)a, (long long)b);
  std::fflush(stdout);
  std::_Exit(1);
}

struct Shared {
  pthread_barrier_t barrier;
  std::vector<int64_t> values;
  uint32_t flags = 0;
};

template <int K>
struct Lanes {
  static constexpr int kThreads = K;
  int32_t tid;
  uint32_t block, blocks;
  Shared* s;
  void sync() { pthread_barrier_wait(&s->barrier); }
  void load4(const int32_t* p, int32_t at, int32_t n, int32_t (&r)[4]) {
    for (int i = 0; i < 4; ++i) r[i] = at + i < n ? p[at + i] : 1;
  }
  template <class V>
  V scan(V v, V* total) {
    s->values[tid] = v;
    sync();
    V before = 0, all = 0;
    for (int i = 0; i < K; ++i) {
      if (i < tid) before += static_cast<V>(s->values[i]);
      all += static_cast<V>(s->values[i]);
    }
    sync();
    *total = all;
    return before;
  }
  uint32_t any(uint32_t f) {
    if (tid == 0) s->flags = 0;
    sync();
    __atomic_fetch_or(&s->flags, f, __ATOMIC_SEQ_CST);
    sync();
    const uint32_t all = __atomic_load_n(&s->flags, __ATOMIC_SEQ_CST);
    sync();
    return all;
  }
  bool all(bool v) { return v; }  // a lane is a wave of its own here
  int32_t ended(const int32_t* ends, int32_t n, int32_t t) {
    int32_t count = 0;
    while (count < n && ends[count] <= t) ++count;
    return count;
  }
  int32_t atomic_add(int32_t* p, int32_t v) { return __atomic_fetch_add(p, v, __ATOMIC_SEQ_CST); }
  int32_t atomic_exch(int32_t* p, int32_t v) { return __atomic_exchange_n(p, v, __ATOMIC_SEQ_CST); }
  void atomic_or(int32_t* p, int32_t v) { __atomic_fetch_or(p, v, __ATOMIC_SEQ_CST); }
};

// `blocks` workgroups of K lanes, one after the other.
template <int K>
void launch(uint32_t blocks, const std::function<void(Lanes<K>&)>& body) {
  Shared s;
  s.values.resize(K);
  pthread_barrier_init(&s.barrier, nullptr, K);
  std::vector<std::thread> threads;
  for (int t = 0; t < K; ++t)
    threads.emplace_back([&, t] {
      for (uint32_t b = 0; b < blocks; ++b) {
        Lanes<K> x{t, b, blocks, &s};
        body(x);
        x.sync();
      }
    });
  for (auto& t : threads) t.join();
  pthread_barrier_destroy(&s.barrier);
}

struct Mem {
  typedef const char* cptr;
  typedef char* ptr;
  static cptr cplace(const char* p) { return p; }
  static ptr place(char* p) { return p; }
  static void aligned(const void* p) {
    if (reinterpret_cast<uintptr_t>(p) % 16) die("an aligned access is not aligned");
  }
  static V16 load16(cptr p) {
    aligned(p);
    return load16u(p);
  }
  static V16 load16u(cptr p) {
    V16 v;
    std::memcpy(&v, p, 16);
    return v;
  }
  static void store16(ptr p, V16 v) {
    aligned(p);
    std::memcpy(p, &v, 16);
  }
  template <class T>
  static T loadu(cptr p) {
    T v;
    std::memcpy(&v, p, sizeof(T));
    return v;
  }
  template <class T>
  static void storeu(ptr p, T v) {
    std::memcpy(p, &v, sizeof(T));
  }
};

constexpr int K = 16;  // lanes of a plan's workgroup here: segments of 64 pages
constexpr int32_t kSegment = K * kPagesPerThread;

// A heap block of exactly n values.
template <class T>
struct Exact {
  T* p;
  size_t n;
  explicit Exact(size_t n_, int fill = 0) : p(static_cast<T*>(std::aligned_alloc(16, (n_ * sizeof(T) + 15) / 16 * 16))), n(n_) {
    std::free(p);
    p = static_cast<T*>(std::malloc(std::max<size_t>(n * sizeof(T), 1)));  // at least 16-byte aligned
    std::memset(p, fill, n * sizeof(T));
  }
  ~Exact() { std::free(p); }
  Exact(const Exact&) = delete;
  T& operator[](size_t i) { return p[i]; }
  std::vector<T> copy() const { return std::vector<T>(p, p + n); }
};

struct Model {
  std::vector<int32_t> table, lengths, refs;
  std::vector<std::vector<std::vector<char>>> pools;  // [buffer][page]
};

struct Cache {
  int32_t S, B, P, T;
  std::vector<uint64_t> page_bytes;
  Exact<int32_t> table, lengths, refs;
  std::vector<std::unique_ptr<Exact<char>>> pools;
  Exact<int32_t> header, seg_free, seg_before, free_ids, live_ids, mark, len, rank, map;
  Exact<PageMove> moves;
  Exact<PageBuffer> buffers;
  PageState st;
  PageWork w;
  PageMover mover;
  bool aligned = true;

  Cache(int32_t s, int32_t b, int32_t p, int32_t t, const std::vector<uint64_t>& bytes)
      : S(s), B(b), P(p), T(t), page_bytes(bytes), table(static_cast<size_t>(s) * b, 0x7b), lengths(s), refs(p), header(kPageHeaderInts),
        seg_free(segs(p), 0x55), seg_before(segs(p), 0x55), free_ids(segs(p) * kSegment, 0x55), live_ids(segs(p) * kSegment, 0x55), mark(std::max(s, p)),
        len(s, 0x55), rank(s, 0x55), map(p, 0x55), moves(std::max(s, p), 0x55), buffers(bytes.size()) {
    uint64_t largest = 0;
    for (size_t i = 0; i < bytes.size(); ++i) {
      pools.push_back(std::make_unique<Exact<char>>(bytes[i] * p));
      buffers[i] = {pools[i]->p, bytes[i]};
      largest = std::max(largest, bytes[i]);
      aligned &= bytes[i] % 16 == 0;
    }
    const uint32_t chunks = static_cast<uint32_t>((largest + kPageChunkBytes - 1) / kPageChunkBytes);
    const int32_t capacity = static_cast<int32_t>(std::min<int64_t>(static_cast<int64_t>(B) * T, 0x7fffffff));
    st = {table.p, lengths.p, refs.p, S, B, P, T, capacity, make_fastdiv(static_cast<uint32_t>(T))};
    w = {header.p, seg_free.p, seg_before.p, free_ids.p, live_ids.p, mark.p, len.p, rank.p, moves.p, map.p, segs(p)};
    mover = {buffers.p, static_cast<uint32_t>(bytes.size()), chunks, make_fastdiv(chunks), page_lane_bits(largest)};
  }
  static int32_t segs(int32_t p) { return (p + kSegment - 1) / kSegment; }

  Model snapshot() const {
    Model m{table.copy(), lengths.copy(), refs.copy(), {}};
    for (size_t i = 0; i < pools.size(); ++i) {
      m.pools.emplace_back();
      for (int32_t p = 0; p < P; ++p)
        m.pools[i].emplace_back(pools[i]->p + p * page_bytes[i], pools[i]->p + (p + 1) * page_bytes[i]);
    }
    return m;
  }
  void check(const Model& m, const char* what) {
    const Model now = snapshot();
    if (now.lengths != m.lengths) die(what, 1);
    if (now.refs != m.refs) die(what, 2);
    if (now.table != m.table) die(what, 3);
    if (now.pools != m.pools) die(what, 4);
    for (size_t i = 0; i < mark.n; ++i)
      if (mark[i]) die("a mark is left", i);
  }
  uint32_t status() {
    const uint32_t s = static_cast<uint32_t>(header[kPageStatus]);
    header[kPageStatus] = 0;
    return s;
  }
  template <class Move>
  void chunk(uint32_t item, uint32_t n, uint32_t tid, Move m, bool packed) {
    if (aligned && packed) page_move_chunk<Mem, true, true>(mover, m, n, item, tid);
    else if (aligned) page_move_chunk<Mem, true, false>(mover, m, n, item, tid);
    else if (packed) page_move_chunk<Mem, false, true>(mover, m, n, item, tid);
    else page_move_chunk<Mem, false, false>(mover, m, n, item, tid);
  }
  void move(std::mt19937_64& rng) {
    if (!header[kPageOk]) return;
    const bool packed = (1 << mover.lane_bits) < kPageThreads && rng() % 4;
    const uint32_t n = static_cast<uint32_t>(header[kPageMoves]), items = packed ? page_items<true>(mover, n) : page_items<false>(mover, n);
    const uint32_t blocks = 1 + static_cast<uint32_t>(rng() % 5);
    for (uint32_t b = 0; b < blocks; ++b)
      for (uint32_t item = b; item < items; item += blocks)
        for (uint32_t tid = 0; tid < kPageThreads; ++tid)
          chunk(item, n, tid, [&](uint32_t i) { return moves[i]; }, packed);
  }
};

int32_t blocks_of(int32_t tokens, int32_t T) { return (tokens + T - 1) / T; }

std::vector<int32_t> lowest_free(const Model& m) {
  std::vector<int32_t> f;
  for (size_t p = 0; p < m.refs.size(); ++p)
    if (m.refs[p] == 0) f.push_back(static_cast<int32_t>(p));
  return f;
}

uint32_t model_extend(const Cache& c, Model* m, const std::vector<int32_t>& s, const std::vector<int32_t>& n) {
  uint32_t bad = 0;
  std::set<int32_t> seen;
  int64_t need = 0;
  for (size_t e = 0; e < s.size(); ++e) {
    if (s[e] == MMR_PAGES_NONE) continue;
    if (s[e] < 0 || s[e] >= c.S) {
      bad |= MMR_PAGES_BAD_SEQUENCE;
      continue;
    }
    if (!seen.insert(s[e]).second) bad |= MMR_PAGES_REPEATED;
    const int32_t old = m->lengths[s[e]];
    if (n[e] < 0 || old < 0 || old > c.st.capacity || n[e] > c.st.capacity - old) {
      bad |= MMR_PAGES_TOO_LONG;
      continue;
    }
    need += blocks_of(old + n[e], c.T) - blocks_of(old, c.T);
    if (n[e] > 0 && old % c.T) {
      const int32_t page = m->table[static_cast<size_t>(s[e]) * c.B + old / c.T];
      if (page < 0 || page >= c.P) bad |= MMR_PAGES_BAD_PAGE;
      else if (m->refs[page] != 1) bad |= MMR_PAGES_SHARED_TAIL;
    }
  }
  const std::vector<int32_t> f = lowest_free(*m);
  if (need > static_cast<int64_t>(f.size())) bad |= MMR_PAGES_OUT_OF_PAGES;
  if (bad) return bad;
  size_t k = 0;
  for (size_t e = 0; e < s.size(); ++e) {
    if (s[e] == MMR_PAGES_NONE) continue;
    const int32_t old = m->lengths[s[e]];
    for (int32_t b = blocks_of(old, c.T); b < blocks_of(old + n[e], c.T); ++b) {
      m->table[static_cast<size_t>(s[e]) * c.B + b] = f[k];
      m->refs[f[k++]] = 1;
    }
    m->lengths[s[e]] = old + n[e];
  }
  return 0;
}

uint32_t model_fork(const Cache& c, Model* m, const std::vector<int32_t>& p, const std::vector<int32_t>& ch) {
  uint32_t bad = 0;
  std::set<int32_t> seen;
  size_t need = 0;
  const std::vector<int32_t> lengths = m->lengths;
  for (size_t e = 0; e < p.size(); ++e) {
    if (ch[e] == MMR_PAGES_NONE) continue;
    if (p[e] < 0 || p[e] >= c.S || ch[e] < 0 || ch[e] >= c.S) {
      bad |= MMR_PAGES_BAD_SEQUENCE;
      continue;
    }
    if (lengths[p[e]] < 0 || lengths[p[e]] > c.st.capacity) {
      bad |= MMR_PAGES_TOO_LONG;
      continue;
    }
    if (lengths[ch[e]] != 0) bad |= MMR_PAGES_NOT_EMPTY;
    if (!seen.insert(ch[e]).second) bad |= MMR_PAGES_REPEATED;
    if (lengths[p[e]] % c.T) {
      const int32_t page = m->table[static_cast<size_t>(p[e]) * c.B + lengths[p[e]] / c.T];
      if (page < 0 || page >= c.P) bad |= MMR_PAGES_BAD_PAGE;
      else ++need;  // (bad either way below)
    }
  }
  const std::vector<int32_t> f = lowest_free(*m);
  if (need > f.size()) bad |= MMR_PAGES_OUT_OF_PAGES;
  if (bad) return bad;
  size_t k = 0;
  for (size_t e = 0; e < p.size(); ++e) {
    if (ch[e] == MMR_PAGES_NONE) continue;
    const int32_t l = lengths[p[e]], full = l / c.T;
    const size_t from = static_cast<size_t>(p[e]) * c.B, to = static_cast<size_t>(ch[e]) * c.B;
    for (int32_t i = 0; i < full; ++i) {
      m->table[to + i] = m->table[from + i];
      m->refs[m->table[from + i]] += 1;
    }
    if (l % c.T) {
      for (auto& pool : m->pools) pool[f[k]] = pool[m->table[from + full]];
      m->table[to + full] = f[k];
      m->refs[f[k++]] = 1;
    }
    m->lengths[ch[e]] = l;
  }
  return 0;
}

uint32_t model_free(const Cache& c, Model* m, const std::vector<int32_t>& s) {
  uint32_t bad = 0;
  for (int32_t q : s) {
    if (q == MMR_PAGES_NONE) continue;
    if (q < 0 || q >= c.S) {
      bad |= MMR_PAGES_BAD_SEQUENCE;
      continue;
    }
    for (int32_t i = 0; i < blocks_of(m->lengths[q], c.T); ++i) m->refs[m->table[static_cast<size_t>(q) * c.B + i]] -= 1;
    m->lengths[q] = 0;
  }
  return bad;
}

void model_compact(const Cache& c, Model* m) {
  int32_t live = 0;
  for (int32_t r : m->refs) live += r != 0;
  std::vector<int32_t> name(c.P);
  int32_t dst = 0;
  for (int32_t p = 0; p < c.P; ++p) {
    name[p] = p;
    if (p < live || m->refs[p] == 0) continue;
    while (m->refs[dst] != 0) ++dst;
    name[p] = dst;
    for (auto& pool : m->pools) pool[dst] = pool[p];
    m->refs[dst] = m->refs[p];
    m->refs[p] = 0;
  }
  for (int32_t s = 0; s < c.S; ++s)
    for (int32_t i = 0; i < blocks_of(m->lengths[s], c.T); ++i) {
      int32_t& id = m->table[static_cast<size_t>(s) * c.B + i];
      id = name[id];
    }
}

uint32_t model_copy(const Cache& c, Model* m, const std::vector<int32_t>& s, const std::vector<int32_t>& d) {
  uint32_t bad = 0;
  std::set<int32_t> dsts;
  for (size_t e = 0; e < s.size(); ++e) {
    if (d[e] == MMR_PAGES_NONE) continue;
    if (s[e] < 0 || s[e] >= c.P || d[e] < 0 || d[e] >= c.P) bad |= MMR_PAGES_BAD_PAGE;
    else if (s[e] != d[e] && !dsts.insert(d[e]).second) bad |= MMR_PAGES_REPEATED;
  }
  for (size_t e = 0; e < s.size(); ++e)
    if (s[e] >= 0 && s[e] < c.P && d[e] >= 0 && d[e] < c.P && s[e] != d[e] && dsts.count(s[e])) bad |= MMR_PAGES_OVERLAP;
  if (bad) return bad;
  for (auto& pool : m->pools) {
    const auto before = pool;
    for (size_t e = 0; e < s.size(); ++e)
      if (d[e] != MMR_PAGES_NONE) pool[d[e]] = before[s[e]];
  }
  return 0;
}

void scan(const Cache& c, bool live) {
  if (c.w.n_segments <= kPlanScans) return;
  launch<K>(static_cast<uint32_t>(c.w.n_segments), [&](Lanes<K>& x) { page_scan_segment(x, c.st, c.w, static_cast<int32_t>(x.block), live); });
}

void cache_case(uint64_t seed) {
  std::mt19937_64 rng(seed);
  auto pick = [&](int32_t lo, int32_t hi) { return lo + static_cast<int32_t>(rng() % static_cast<uint64_t>(hi - lo + 1)); };
  const int32_t T = pick(1, 3) == 1 ? 1 : pick(2, 9), S = pick(1, 40);
  const bool big = pick(0, 11) == 0;  // enough pages for the second launch of extend to have work
  const int32_t B = big ? 400 : pick(1, 12), P = big ? pick(5000, 9000) : pick(1, 260);
  std::vector<uint64_t> bytes;
  const int kind = big ? 2 : pick(0, 3);
  for (int i = pick(1, 3); i > 0; --i)
    bytes.push_back(kind == 0 ? 16u * pick(1, 40) : kind == 1 ? 16u * pick(500, 600) : kind == 2 ? pick(1, 40) : pick(8190, 8300));
  Cache c(S, B, P, T, bytes);
  for (auto& p : c.pools)
    for (size_t i = 0; i < p->n; ++i) (*p)[i] = static_cast<char>(rng());
  for (int step = 0; step < 14; ++step) {
    Model m = c.snapshot();
    const int op = pick(0, 4);
    const bool wild = pick(0, 5) == 0;  // entries at random, bad ones among them
    std::vector<int32_t> a, b;
    std::vector<int32_t> seqs(S);
    for (int32_t i = 0; i < S; ++i) seqs[i] = i;
    std::shuffle(seqs.begin(), seqs.end(), rng);
    if (op == 0 || op == 1) {
      int n = pick(0, S);
      for (int e = 0; e < n; ++e) {
        a.push_back(wild ? pick(-2, S) : pick(0, 9) ? seqs[e] : MMR_PAGES_NONE);
        const int32_t room = c.st.capacity - std::min(c.st.capacity, c.lengths[seqs[e]]);
        b.push_back(wild ? pick(-1, 2 * T) : pick(0, std::max(0, room) ? std::min(room, pick(0, 2) ? 2 * T : B * T) : 0));
      }
      const uint32_t want = model_extend(c, &m, a, b);
      Exact<int32_t> sa(a.size()), sb(b.size());
      std::copy(a.begin(), a.end(), sa.p);
      std::copy(b.begin(), b.end(), sb.p);
      std::vector<int32_t> shared(kMaxPageSegments);
      const bool whole = pick(0, 1);
      if (n) {
        scan(c, false);
        launch<K>(1, [&](Lanes<K>& x) { page_extend_plan(x, c.st, c.w, shared.data(), sa.p, sb.p, n, whole); });
        if (!whole)
          launch<8>(3, [&](Lanes<8>& x) { page_extend_rows<Lanes<8>, kSegment>(x, c.st, c.w, shared.data(), sa.p, sb.p, n); });
      }
      if (c.status() != want) die("extend: status", want, seed);
      c.check(m, "extend");
    } else if (op == 2) {
      std::vector<int32_t> empty;
      for (int32_t q : seqs)
        if (c.lengths[q] == 0) empty.push_back(q);
      const int n = wild ? pick(0, S) : pick(0, static_cast<int32_t>(empty.size()));
      for (int e = 0; e < n; ++e) {
        a.push_back(pick(wild ? -1 : 0, wild ? S : S - 1));
        b.push_back(wild ? pick(-2, S) : pick(0, 9) ? empty[e] : MMR_PAGES_NONE);
      }
      const uint32_t want = model_fork(c, &m, a, b);
      Exact<int32_t> sa(a.size()), sb(b.size());
      std::copy(a.begin(), a.end(), sa.p);
      std::copy(b.begin(), b.end(), sb.p);
      std::vector<int32_t> shared(kMaxPageSegments);
      if (n) {
        scan(c, false);
        launch<K>(1, [&](Lanes<K>& x) { page_fork_plan(x, c.st, c.w, shared.data(), sa.p, sb.p, n); });
        if (c.header[kPageOk]) {
          const uint32_t rows = 1 + static_cast<uint32_t>(rng() % 4);
          launch<K>(rows, [&](Lanes<K>& x) { page_fork_rows(x, c.st, c.w, sa.p, sb.p, n, x.block, x.blocks); });
        }
        c.move(rng);
      }
      const uint32_t got = c.status();
      if (got != want) die("fork: status", want, got);
      c.check(m, "fork");
    } else if (op == 3) {
      const int n = pick(0, S);
      for (int e = 0; e < n; ++e) a.push_back(wild ? pick(-2, S) : pick(-1, 0) ? MMR_PAGES_NONE : seqs[pick(0, S - 1)]);
      const uint32_t want = model_free(c, &m, a);
      Exact<int32_t> sa(a.size());
      std::copy(a.begin(), a.end(), sa.p);
      int32_t shared[1];
      if (n) launch<K>(n, [&](Lanes<K>& x) { page_free(x, c.st, c.w, shared, sa.p); });
      if (c.status() != want) die("free: status", want, seed);
      c.check(m, "free");
    } else if (pick(0, 1)) {
      model_compact(c, &m);
      std::vector<int32_t> shared(kMaxPageSegments);
      const bool whole = pick(0, 1);
      scan(c, true);
      launch<K>(1, [&](Lanes<K>& x) { page_compact_plan(x, c.st, c.w, shared.data(), whole); });
      if (!whole) launch<8>(3, [&](Lanes<8>& x) { page_compact_list<Lanes<8>, kSegment>(x, c.st, c.w, shared.data()); });
      const uint32_t rows = 1 + static_cast<uint32_t>(rng() % 4);
      launch<K>(rows, [&](Lanes<K>& x) { page_compact_rows(x, c.st, c.w, x.block, x.blocks); });
      c.move(rng);
      if (c.status()) die("compact: status");
      // compact leaves old contents in the pages it moved away from
      c.check(m, "compact");
    } else {
      const int n = pick(0, P);
      std::vector<int32_t> ids(P);
      for (int32_t i = 0; i < P; ++i) ids[i] = i;
      std::shuffle(ids.begin(), ids.end(), rng);
      const int32_t cut = pick(0, P);  // sources from one side, destinations from the other
      for (int e = 0; e < n && (wild || (cut > 0 && cut + e < P)); ++e) {
        a.push_back(wild ? pick(-1, P) : pick(0, 9) == 0 ? ids[cut + e] : ids[pick(0, cut - 1)]);
        b.push_back(wild ? pick(-2, P) : pick(0, 9) ? ids[cut + e] : MMR_PAGES_NONE);
      }
      const uint32_t want = model_copy(c, &m, a, b);
      const int32_t count = static_cast<int32_t>(a.size());
      Exact<int32_t> sa(a.size()), sb(b.size());
      std::copy(a.begin(), a.end(), sa.p);
      std::copy(b.begin(), b.end(), sb.p);
      if (count && count <= kFewPairs && pick(0, 1)) {
        int32_t pairs[2 * kFewPairs];
        const uint32_t items = static_cast<uint32_t>(count) * c.mover.n_buffers * c.mover.chunks;
        std::vector<char> ok(std::min(items, 5u));  // the first workgroups check, one after the other
        launch<kFewPairs>(static_cast<uint32_t>(ok.size()), [&](Lanes<kFewPairs>& x) {
          const bool go = page_copy_few(x, c.st, c.w, pairs, sa.p, sb.p, count);
          if (x.tid == 0) ok[x.block] = go;
        });
        for (char g : ok)
          if (g != ok[0]) die("workgroups disagree");
        for (uint32_t item = 0; ok[0] && item < items; ++item)
          for (uint32_t t = 0; t < static_cast<uint32_t>(kPageThreads); ++t)
            c.chunk(item, static_cast<uint32_t>(count), t, [&](uint32_t i) { return PageMove{pairs[i], pairs[kFewPairs + i]}; }, false);
      } else if (count) {
        const bool sorted = pick(0, 1);
        launch<K>(1, [&](Lanes<K>& x) { page_copy_plan(x, c.st, c.w, sa.p, sb.p, count, sorted); });
        c.move(rng);
      }
      if (c.status() != want) die("copy: status", want, seed);
      c.check(m, "copy");
    }
  }
  std::vector<int32_t> shared(kMaxPageSegments);
  scan(c, false);
  launch<K>(1, [&](Lanes<K>& x) { page_count(x, c.st, c.w, shared.data()); });
  int32_t live = 0;
  for (int32_t i = 0; i < P; ++i) live += c.refs[i] != 0;
  if (c.header[kPageLive] != live) die("count", live, c.header[kPageLive]);
}

// Tables that are out of step with themselves: nothing may be touched out of bounds, and the status says so.
void corrupt_case(uint64_t seed) {
  std::mt19937_64 rng(seed);
  const int32_t S = 7, B = 5, P = 90, T = 3;
  Cache c(S, B, P, T, {48});
  for (int32_t s = 0; s < S; ++s) c.lengths[s] = static_cast<int32_t>(rng() % 24) - 4 + (s == 0 ? 1000000 : 0);
  for (size_t i = 0; i < c.table.n; ++i) c.table[i] = static_cast<int32_t>(rng() % 120) - 15;
  for (int32_t p = 0; p < P; ++p) c.refs[p] = static_cast<int32_t>(rng() % 4) - 1;
  std::vector<int32_t> shared(kMaxPageSegments);
  Exact<int32_t> a(S), b(S);
  for (int32_t s = 0; s < S; ++s) a[s] = s, b[s] = (s + 1) % S;
  scan(c, false);
        launch<K>(1, [&](Lanes<K>& x) { page_extend_plan(x, c.st, c.w, shared.data(), a.p, b.p, S, true); });
  scan(c, false);
        launch<K>(1, [&](Lanes<K>& x) { page_fork_plan(x, c.st, c.w, shared.data(), a.p, b.p, S); });
  if (c.header[kPageOk]) die("a corrupt fork is taken");
  scan(c, true);
      launch<K>(1, [&](Lanes<K>& x) { page_compact_plan(x, c.st, c.w, shared.data(), true); });
  launch<K>(3, [&](Lanes<K>& x) { page_compact_rows(x, c.st, c.w, x.block, x.blocks); });
  c.move(rng);
  launch<K>(S, [&](Lanes<K>& x) { page_free(x, c.st, c.w, shared.data(), a.p); });
  if (!(c.status() & (MMR_PAGES_TOO_LONG | MMR_PAGES_BAD_PAGE))) die("corrupt tables pass");
  for (int32_t s = 0; s < S; ++s)
    if (c.lengths[s] != 0) die("free left a length");
}

template <class T>
double value_of(const char* p) {
  if constexpr (T::kBytes == 1) return 0;
  else if constexpr (T::kBytes == 4) return T::get(Mem::loadu<uint32_t>(p));
  else return T::get(Mem::loadu<uint16_t>(p));
}

// Rotation of random shapes, paged or not, against the formula in 64 bits.
template <class T, int VEC, bool INTERLEAVED>
void rotary_case(uint64_t seed, double eps) {
  std::mt19937_64 rng(seed);
  auto pick = [&](int32_t lo, int32_t hi) { return lo + static_cast<int32_t>(rng() % static_cast<uint64_t>(hi - lo + 1)); };
  constexpr bool kWide = VEC * T::kBytes == 16, kRaw = T::kBytes == 1;
  const int half = kRaw ? 0 : (INTERLEAVED ? VEC / 2 : VEC) * pick(1, VEC == 1 ? 9 : 4);
  const int dim = kWide ? (2 * half + VEC - 1) / VEC * VEC + VEC * pick(kRaw, 3) : 2 * half + pick(kRaw, pick(0, 1) ? 40 : 5);
  const int outer = pick(1, 2), seq = pick(1, 40), heads = pick(1, 11), paged = pick(0, 2);
  const bool in_place = !kRaw && paged != 1 && pick(0, 2) == 0, turn = !kRaw && !(paged && pick(0, 3) == 0), spread = pick(0, 1);
  const bool heads_minor = paged || pick(0, 1);
  const int tokens = paged ? seq : outer * seq;
  Exact<uint64_t> freq(std::max(half, 1));
  for (int i = 0; i < half; ++i) freq[i] = static_cast<uint64_t>(std::ldexp(std::pow(100.0, -static_cast<double>(i) / half) / 6.283185307179586, 62)) * 4;
  const int64_t row = static_cast<int64_t>(dim) * T::kBytes;
  RotaryAngles a{};
  RotaryPages pages{};
  RotaryShape j{};
  RotaryBuffer buf{};
  a.frequency = freq.p;
  a.magnitude = 1.25f;
  a.sine = pick(0, 1) ? 1.25f : -1.25f;
  a.half = half;
  Exact<char> x(static_cast<size_t>(tokens) * heads * row);
  std::normal_distribution<float> normal;
  for (int64_t i = 0; i < static_cast<int64_t>(tokens) * heads * dim; ++i) {
    const uint32_t v = kRaw ? static_cast<uint32_t>(rng()) : T::put(normal(rng));
    std::memcpy(x.p + i * T::kBytes, &v, T::kBytes);
  }
  j.tokens = tokens, j.seq = seq, j.heads = heads, j.paged = paged;
  j.src_head = heads_minor ? row : row * seq;
  j.src_seq = heads_minor ? row * heads : row;
  j.src_outer = row * heads * seq;
  // pages
  const int32_t Tk = pick(1, 5), n = pick(1, 6), S = n + 2, B = 12, P = S * B;
  Exact<int32_t> table(S * B), lengths(S), slots(n), begins(n + 1), status(1), positions(tokens);
  Exact<char> pool(paged == 1 ? static_cast<size_t>(P) * Tk * heads * row : 0), out(paged == 1 || in_place ? 0 : x.n, 0x11);
  std::vector<int32_t> where(tokens, -1), page_of(tokens, -1), row_of(tokens, 0);
  buf.src = x.p;
  uint32_t want_status = 0;
  if (paged) {
    std::vector<int32_t> ids(P);
    for (int i = 0; i < P; ++i) ids[i] = i;
    std::shuffle(ids.begin(), ids.end(), rng);
    std::copy(ids.begin(), ids.end(), table.p);
    std::vector<int32_t> order(S);
    for (int i = 0; i < S; ++i) order[i] = i;
    std::shuffle(order.begin(), order.end(), rng);
    std::vector<int32_t> cuts(n + 1);
    for (auto& q : cuts) q = pick(0, seq);
    std::sort(cuts.begin(), cuts.end());
    for (int e = 0; e <= n; ++e) begins[e] = cuts[e];
    for (int e = 0; e < n; ++e) {
      slots[e] = pick(0, 12) == 0 ? (pick(0, 1) ? -2 : S) : pick(0, 12) == 0 ? MMR_PAGES_NONE : order[e];
      const int32_t count = begins[e + 1] - begins[e];
      if (slots[e] >= 0 && slots[e] < S) {
        lengths[slots[e]] = count + pick(0, 9);
        if (pick(0, 9) == 0) table[slots[e] * B] = pick(0, 1) ? -3 : P;
      }
      for (int32_t t = begins[e]; t < begins[e + 1]; ++t) {
        if (slots[e] < 0 || slots[e] >= S) {
          if (slots[e] != MMR_PAGES_NONE) want_status |= MMR_PAGES_BAD_SEQUENCE;
          continue;
        }
        const int32_t p = lengths[slots[e]] - count + (t - begins[e]);
        if (p < 0 || p >= B * Tk) {
          want_status |= MMR_PAGES_TOO_LONG;
          continue;
        }
        const int32_t page = table[slots[e] * B + p / Tk];
        if (page < 0 || page >= P) {
          want_status |= MMR_PAGES_BAD_PAGE;
          continue;
        }
        where[t] = p, page_of[t] = page, row_of[t] = p % Tk;
      }
    }
    pages = {table.p, lengths.p, slots.p, begins.p, status.p, n, S, B, P, Tk, B * Tk, make_fastdiv(static_cast<uint32_t>(Tk))};
    buf.dst = paged == 1 ? pool.p : in_place ? x.p : out.p;
    if (paged == 1) j.dst_outer = Tk * heads * row, j.dst_seq = heads * row, j.dst_head = row;
    else j.dst_seq = j.src_seq, j.dst_head = j.src_head;
  } else {
    buf.dst = in_place ? x.p : out.p;
    j.dst_outer = j.src_outer, j.dst_seq = j.src_seq, j.dst_head = j.src_head;
    const bool given = pick(0, 1);
    buf.base = pick(-100, 1000000);
    j.pos_outer = seq, j.pos_seq = 1;
    if (given) buf.positions = positions.p;
    for (int t = 0; t < tokens; ++t) {
      positions[t] = pick(-5, 70000);
      where[t] = given ? positions[t] : static_cast<int32_t>(buf.base + t % seq);
    }
  }
  const auto before = x.copy();
  const bool same = buf.dst == x.p;
  rotary_units(&j, static_cast<uint32_t>(row), turn ? static_cast<uint32_t>(2 * half * T::kBytes) : 0,
               static_cast<uint32_t>(VEC * T::kBytes * (INTERLEAVED ? 1 : 2)), T::kBytes, turn && same);
  rotary_shape(&j, j.src_head <= j.src_seq, spread);
  // in some cases a part of the tile is padding, which stays as it is
  buf.outer = paged ? 1 : pick(1, outer), buf.seq = paged || pick(0, 1) ? seq : pick(1, seq), buf.heads = pick(0, 1) ? heads : pick(1, heads);
  for (uint32_t b = 0; b < j.blocks; ++b)  // its lanes wait for nothing, so that one thread can be all of them in turn
    for (int32_t t = 0; t < kRotaryThreads; ++t) {
      Lanes<kRotaryThreads> l{t, b, j.blocks, nullptr};
      rotary_block<Mem, T, VEC, INTERLEAVED>(l, a, pages, j, buf);
    }
  if (static_cast<uint32_t>(status[0]) != want_status) die("rotary: status", want_status, status[0]);
  std::set<std::pair<int32_t, int32_t>> written;
  for (int t = 0; t < tokens; ++t)
    for (int h = 0; h < heads; ++h) {
      const int64_t at = (t / seq) * j.src_outer + (t % seq) * j.src_seq + h * j.src_head;
      const char* to;
      const bool pad = static_cast<uint32_t>(h) >= buf.heads || static_cast<uint32_t>(t % seq) >= buf.seq || static_cast<uint32_t>(t / seq) >= buf.outer;
      const bool skip = (paged && page_of[t] < 0) || pad;
      if (paged == 1) {
        if (skip) continue;
        to = pool.p + page_of[t] * j.dst_outer + row_of[t] * j.dst_seq + h * j.dst_head;
      } else {
        to = (same ? x.p : out.p) + at;
      }
      for (int d = 0; d < dim; ++d) {
        if (skip) {
          const char old = same ? before[at + d * T::kBytes] : 0x11;
          if (to[d * T::kBytes] != old) die("a skipped row is written", t, d);
          continue;
        }
        if (!turn || d >= 2 * half) {
          if (std::memcmp(to + d * T::kBytes, before.data() + at + d * T::kBytes, T::kBytes)) die("a value that passes through changed", t, d);
          continue;
        }
        const double own = value_of<T>(before.data() + at + d * T::kBytes);
        const int i = INTERLEAVED ? d / 2 : d % half;
        const bool second = INTERLEAVED ? d % 2 : d >= half;
        const int other = INTERLEAVED ? d ^ 1 : second ? d - half : d + half;
        const double y = value_of<T>(before.data() + at + other * T::kBytes);
        const double turns = std::ldexp(static_cast<double>(static_cast<int64_t>(static_cast<uint64_t>(static_cast<int64_t>(where[t])) * freq[i])), -64);
        const double c = 1.25 * std::cos(turns * 6.283185307179586476925), s = a.sine * std::sin(turns * 6.283185307179586476925);
        const double want = second ? own * c + y * s : own * c - y * s;
        const double got = value_of<T>(to + d * T::kBytes);
        // half a step of the type; 4 roundings of 2^-24 and the angle's 2^-24 on each product
        const double tol = eps / 2 * std::fabs(want) + 1.25 * 8 * 5.97e-8 * (std::fabs(own) + std::fabs(y)) + (T::kBytes == 2 ? 6e-8 : 0);
        if (std::fabs(got - want) > tol) die("rotary value", t, d);
      }
    }
}

// turn_sincos over the circle against the C library in 64 bits
void sincos_case() {
  double worst = 0;
  for (uint64_t i = 0; i < 2000003; ++i) {
    const uint32_t turns = static_cast<uint32_t>(i * 2147000911u + 17);
    float s, c;
    turn_sincos(turns, &s, &c);
    const double a = std::ldexp(static_cast<double>(turns), -32) * 6.283185307179586476925;
    worst = std::max({worst, std::fabs(s - std::sin(a)), std::fabs(c - std::cos(a))});
  }
  std::printf("sincos: largest error %.3g\n", worst);
  // 2^-25 of the rest's rounding (times pi/4), 2^-24.5 of the last addition, the cut-off terms: under 2^-23
  if (worst > 1.2e-7) die("sincos");
}

}  // namespace

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? std::atoi(argv[1]) : 40;
  sincos_case();
  for (int i = 0; i < rounds; ++i) cache_case(1000 + i);
  std::printf("page operators: %d sweeps\n", rounds);
  for (int i = 0; i < rounds / 4 + 1; ++i) corrupt_case(5000 + i);
  std::printf("corrupt tables: %d\n", rounds / 4 + 1);
  std::fflush(stdout);
  int shapes = 0;
  for (int i = 0; i < rounds / 4 + 1; ++i) {
    const auto seed = [&] { return static_cast<uint64_t>(++shapes); };
    rotary_case<RotaryF32, 4, false>(seed(), 1.2e-7);
    rotary_case<RotaryF32, 4, true>(seed(), 1.2e-7);
    rotary_case<RotaryF32, 2, false>(seed(), 1.2e-7);
    rotary_case<RotaryF32, 2, true>(seed(), 1.2e-7);
    rotary_case<RotaryF32, 1, false>(seed(), 1.2e-7);
    rotary_case<RotaryBF16, 8, false>(seed(), 0.0078125);
    rotary_case<RotaryBF16, 8, true>(seed(), 0.0078125);
    rotary_case<RotaryBF16, 4, false>(seed(), 0.0078125);
    rotary_case<RotaryBF16, 4, true>(seed(), 0.0078125);
    rotary_case<RotaryBF16, 2, false>(seed(), 0.0078125);
    rotary_case<RotaryBF16, 2, true>(seed(), 0.0078125);
    rotary_case<RotaryBF16, 1, false>(seed(), 0.0078125);
    rotary_case<RotaryF16, 8, false>(seed(), 0.0009765625);
    rotary_case<RotaryF16, 2, true>(seed(), 0.0009765625);
    rotary_case<RotaryRaw, 16, false>(seed(), 0);
    rotary_case<RotaryRaw, 1, false>(seed(), 0);
  }
  std::printf("rotary: %d shapes\nOK\n", shapes);
  return 0;
}
