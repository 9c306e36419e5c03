// Tables that are out of step with themselves, for tests only: one fault a case in an otherwise valid call, with the
// exact status, tables and pages that the call must leave.  The kernels' per-workgroup routines with host threads as
// lanes, on buffers of exactly their size, as in page_sweep.cc, whose cache this builds on.
#define main page_sweep_main
#include "page_sweep.cc"
#undef main

namespace {

struct FaultCase {
  Cache c;
  std::vector<int32_t> shared = std::vector<int32_t>(kMaxPageSegments);
  std::mt19937_64 rng{1};
  bool prepared;  // which form of the call: see page_fork_plan

  // 4 tokens a page, 8 sequences of up to 6 pages; no two pages hold the same.
  FaultCase(int32_t P, bool prepared_) : c(8, 6, P, 4, {48, 5}), prepared(prepared_) {
    for (auto& pool : c.pools)
      for (int32_t p = 0; p < P; ++p)
        for (size_t i = 0; i < pool->n / P; ++i) (*pool)[p * (pool->n / P) + i] = static_cast<char>(i < 2 ? p >> (8 * i) : i);
  }
  // Sequence s holds `tokens` in the pages `row`, each with a user more.
  void holds(int32_t s, int32_t tokens, const std::vector<int32_t>& row) {
    c.lengths[s] = tokens;
    for (size_t i = 0; i < row.size(); ++i) {
      at(s, static_cast<int32_t>(i)) = row[i];
      if (row[i] >= 0 && row[i] < c.P) c.refs[row[i]] += 1;
    }
  }
  int32_t& at(int32_t s, int32_t i) { return c.table[static_cast<size_t>(s) * c.B + i]; }
  void expect(const char* what, uint32_t status, const Model& m) {
    const uint32_t got = c.status();
    if (got != status) die(what, status, got);
    c.check(m, what);
  }
  void fork(const std::vector<int32_t>& parents, const std::vector<int32_t>& children) {
    const int32_t n = static_cast<int32_t>(parents.size());
    Exact<int32_t> a(n), b(n);
    std::copy(parents.begin(), parents.end(), a.p);
    std::copy(children.begin(), children.end(), b.p);
    if (prepared) {
      const uint32_t segments = static_cast<uint32_t>(c.w.n_segments), checks = 1 + static_cast<uint32_t>(rng() % n);
      launch<K>(segments, [&](Lanes<K>& x) { page_scan_segment(x, c.st, c.w, static_cast<int32_t>(x.block), false); });
      launch<K>(checks, [&](Lanes<K>& x) { page_fork_check(x, c.st, c.w, a.p, b.p, n, x.block, x.blocks); });
    } else {
      scan(c, false);
    }
    launch<K>(1, [&](Lanes<K>& x) { page_fork_plan(x, c.st, c.w, shared.data(), a.p, b.p, n, prepared); });
    if (c.header[kPageForkBad]) die("what the check found is left");
    if (!c.header[kPageOk]) return;
    launch<K>(2, [&](Lanes<K>& x) { page_fork_rows(x, c.st, c.w, a.p, b.p, n, x.block, x.blocks); });
    c.move(rng);
  }
  void compact(bool whole) {
    scan(c, true);
    launch<K>(1, [&](Lanes<K>& x) { page_compact_plan(x, c.st, c.w, shared.data(), whole); });
    if (!whole) launch<8>(3, [&](Lanes<8>& x) { page_compact_list<Lanes<8>, kSegment>(x, c.st, c.w, shared.data()); });
    launch<K>(3, [&](Lanes<K>& x) { page_compact_rows(x, c.st, c.w, x.block, x.blocks); });
    c.move(rng);
  }
};

// A fork whose parent's row names a page that is not there, or that nobody uses, changes nothing and says so.
void fork_cases(int32_t P, bool prepared) {
  for (const int32_t last : {0, 2}) {  // the parent's last page is full, or holds two of four tokens
    for (int32_t i = 0; i < (last ? 3 : 2); ++i) {
      for (const int32_t bad : {-1, -5, P, P + 1000, 2147483647}) {
        FaultCase f(P, prepared);
        f.holds(0, 5, {3, 4});
        f.holds(1, 8 + last, last ? std::vector<int32_t>{8, 9, 10} : std::vector<int32_t>{8, 9});
        f.c.refs[f.at(1, i)] = 0;
        f.at(1, i) = bad;
        const Model m = f.c.snapshot();
        f.fork({0, 1, 0}, {2, 3, 4});
        f.expect("fork: an id outside the pool", MMR_PAGES_BAD_PAGE, m);
      }
      for (const int32_t users : {0, -2}) {
        FaultCase f(P, prepared);
        f.holds(0, 5, {3, 4});
        f.holds(1, 8 + last, last ? std::vector<int32_t>{0, 1, 2} : std::vector<int32_t>{0, 1});
        f.c.refs[f.at(1, i)] = users;  // the lowest free page, the first to be given out
        const Model m = f.c.snapshot();
        f.fork({0, 1}, {2, 3});
        f.expect("fork: a page that nobody uses", MMR_PAGES_BAD_COUNT, m);
      }
    }
  }
  // what stands behind the parent's tokens, in entries that are none, and in other rows means nothing
  FaultCase f(P, prepared);
  f.holds(0, 6, {3, 4});
  f.at(0, 2) = -7;
  f.holds(1, 6, {-9, -1});
  Model m = f.c.snapshot();
  if (model_fork(f.c, &m, {0, 1}, {2, MMR_PAGES_NONE})) die("fork: the model refuses");
  f.fork({0, 1}, {2, MMR_PAGES_NONE});
  f.expect("fork: a valid one beside bad rows", 0, m);
}

// A row that names a page nobody uses keeps that id through a compact, everything else moves, and the status tells.
void compact_cases(int32_t P, bool whole) {
  struct Fault {
    int32_t id;
    uint32_t flag;
  };
  // 7 pages are in use, so 0 .. 6 are live afterwards: pages 0, 2, 4 and 5 are given to the pages beyond
  for (const Fault fault : {Fault{0, MMR_PAGES_BAD_COUNT}, Fault{4, MMR_PAGES_BAD_COUNT}, Fault{5, MMR_PAGES_BAD_COUNT},
                            Fault{7, MMR_PAGES_BAD_COUNT}, Fault{P - 1, MMR_PAGES_BAD_COUNT}, Fault{P, MMR_PAGES_BAD_PAGE},
                            Fault{-1, MMR_PAGES_BAD_PAGE}, Fault{6, 0}, Fault{P - 2, 0}}) {
    FaultCase f(P, false);
    f.holds(0, 14, {1, P - 2, 8, 3});
    f.holds(3, 9, {P - 3, 6, P - 5});
    f.compact(whole);  // so that what the calls below find from earlier ones is not zeros
    if (f.c.status()) die("compact: a valid one");
    for (size_t i = 0; i < f.c.table.n; ++i) f.c.table[i] = 0x7b7b7b7b;
    for (int32_t i = 0; i < P; ++i) f.c.refs[i] = 0;
    f.holds(0, 14, {1, P - 2, 8, 3});
    f.holds(3, 9, {P - 3, 6, P - 5});
    f.c.lengths[5] = 4;
    f.at(5, 0) = fault.id;
    Model m = f.c.snapshot();
    int32_t& id = m.table[5 * static_cast<size_t>(f.c.B)];
    if (fault.flag == MMR_PAGES_BAD_PAGE) id = 0;
    model_compact(f.c, &m);
    if (fault.flag) id = fault.id;
    f.compact(whole);
    f.expect("compact: a row in error", fault.flag, m);
  }
}

// What free takes from a row in error, beside what is right.
void free_cases(int32_t P) {
  auto run = [&](FaultCase& f, const std::vector<int32_t>& a) {
    Exact<int32_t> ids(a.size());
    std::copy(a.begin(), a.end(), ids.p);
    launch<K>(static_cast<uint32_t>(a.size()), [&](Lanes<K>& x) { page_free(x, f.c.st, f.c.w, f.shared.data(), ids.p); });
  };
  for (const int32_t bad : {-1, P, 2147483647}) {
    FaultCase f(P, false);
    f.holds(2, 12, {4, 9, 6});
    f.c.refs[9] = 0;
    f.at(2, 1) = bad;
    Model m = f.c.snapshot();
    m.lengths[2] = m.refs[4] = m.refs[6] = 0;
    run(f, {2, 2});
    f.expect("free: an id outside the pool", MMR_PAGES_BAD_PAGE, m);
  }
  for (const int32_t users : {0, -3}) {
    FaultCase f(P, false);
    f.holds(2, 12, {4, 9, 6});
    f.c.refs[9] = users;
    Model m = f.c.snapshot();
    m.lengths[2] = m.refs[4] = m.refs[6] = 0;
    run(f, {2});
    f.expect("free: a page that nobody uses", MMR_PAGES_BAD_COUNT, m);
  }
  FaultCase f(P, false);  // three rows name page 9, which has two users
  f.holds(2, 12, {4, 9, 6});
  f.holds(1, 6, {9, 7});
  f.holds(0, 2, {9});
  f.c.refs[9] = 2;
  Model m = f.c.snapshot();
  for (int32_t page : {4, 9, 6, 7}) m.refs[page] = 0;
  for (int32_t s : {0, 1, 2}) m.lengths[s] = 0;
  run(f, {0, 1, 2});
  f.expect("free: more rows than users", MMR_PAGES_BAD_COUNT, m);
}

// An extend into a partly filled page that is not there, or whose only user is not this sequence.
void extend_cases(int32_t P) {
  struct Fault {
    int32_t id, users;
    uint32_t flag;
  };
  for (const Fault fault : {Fault{-1, 1, MMR_PAGES_BAD_PAGE}, Fault{P, 1, MMR_PAGES_BAD_PAGE}, Fault{9, 0, MMR_PAGES_SHARED_TAIL},
                            Fault{9, 2, MMR_PAGES_SHARED_TAIL}}) {
    FaultCase f(P, false);
    f.holds(2, 6, {4, 9});
    f.c.refs[9] = fault.users;
    f.at(2, 1) = fault.id;
    const Model m = f.c.snapshot();
    Exact<int32_t> a(2), b(2);
    a[0] = 0, b[0] = 5, a[1] = 2, b[1] = 1;
    scan(f.c, false);
    launch<K>(1, [&](Lanes<K>& x) { page_extend_plan(x, f.c.st, f.c.w, f.shared.data(), a.p, b.p, 2, true); });
    f.expect("extend: a bad last page", fault.flag, m);
  }
}

}  // namespace

int main() {
  for (const int32_t P : {24, 3 * kSegment + 9})
    for (const bool form : {false, true}) {
      fork_cases(P, form);
      compact_cases(P, form);
      free_cases(P);
      extend_cases(P);
    }
  std::printf("OK\n");
  return 0;
}
