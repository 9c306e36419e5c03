// Page cache and rotary positions: argument checks and launches of the C entry points.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <limits>
#include <new>
#include <set>
#include <vector>

#include "context_access.h"
#include "page_kernels.h"

using mmr::fail;
using mmr::Side;

#define MMR_HIP(expr)                                                                             \
  do {                                                                                            \
    hipError_t e_ = (expr);                                                                       \
    if (e_ != hipSuccess)                                                                         \
      return fail(e_ == hipErrorOutOfMemory ? MMR_OUT_OF_MEMORY : MMR_HIP_ERROR, "%s failed: %s", #expr, \
                  hipGetErrorString(e_));                                                         \
  } while (0)

struct mmr_pages : mmr::Attachment {
  struct Pool {
    int64_t id;
    Side side;
    std::vector<char*> tiles;  // buffers the device table was written with
  };
  std::vector<Pool> pools;
  int64_t table_id = 0, lengths_id = 0, refs_id = 0;
  mmr::PageState state{};
  mmr::PageWork work{};
  mmr::PageMoveLaunch move{};
  char* block = nullptr;  // workspace and buffer table
  size_t capacity = 0;
  size_t buffers_at = 0;
  uint64_t epoch = 0;
  ~mmr_pages() override {
    if (block) mmr::context_give_block(owner, block, capacity);
  }
};

struct mmr_rotary : mmr::Attachment {
  int32_t dim = 0;  // R
  bool interleaved = false;
  float magnitude = 1.0f;
  char* block = nullptr;  // R / 2 frequencies
  size_t capacity = 0;
  ~mmr_rotary() override {
    if (block) mmr::context_give_block(owner, block, capacity);
  }
};

namespace {

// Device memory the caller names by address: 4-byte aligned and not null where there is something to read.
int check_ids(const void* p, int32_t n, const char* what) {
  if (n > 0 && !p) return fail(MMR_INVALID_ARGUMENT, "%s is null", what);
  if (reinterpret_cast<uintptr_t>(p) % 4) return fail(MMR_INVALID_ARGUMENT, "%s is not 4-byte aligned", what);
  return MMR_OK;
}

// A store of int32 in one whole buffer, row-major.
int check_table(mmr_context* ctx, const mmr_store* s, int rank, const char* what) {
  if (int rc = mmr::context_check_store(ctx, s, what)) return rc;
  const Side& d = mmr::store_side(s);
  if (d.dtype != MMR_S32) return fail(MMR_INVALID_ARGUMENT, "%s store is not S32", what);
  if (d.rank != rank) return fail(MMR_INVALID_ARGUMENT, "%s store has rank %d, not %d", what, d.rank, rank);
  if (d.dev_count != 1) return fail(MMR_INVALID_ARGUMENT, "%s store is spread over %lld devices", what, (long long)d.dev_count);
  if (d.stride[rank - 1] != 1 && d.ext[rank - 1] > 1) return fail(MMR_INVALID_ARGUMENT, "%s store is not row-major", what);
  for (int i = 0; i < rank; ++i)
    if (d.size[i] < 1 || d.size[i] > 0x7fffffff)
      return fail(MMR_INVALID_ARGUMENT, "%s store has extent %lld along dim %d", what, (long long)d.size[i], i);
  return MMR_OK;
}

// No C++ exception leaves a C entry point (what can throw here is host memory running out).
int exception_status() {
  try {
    throw;
  } catch (const std::bad_alloc&) {
    return fail(MMR_OUT_OF_MEMORY, "out of host memory");
  } catch (const std::exception& e) {
    return fail(MMR_INTERNAL, "%s", e.what());
  } catch (...) {
    return fail(MMR_INTERNAL, "unknown exception");
  }
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

std::vector<char*> tiles_of(const mmr_store* s) {
  std::vector<char*> t;
  for (int64_t k = 0; k < mmr::store_side(s).dev_count; ++k) t.push_back(mmr::store_tile(s, k));
  return t;
}

int upload_buffers(mmr_context* ctx, mmr_pages* p) {
  std::vector<mmr::PageBuffer> b;
  for (const auto& pool : p->pools)
    for (char* t : pool.tiles) b.push_back({t, static_cast<uint64_t>(pool.side.shard_bytes / pool.side.size[0])});
  return mmr::context_upload(ctx, p->block + p->buffers_at, b.data(), b.size() * sizeof(b[0]));
}

// The stores of the cache are still there and where they were; a pool that was offloaded and reloaded has its buffers
// entered anew.
int refresh(mmr_context* ctx, mmr_pages* p) {
  const uint64_t epoch = mmr::context_store_epoch(ctx);
  if (epoch == p->epoch) return MMR_OK;
  auto find = [&](int64_t id, const char* what, mmr_store** out) {
    *out = mmr::context_find_store(ctx, id);
    if (!*out) return fail(MMR_NOT_FOUND, "the %s store %lld of the page cache was freed", what, (long long)id);
    return mmr::context_check_store(ctx, *out, what);
  };
  mmr_store* s = nullptr;
  if (int rc = find(p->table_id, "table", &s)) return rc;
  int32_t* table = reinterpret_cast<int32_t*>(mmr::store_tile(s, 0));
  if (int rc = find(p->lengths_id, "lengths", &s)) return rc;
  int32_t* lengths = reinterpret_cast<int32_t*>(mmr::store_tile(s, 0));
  if (int rc = find(p->refs_id, "refs", &s)) return rc;
  int32_t* refs = reinterpret_cast<int32_t*>(mmr::store_tile(s, 0));
  std::vector<std::vector<char*>> tiles;
  bool moved = false;
  for (const auto& pool : p->pools) {
    if (int rc = find(pool.id, "pool", &s)) return rc;
    tiles.push_back(tiles_of(s));
    moved |= tiles.back() != pool.tiles;
  }
  if (moved) {
    if (int rc = mmr::context_refuse_capture(ctx, "the first call on a page cache whose pools have moved")) return rc;
    for (size_t i = 0; i < tiles.size(); ++i) p->pools[i].tiles = tiles[i];
    if (int rc = upload_buffers(ctx, p)) {
      p->pools[0].tiles.clear();  // entered again by the next call
      return rc;
    }
  }
  p->state.table = table, p->state.lengths = lengths, p->state.refs = refs;
  p->epoch = epoch;
  return MMR_OK;
}

// Common start of the operators on a cache.
int begin(mmr_pages* p, int32_t n, int32_t limit, const char* of) {
  if (n < 0 || n > limit) return fail(MMR_INVALID_ARGUMENT, "%d entries, at most %d (%s)", n, limit, of);
  if (int rc = mmr::context_use_device(p->owner)) return rc;
  return refresh(p->owner, p);
}

mmr::PageMoveLaunch moves_up_to(const mmr_pages* p, int64_t most) {
  mmr::PageMoveLaunch m = p->move;
  m.max_moves = static_cast<uint32_t>(std::min<int64_t>(most, p->state.P));
  return m;
}

// Tile coordinate of relative device k along dim i.
int64_t tile_at(const Side& s, int64_t k, int i) { return k / s.dev_stride[i] % s.tiles[i]; }
int64_t tile_start(const Side& s, int64_t k, int i) { return tile_at(s, k, i) * s.ext[i]; }
int64_t tile_valid(const Side& s, int64_t k, int i) {
  return std::max<int64_t>(0, std::min(s.ext[i], s.size[i] - tile_start(s, k, i)));
}

bool tile_empty(const Side& s, int64_t k) {
  for (int i = 0; i < s.rank; ++i)
    if (tile_valid(s, k, i) == 0) return true;
  return false;
}

// Replicas that the caller keeps in one buffer are turned once: *again says that an earlier device than k writes k's tile.
// Tiles that lie over one another in any other way are refused, as their writes have no order.
int check_again(const mmr_store* out, int64_t k, bool* again) {
  *again = false;
  if (!mmr::store_tiles_overlap(out)) return MMR_OK;
  const Side& s = mmr::store_side(out);
  const char* mine = mmr::store_tile(out, k);
  for (int64_t m = 0; m < k; ++m) {
    const char* other = mmr::store_tile(out, m);
    if (mine + s.shard_bytes <= other || other + s.shard_bytes <= mine || tile_empty(s, m)) continue;
    bool same = mine == other;
    for (int i = 0; i < s.rank; ++i) same &= tile_at(s, k, i) == tile_at(s, m, i);
    if (!same)
      return fail(MMR_INVALID_ARGUMENT, "the buffers of devices %lld and %lld of the output store overlap", (long long)(s.dev_start + m),
                  (long long)(s.dev_start + k));
    *again = true;
  }
  return MMR_OK;
}

int check_row(const Side& s, const char* what) {
  const int d = s.rank - 1;
  if (s.tiles[d] != 1) return fail(MMR_INVALID_ARGUMENT, "the last dim of the %s store is sharded", what);
  if (s.size[d] > 1 && s.stride[d] != 1) return fail(MMR_INVALID_ARGUMENT, "the last dim of the %s store is not its minor-most", what);
  if (s.size[d] < 1 || s.size[d] > (1 << 20)) return fail(MMR_INVALID_ARGUMENT, "rows of %lld elements", (long long)s.size[d]);
  return MMR_OK;
}

int check_rotary(mmr_context* ctx, const mmr_rotary* r, int64_t dim, int32_t dtype) {
  if (r->owner != ctx) return fail(MMR_INVALID_ARGUMENT, "the rotary plan belongs to another context");
  if (dtype != MMR_F32 && dtype != MMR_BF16 && dtype != MMR_F16)
    return fail(MMR_UNSUPPORTED, "rotary positions turn F32, BF16 and F16, not type %d", dtype);
  if (r->dim > dim) return fail(MMR_INVALID_ARGUMENT, "the rotary plan turns %d elements of rows of %lld", r->dim, (long long)dim);
  return MMR_OK;
}

constexpr uint64_t kMaxRotaryBlocks = (1u << 24) - 1;  // a grid has fewer than 2^32 threads

constexpr int64_t kL2Bytes = int64_t{32} << 20;  // eight XCDs of 4 MiB

void set_plan(mmr::RotaryLaunch* l, const mmr_rotary* r, bool backward) {
  if (!r) return;
  l->angles = {reinterpret_cast<const uint64_t*>(r->block), r->magnitude, backward ? -r->magnitude : r->magnitude,
               static_cast<uint32_t>(r->dim / 2)};
  l->interleaved = r->interleaved;
}

// What of a row a call does: its length in elements, and whether it is turned and in place.
struct Row {
  int64_t dim;
  bool turned, in_place;
};

// Bytes of the vectors a lane turns: 16 where every row, its turned part (its two halves, unless interleaved) and with
// them every stride are whole vectors, else the widest that divides the turned part - these may stand at any address.
int vector_bytes(const mmr::RotaryLaunch& l, const std::vector<Row>& rows, int itemsize) {
  const int64_t part = static_cast<int64_t>(l.angles.half) * itemsize * (l.interleaved ? 2 : 1);
  bool wide = true, turned = false;
  for (const Row& r : rows) {
    wide &= r.dim * itemsize % 16 == 0;
    turned |= r.turned;
  }
  if (!turned) return wide ? 16 : 1;
  if (wide && part % 16 == 0) return 16;
  for (int bytes = 8; bytes > itemsize; bytes /= 2)
    if (part % bytes == 0) return bytes;
  return itemsize;
}

// Whether every piece of a row that one store instruction writes is whole 128-byte lines.
bool whole_lines(const mmr::RotaryLaunch& l, const std::vector<Row>& rows, int itemsize) {
  const int64_t part = static_cast<int64_t>(l.angles.half) * itemsize * (l.interleaved ? 2 : 1);
  for (const Row& r : rows)
    if (r.dim * itemsize % 128 || (r.turned && part % 128)) return false;
  return true;
}

// Units of the shapes, and the launches.  A call of few rows takes one head a lane, so that its latency is one row's and
// not four.
int launch_rows(mmr_context* ctx, mmr::RotaryLaunch* l, const std::vector<Row>& rows, int itemsize) {
  l->vector_bytes = vector_bytes(*l, rows, itemsize);
  for (size_t i = 0; i < rows.size(); ++i) {
    const int64_t turned = rows[i].turned ? static_cast<int64_t>(l->angles.half) * 2 * itemsize : 0;
    const int64_t unit = static_cast<int64_t>(l->vector_bytes) * (l->interleaved ? 1 : 2);
    mmr::rotary_units(&l->shapes[i], static_cast<uint32_t>(rows[i].dim * itemsize), static_cast<uint32_t>(turned),
                      static_cast<uint32_t>(unit), static_cast<uint32_t>(l->type < 0 ? 1 : itemsize), rows[i].in_place);
  }
  int64_t lanes = 0, bytes = 0;
  for (const mmr::RotaryBuffer& b : l->buffers) {
    const int64_t n = static_cast<int64_t>(b.outer) * b.seq * b.heads;
    lanes += n * l->shapes[b.shape].units;
    bytes += n * rows[b.shape].dim * itemsize;
  }
  const bool spread = lanes < 256 * 1024;  // a lane each would leave the 256 CUs under four workgroups
  for (size_t i = 0; i < l->shapes.size(); ++i) {
    mmr::RotaryShape& j = l->shapes[i];
    if (mmr::rotary_shape(&j, j.src_head <= j.src_seq, spread) > kMaxRotaryBlocks)
      return fail(MMR_UNSUPPORTED, "a tile of %u tokens of %u heads is more than a launch takes", j.tokens, j.heads);
  }
  l->past_caches = bytes > kL2Bytes && whole_lines(*l, rows, itemsize);
  int launches = 0;
  const hipError_t e = mmr::launch_rotary(*l, &launches, mmr::context_stream(ctx));
  mmr::context_count(ctx, launches);
  MMR_HIP(e);
  return MMR_OK;
}

}  // namespace

extern "C" {

int mmr_pages_create(mmr_context* ctx, mmr_store* const* pools, int32_t n_pools, mmr_store* table, mmr_store* lengths,
                     mmr_store* refs, int32_t page_tokens, mmr_pages** out) try {
  if (!ctx || !out || (n_pools > 0 && !pools)) return fail(MMR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  mmr::ContextLock lock(ctx);
  if (int rc = mmr::context_use_device(ctx)) return rc;
  if (n_pools < 1 || n_pools > 65536) return fail(MMR_INVALID_ARGUMENT, "%d pools", n_pools);
  if (page_tokens < 1) return fail(MMR_INVALID_ARGUMENT, "pages of %d tokens", page_tokens);
  if (int rc = check_table(ctx, table, 2, "table")) return rc;
  if (int rc = check_table(ctx, lengths, 1, "lengths")) return rc;
  if (int rc = check_table(ctx, refs, 1, "refs")) return rc;
  if (table == lengths || table == refs || lengths == refs)
    return fail(MMR_INVALID_ARGUMENT, "table, lengths and refs are stores of their own");
  const Side& t = mmr::store_side(table);
  const int64_t S = t.size[0], B = t.size[1], P = mmr::store_side(refs).size[0];
  if (mmr::store_side(lengths).size[0] != S)
    return fail(MMR_INVALID_ARGUMENT, "table of %lld sequences, lengths of %lld", (long long)S,
                (long long)mmr::store_side(lengths).size[0]);
  if (S > (1 << 21)) return fail(MMR_UNSUPPORTED, "%lld sequences, at most %d", (long long)S, 1 << 21);
  if (P > mmr::kMaxPages) return fail(MMR_UNSUPPORTED, "%lld pages, at most %d", (long long)P, mmr::kMaxPages);
  auto p = std::make_unique<mmr_pages>();
  int64_t buffers = 0, largest = 0;
  bool aligned = true;
  std::set<const mmr_store*> seen;
  for (int32_t i = 0; i < n_pools; ++i) {
    if (int rc = mmr::context_check_store(ctx, pools[i], "pool")) return rc;
    if (pools[i] == table || pools[i] == lengths || pools[i] == refs)
      return fail(MMR_INVALID_ARGUMENT, "pool %d is one of the tables", i);
    if (!seen.insert(pools[i]).second) return fail(MMR_INVALID_ARGUMENT, "pool %d is the same store as an earlier one", i);
    const Side& s = mmr::store_side(pools[i]);
    if (s.rank < 1 || s.size[0] != P || s.tiles[0] != 1)
      return fail(MMR_INVALID_ARGUMENT, "dim 0 of pool %d is not the %lld pages, unsharded", i, (long long)P);
    if (s.shard_bytes < 1 || (P > 1 && s.stride[0] != s.shard_elems / P))
      return fail(MMR_INVALID_ARGUMENT, "the pages of pool %d are not the slowest dim of its buffers, or are empty", i);
    buffers += s.dev_count;
    largest = std::max(largest, s.shard_bytes / P);
    aligned &= s.shard_bytes / P % 16 == 0;
    p->pools.push_back({mmr_store_id(pools[i]), s, tiles_of(pools[i])});
  }
  const int64_t chunks = (largest + mmr::kPageChunkBytes - 1) / mmr::kPageChunkBytes;
  if (chunks > 0x7fffffff / P || buffers > 0x7fffffff / (P * chunks))
    return fail(MMR_UNSUPPORTED, "%lld pages of %lld bytes in %lld buffers are more pieces than a launch numbers", (long long)P,
                (long long)largest, (long long)buffers);
  if (int rc = mmr::context_refuse_capture(ctx, "creating a page cache")) return rc;
  // one block: header, then the arrays of PageWork, then the buffer table
  const int64_t segments = (P + mmr::kPageSegment - 1) / mmr::kPageSegment;
  const int64_t ids = segments * mmr::kPageSegment;
  size_t at = 0;
  auto take = [&at](int64_t n, size_t size) {
    const size_t here = at;
    at = align256(at + static_cast<size_t>(n) * size);
    return here;
  };
  const size_t header = take(mmr::kPageHeaderInts, 4), mark = take(std::max(S, P), 4), cleared = at;
  const size_t seg_free = take(segments, 4), seg_before = take(segments, 4), free_ids = take(ids, 4), live_ids = take(ids, 4);
  const size_t len = take(S, 4), rank = take(S, 4);
  const size_t moves = take(std::max(S, P), sizeof(mmr::PageMove)), map = take(P, 4);
  p->buffers_at = take(buffers, sizeof(mmr::PageBuffer));
  p->owner = ctx;
  if (int rc = mmr::context_take_block(ctx, at, &p->block, &p->capacity)) return rc;
  MMR_HIP(hipMemsetAsync(p->block, 0, cleared, mmr::context_stream(ctx)));
  if (int rc = upload_buffers(ctx, p.get())) return rc;
  auto ints = [&](size_t offset) { return reinterpret_cast<int32_t*>(p->block + offset); };
  p->work = {ints(header), ints(seg_free), ints(seg_before), ints(free_ids), ints(live_ids), ints(mark), ints(len), ints(rank),
             reinterpret_cast<mmr::PageMove*>(p->block + moves), ints(map), static_cast<int32_t>(segments)};
  const int64_t capacity = std::min<int64_t>(B * page_tokens, 0x7fffffff);
  p->state = {reinterpret_cast<int32_t*>(mmr::store_tile(table, 0)), reinterpret_cast<int32_t*>(mmr::store_tile(lengths, 0)),
              reinterpret_cast<int32_t*>(mmr::store_tile(refs, 0)), static_cast<int32_t>(S), static_cast<int32_t>(B),
              static_cast<int32_t>(P), page_tokens, static_cast<int32_t>(capacity), mmr::make_fastdiv(static_cast<uint32_t>(page_tokens))};
  p->move.mover = {reinterpret_cast<const mmr::PageBuffer*>(p->block + p->buffers_at), static_cast<uint32_t>(buffers),
                   static_cast<uint32_t>(chunks), mmr::make_fastdiv(static_cast<uint32_t>(chunks)),
                   mmr::page_lane_bits(static_cast<uint64_t>(largest))};
  p->move.aligned = aligned;
  p->move.packed = (1 << p->move.mover.lane_bits) < mmr::kPageThreads;
  p->table_id = mmr_store_id(table), p->lengths_id = mmr_store_id(lengths), p->refs_id = mmr_store_id(refs);
  for (int32_t i = 0; i < n_pools; ++i) mmr::context_watch(pools[i]);
  for (mmr_store* t : {table, lengths, refs}) mmr::context_watch(t);
  p->epoch = mmr::context_store_epoch(ctx);
  mmr_pages* handle = p.get();
  mmr::context_attach(ctx, std::move(p));
  *out = handle;
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_pages_destroy(mmr_pages* pages) try {
  if (!pages) return fail(MMR_INVALID_ARGUMENT, "null page cache");
  mmr_context* ctx = pages->owner;
  mmr::ContextLock lock(ctx);
  mmr::context_detach(ctx, pages);
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_pages_extend(mmr_pages* pages, const int32_t* sequences, const int32_t* tokens, int32_t n) try {
  if (!pages) return fail(MMR_INVALID_ARGUMENT, "null page cache");
  mmr::ContextLock lock(pages->owner);
  if (int rc = begin(pages, n, pages->state.S, "the sequences of the table")) return rc;
  if (int rc = check_ids(sequences, n, "sequences")) return rc;
  if (int rc = check_ids(tokens, n, "tokens")) return rc;
  if (n == 0) return MMR_OK;
  mmr::context_hash(pages->owner, 16, {static_cast<uint64_t>(n)});
  int launches = 0;
  const hipError_t e = mmr::launch_page_extend(pages->state, pages->work, sequences, tokens, n, mmr::context_stream(pages->owner), &launches);
  mmr::context_count(pages->owner, launches);
  MMR_HIP(e);
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_pages_free(mmr_pages* pages, const int32_t* sequences, int32_t n) try {
  if (!pages) return fail(MMR_INVALID_ARGUMENT, "null page cache");
  mmr::ContextLock lock(pages->owner);
  if (int rc = begin(pages, n, pages->state.S, "the sequences of the table")) return rc;
  if (int rc = check_ids(sequences, n, "sequences")) return rc;
  if (n == 0) return MMR_OK;
  mmr::context_hash(pages->owner, 17, {static_cast<uint64_t>(n)});
  int launches = 0;
  const hipError_t e = mmr::launch_page_free(pages->state, pages->work, sequences, n, mmr::context_stream(pages->owner), &launches);
  mmr::context_count(pages->owner, launches);
  MMR_HIP(e);
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_pages_fork(mmr_pages* pages, const int32_t* parents, const int32_t* children, int32_t n) try {
  if (!pages) return fail(MMR_INVALID_ARGUMENT, "null page cache");
  mmr::ContextLock lock(pages->owner);
  if (int rc = begin(pages, n, pages->state.S, "the sequences of the table")) return rc;
  if (int rc = check_ids(parents, n, "parents")) return rc;
  if (int rc = check_ids(children, n, "children")) return rc;
  if (n == 0) return MMR_OK;
  mmr::context_hash(pages->owner, 18, {static_cast<uint64_t>(n)});
  int launches = 0;
  const hipError_t e = mmr::launch_page_fork(pages->state, pages->work, parents, children, n, moves_up_to(pages, n),
                                mmr::context_stream(pages->owner), &launches);
  mmr::context_count(pages->owner, launches);
  MMR_HIP(e);
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_pages_compact(mmr_pages* pages) try {
  if (!pages) return fail(MMR_INVALID_ARGUMENT, "null page cache");
  mmr::ContextLock lock(pages->owner);
  if (int rc = begin(pages, 0, 0, "")) return rc;
  mmr::context_hash(pages->owner, 19, {});
  int launches = 0;
  const hipError_t e = mmr::launch_page_compact(pages->state, pages->work, moves_up_to(pages, pages->state.P / 2),
                                   mmr::context_stream(pages->owner), &launches);
  mmr::context_count(pages->owner, launches);
  MMR_HIP(e);
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_pages_copy(mmr_pages* pages, const int32_t* sources, const int32_t* destinations, int32_t n) try {
  if (!pages) return fail(MMR_INVALID_ARGUMENT, "null page cache");
  mmr::ContextLock lock(pages->owner);
  if (int rc = begin(pages, n, pages->state.P, "the pages of the pools")) return rc;
  if (int rc = check_ids(sources, n, "sources")) return rc;
  if (int rc = check_ids(destinations, n, "destinations")) return rc;
  if (n == 0) return MMR_OK;
  mmr::context_hash(pages->owner, 20, {static_cast<uint64_t>(n)});
  int launches = 0;
  const hipError_t e = mmr::launch_page_copy(pages->state, pages->work, sources, destinations, n, moves_up_to(pages, n),
                                mmr::context_stream(pages->owner), &launches);
  mmr::context_count(pages->owner, launches);
  MMR_HIP(e);
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_pages_status(mmr_pages* pages, uint32_t* flags, int64_t* pages_in_use) try {
  if (!pages || !flags) return fail(MMR_INVALID_ARGUMENT, "null argument");
  mmr_context* ctx = pages->owner;
  mmr::ContextLock lock(ctx);
  if (int rc = begin(pages, 0, 0, "")) return rc;
  if (int rc = mmr::context_refuse_capture(ctx, "reading the status of a page cache")) return rc;
  hipStream_t stream = mmr::context_stream(ctx);
  int launches = 0;
  const hipError_t e = mmr::launch_page_count(pages->state, pages->work, stream, &launches);
  mmr::context_count(ctx, launches);
  MMR_HIP(e);
  int32_t header[8] = {};
  MMR_HIP(hipMemcpyAsync(header, pages->work.header, sizeof(header), hipMemcpyDeviceToHost, stream));
  MMR_HIP(hipMemsetAsync(pages->work.header + mmr::kPageStatus, 0, 4, stream));
  if (int rc = mmr::context_wait(ctx)) return rc;
  *flags = static_cast<uint32_t>(header[mmr::kPageStatus]);
  if (pages_in_use) *pages_in_use = header[mmr::kPageLive];
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_rotary_create(mmr_context* ctx, const mmr_rotary_options* o, mmr_rotary** out) try {
  if (!ctx || !o || !out) return fail(MMR_INVALID_ARGUMENT, "null argument");
  *out = nullptr;
  mmr::ContextLock lock(ctx);
  if (int rc = mmr::context_use_device(ctx)) return rc;
  if (o->rotary_dim < 2 || o->rotary_dim % 2 || o->rotary_dim > (1 << 20))
    return fail(MMR_INVALID_ARGUMENT, "rotary dim %d is not even and in [2, 2^20]", o->rotary_dim);
  if (!o->frequencies && !(o->base > 0 && std::isfinite(o->base))) return fail(MMR_INVALID_ARGUMENT, "base %g", o->base);
  // held in 32 bits
  if (!(o->magnitude >= 0 && o->magnitude <= std::numeric_limits<float>::max())) return fail(MMR_INVALID_ARGUMENT, "magnitude %g", o->magnitude);
  if (o->scaling < MMR_ROTARY_UNSCALED || o->scaling > MMR_ROTARY_BY_PARTS)
    return fail(MMR_INVALID_ARGUMENT, "scaling %d", o->scaling);
  if (o->scaling != MMR_ROTARY_UNSCALED && !(o->factor > 0 && std::isfinite(o->factor)))
    return fail(MMR_INVALID_ARGUMENT, "factor %g", o->factor);
  if (o->scaling == MMR_ROTARY_BY_PARTS &&
      !(o->original_positions > 0 && o->low_turns >= 0 && o->high_turns > o->low_turns && std::isfinite(o->high_turns)))
    return fail(MMR_INVALID_ARGUMENT, "parts from %g to %g turns over %lld positions", o->low_turns, o->high_turns,
                (long long)o->original_positions);
  const int half = o->rotary_dim / 2;
  std::vector<uint64_t> turns(static_cast<size_t>(half));
  const long double tau = 6.283185307179586476925286766559005768L;
  for (int i = 0; i < half; ++i) {
    if (o->frequencies && !std::isfinite(o->frequencies[i])) return fail(MMR_INVALID_ARGUMENT, "frequency %d is not finite", i);
    long double f = o->frequencies ? static_cast<long double>(o->frequencies[i])
                                   : std::pow(static_cast<long double>(o->base), -2.0L * i / o->rotary_dim);
    f /= tau;
    if (o->scaling == MMR_ROTARY_LINEAR) f /= o->factor;
    if (o->scaling == MMR_ROTARY_BY_PARTS) {
      const long double n = o->original_positions * std::fabs(f);
      const long double w = std::min(1.0L, std::max(0.0L, (n - o->low_turns) / (static_cast<long double>(o->high_turns) - o->low_turns)));
      f *= w + (1.0L - w) / o->factor;
    }
    f -= std::floor(f);  // positions are whole: whole turns drop out
    const long double scaled = f * 18446744073709551616.0L + 0.5L;
    turns[static_cast<size_t>(i)] = scaled >= 18446744073709551616.0L ? 0 : static_cast<uint64_t>(scaled);
  }
  if (int rc = mmr::context_refuse_capture(ctx, "creating a rotary plan")) return rc;
  auto r = std::make_unique<mmr_rotary>();
  r->owner = ctx;
  r->dim = o->rotary_dim;
  r->interleaved = o->interleaved != 0;
  r->magnitude = static_cast<float>(o->magnitude);
  if (int rc = mmr::context_take_block(ctx, turns.size() * 8, &r->block, &r->capacity)) return rc;
  if (int rc = mmr::context_upload(ctx, r->block, turns.data(), turns.size() * 8)) return rc;
  mmr_rotary* handle = r.get();
  mmr::context_attach(ctx, std::move(r));
  *out = handle;
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_rotary_destroy(mmr_rotary* rotary) try {
  if (!rotary) return fail(MMR_INVALID_ARGUMENT, "null rotary plan");
  mmr_context* ctx = rotary->owner;
  mmr::ContextLock lock(ctx);
  mmr::context_detach(ctx, rotary);
  return MMR_OK;
} catch (...) {
  return exception_status();
}

int mmr_rotary_apply(mmr_rotary* rotary, mmr_store* x, mmr_store* out, int32_t seq_dim, mmr_store* positions, int64_t offset,
                     uint32_t flags) try {
  if (!rotary) return fail(MMR_INVALID_ARGUMENT, "null rotary plan");
  mmr_context* ctx = rotary->owner;
  mmr::ContextLock lock(ctx);
  if (flags & ~MMR_ROTARY_BACKWARD) return fail(MMR_INVALID_ARGUMENT, "unknown flags %#x", flags);
  if (int rc = mmr::context_use_device(ctx)) return rc;
  if (int rc = mmr::context_check_store(ctx, x, "input")) return rc;
  if (int rc = mmr::context_check_store(ctx, out, "output")) return rc;
  if (x != out && mmr::store_key(x) != mmr::store_key(out))
    return fail(MMR_INVALID_ARGUMENT, "input and output stores have different descriptors");
  const Side& s = mmr::store_side(x);
  if (s.rank < 2 || s.rank > 4) return fail(MMR_INVALID_ARGUMENT, "rank %d, not 2 to 4", s.rank);
  if (seq_dim < 0 || seq_dim >= s.rank - 1) return fail(MMR_INVALID_ARGUMENT, "seq_dim %d of rank %d", seq_dim, s.rank);
  if (int rc = check_row(s, "input")) return rc;
  if (int rc = check_rotary(ctx, rotary, s.size[s.rank - 1], s.dtype)) return rc;
  if (offset < INT32_MIN || offset > INT32_MAX) return fail(MMR_INVALID_ARGUMENT, "offset %lld", (long long)offset);
  // the other dims: heads, and an outer one; -1 is a dim of extent 1
  int other[2] = {-1, -1};
  for (int i = 0, k = 0; i < s.rank - 1; ++i)
    if (i != seq_dim) other[k++] = i;
  int outer = -1, head = other[0];
  if (other[1] >= 0) outer = other[0], head = other[1];
  if (outer >= 0 && s.stride[outer] < s.stride[head]) std::swap(outer, head);  // heads: the one closer to the rows
  const Side* ps = nullptr;
  if (positions) {
    if (int rc = mmr::context_check_store(ctx, positions, "positions")) return rc;
    ps = &mmr::store_side(positions);
    if (ps->dtype != MMR_S32) return fail(MMR_INVALID_ARGUMENT, "positions store is not S32");
    if (offset) return fail(MMR_INVALID_ARGUMENT, "positions and an offset");
    if (ps->rank < 1 || ps->rank > 2) return fail(MMR_INVALID_ARGUMENT, "positions of rank %d, not 1 or 2", ps->rank);
    if (ps->dev_count != s.dev_count)
      return fail(MMR_INVALID_ARGUMENT, "positions on %lld devices, input on %lld", (long long)ps->dev_count, (long long)s.dev_count);
    if (ps->rank == 2) {
      if (s.rank < 3 || seq_dim == 0) return fail(MMR_INVALID_ARGUMENT, "positions of rank 2 take dim 0 of the input as their first");
      if (head == 0) std::swap(outer, head);
      if (ps->size[0] != s.size[0]) return fail(MMR_INVALID_ARGUMENT, "positions of %lld, dim 0 of %lld", (long long)ps->size[0], (long long)s.size[0]);
    }
    if (ps->size[ps->rank - 1] != s.size[seq_dim])
      return fail(MMR_INVALID_ARGUMENT, "positions of %lld, sequence of %lld", (long long)ps->size[ps->rank - 1], (long long)s.size[seq_dim]);
  }
  mmr::RotaryLaunch l;
  set_plan(&l, rotary, flags & MMR_ROTARY_BACKWARD);
  l.type = s.dtype;
  const int64_t all_outer = outer >= 0 ? s.ext[outer] : 1, all_heads = head >= 0 ? s.ext[head] : 1, all_seq = s.ext[seq_dim];
  if (all_outer == 0 || all_heads == 0 || all_seq == 0) return MMR_OK;  // an empty array
  if (all_outer > 0x7fffffff / all_seq || all_heads > 0x7fffffff) return fail(MMR_UNSUPPORTED, "a tile of more than 2^31 rows");
  mmr::RotaryShape shape{};
  shape.tokens = static_cast<uint32_t>(all_outer * all_seq), shape.seq = static_cast<uint32_t>(all_seq);
  shape.heads = static_cast<uint32_t>(all_heads);
  shape.src_seq = shape.dst_seq = s.stride[seq_dim] * s.itemsize;
  shape.src_outer = shape.dst_outer = outer >= 0 ? s.stride[outer] * s.itemsize : 0;
  shape.src_head = shape.dst_head = head >= 0 ? s.stride[head] * s.itemsize : 0;
  if (ps) {
    shape.pos_seq = ps->stride[ps->rank - 1];
    shape.pos_outer = ps->rank == 2 ? ps->stride[0] : 0;
  }
  l.shapes.push_back(shape);
  bool in_place = true;
  for (int64_t k = 0; k < s.dev_count; ++k) {
    mmr::RotaryBuffer b{};
    b.src = mmr::store_tile(x, k);
    b.dst = mmr::store_tile(out, k);
    b.outer = static_cast<uint32_t>(outer >= 0 ? tile_valid(s, k, outer) : 1);
    b.heads = static_cast<uint32_t>(head >= 0 ? tile_valid(s, k, head) : 1);
    b.seq = static_cast<uint32_t>(tile_valid(s, k, seq_dim));
    if (b.outer == 0 || b.heads == 0 || b.seq == 0) continue;  // a tile of padding
    b.base = offset + tile_start(s, k, seq_dim);
    if (ps) {
      const int q = ps->rank - 1;
      // this device's positions cover its part of the sequence (and of dim 0)
      const int64_t at = tile_start(s, k, seq_dim) - tile_start(*ps, k, q);
      bool covered = at >= 0 && at + b.seq <= tile_valid(*ps, k, q);
      int64_t first = at * ps->stride[q];
      if (ps->rank == 2) {
        const int64_t row = tile_start(s, k, 0) - tile_start(*ps, k, 0);
        covered &= row >= 0 && row + tile_valid(s, k, 0) <= tile_valid(*ps, k, 0);
        first += row * ps->stride[0];
      }
      if (!covered)
        return fail(MMR_INVALID_ARGUMENT, "device %lld holds positions of another part of the sequence than its tile",
                    (long long)(s.dev_start + k));
      b.positions = reinterpret_cast<const int32_t*>(mmr::store_tile(positions, k)) + first;
    }
    bool again = false;
    if (int rc = check_again(out, k, &again)) return rc;
    if (again) continue;
    in_place &= b.src == b.dst;
    l.buffers.push_back(b);
  }
  mmr::context_hash(ctx, 21, {static_cast<uint64_t>(mmr::store_ordinal(x)), static_cast<uint64_t>(mmr::store_ordinal(out)), flags});
  return launch_rows(ctx, &l, {Row{s.size[s.rank - 1], true, in_place}}, s.itemsize);
} catch (...) {
  return exception_status();
}

int mmr_pages_write(mmr_pages* pages, const int32_t* sequences, const int32_t* begins, int32_t n, int32_t k_pool, mmr_store* k,
                    int32_t v_pool, mmr_store* v, mmr_rotary* rotary, mmr_store* q, mmr_store* q_out) try {
  if (!pages) return fail(MMR_INVALID_ARGUMENT, "null page cache");
  mmr_context* ctx = pages->owner;
  mmr::ContextLock lock(ctx);
  if (int rc = begin(pages, n, pages->state.S, "the sequences of the table")) return rc;
  if (int rc = check_ids(sequences, n, "sequences")) return rc;
  if (int rc = check_ids(begins, n, "begins")) return rc;
  if (!k) return fail(MMR_INVALID_ARGUMENT, "k store is null");
  if ((q == nullptr) != (q_out == nullptr)) return fail(MMR_INVALID_ARGUMENT, "q and q_out come together");
  if (q && !rotary) return fail(MMR_INVALID_ARGUMENT, "q without a rotary plan");
  if (v && v_pool == k_pool) return fail(MMR_INVALID_ARGUMENT, "k and v go to the same pool");
  mmr::RotaryLaunch l;
  set_plan(&l, rotary, false);
  std::vector<Row> rows;
  int64_t tokens = -1;
  int32_t dtype = -1;
  int itemsize = 0;
  // a new-token store: [tokens, heads, dim], tokens unsharded, every part of one call of the same type and length
  auto check_new = [&](const mmr_store* s, const char* what) {
    if (int rc = mmr::context_check_store(ctx, s, what)) return rc;
    const Side& d = mmr::store_side(s);
    if (d.rank != 3) return fail(MMR_INVALID_ARGUMENT, "%s store has rank %d, not [tokens, heads, dim]", what, d.rank);
    if (int rc = check_row(d, what)) return rc;
    if (d.tiles[0] != 1) return fail(MMR_INVALID_ARGUMENT, "the tokens of the %s store are sharded", what);
    if (d.size[0] > 0x7fffffff || d.size[1] > 0x7fffffff) return fail(MMR_UNSUPPORTED, "%s store of more than 2^31 rows", what);
    if (tokens >= 0 && d.size[0] != tokens) return fail(MMR_INVALID_ARGUMENT, "%s store of %lld tokens, another of %lld", what, (long long)d.size[0], (long long)tokens);
    if (dtype >= 0 && d.dtype != dtype) return fail(MMR_INVALID_ARGUMENT, "the %s store is of another type", what);
    tokens = d.size[0], dtype = d.dtype, itemsize = d.itemsize;
    return static_cast<int>(MMR_OK);
  };
  auto add = [&](const mmr_store* s, const Side* pool, const std::vector<char*>* pool_tiles, const mmr_store* out, bool turn) {
    const Side& d = mmr::store_side(s);
    if (d.size[0] == 0 || d.size[1] == 0) return static_cast<int>(MMR_OK);
    mmr::RotaryShape j{};
    j.tokens = j.seq = static_cast<uint32_t>(d.size[0]);
    j.heads = static_cast<uint32_t>(d.ext[1]);
    j.src_seq = d.stride[0] * d.itemsize, j.src_head = d.stride[1] * d.itemsize;
    if (pool) {
      j.paged = 1;
      j.dst_outer = pool->shard_bytes / pool->size[0];
      j.dst_seq = pool->stride[1] * pool->itemsize, j.dst_head = pool->stride[2] * pool->itemsize;
    } else {
      j.paged = 2;
      j.dst_seq = j.src_seq, j.dst_head = j.src_head;
    }
    bool in_place = !pool;
    for (int64_t dev = 0; dev < d.dev_count; ++dev) {
      mmr::RotaryBuffer b{};
      b.src = mmr::store_tile(s, dev);
      b.dst = pool ? (*pool_tiles)[static_cast<size_t>(dev)] : mmr::store_tile(out, dev);
      b.outer = 1, b.seq = j.seq, b.heads = static_cast<uint32_t>(tile_valid(d, dev, 1));
      b.shape = static_cast<uint32_t>(l.shapes.size());
      if (b.heads == 0) continue;
      bool again = false;
      if (out)
        if (int rc = check_again(out, dev, &again)) return rc;
      if (again) continue;
      in_place &= b.src == b.dst;
      l.buffers.push_back(b);
    }
    l.shapes.push_back(j);
    rows.push_back(Row{d.size[2], turn, in_place});
    return static_cast<int>(MMR_OK);
  };
  auto add_pool = [&](const mmr_store* s, int32_t pool, bool turn, const char* what) {
    if (int rc = check_new(s, what)) return rc;
    if (pool < 0 || pool >= static_cast<int32_t>(pages->pools.size()))
      return fail(MMR_INVALID_ARGUMENT, "%s pool %d of %zu", what, pool, pages->pools.size());
    const Side& d = mmr::store_side(s);
    const Side& p = pages->pools[static_cast<size_t>(pool)].side;
    if (p.rank != 4 || p.size[1] != pages->state.T || p.size[2] != d.size[1] || p.size[3] != d.size[2] || p.dtype != d.dtype ||
        p.tiles[1] != 1)
      return fail(MMR_INVALID_ARGUMENT, "pool %d is not [pages, %d, %lld, %lld] of the type of the %s store, heads alone sharded", pool,
                  pages->state.T, (long long)d.size[1], (long long)d.size[2], what);
    if (int rc = check_row(p, "pool")) return rc;
    if (p.dev_count != d.dev_count) return fail(MMR_INVALID_ARGUMENT, "%s store and pool %d are on different devices", what, pool);
    for (int64_t dev = 0; dev < d.dev_count; ++dev)
      if (tile_at(p, dev, 2) != tile_at(d, dev, 1) || p.tiles[2] != d.tiles[1])
        return fail(MMR_INVALID_ARGUMENT, "the heads of the %s store and of pool %d are sharded differently", what, pool);
    if (turn)
      if (int rc = check_rotary(ctx, rotary, d.size[2], d.dtype)) return rc;
    return add(s, &p, &pages->pools[static_cast<size_t>(pool)].tiles, nullptr, turn);
  };
  if (q) {
    if (int rc = check_new(q, "q")) return rc;
    if (int rc = mmr::context_check_store(ctx, q_out, "q_out")) return rc;
    if (q != q_out && mmr::store_key(q) != mmr::store_key(q_out))
      return fail(MMR_INVALID_ARGUMENT, "q and q_out have different descriptors");
    if (q_out == k || q_out == v) return fail(MMR_INVALID_ARGUMENT, "q_out is also the %s store", q_out == k ? "k" : "v");
    if (int rc = check_rotary(ctx, rotary, mmr::store_side(q).size[2], dtype)) return rc;
    if (int rc = add(q, nullptr, nullptr, q_out, true)) return rc;
  }
  if (int rc = add_pool(k, k_pool, rotary != nullptr, "k")) return rc;
  if (v)
    if (int rc = add_pool(v, v_pool, false, "v")) return rc;
  if (n == 0 || l.buffers.empty()) return MMR_OK;
  l.type = rotary ? dtype : -1;
  const mmr::PageState& st = pages->state;
  l.pages = {st.table, st.lengths, sequences, begins, pages->work.header + mmr::kPageStatus, n, st.S, st.B, st.P, st.T,
                  st.capacity, st.div_T};
  mmr::context_hash(ctx, 22, {static_cast<uint64_t>(mmr::store_ordinal(k)), static_cast<uint64_t>(k_pool), static_cast<uint64_t>(n)});
  return launch_rows(ctx, &l, rows, itemsize);
} catch (...) {
  return exception_status();
}

}  // extern "C"
