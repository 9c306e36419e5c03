// gfx950 kernels of the page cache and of rotary positions.  What a workgroup does stands in page_ops.h and
// rotary_ops.h, shared with the host emulation of the tests; here is how a workgroup synchronises, and the launches.
#include <hip/hip_runtime.h>

#include "device_mem.h"
#include "page_kernels.h"

namespace mmr {
namespace {

typedef RowMem<true, true> StreamMem;  // every byte is touched once

// A workgroup of K threads.
template <int K>
struct Workgroup {
  static constexpr int kThreads = K;
  int32_t tid;
  uint32_t block, blocks;
  int32_t* shared;  // K / 64 + 1 words for the scan

  __device__ __forceinline__ Workgroup(int32_t* lds) : tid(threadIdx.x), block(blockIdx.x), blocks(gridDim.x), shared(lds) {}
  __device__ __forceinline__ void sync() { __syncthreads(); }

  __device__ __forceinline__ void load4(const int32_t* p, int32_t at, int32_t n, int32_t (&r)[4]) {
    if (at + 3 < n) {
      const int4 v = *reinterpret_cast<const int4*>(p + at);  // the buffer and `at` are 16-byte aligned
      r[0] = v.x, r[1] = v.y, r[2] = v.z, r[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = at + i < n ? p[at + i] : 1;
    }
  }

  template <class V>
  __device__ __forceinline__ V scan(V v, V* total) {
    V* sums = reinterpret_cast<V*>(shared);
    const int lane = tid & 63, wave = tid >> 6;
    V in = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const V other = __shfl_up(in, d, 64);
      if (lane >= d) in += other;
    }
    if (lane == 63) sums[wave] = in;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < K / 64; ++i) {
      const V s = sums[i];
      before += i < wave ? s : 0;
      all += s;
    }
    __syncthreads();
    *total = all;
    return before + in - v;
  }

  __device__ __forceinline__ uint32_t any(uint32_t flags) {
    if (tid == 0) shared[0] = 0;
    __syncthreads();
    if (flags) atomicOr(&shared[0], static_cast<int32_t>(flags));
    __syncthreads();
    const uint32_t all = static_cast<uint32_t>(shared[0]);
    __syncthreads();
    return all;
  }

  __device__ __forceinline__ bool all(bool v) { return __all(v); }  // over the wave

  // Of n ascending values, how many are at most t; t and the call are uniform over the wave.
  __device__ __forceinline__ int32_t ended(const int32_t* ends, int32_t n, int32_t t) {
    int32_t count = 0;
    for (int32_t base = 0; base < n; base += 64) {
      const int32_t i = base + (tid & 63);
      const uint64_t below = __ballot(i < n && ends[i < n ? i : n - 1] <= t);
      count += __popcll(below);
      if (~below) break;
    }
    return count;
  }

  __device__ __forceinline__ int32_t atomic_add(int32_t* p, int32_t v) { return atomicAdd(p, v); }
  __device__ __forceinline__ int32_t atomic_exch(int32_t* p, int32_t v) { return atomicExch(p, v); }
  __device__ __forceinline__ void atomic_or(int32_t* p, int32_t v) { atomicOr(p, v); }
};

constexpr int kScanInts = 2 * (kPagePlanThreads / 64) + 2;
typedef Workgroup<kPagePlanThreads> PlanGroup;
typedef Workgroup<kPageThreads> ApplyGroup;

#define MMR_PLAN_SHARED                                              \
  __shared__ __attribute__((aligned(16))) int32_t scan[kScanInts];   \
  __shared__ int32_t prefix[kMaxPageSegments];                       \
  PlanGroup x(scan)

__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_scan_kernel(PageState st, PageWork w, bool live) {
  __shared__ __attribute__((aligned(16))) int32_t scan[kScanInts];
  PlanGroup x(scan);
  page_scan_segment(x, st, w, static_cast<int32_t>(x.block), live);
}

__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_extend_kernel(PageState st, PageWork w, const int32_t* slots,
                                                                           const int32_t* counts, int32_t n, bool whole) {
  MMR_PLAN_SHARED;
  page_extend_plan(x, st, w, prefix, slots, counts, n, whole);
}

#define MMR_ROWS_SHARED                                                                    \
  __shared__ __attribute__((aligned(16))) int32_t scan[2 * (kPageThreads / 64) + 2];       \
  __shared__ int32_t prefix[kMaxPageSegments];                                             \
  ApplyGroup x(scan)

__global__ __launch_bounds__(kPageThreads) void mmr_page_extend_rows_kernel(PageState st, PageWork w, const int32_t* slots,
                                                                            const int32_t* counts, int32_t n) {
  MMR_ROWS_SHARED;
  page_extend_rows<ApplyGroup, kPageSegment>(x, st, w, prefix, slots, counts, n);
}

__global__ __launch_bounds__(kPageThreads) void mmr_page_compact_list_kernel(PageState st, PageWork w) {
  MMR_ROWS_SHARED;
  page_compact_list<ApplyGroup, kPageSegment>(x, st, w, prefix);
}

// The first workgroups scan, the others check the pages that the children will share.
__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_fork_scan_kernel(PageState st, PageWork w, const int32_t* parents,
                                                                              const int32_t* children, int32_t n) {
  __shared__ __attribute__((aligned(16))) int32_t scan[kScanInts];
  PlanGroup x(scan);
  const uint32_t segments = static_cast<uint32_t>(w.n_segments);
  if (x.block < segments) page_scan_segment(x, st, w, static_cast<int32_t>(x.block), false);
  else page_fork_check(x, st, w, parents, children, n, x.block - segments, x.blocks - segments);
}

__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_fork_plan_kernel(PageState st, PageWork w, const int32_t* parents,
                                                                              const int32_t* children, int32_t n, bool prepared) {
  MMR_PLAN_SHARED;
  page_fork_plan(x, st, w, prefix, parents, children, n, prepared);
}

__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_compact_plan_kernel(PageState st, PageWork w, bool whole) {
  MMR_PLAN_SHARED;
  page_compact_plan(x, st, w, prefix, whole);
}

__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_count_kernel(PageState st, PageWork w) {
  MMR_PLAN_SHARED;
  page_count(x, st, w, prefix);
}

__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_copy_plan_kernel(PageState st, PageWork w, const int32_t* src,
                                                                              const int32_t* dst, int32_t n, bool sorted) {
  __shared__ __attribute__((aligned(16))) int32_t scan[kScanInts];
  PlanGroup x(scan);
  page_copy_plan(x, st, w, src, dst, n, sorted);
}

template <bool ALIGNED>
__global__ __launch_bounds__(kPageThreads) void mmr_page_copy_few_kernel(PageState st, PageWork w, PageMover mv, const int32_t* src,
                                                                         const int32_t* dst, int32_t n) {
  __shared__ __attribute__((aligned(16))) int32_t scan[2 * (kPageThreads / 64) + 2];
  __shared__ int32_t pairs[2 * kFewPairs];
  ApplyGroup x(scan);
  if (!page_copy_few(x, st, w, pairs, src, dst, n)) return;
  page_move_chunk<StreamMem, ALIGNED, false>(mv, [&](uint32_t i) { return PageMove{pairs[i], pairs[kFewPairs + i]}; },
                                      static_cast<uint32_t>(n), blockIdx.x, threadIdx.x);
}

__global__ __launch_bounds__(kPagePlanThreads) void mmr_page_free_kernel(PageState st, PageWork w, const int32_t* slots) {
  __shared__ __attribute__((aligned(16))) int32_t scan[kScanInts];
  PlanGroup x(scan);
  page_free(x, st, w, scan, slots);
}

// The first `row_blocks` workgroups write tables (KIND 1: fork, 2: compact; 0: none), the others move pages.  The page that
// a fork copies is often the last one of several entries: its loads go through the caches (256 sequences forked from 16,
// 402 MB written: 82 us; past the caches 131 us).  A copy or a compact reads every page once, past the caches (copy of
// 805 MB 308 us, through them 311; compact 719 and 728).
template <int KIND, bool ALIGNED, bool PACKED>
__global__ __launch_bounds__(kPageThreads) void mmr_page_apply_kernel(PageState st, PageWork w, PageMover mv,
                                                                      const int32_t* parents, const int32_t* children, int32_t n,
                                                                      uint32_t row_blocks) {
  if (!w.header[kPageOk]) return;
  if (KIND != 0 && blockIdx.x < row_blocks) {
    __shared__ __attribute__((aligned(16))) int32_t scan[2 * (kPageThreads / 64) + 2];
    ApplyGroup x(scan);
    if (KIND == 1) page_fork_rows(x, st, w, parents, children, n, blockIdx.x, row_blocks);
    else page_compact_rows(x, st, w, blockIdx.x, row_blocks);
    return;
  }
  const uint32_t moves = static_cast<uint32_t>(w.header[kPageMoves]), items = page_items<PACKED>(mv, moves);
  const uint32_t step = gridDim.x - row_blocks;
  for (uint32_t at = blockIdx.x - row_blocks; at < (items + 511u) / 512u * 512u; at += step) {
    const uint32_t item = chunk_index(at, 64);  // runs of 64 neighbours share an XCD
    typedef RowMem<KIND != 1, true> M;
    if (item < items) page_move_chunk<M, ALIGNED, PACKED>(mv, [&](uint32_t i) { return w.moves[i]; }, moves, item, threadIdx.x);
  }
}

// STREAM: a launch that writes more than the caches keep for a reader writes past them, if its stores are whole lines
// (queries, keys and values of 18,001 tokens, 443 MB in all: 82.4 -> 79.3 us; the gradient of bf16 [4,32,2048,128] 23.9 ->
// 20.7 us; parts of lines meet in the L2 instead: bf16 rows of 80 with halves of 80 bytes 32.1 us through it, 42.5 past
// it); what a small one writes, a decode step's queries and keys, stays for the kernel that reads it next.
template <class T, int VEC, bool INTERLEAVED, bool STREAM, class Args>
__global__ __launch_bounds__(kRotaryThreads) void mmr_rotary_kernel(Args a) {
  Workgroup<kRotaryThreads> x(nullptr);
  const RotaryBuffer& b = a.buffers[blockIdx.y];
  const RotaryShape& j = a.shapes[Args::kShapes == 1 ? 0 : b.shape];
  if (x.block >= j.blocks) return;  // uniform over the workgroup
  rotary_block<RowMem<false, STREAM>, T, VEC, INTERLEAVED>(x, a.angles, a.pages, j, b);
}

template <class Args>
hipError_t launch_rotary_args(const RotaryLaunch& l, const Args& args, uint32_t blocks, int n, hipStream_t stream) {
  const dim3 grid(blocks, static_cast<uint32_t>(n)), threads(kRotaryThreads);
#define MMR_ROTARY(T, V, I, S) hipLaunchKernelGGL((mmr_rotary_kernel<T, V, I, S, Args>), grid, threads, 0, stream, args)
#define MMR_ROTARY_WIDE(T, V, I)                      \
  do {                                                \
    if (l.past_caches) MMR_ROTARY(T, V, I, true);     \
    else MMR_ROTARY(T, V, I, false);                  \
  } while (0)
// narrower vectors: 8 bytes, 4 bytes, or a single element where the halves of the rotated part are of odd length
#define MMR_ROTARY_16(T)                                                          \
  do {                                                                            \
    if (l.vector_bytes == 16 && l.interleaved) MMR_ROTARY_WIDE(T, 8, true);       \
    else if (l.vector_bytes == 16) MMR_ROTARY_WIDE(T, 8, false);                  \
    else if (l.vector_bytes == 8 && l.interleaved) MMR_ROTARY(T, 4, true, false); \
    else if (l.vector_bytes == 8) MMR_ROTARY(T, 4, false, false);                 \
    else if (l.interleaved) MMR_ROTARY(T, 2, true, false);                        \
    else if (l.vector_bytes == 4) MMR_ROTARY(T, 2, false, false);                 \
    else MMR_ROTARY(T, 1, false, false);                                          \
  } while (0)
  switch (l.type) {
    case MMR_F32:
      if (l.vector_bytes == 16 && l.interleaved) MMR_ROTARY_WIDE(RotaryF32, 4, true);
      else if (l.vector_bytes == 16) MMR_ROTARY_WIDE(RotaryF32, 4, false);
      else if (l.interleaved) MMR_ROTARY(RotaryF32, 2, true, false);
      else if (l.vector_bytes == 8) MMR_ROTARY(RotaryF32, 2, false, false);
      else MMR_ROTARY(RotaryF32, 1, false, false);
      break;
    case MMR_BF16: MMR_ROTARY_16(RotaryBF16); break;
    case MMR_F16: MMR_ROTARY_16(RotaryF16); break;
    default:
      if (l.vector_bytes == 16) MMR_ROTARY_WIDE(RotaryRaw, 16, false);
      else MMR_ROTARY(RotaryRaw, 1, false, false);
  }
#undef MMR_ROTARY_16
#undef MMR_ROTARY_WIDE
#undef MMR_ROTARY
  return hipGetLastError();
}

// Buffers [at, at + n) of a launch, with the shapes they have.
template <class Args>
hipError_t launch_rotary_part(const RotaryLaunch& l, size_t at, int n, hipStream_t stream) {
  Args args;
  args.angles = l.angles;
  args.pages = l.pages;
  for (int i = 0; i < Args::kShapes; ++i) args.shapes[i] = i < static_cast<int>(l.shapes.size()) ? l.shapes[static_cast<size_t>(i)] : RotaryShape{};
  uint32_t blocks = 0;
  for (int i = 0; i < Args::kBuffers; ++i) {
    args.buffers[i] = i < n ? l.buffers[at + static_cast<size_t>(i)] : RotaryBuffer{};
    if (i >= n) continue;
    const uint32_t mine = l.shapes[args.buffers[i].shape].blocks;
    blocks = mine > blocks ? mine : blocks;
  }
  return launch_rotary_args(l, args, blocks, n, stream);
}

hipError_t launched(int* launches) {
  *launches += 1;
  return hipGetLastError();
}

// The launch before a plan, where the pool is more than a plan scans itself.
hipError_t launch_scan(const PageState& st, const PageWork& w, bool live, hipStream_t stream, int* launches) {
  if (w.n_segments <= kPlanScans) return hipSuccess;
  hipLaunchKernelGGL(mmr_page_scan_kernel, dim3(static_cast<uint32_t>(w.n_segments)), dim3(kPagePlanThreads), 0, stream, st, w, live);
  return launched(launches);
}

// Workgroups of a move: one per chunk up to this many, which then loop.
constexpr uint64_t kMaxMoveBlocks = 1u << 18;

// Up to so many pages the plan of a compact lists the moves itself, in at most 8 rounds (compact of 16,384 pages of 256
// bytes: 19.9 us, with a launch for the list 21.8; of 32,768: 30.1 and 23.7).
constexpr int32_t kCompactWhole = 16384;
// A copy of few pairs is one launch, whose workgroups (one a chunk) each check all pairs, up to so many workgroups times
// pairs: 4 pairs of 1,024 chunks 4.6 us, in two launches 7.7; 16 of 1,024 5.5 and 7.5; 32 of 512 5.9 and 7.9; but 64 of
// 1,024 9.7 and 8.8, 32 of 8,192 32.5 and 29.2.  The product is a rough measure: 32 of 2,048, as many checks as 64 of 1,024,
// would take 9.8 and go in two launches at 13.1.
constexpr uint64_t kFewChecks = 48 * 1024;

template <int KIND>
hipError_t launch_apply(const PageState& st, const PageWork& w, const PageMoveLaunch& mv, const int32_t* parents,
                        const int32_t* children, int32_t n, uint32_t row_blocks, hipStream_t stream, int* launches) {
  const uint64_t items = mv.packed ? page_items<true>(mv.mover, mv.max_moves) : page_items<false>(mv.mover, mv.max_moves);
  const uint32_t movers = static_cast<uint32_t>(items < kMaxMoveBlocks ? (items + 511) / 512 * 512 : kMaxMoveBlocks);
  if (movers + row_blocks == 0) return hipSuccess;
#define MMR_APPLY(A, P)                                                                                                          \
  hipLaunchKernelGGL((mmr_page_apply_kernel<KIND, A, P>), dim3(movers + row_blocks), dim3(kPageThreads), 0, stream, st, w, mv.mover, \
                     parents, children, n, row_blocks)
  if (mv.aligned && mv.packed) MMR_APPLY(true, true);
  else if (mv.aligned) MMR_APPLY(true, false);
  else if (mv.packed) MMR_APPLY(false, true);
  else MMR_APPLY(false, false);
#undef MMR_APPLY
  return launched(launches);
}

}  // namespace

// Extend is one launch (besides the scan's) where no call of this size can give out more pages than the plan's workgroup
// writes in 16 rounds; else another one follows it, which does the writing if there is more than kExtendFew (768 prompts of
// 128 pages each: 97 us by one workgroup) and otherwise ends at once.
constexpr int64_t kExtendWhole = 16384;

hipError_t launch_page_extend(const PageState& st, const PageWork& w, const int32_t* slots, const int32_t* counts, int32_t n,
                              hipStream_t stream, int* launches) {
  const int64_t most = static_cast<int64_t>(n) * st.B;
  const bool whole = (most < st.P ? most : st.P) <= kExtendWhole;
  if (hipError_t e = launch_scan(st, w, false, stream, launches)) return e;
  hipLaunchKernelGGL(mmr_page_extend_kernel, dim3(1), dim3(kPagePlanThreads), 0, stream, st, w, slots, counts, n, whole);
  if (hipError_t e = launched(launches)) return e;
  if (whole) return hipSuccess;
  hipLaunchKernelGGL(mmr_page_extend_rows_kernel, dim3(static_cast<uint32_t>(n < 4096 ? n : 4096)), dim3(kPageThreads), 0, stream, st,
                     w, slots, counts, n);
  return launched(launches);
}

hipError_t launch_page_free(const PageState& st, const PageWork& w, const int32_t* slots, int32_t n, hipStream_t stream, int* launches) {
  hipLaunchKernelGGL(mmr_page_free_kernel, dim3(static_cast<uint32_t>(n)), dim3(kPagePlanThreads), 0, stream, st, w, slots);
  return launched(launches);
}

// Places of the parents' rows (children times pages a row) up to which the plan of a fork checks them itself, in at most 4
// rounds: a call of 4,096 places, copying its tables included, 16.4 us, with a launch for the check 18.9; of 8,192 19.3 and
// 18.9; of 32,768 36.5 and 18.9.  Where the pool has more segments than the plan scans, the launch is there already.
constexpr int64_t kForkWhole = 4096;

hipError_t launch_page_fork(const PageState& st, const PageWork& w, const int32_t* parents, const int32_t* children, int32_t n,
                            const PageMoveLaunch& mv, hipStream_t stream, int* launches) {
  const bool prepared = w.n_segments > kPlanScans || static_cast<int64_t>(n) * st.B > kForkWhole;
  if (prepared) {
    const uint32_t blocks = static_cast<uint32_t>(w.n_segments) + static_cast<uint32_t>(n < 4096 ? n : 4096);
    hipLaunchKernelGGL(mmr_page_fork_scan_kernel, dim3(blocks), dim3(kPagePlanThreads), 0, stream, st, w, parents, children, n);
    if (hipError_t e = launched(launches)) return e;
  }
  hipLaunchKernelGGL(mmr_page_fork_plan_kernel, dim3(1), dim3(kPagePlanThreads), 0, stream, st, w, parents, children, n, prepared);
  if (hipError_t e = launched(launches)) return e;
  return launch_apply<1>(st, w, mv, parents, children, n, static_cast<uint32_t>(n < 4096 ? n : 4096), stream, launches);
}

hipError_t launch_page_compact(const PageState& st, const PageWork& w, const PageMoveLaunch& mv, hipStream_t stream, int* launches) {
  const bool whole = st.P <= kCompactWhole;
  if (hipError_t e = launch_scan(st, w, true, stream, launches)) return e;
  hipLaunchKernelGGL(mmr_page_compact_plan_kernel, dim3(1), dim3(kPagePlanThreads), 0, stream, st, w, whole);
  if (hipError_t e = launched(launches)) return e;
  if (!whole) {
    const uint32_t blocks = (mv.max_moves + kPageThreads - 1) / kPageThreads;
    hipLaunchKernelGGL(mmr_page_compact_list_kernel, dim3(blocks < 1024 ? blocks : 1024), dim3(kPageThreads), 0, stream, st, w);
    if (hipError_t e = launched(launches)) return e;
  }
  return launch_apply<2>(st, w, mv, nullptr, nullptr, 0, static_cast<uint32_t>(st.S < 4096 ? st.S : 4096), stream, launches);
}

hipError_t launch_page_copy(const PageState& st, const PageWork& w, const int32_t* src, const int32_t* dst, int32_t n,
                            const PageMoveLaunch& mv, hipStream_t stream, int* launches) {
  const uint64_t items = static_cast<uint64_t>(n) * mv.mover.n_buffers * mv.mover.chunks;
  if (n <= kFewPairs && items * static_cast<uint64_t>(n) <= kFewChecks) {
    const dim3 grid(static_cast<uint32_t>(items));
    if (mv.aligned) hipLaunchKernelGGL(mmr_page_copy_few_kernel<true>, grid, dim3(kPageThreads), 0, stream, st, w, mv.mover, src, dst, n);
    else hipLaunchKernelGGL(mmr_page_copy_few_kernel<false>, grid, dim3(kPageThreads), 0, stream, st, w, mv.mover, src, dst, n);
    return launched(launches);
  }
  // in the order of the destinations 512 pages of 32 KiB in each of 48 buffers take 293 us, in the caller's 308; where the pairs
  // are few among the pages the pass over these costs more than it gives (512 of 20,000: 59 us, sorted 69)
  const bool sorted = st.P / 8 <= n;
  hipLaunchKernelGGL(mmr_page_copy_plan_kernel, dim3(1), dim3(kPagePlanThreads), 0, stream, st, w, src, dst, n, sorted);
  if (hipError_t e = launched(launches)) return e;
  return launch_apply<0>(st, w, mv, nullptr, nullptr, 0, 0, stream, launches);
}

hipError_t launch_page_count(const PageState& st, const PageWork& w, hipStream_t stream, int* launches) {
  if (hipError_t e = launch_scan(st, w, false, stream, launches)) return e;
  hipLaunchKernelGGL(mmr_page_count_kernel, dim3(1), dim3(kPagePlanThreads), 0, stream, st, w);
  return launched(launches);
}

hipError_t launch_rotary(const RotaryLaunch& l, int* launches, hipStream_t stream) {
  *launches = 0;
  for (size_t at = 0; at < l.buffers.size();) {
    const size_t left = l.buffers.size() - at;
    const int n = static_cast<int>(left < RotaryManyBuffers::kBuffers ? left : RotaryManyBuffers::kBuffers);
    hipError_t e;
    if (l.shapes.size() == 1 && n <= RotaryOneShape::kBuffers) e = launch_rotary_part<RotaryOneShape>(l, at, n, stream);
    else if (n <= RotaryFewBuffers::kBuffers) e = launch_rotary_part<RotaryFewBuffers>(l, at, n, stream);
    else e = launch_rotary_part<RotaryManyBuffers>(l, at, n, stream);
    if (e) return e;
    *launches += 1;
    at += static_cast<size_t>(n);
  }
  return hipSuccess;
}

}  // namespace mmr
