// Launchers of the page-cache and rotary kernels (page_ops.h, rotary_ops.h).
#ifndef MMR_CSRC_PAGE_KERNELS_H_
#define MMR_CSRC_PAGE_KERNELS_H_

#include <hip/hip_runtime_api.h>

#include <vector>

#include "page_ops.h"
#include "rotary_ops.h"

namespace mmr {

constexpr int kPagePlanThreads = 1024;
constexpr int32_t kPageSegment = kPagesPerThread * kPagePlanThreads;  // pages a workgroup of a plan scans
constexpr int32_t kMaxPages = kPageSegment * kMaxPageSegments;

// Chunks are numbered with 31 bits; `max_moves` bounds the moves a call can make.
struct PageMoveLaunch {
  PageMover mover;
  uint32_t max_moves;
  bool aligned;  // every page is a multiple of 16 bytes
  bool packed;   // a page takes at most half a workgroup, 16 bytes a lane
};

// All of them add the launches they make to *launches.
hipError_t launch_page_extend(const PageState& st, const PageWork& w, const int32_t* slots, const int32_t* counts, int32_t n,
                              hipStream_t stream, int* launches);
hipError_t launch_page_free(const PageState& st, const PageWork& w, const int32_t* slots, int32_t n, hipStream_t stream, int* launches);
hipError_t launch_page_fork(const PageState& st, const PageWork& w, const int32_t* parents, const int32_t* children, int32_t n,
                            const PageMoveLaunch& mv, hipStream_t stream, int* launches);
hipError_t launch_page_compact(const PageState& st, const PageWork& w, const PageMoveLaunch& mv, hipStream_t stream, int* launches);
hipError_t launch_page_copy(const PageState& st, const PageWork& w, const int32_t* src, const int32_t* dst, int32_t n,
                            const PageMoveLaunch& mv, hipStream_t stream, int* launches);
hipError_t launch_page_count(const PageState& st, const PageWork& w, hipStream_t stream, int* launches);

// One call's rows: at most kRotaryShapes shapes, any number of buffers (several launches if there are many).
struct RotaryLaunch {
  RotaryAngles angles{};
  RotaryPages pages{};
  std::vector<RotaryShape> shapes;
  std::vector<RotaryBuffer> buffers;
  int type = -1;  // MMR_F32, MMR_BF16 or MMR_F16; -1: rows only move (nothing is turned)
  int vector_bytes = 0;  // 16: rows, turned parts and strides are whole vectors; else what divides the turned part
  bool interleaved = false;
  bool past_caches = false;  // how results are stored (16-byte vectors alone)
};
hipError_t launch_rotary(const RotaryLaunch& l, int* launches, hipStream_t stream);

}  // namespace mmr

#endif  // MMR_CSRC_PAGE_KERNELS_H_
