// Memory policy of the page and rotary kernels for the routines of page_ops.h and rotary_ops.h (device code only).
#ifndef MMR_CSRC_DEVICE_MEM_H_
#define MMR_CSRC_DEVICE_MEM_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "chunk_ops.h"

namespace mmr {
namespace {

// Pools and stores are always device (global) memory: address space 1 makes every access a global_* instruction, where
// a pointer read from a table would compile to flat_*.  NTL / NTS: loads / stores past the caches.  Accesses other than
// load16 / store16 may stand at any address, which gfx950 takes as a single access under the HSA runtime.
template <bool NTL, bool NTS>
struct RowMem {
  typedef __attribute__((address_space(1))) const char* cptr;
  typedef __attribute__((address_space(1))) char* ptr;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

  static __device__ __forceinline__ cptr cplace(const char* p) { return (cptr)p; }
  static __device__ __forceinline__ ptr place(char* p) { return (ptr)p; }

  template <typename T, int ALIGN>
  static __device__ __forceinline__ T ld(cptr p) {
    typedef __attribute__((address_space(1))) const T __attribute__((aligned(ALIGN))) at;
    if constexpr (NTL) return __builtin_nontemporal_load(reinterpret_cast<at*>(p));
    else return *reinterpret_cast<at*>(p);
  }
  template <typename T, int ALIGN>
  static __device__ __forceinline__ void st(ptr p, T v) {
    typedef __attribute__((address_space(1))) T __attribute__((aligned(ALIGN))) at;
    if constexpr (NTS) __builtin_nontemporal_store(v, reinterpret_cast<at*>(p));
    else *reinterpret_cast<at*>(p) = v;
  }
  static __device__ __forceinline__ V16 load16(cptr p) {
    const u32x4 v = ld<u32x4, 16>(p);
    return V16{v.x, v.y, v.z, v.w};
  }
  static __device__ __forceinline__ void store16(ptr p, V16 v) { st<u32x4, 16>(p, u32x4{v.x, v.y, v.z, v.w}); }
  static __device__ __forceinline__ V16 load16u(cptr p) {
    const u32x4 v = ld<u32x4, 1>(p);
    return V16{v.x, v.y, v.z, v.w};
  }
  template <typename T>
  static __device__ __forceinline__ T loadu(cptr p) {
    return ld<T, 1>(p);
  }
  template <typename T>
  static __device__ __forceinline__ void storeu(ptr p, T v) {
    if constexpr (sizeof(T) == 16) st<u32x4, 1>(p, u32x4{v.x, v.y, v.z, v.w});
    else st<T, 1>(p, v);
  }
};

}  // namespace
}  // namespace mmr

#endif  // MMR_CSRC_DEVICE_MEM_H_
