// Memory policy of the kernels for the routines of chunk_ops.h and page_ops.h (device code only).
#ifndef MMR_CSRC_DEVICE_MEM_H_
#define MMR_CSRC_DEVICE_MEM_H_

#include <hip/hip_runtime.h>

#include <cstdint>

#include "chunk_ops.h"

namespace mmr {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Shard buffers are always device (global) memory.  Pointers read from the
// pointer table would otherwise be generic and compile to flat_* accesses;
// address space 1 makes every access a global_* instruction.
#define MMR_GLOBAL __attribute__((address_space(1)))
typedef MMR_GLOBAL char gchar;
typedef MMR_GLOBAL const char gcchar;

// Device memory policy for chunk_ops.h.  NTL / NTS: nontemporal loads / stores
// (every byte is touched exactly once, keep it out of the caches' way), or
// plain cacheable ones (ragged rows: a line shared by two rows or two chunks
// is fetched once and its pieces merge in the L2).  gfx950 under the HSA
// runtime runs with unaligned global access enabled and the compiler emits a
// single access for the aligned(1) types below.
template <bool NTL, bool NTS>
struct DeviceMem {
  typedef gcchar* cptr;
  typedef gchar* ptr;

  template <typename T, int ALIGN>
  static __device__ __forceinline__ T ld(cptr p) {
    typedef MMR_GLOBAL const T __attribute__((aligned(ALIGN))) gt;
    if constexpr (NTL) return __builtin_nontemporal_load(reinterpret_cast<gt*>(p));
    else return *reinterpret_cast<gt*>(p);
  }
  template <typename T, int ALIGN>
  static __device__ __forceinline__ void st(ptr p, T v) {
    typedef MMR_GLOBAL T __attribute__((aligned(ALIGN))) gt;
    if constexpr (NTS) __builtin_nontemporal_store(v, reinterpret_cast<gt*>(p));
    else *reinterpret_cast<gt*>(p) = v;
  }
  static __device__ __forceinline__ V16 pack(u32x4 v) { return V16{v.x, v.y, v.z, v.w}; }
  static __device__ __forceinline__ u32x4 unpack(V16 v) { return u32x4{v.x, v.y, v.z, v.w}; }

  static __device__ __forceinline__ V16 load16(cptr p) { return pack(ld<u32x4, 16>(p)); }
  static __device__ __forceinline__ V16 load16u(cptr p) { return pack(ld<u32x4, 1>(p)); }
  // 16 bytes at any alignment that other workgroups read too: an ordinary cacheable load whatever NTL says
  static __device__ __forceinline__ V16 load16u_keep(cptr p) {
    typedef MMR_GLOBAL const u32x4 __attribute__((aligned(1))) gt;
    return pack(*reinterpret_cast<gt*>(p));
  }
  static __device__ __forceinline__ void store16(ptr p, V16 v) { st<u32x4, 16>(p, unpack(v)); }
  template <typename T>
  static __device__ __forceinline__ T loadu(cptr p) {
    if constexpr (sizeof(T) == 16) return load16u(p);
    else return ld<T, 1>(p);
  }
  template <typename T>
  static __device__ __forceinline__ void storeu(ptr p, T v) {
    if constexpr (sizeof(T) == 16) st<u32x4, 1>(p, unpack(v));
    else st<T, 1>(p, v);
  }
  // a plain pointer to device memory in this policy's terms
  static __device__ __forceinline__ cptr cplace(const char* p) { return (cptr)p; }
  static __device__ __forceinline__ ptr place(char* p) { return (ptr)p; }
  static __device__ __forceinline__ uintptr_t addr(ptr p) { return reinterpret_cast<uintptr_t>(p); }
  static __device__ __forceinline__ uintptr_t caddr(cptr p) { return reinterpret_cast<uintptr_t>(p); }
};

}  // namespace
}  // namespace mmr

#endif  // MMR_CSRC_DEVICE_MEM_H_
