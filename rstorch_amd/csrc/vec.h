// Pairs of doubles at any 8-byte aligned address: one 16-byte global access either way (the hardware
// asks for no more than 4-byte alignment), so odd extents and offset views travel like aligned ones.
#pragma once

#include <hip/hip_runtime.h>

namespace rst {

typedef double v2u __attribute__((ext_vector_type(2), aligned(8)));

__device__ __forceinline__ v2u load2(const double* p) { return *reinterpret_cast<const v2u*>(p); }
// for arrays that are read once: past the caches
__device__ __forceinline__ v2u load2_stream(const double* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const v2u*>(p));
}
__device__ __forceinline__ void store2(double* p, v2u v) { *reinterpret_cast<v2u*>(p) = v; }

}  // namespace rst
