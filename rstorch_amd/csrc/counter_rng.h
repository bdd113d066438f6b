// The counter-based generator: value(seed, stream, index) is a pure function, a splitmix64 finaliser
// over a per-tensor key, so what a kernel draws does not depend on launch geometry.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace rst {

__host__ __device__ inline uint64_t mix64(uint64_t z) {
  z += 0x9E3779B97F4A7C15ULL;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ULL;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBULL;
  return z ^ (z >> 31);
}

__host__ __device__ inline uint64_t tensor_key(uint64_t seed, uint64_t stream) {
  return mix64(mix64(seed) ^ (stream * 0xD1342543DE82EF95ULL));
}

__device__ inline uint64_t draw(uint64_t key, uint64_t index) {
  return mix64(key + index * 0x9E3779B97F4A7C15ULL);
}

}  // namespace rst
