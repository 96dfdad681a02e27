// How the streaming kernels divide their list of weight rows: host-compilable, no CUDA types.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define B200_LIST_FN __host__ __device__ __forceinline__
#else
#define B200_LIST_FN inline
#endif

namespace b200 {

// ceil(total / parts), total >= 0, parts > 0. The 32-bit division is for speed (a 64-bit one is some hundred cycles at the start
// of a kernel that runs for ten microseconds); it is taken where the sum that it divides fits 32 bits.
B200_LIST_FN int64_t list_share(int64_t total, uint32_t parts) {
  const int64_t sum = total + parts - 1;
  return sum >> 32 ? sum / parts : static_cast<uint32_t>(sum) / parts;
}

}  // namespace b200
