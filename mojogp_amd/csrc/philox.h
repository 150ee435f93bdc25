// Counter-based random numbers on the device: the Philox4x32-10 block of counter
// (block, step) and key seed (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", 2011).
#pragma once

#include "mgp_common.h"

namespace mgp {

struct Draws {
  uint32_t w[4];
  __device__ __forceinline__ uint32_t half(int i) const {
    return (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
  }
};

__device__ __forceinline__ Draws philox(uint64_t block, uint64_t seed, uint64_t step = 0) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

}  // namespace mgp
