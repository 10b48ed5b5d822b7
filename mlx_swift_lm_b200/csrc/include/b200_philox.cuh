// Philox-4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", SC'11): ten rounds of two 32 x 32 -> 64 bit products turn a
// 128-bit counter and a 64-bit key into 128 random bits.
#pragma once

#include <cstdint>

namespace b200 {

__host__ __device__ __forceinline__ void philox_round(uint32_t c[4], uint32_t k[2]) {
  const uint64_t p0 = (uint64_t)0xD2511F53u * c[0];
  const uint64_t p1 = (uint64_t)0xCD9E8D57u * c[2];
  const uint32_t hi0 = (uint32_t)(p0 >> 32), lo0 = (uint32_t)p0;
  const uint32_t hi1 = (uint32_t)(p1 >> 32), lo1 = (uint32_t)p1;
  const uint32_t n0 = hi1 ^ c[1] ^ k[0];
  const uint32_t n2 = hi0 ^ c[3] ^ k[1];
  c[0] = n0;
  c[1] = lo1;
  c[2] = n2;
  c[3] = lo0;
}

// c: counter in, random words out.
__host__ __device__ __forceinline__ void philox_4x32_10(uint32_t c[4], uint64_t key) {
  uint32_t k[2] = {(uint32_t)key, (uint32_t)(key >> 32)};
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    philox_round(c, k);
    k[0] += 0x9E3779B9u;
    k[1] += 0xBB67AE85u;
  }
}

}  // namespace b200
