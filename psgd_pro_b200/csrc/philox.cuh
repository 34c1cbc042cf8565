// The counter-based generator of the library: Philox4x32-10, shared by the staging kernels' damping noise and by dropout.
#pragma once
#include "common.cuh"

namespace psgd {

// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC'11): ten rounds of
// two 32 x 32 -> 64-bit multiplications on a 4-word counter, the 2-word key bumped by Weyl constants between
// rounds.
PSGD_DEVI uint4 philox4x32_10(uint4 c, uint32_t k0, uint32_t k1) {
  constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)M0 * c.x, p1 = (uint64_t)M1 * c.z;  // (one wide product each)
    c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k0, (uint32_t)p1, (uint32_t)(p0 >> 32) ^ c.w ^ k1, (uint32_t)p0);
    k0 += W0;
    k1 += W1;
  }
  return c;
}

// The ten round keys of a key (k0, k1), formed once per thread: the generator's rounds then take them as operands
// instead of bumping the key between rounds.
struct PhiloxKeys {
  uint32_t k0[10], k1[10];
};
PSGD_DEVI PhiloxKeys philox_keys(uint32_t k0, uint32_t k1) {
  PhiloxKeys ks;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    ks.k0[r] = k0 + (uint32_t)r * 0x9E3779B9u;
    ks.k1[r] = k1 + (uint32_t)r * 0xBB67AE85u;
  }
  return ks;
}
PSGD_DEVI uint4 philox4x32_10(uint4 c, const PhiloxKeys& ks) {
  constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint32_t hi0 = __umulhi(M0, c.x), lo0 = M0 * c.x;
    const uint32_t hi1 = __umulhi(M1, c.z), lo1 = M1 * c.z;
    c = make_uint4(hi1 ^ c.y ^ ks.k0[r], lo1, hi0 ^ c.w ^ ks.k1[r], lo0);
  }
  return c;
}

}  // namespace psgd
