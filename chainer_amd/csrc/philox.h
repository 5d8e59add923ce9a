// The counter-based generator of the kernels that draw random numbers.
#pragma once

#include "common.h"

namespace hipcx {

// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): 128 bits that depend on a counter and a key alone.
__device__ __forceinline__ void Philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = uint64_t{0xD2511F53u} * c[0], p1 = uint64_t{0xCD9E8D57u} * c[2];
        const uint32_t c1 = c[1], c3 = c[3];
        c[0] = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0, c[1] = static_cast<uint32_t>(p1);
        c[2] = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1, c[3] = static_cast<uint32_t>(p0);
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
}

}  // namespace hipcx
