// Philox4x32-10 is the counter-based generator of Salmon, Moraes, Dror and Shaw ("Parallel random numbers: as
// easy as 1, 2, 3", SC 2011; Random123): ten rounds of two 32x32 -> 64-bit multiplications (0xD2511F53,
// 0xCD9E8D57) with the key bumped by the Weyl constants (0x9E3779B9, 0xBB67AE85) between rounds.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace efgs {

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint2 k) {
#pragma unroll
    for (int r = 0; r < 10; r++) {
        if (r > 0) {
            k.x += 0x9E3779B9u;
            k.y += 0xBB67AE85u;
        }
        const uint32_t lo0 = 0xD2511F53u * c.x, hi0 = __umulhi(0xD2511F53u, c.x);
        const uint32_t lo1 = 0xCD9E8D57u * c.z, hi1 = __umulhi(0xCD9E8D57u, c.z);
        c = make_uint4(hi1 ^ c.y ^ k.x, lo1, hi0 ^ c.w ^ k.y, lo0);
    }
    return c;
}

}  // namespace efgs
