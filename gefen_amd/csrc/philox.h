// Dropout's factors from a counter: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", 2011) with key = seed and counter = (element / 8,
// offset).  A block's four words serve eight elements with 16 bits each, low half first, and
// an element is kept where its 16 bits are at least `cut`: a probability is a multiple of
// 2^-16.  Ten rounds for eight elements instead of four keep the generator (20 wide
// multiplications a block) below the time that 16-bit elements take to move.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_internal.h"

namespace gefen {

struct Dropout {
    const int64_t* seed_at;  // device; NULL: seed
    int64_t seed, offset;
    uint32_t cut;            // 65536 p, 0: nothing is dropped
    float scale;             // 1 / (1 - p)
};

inline bool dropout_of(double p, const int64_t* seed_at, int64_t seed, int64_t offset, Dropout* out) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    out->seed_at = seed_at;
    out->seed = seed;
    out->offset = offset;
    out->cut = (uint32_t)nearbyint(p * 65536.0);
    out->scale = out->cut == 65536u ? 0.0f : (float)(65536.0 / (65536.0 - out->cut));
    return true;
}

__device__ __forceinline__ uint64_t dropout_seed(const Dropout& d) {
    return (uint64_t)(d.seed_at ? *d.seed_at : d.seed);
}

// Which of the eight elements of a block are kept, bit by bit.
__device__ __forceinline__ uint32_t philox_keep(uint64_t block, uint64_t offset, uint64_t seed, uint32_t cut) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    const uint32_t w[4] = {c0, c1, c2, c3};
    uint32_t keep = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        keep |= (w[i] & 0xffffu) >= cut ? 1u << (2 * i) : 0u;
        keep |= (w[i] >> 16) >= cut ? 2u << (2 * i) : 0u;
    }
    return keep;
}
// The same of the eight elements from e on.
__device__ __forceinline__ uint32_t dropout_keep(const Dropout& d, uint64_t seed, int64_t e) {
    const uint32_t at = (uint32_t)e & 7u;
    const uint32_t low = philox_keep((uint64_t)e >> 3, (uint64_t)d.offset, seed, d.cut);
    if (at == 0) return low;
    return (low | philox_keep(((uint64_t)e >> 3) + 1, (uint64_t)d.offset, seed, d.cut) << 8) >> at;
}
// An element that is dropped counts as zero whatever it holds.
__device__ __forceinline__ float dropped(float v, uint32_t keep, int k, float scale) {
    return keep >> k & 1u ? v * scale : 0.0f;
}

}  // namespace gefen
