// The dropout mask: a function of (seed, offset, element index), computed where
// it is needed and never stored.
//
// Element i of a tensor in its logical (row-major) order compares 16 bits with a
// threshold t = round(65536 p): half i % 8 of the 128 bits that Philox4x32-10
// (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC
// 2011) gives for the counter (i / 8, offset) and the key seed.  16 bits an element
// make the rate a multiple of 2^-16 (what is kept is divided by the rate that the
// threshold gives, so the mean stays exact) and one block serves the eight
// elements that a lane holds: 20 products of 32 bits for eight elements.
#pragma once

#include "elements.hpp"

namespace p3d {

struct MaskDev {
    const int64_t* state;  // (seed, offset) on the device, or NULL
    uint64_t seed, offset;
    uint32_t threshold;  // 0: nothing is dropped
    float inv;           // 1 / (share that is kept)
};

inline MaskDev mask_dev(const p3d_dropout& d) {
    return MaskDev{d.state, (uint64_t)d.seed, (uint64_t)d.offset, (uint32_t)d.threshold,
                   65536.f / (float)(65536 - d.threshold)};
}
inline bool mask_ok(const p3d_dropout& d) { return d.threshold >= 0 && d.threshold <= 65535; }

// The state read into registers (uniform over the launch).
__device__ __forceinline__ void mask_begin(MaskDev& m) {
    if (m.threshold && m.state) {
        m.seed = (uint64_t)m.state[0];
        m.offset = (uint64_t)m.state[1];
    }
}

// Philox4x32-10 of the counter (group, offset).
__device__ __forceinline__ void philox(uint64_t group, uint64_t offset, uint64_t seed, uint32_t (&c)[4]) {
    c[0] = (uint32_t)group;
    c[1] = (uint32_t)(group >> 32);
    c[2] = (uint32_t)offset;
    c[3] = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
        const uint32_t c1 = c[1], c3 = c[3];
        c[0] = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c[1] = (uint32_t)b;
        c[2] = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// Bit e set: element 8 group + e stays.
__device__ __forceinline__ uint32_t keep_group(const MaskDev& m, uint64_t group) {
    uint32_t c[4];
    philox(group, m.offset, m.seed, c);
    uint32_t bits = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        bits |= ((c[w] & 0xffffu) >= m.threshold ? 1u : 0u) << (2 * w);
        bits |= ((c[w] >> 16) >= m.threshold ? 1u : 0u) << (2 * w + 1);
    }
    return bits;
}

// Bit e set: element first + e stays, e < 8.  Rows of a width that is no multiple
// of 8 start inside a group and take two of them.
__device__ __forceinline__ uint32_t keep8(const MaskDev& m, uint64_t first) {
    const uint32_t shift = (uint32_t)first & 7;
    uint32_t bits = keep_group(m, first >> 3);
    if (shift) bits = (bits | keep_group(m, (first >> 3) + 1) << 8) >> shift;
    return bits & 0xff;
}

}  // namespace p3d
