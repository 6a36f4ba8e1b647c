// The dropout mask: a function of (seed, offset, element index), computed where
// it is needed and never stored.
//
// Element i of a tensor in its logical (row-major) order compares 16 bits with a
// threshold t = round(65536 p): half i % 8 of the 128 bits that Philox4x32-10
// (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC
// 2011) gives for the counter (i / 8, offset) and the key seed.  16 bits an element
// make the rate a multiple of 2^-16 (what is kept is divided by the rate that the
// threshold gives, so the mean stays exact) and one block serves eight elements:
// 20 products of 32 bits for eight elements.
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

// a ^ b ^ c in one instruction (0x96 is its truth table).
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
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
        c[0] = xor3((uint32_t)(b >> 32), c1, k0);
        c[1] = (uint32_t)b;
        c[2] = xor3((uint32_t)(a >> 32), c3, k1);
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

// Bits of a lane's E <= 8 elements, from channel c of row `row` on, in a tensor of rows
// of dim.  TPR lanes (every one of them here) hold the row, lane `sub` of them from
// channel E sub on or less.
//
// Where runs of eight and groups coincide each lane computes its own group.  Else the
// row's groups are dealt out over its lanes and passed between them: a run overlaps two
// groups, and computing both in each lane took twice the generator's time.  Rows wider
// than a wave do that all the same.
template <int TPR, int E>
__device__ __forceinline__ uint32_t keep_run(const MaskDev& m, uint32_t row, int dim, int c, int sub) {
    if (E == 8 && dim % 8 == 0) return keep_group(m, (uint64_t)row * (uint32_t)(dim / 8) + (c >> 3));
    const uint64_t start = (uint64_t)row * (uint32_t)dim;
    if constexpr (TPR > 64) {
        const uint64_t first = start + c;
        const uint32_t shift = (uint32_t)first & 7;
        uint32_t bits = keep_group(m, first >> 3);
        if (shift + E > 8) bits |= keep_group(m, (first >> 3) + 1) << 8;
        return bits >> shift;
    } else {
        const uint64_t group = start >> 3;
        const uint32_t at = (uint32_t)(start & 7) + c, g = at >> 3;
        const uint32_t mine = keep_group(m, group + sub);
        uint32_t low = __shfl(mine, (int)g, TPR), high = __shfl(mine, (int)g + 1, TPR);
        // Rows that fill their lanes and start inside a group reach one group past them.
        if (E * TPR / 8 >= TPR && (at & 7) + E > 8 && g + 1 == TPR) high = keep_group(m, group + TPR);
        return (low | high << 8) >> (at & 7);
    }
}

// Bit e of bits as a word: all ones where it is set.  (The instruction by name: the
// compiler makes a comparison and a select, with a wait between them, of the builtin.)
__device__ __forceinline__ uint32_t bit_word(uint32_t bits, int e) {
    uint32_t w;
    asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(w) : "v"(bits), "n"(e));
    return w;
}
__device__ __forceinline__ float and_word(float x, uint32_t w) { return __uint_as_float(__float_as_uint(x) & w); }

}  // namespace p3d
