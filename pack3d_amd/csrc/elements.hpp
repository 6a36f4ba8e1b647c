// Runs of consecutive elements at any element alignment, and sums over the lanes of
// a row.
#pragma once

#include "common.hpp"

namespace p3d {

// E elements as they lie in memory.  Copied with the alignment of one element: global
// memory takes accesses of up to 16 bytes at any element address, so odd widths and
// strides run the same wide instructions.
template <typename T, int E>
struct Run {
    T v[E];
    __device__ __forceinline__ void load(const void* p) { __builtin_memcpy(v, p, sizeof(v)); }
    __device__ __forceinline__ void store(void* p) const { __builtin_memcpy(p, v, sizeof(v)); }
    __device__ __forceinline__ void to(float (&f)[E]) const {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = to_f32(v[e]);
    }
    __device__ __forceinline__ void from(const float (&f)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = from_f32<T>(f[e]);
    }
};

__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float x) {
    if (dtype == P3D_F32) reinterpret_cast<float*>(p)[i] = x;
    else if (dtype == P3D_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)x;
    else reinterpret_cast<__bf16*>(p)[i] = (__bf16)x;
}

// base + row * stride bytes, with both below 2^32: one multiply-add.  Addresses stay
// pointers of the kernel's arguments: ones made from integers compile to flat accesses,
// whose waits are the LDS's too, and no load is then ahead of a reduction.
__device__ __forceinline__ const char* row_address(const char* base, uint32_t row, uint32_t stride) {
    return base + (uint64_t)row * stride;
}
__device__ __forceinline__ char* row_address(char* base, uint32_t row, uint32_t stride) {
    return base + (uint64_t)row * stride;
}

// Sum over an aligned group of LANES lanes (a power of two from 2 to 64); every lane of
// the group ends with the same bits.
template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
    x += dpp_move<0xB1>(x);
    if constexpr (LANES >= 4) x += dpp_move<0x4E>(x);
    if constexpr (LANES >= 8) x += dpp_move<0x141>(x);
    if constexpr (LANES >= 16) x += dpp_move<0x140>(x);
    // The row swaps give x of the even and of the odd rows (halves), in every lane.
    if constexpr (LANES >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (LANES >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return x;
}

// Sums of N values over the TPR threads of a row.  Rows of more than one wave
// meet in LDS: the two buffers take turns, so that one barrier a sum is enough
// (a buffer is written again only past the next sum's barrier, by when every
// wave has read it).
template <int TPR>
struct RowSum {
    static constexpr int WAVES = TPR > 64 ? TPR / 64 : 1;
    // Lanes that add the waves' sums: the next power of two, the last ones adding nothing.
    static constexpr int SLOTS = WAVES <= 2 ? 2 : (WAVES <= 4 ? 4 : (WAVES <= 8 ? 8 : 16));
    static constexpr int LDS = TPR > 64 ? 2 * SLOTS * 3 : 1;
    float* lds;  // LDS floats
    int turn = 0;

    template <int N>
    __device__ __forceinline__ void sum(float (&x)[N]) {
        static_assert(N <= 3, "room for three values");
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = group_sum<(TPR > 64 ? 64 : TPR)>(x[i]);
        if constexpr (TPR > 64) {
            float* buf = lds + turn * SLOTS * 3;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) buf[i * SLOTS + (threadIdx.x >> 6)] = x[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int slot = threadIdx.x % SLOTS;
                const float s = buf[i * SLOTS + slot];
                x[i] = group_sum<SLOTS>(SLOTS == WAVES || slot < WAVES ? s : 0.f);
            }
        }
    }
};

}  // namespace p3d
