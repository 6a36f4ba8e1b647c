// Eight consecutive elements at a time, at any element alignment, and sums over
// the lanes of a row.
#pragma once

#include "common.hpp"

namespace p3d {

constexpr int kPiece = 8;  // elements that a lane holds of a row: 16 bytes of a 16-bit type, 32 of fp32

template <typename T>
struct Eight {
    // Aligned as one element only: global memory takes 16-byte accesses at any
    // element address, so odd widths and strides run the same instructions.
    typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// v = the first `count` of eight elements at p, zero past them.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int count, float (&v)[kPiece]) {
    if (count >= kPiece) {
        const typename Eight<T>::type raw = *reinterpret_cast<const typename Eight<T>::type*>(p);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) v[e] = to_f32(raw[e]);
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) v[e] = e < count ? to_f32(p[e]) : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int count, const float (&v)[kPiece]) {
    if (count >= kPiece) {
        typename Eight<T>::type raw;
#pragma unroll
        for (int e = 0; e < kPiece; ++e) raw[e] = from_f32<T>(v[e]);
        *reinterpret_cast<typename Eight<T>::type*>(p) = raw;
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
            if (e < count) p[e] = from_f32<T>(v[e]);
    }
}

// The same for a tensor of a runtime dtype, from element i on.
__device__ __forceinline__ void load8_any(const void* p, int64_t i, int dtype, int count, float (&v)[kPiece]) {
    if (dtype == P3D_F32) load8(reinterpret_cast<const float*>(p) + i, count, v);
    else if (dtype == P3D_F16) load8(reinterpret_cast<const _Float16*>(p) + i, count, v);
    else load8(reinterpret_cast<const __bf16*>(p) + i, count, v);
}
__device__ __forceinline__ void store8_any(void* p, int64_t i, int dtype, int count, const float (&v)[kPiece]) {
    if (dtype == P3D_F32) store8(reinterpret_cast<float*>(p) + i, count, v);
    else if (dtype == P3D_F16) store8(reinterpret_cast<_Float16*>(p) + i, count, v);
    else store8(reinterpret_cast<__bf16*>(p) + i, count, v);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int dtype, float x) {
    if (dtype == P3D_F32) reinterpret_cast<float*>(p)[i] = x;
    else if (dtype == P3D_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)x;
    else reinterpret_cast<__bf16*>(p)[i] = (__bf16)x;
}

// Sum over an aligned group of LANES lanes (8, 16, 32 or 64); every lane of the
// group ends with the same bits.
template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
    x += dpp_move<0xB1>(x);
    x += dpp_move<0x4E>(x);
    x += dpp_move<0x141>(x);
    if constexpr (LANES >= 16) x += dpp_move<0x140>(x);
    if constexpr (LANES >= 32) x += lane_xor16(x);
    if constexpr (LANES >= 64) x += lane_xor32(x);
    return x;
}

// Sums of N values over the TPR threads of a row.  Rows of more than one wave
// meet in LDS: the two buffers take turns, so that one barrier a sum is enough
// (a buffer is written again only past the next sum's barrier, by when every
// wave has read it).
template <int TPR>
struct RowSum {
    static constexpr int WAVES = TPR > 64 ? TPR / 64 : 1;
    float* lds;  // [2][WAVES][4], with more than one wave
    int turn = 0;

    template <int N>
    __device__ __forceinline__ void sum(float (&x)[N]) {
        static_assert(N <= 4, "room for four values");
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = group_sum<(TPR > 64 ? 64 : TPR)>(x[i]);
        if constexpr (TPR > 64) {
            float* buf = lds + turn * WAVES * 4;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < N; ++i) buf[(threadIdx.x >> 6) * 4 + i] = x[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) s += buf[w * 4 + i];
                x[i] = s;
            }
        }
    }
};

}  // namespace p3d
