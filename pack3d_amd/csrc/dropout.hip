// Dropout of a contiguous tensor: y = x / (1 - p) where the mask of philox.hpp
// keeps the element, else 0 (a select: what is dropped may be infinite or NaN).
// The backward is the same pass over the output's gradient.  Bound by memory: 4
// bytes an element in 16 bits, next to about 17 VALU issues for its share of the
// generator (134 million elements in bf16: 537 MB in 87 us, 6.1 TB/s).  A thread takes
// the eight elements of one run of the generator, so that no lane works out bits that
// another one uses.
#include "philox.hpp"

namespace p3d {
namespace {

constexpr int kRun = 8;

template <typename T>
__global__ __launch_bounds__(256) void k_dropout(const T* x, T* y, int64_t count, MaskDev m) {
    mask_begin(m);
    const int64_t group = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t first = group * kRun;
    if (first >= count) return;
    const bool whole = first + kRun <= count;
    Run<T, kRun> r;
    if (whole) {
        r.load(x + first);
    } else {
#pragma unroll
        for (int e = 0; e < kRun; ++e) r.v[e] = first + e < count ? x[first + e] : from_f32<T>(0.f);
    }
    const uint32_t keep = keep_group(m, (uint64_t)group);
    float v[kRun];
    r.to(v);
#pragma unroll
    for (int e = 0; e < kRun; ++e) v[e] = and_word(v[e] * m.inv, bit_word(keep, e));
    r.from(v);
    if (whole) {
        r.store(y + first);
    } else {
#pragma unroll
        for (int e = 0; e < kRun; ++e)
            if (first + e < count) y[first + e] = r.v[e];
    }
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_dropout_apply(const void* x, void* y, int64_t count, int32_t dtype, const p3d_dropout* dropout,
                                 void* stream) {
    P3D_REQUIRE(x && y && dropout, "null pointer argument");
    P3D_REQUIRE(dtype >= P3D_F32 && dtype <= P3D_BF16, "unknown dtype");
    P3D_REQUIRE(count >= 1 && cdiv(count, 256 * kRun) < (1LL << 31), "element count out of range");
    P3D_REQUIRE(mask_ok(*dropout), "threshold must be in [0, 65535]");
    const MaskDev m = mask_dev(*dropout);
    const unsigned blocks = (unsigned)cdiv(count, 256 * kRun);
    hipStream_t s = as_stream(stream);
    switch (dtype) {
        case P3D_F32: k_dropout<float><<<blocks, 256, 0, s>>>((const float*)x, (float*)y, count, m); break;
        case P3D_F16: k_dropout<_Float16><<<blocks, 256, 0, s>>>((const _Float16*)x, (_Float16*)y, count, m); break;
        default: k_dropout<__bf16><<<blocks, 256, 0, s>>>((const __bf16*)x, (__bf16*)y, count, m); break;
    }
    return check_launch("p3d_dropout_apply");
}
