// Dropout of a contiguous tensor: y = x / (1 - p) where the mask of philox.hpp
// keeps the element, else 0 (a select: what is dropped may be infinite or NaN).
// The backward is the same pass over the output's gradient.  Bound by memory: 4
// bytes an element in 16 bits, next to about 17 VALU issues for its share of the
// generator.
#include "philox.hpp"

namespace p3d {
namespace {

template <typename T>
__global__ __launch_bounds__(256) void k_dropout(const T* x, T* y, int64_t count, MaskDev m) {
    mask_begin(m);
    const int64_t group = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t first = group * kPiece;
    if (first >= count) return;
    const int n = (int)min((int64_t)kPiece, count - first);
    float v[kPiece];
    load8(x + first, n, v);
    const uint32_t keep = keep_group(m, (uint64_t)group);
#pragma unroll
    for (int e = 0; e < kPiece; ++e) v[e] = keep >> e & 1 ? v[e] * m.inv : 0.f;
    store8(y + first, n, v);
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_dropout_apply(const void* x, void* y, int64_t count, int32_t dtype, const p3d_dropout* dropout,
                                 void* stream) {
    P3D_REQUIRE(x && y && dropout, "null pointer argument");
    P3D_REQUIRE(dtype >= P3D_F32 && dtype <= P3D_BF16, "unknown dtype");
    P3D_REQUIRE(count >= 1 && cdiv(count, 256 * kPiece) < (1LL << 31), "element count out of range");
    P3D_REQUIRE(mask_ok(*dropout), "threshold must be in [0, 65535]");
    const MaskDev m = mask_dev(*dropout);
    const unsigned blocks = (unsigned)cdiv(count, 256 * kPiece);
    hipStream_t s = as_stream(stream);
    switch (dtype) {
        case P3D_F32: k_dropout<float><<<blocks, 256, 0, s>>>((const float*)x, (float*)y, count, m); break;
        case P3D_F16: k_dropout<_Float16><<<blocks, 256, 0, s>>>((const _Float16*)x, (_Float16*)y, count, m); break;
        default: k_dropout<__bf16><<<blocks, 256, 0, s>>>((const __bf16*)x, (__bf16*)y, count, m); break;
    }
    return check_launch("p3d_dropout_apply");
}
