// What surrounds a block (block_kernels.hpp) as its kernels see it.
#pragma once

#include "philox.hpp"

namespace p3d {

struct NormDev {
    const void* weight;
    const void* bias;
    int kind;
    float eps;
};

struct BlockDev {
    int64_t tokens;
    int rows, samples, splits, dim;  // rows = samples * tokens < 2^31
    int param, gate_dtype, gate_kind;
    const void* x;
    const void* y;
    uint32_t x_stride, y_stride, gate_stride;  // bytes between rows (gate: rows or samples)
    const void* gate;
    const void* scale;
    float alpha;
    NormDev post, next;
    MaskDev mask;
    void* out;
    void* n;
    float* stats;  // [4][rows]: mean and rstd of y, of out; NULL without a backward
    // backward
    const void* dout;
    const void* dn;
    uint32_t dout_stride, dn_stride;
    void* dx;
    void* dy;
    void* dgate;        // per token or per element, in gate_dtype
    float* dgate_part;  // [splits][samples][dim], per sample
    float* part;        // [grid][5][dim]: post weight, post bias, scale, next weight, next bias
};

struct BlockLaunch {
    bool backward;
    unsigned grid;
    hipStream_t stream;
    int32_t* resident;  // not NULL: no launch, the workgroups of the kernel that run at a time
};

// Workgroups of a kernel that the current device runs at a time.
int resident_workgroups(const void* kernel, int threads, int32_t* count);

// Launches the kernels of one pair of types (block_<outer>_<inner>.hip).
template <typename TX, typename TY>
int launch_block(const BlockDev& a, const BlockLaunch& l);

}  // namespace p3d
