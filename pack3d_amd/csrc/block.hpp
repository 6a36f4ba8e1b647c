// What the forward and the backward kernel of a block's end share: the arguments
// as the device sees them, and how rows are dealt out.
//
// Per row of dim channels, all in fp32, each output rounded once:
//   b = norm1(y) w1 + b1 (or y),  z = keep ? b / (1 - p) : 0,
//   out = alpha x + scale gate z,  n = norm2(out) w2 + b2,
// with norm(v) = (v - mean) rstd (LayerNorm, biased variance from the centred
// values) or v rstd (RMSNorm).  Without y, out is x: the norm before a block.
//
// TPR threads share a row and hold eight consecutive channels each; rows of up to
// 512 channels lie within a wave (several to a wave below), wider ones take a
// workgroup, so every row is read once into registers whatever its width.
//
// Rows are dealt out in units: `tokens` rows that share a gate vector (a sample),
// cut into `splits` ranges.  A workgroup takes units blockIdx.x, + gridDim.x, ...,
// so the gate and the parameters stay in registers over a unit's rows.
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
    int64_t rows, tokens;  // rows = samples * tokens
    int samples, splits, dim;
    int param, gate_dtype, gate_kind;
    const void* x;
    const void* y;
    int64_t x_stride, y_stride;
    const void* gate;
    int64_t gate_stride;  // elements between rows (full, token) or samples (sample)
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
    int64_t dout_stride, dn_stride;
    void* dx;
    void* dy;
    void* dgate;       // per token or per element, in gate_dtype
    float* dgate_part;  // [splits][samples][dim], per sample
    float* part;       // [grid][5][dim]: post weight, post bias, scale, next weight, next bias
};

// The rows of unit u: `count` rows from `first` on.
struct Unit {
    int sample;
    int64_t first;
    int64_t count;
};
__device__ __forceinline__ Unit unit_of(const BlockDev& a, int u) {
    const int split = u / a.samples, sample = u - split * a.samples;
    const int64_t per = (a.tokens + a.splits - 1) / a.splits;
    const int64_t at = min(split * per, a.tokens), end = min(at + per, a.tokens);
    return Unit{sample, sample * a.tokens + at, end - at};
}

// Threads of a row for a width, and of its workgroup.
inline int threads_per_row(int dim) {
    const int pieces = (dim + kPiece - 1) / kPiece;
    int t = 8;
    while (t < pieces) t *= 2;
    return t;
}
constexpr int block_threads(int tpr) { return tpr <= 64 ? 256 : tpr; }

// Eight values of a parameter, or `missing` where it has none.
__device__ __forceinline__ void load_param(const void* p, int dtype, int c, int count, float missing,
                                           float (&v)[kPiece]) {
    if (p) load8_any(p, c, dtype, count, v);
    else
#pragma unroll
        for (int e = 0; e < kPiece; ++e) v[e] = missing;
}

int block_dev(const p3d_block_args* args, BlockDev& a);

}  // namespace p3d
