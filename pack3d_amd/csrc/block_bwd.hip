// The gradients of a block's end in one pass over its rows; block.hpp has the
// forward's mathematics and the split.  With go the gradient of out,
//   go = dout + rstd2 (g2 - [layer] mean(g2) - xh2 mean(g2 xh2)),  g2 = dn w2,
//   dx = alpha go,  dscale = sum gate z go,  dgate = sum scale z go,
//   db = keep scale gate go / (1 - p),  g1 = db w1,
//   dy = rstd1 (g1 - [layer] mean(g1) - xh1 mean(g1 xh1)),
// and the weights' and biases' gradients sum xh and 1 times dn (next) and db
// (post) over the rows.  out is formed again from x and y (the same bytes as
// reading it, and not rounded), the statistics come from the forward.
//
// Sums over rows are held in registers over all rows of a workgroup, then added
// over its row groups in LDS in a fixed order; a workgroup writes one row of
// partials, which p3d_sum_rows adds.  No atomics.
//
// Bound by memory: dout, dn, x and y read, dx and dy written once.
#include "block.hpp"

namespace p3d {
namespace {

template <typename TX, typename TY, int TPR>
__global__ __launch_bounds__(block_threads(TPR)) void k_block_bwd(BlockDev a) {
    constexpr int GROUPS = TPR > 64 ? 1 : 256 / TPR;
    __shared__ float lds[TPR > 64 ? 2 * RowSum<TPR>::WAVES * 4 : 256 * kPiece];
    RowSum<TPR> row_sum{lds};
    const int sub = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int c = sub * kPiece, cnt = min(kPiece, a.dim - c);
    const float inv_dim = 1.f / (float)a.dim;
    const bool layer1 = a.post.kind == P3D_NORM_LAYER, layer2 = a.next.kind == P3D_NORM_LAYER;
    MaskDev mask = a.mask;
    mask_begin(mask);
    float w1[kPiece], b1[kPiece], w2[kPiece], sc[kPiece];
    load_param(a.post.weight, a.param, c, cnt, 1.f, w1);
    load_param(a.post.bias, a.param, c, cnt, 0.f, b1);
    load_param(a.next.weight, a.param, c, cnt, 1.f, w2);
    load_param(a.scale, a.param, c, cnt, 1.f, sc);
    // Sums over this thread's rows: dw1, db1, dscale, dw2, db2.
    float acc[5][kPiece], unit_acc[kPiece];
#pragma unroll
    for (int k = 0; k < 5; ++k)
#pragma unroll
        for (int e = 0; e < kPiece; ++e) acc[k][e] = 0.f;
    const bool per_sample = a.gate_kind == P3D_GATE_SAMPLE;

    // Sum over the workgroup's row groups, in order; group 0 ends with it.
    auto over_groups = [&](float(&v)[kPiece]) {
        if constexpr (GROUPS > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kPiece; ++e) lds[e * 256 + threadIdx.x] = v[e];
            __syncthreads();
            if (grp == 0) {
#pragma unroll
                for (int e = 0; e < kPiece; ++e)
                    for (int k = 1; k < GROUPS; ++k) v[e] += lds[e * 256 + k * TPR + sub];
            }
        }
    };

    const int units = a.samples * a.splits;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit unit = unit_of(a, u);
        float gs[kPiece];
        if (per_sample) load8_any(a.gate, unit.sample * a.gate_stride + c, a.gate_dtype, cnt, gs);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) {
            gs[e] = per_sample ? gs[e] : 1.f;
            unit_acc[e] = 0.f;
        }
        for (int64_t i = grp; i - grp < unit.count; i += GROUPS) {
            const bool live = i < unit.count;
            const int64_t row = unit.first + (live ? i : unit.count - 1);
            const int n = live ? cnt : 0;  // rows that are not there read as zeros
            float go[kPiece], z[kPiece], xh1[kPiece], k1[kPiece], g[kPiece];
            uint32_t keep = 0xff;
            if (a.dout) load8(reinterpret_cast<const TX*>(a.dout) + row * a.dout_stride + c, n, go);
            else
#pragma unroll
                for (int e = 0; e < kPiece; ++e) go[e] = 0.f;
            float tok = 1.f;
            if (a.y) {
                load8(reinterpret_cast<const TY*>(a.y) + row * a.y_stride + c, n, xh1);
                if (a.gate_kind == P3D_GATE_FULL) load8_any(a.gate, row * a.gate_stride + c, a.gate_dtype, n, g);
                if (a.gate_kind == P3D_GATE_TOKEN) tok = load_any(a.gate, row * a.gate_stride, a.gate_dtype);
                float mean = 0.f, rstd = 1.f;
                if (a.post.kind) {
                    mean = a.stats[row];
                    rstd = a.stats[a.rows + row];
                }
                if (mask.threshold) keep = keep8(mask, (uint64_t)row * a.dim + c);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    xh1[e] = e < n ? (xh1[e] - mean) * rstd : 0.f;
                    const float b = a.post.kind ? xh1[e] * w1[e] + b1[e] : xh1[e];
                    z[e] = keep >> e & 1 ? b * mask.inv : 0.f;
                    g[e] = a.gate_kind == P3D_GATE_FULL ? g[e] : tok * gs[e];
                    k1[e] = g[e] * sc[e];
                }
            }
            if (a.dn) {
                float xh2[kPiece], g2[kPiece], s[2] = {0.f, 0.f};
                load8(reinterpret_cast<const TX*>(a.x) + row * a.x_stride + c, n, xh2);
                load8(reinterpret_cast<const TY*>(a.dn) + row * a.dn_stride + c, n, g2);
                const float mean = a.stats[2 * a.rows + row], rstd = a.stats[3 * a.rows + row];
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    const float out = a.y ? a.alpha * xh2[e] + k1[e] * z[e] : xh2[e];
                    xh2[e] = e < n ? (out - mean) * rstd : 0.f;
                    acc[3][e] += g2[e] * xh2[e];
                    acc[4][e] += g2[e];
                    g2[e] *= w2[e];
                    s[0] += g2[e];
                    s[1] += g2[e] * xh2[e];
                }
                row_sum.sum(s);
                const float m0 = layer2 ? s[0] * inv_dim : 0.f, m1 = s[1] * inv_dim;
#pragma unroll
                for (int e = 0; e < kPiece; ++e) go[e] += rstd * (g2[e] - m0 - xh2[e] * m1);
            }
            if (a.dx && live) {
                float v[kPiece];
#pragma unroll
                for (int e = 0; e < kPiece; ++e) v[e] = a.alpha * go[e];
                store8(reinterpret_cast<TX*>(a.dx) + row * a.dim + c, cnt, v);
            }
            if (!a.y) continue;
            float s[3] = {0.f, 0.f, 0.f}, db[kPiece], dg[kPiece];
#pragma unroll
            for (int e = 0; e < kPiece; ++e) {
                const float zg = z[e] * go[e];
                dg[e] = e < n ? sc[e] * zg : 0.f;
                s[2] += dg[e];
                if (per_sample) unit_acc[e] += zg;
                else acc[2][e] += g[e] * zg;
                db[e] = keep >> e & 1 ? mask.inv * k1[e] * go[e] : 0.f;
                if (a.post.kind) {
                    db[e] = e < n ? db[e] : 0.f;
                    acc[0][e] += db[e] * xh1[e];
                    acc[1][e] += db[e];
                    db[e] *= w1[e];
                    s[0] += db[e];
                    s[1] += db[e] * xh1[e];
                }
            }
            if (a.post.kind || (a.gate_kind == P3D_GATE_TOKEN && a.dgate)) row_sum.sum(s);
            if (a.post.kind) {
                const float rstd = a.stats[a.rows + row];
                const float m0 = layer1 ? s[0] * inv_dim : 0.f, m1 = s[1] * inv_dim;
#pragma unroll
                for (int e = 0; e < kPiece; ++e) db[e] = rstd * (db[e] - m0 - xh1[e] * m1);
            }
            if (live) {
                if (a.dy) store8(reinterpret_cast<TY*>(a.dy) + row * a.dim + c, cnt, db);
                if (a.dgate && a.gate_kind == P3D_GATE_FULL)
                    store8_any(a.dgate, row * a.dim + c, a.gate_dtype, cnt, dg);
                if (a.dgate && a.gate_kind == P3D_GATE_TOKEN && sub == 0)
                    store_any(a.dgate, row, a.gate_dtype, s[2]);
            }
        }
        if (per_sample) {
            // z go summed over the unit's rows gives the gate's gradient times scale
            // and the scale's times the gate.
#pragma unroll
            for (int e = 0; e < kPiece; ++e) acc[2][e] += gs[e] * unit_acc[e];
            if (a.dgate_part) {
                over_groups(unit_acc);
                if (grp == 0) {
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) unit_acc[e] *= sc[e];
                    store8(a.dgate_part + (int64_t)u * a.dim + c, cnt, unit_acc);
                }
            }
        }
    }
    if (!a.part) return;
    const bool want[5] = {a.post.weight != nullptr, a.post.bias != nullptr, a.scale != nullptr,
                          a.next.weight != nullptr && a.dn, a.next.bias != nullptr && a.dn};
#pragma unroll
    for (int k = 0; k < 5; ++k) {
        if (!want[k]) continue;
        over_groups(acc[k]);
        if (grp == 0) store8(a.part + ((int64_t)blockIdx.x * 5 + k) * a.dim + c, cnt, acc[k]);
    }
}

template <typename TX, typename TY>
int launch_bwd(const BlockDev& a, unsigned grid, hipStream_t s) {
    switch (threads_per_row(a.dim)) {
#define CASE(T) \
    case T: k_block_bwd<TX, TY, T><<<grid, block_threads(T), 0, s>>>(a); break;
        CASE(8) CASE(16) CASE(32) CASE(64) CASE(128) CASE(256) CASE(512) CASE(1024)
#undef CASE
        default: return fail(P3D_EUNSUPPORTED, "dim too large for the block kernels");
    }
    return check_launch("p3d_block_bwd");
}

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_block_bwd(const p3d_block_args* args, void* stream) {
    BlockDev a;
    if (const int rc = block_dev(args, a)) return rc;
    P3D_REQUIRE(a.dout || a.dn, "no upstream gradient");
    P3D_REQUIRE(!a.dn || a.next.kind, "a gradient of n needs the next norm");
    P3D_REQUIRE((!a.post.kind && !a.dn) || a.stats, "the norms' statistics are missing");
    P3D_REQUIRE(!a.dgate || a.gate_kind == P3D_GATE_TOKEN || a.gate_kind == P3D_GATE_FULL, "dgate is per token or element");
    P3D_REQUIRE(!a.dgate_part || a.gate_kind == P3D_GATE_SAMPLE, "dgate_part is per sample");
    P3D_REQUIRE(a.y || !a.dy, "dy without y");
    hipStream_t s = as_stream(stream);
    const unsigned grid = (unsigned)args->grid;
    if (args->outer == P3D_F16) return launch_bwd<_Float16, _Float16>(a, grid, s);
    if (args->outer == P3D_BF16) return launch_bwd<__bf16, __bf16>(a, grid, s);
    if (args->inner == P3D_F16) return launch_bwd<float, _Float16>(a, grid, s);
    if (args->inner == P3D_BF16) return launch_bwd<float, __bf16>(a, grid, s);
    return launch_bwd<float, float>(a, grid, s);
}
