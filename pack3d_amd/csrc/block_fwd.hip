// The end of a block (and the norm before one) in one pass over its rows; block.hpp
// has the mathematics and the split.
//
// Bound by memory: x and y read, out and n written once, 8 bytes an element in 16
// bits.
#include "block.hpp"

namespace p3d {
namespace {

template <typename TX, typename TY, int TPR>
__global__ __launch_bounds__(block_threads(TPR)) void k_block_fwd(BlockDev a) {
    constexpr int GROUPS = TPR > 64 ? 1 : 256 / TPR;
    __shared__ float lds[TPR > 64 ? 2 * RowSum<TPR>::WAVES * 4 : 1];
    RowSum<TPR> row_sum{lds};
    const int sub = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int c = sub * kPiece, cnt = min(kPiece, a.dim - c);  // <= 0 for lanes past the row
    const float inv_dim = 1.f / (float)a.dim;
    MaskDev mask = a.mask;
    mask_begin(mask);
    float w1[kPiece], b1[kPiece], w2[kPiece], b2[kPiece], sc[kPiece], gs[kPiece];
    load_param(a.post.weight, a.param, c, cnt, 1.f, w1);
    load_param(a.post.bias, a.param, c, cnt, 0.f, b1);
    load_param(a.next.weight, a.param, c, cnt, 1.f, w2);
    load_param(a.next.bias, a.param, c, cnt, 0.f, b2);
    load_param(a.scale, a.param, c, cnt, 1.f, sc);
    const int units = a.samples * a.splits;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit unit = unit_of(a, u);
        if (a.gate_kind == P3D_GATE_SAMPLE)
            load8_any(a.gate, unit.sample * a.gate_stride + c, a.gate_dtype, cnt, gs);
#pragma unroll
        for (int e = 0; e < kPiece; ++e) gs[e] = a.gate_kind == P3D_GATE_SAMPLE ? gs[e] * sc[e] : sc[e];
        // Every thread of a workgroup that shares a row makes the same steps; groups
        // of a wave that have no row left read the unit's last one and write nothing.
        for (int64_t i = grp; i - grp < unit.count; i += GROUPS) {
            const bool live = i < unit.count;
            const int64_t row = unit.first + (live ? i : unit.count - 1);
            float v[kPiece], z[kPiece], g[kPiece];
            load8(reinterpret_cast<const TX*>(a.x) + row * a.x_stride + c, cnt, v);
            if (a.y) {
                load8(reinterpret_cast<const TY*>(a.y) + row * a.y_stride + c, cnt, z);
                if (a.gate_kind == P3D_GATE_FULL)
                    load8_any(a.gate, row * a.gate_stride + c, a.gate_dtype, cnt, g);
                float tok = 1.f;
                if (a.gate_kind == P3D_GATE_TOKEN) tok = load_any(a.gate, row * a.gate_stride, a.gate_dtype);
                if (a.post.kind) {
                    float mean = 0.f;
                    if (a.post.kind == P3D_NORM_LAYER) {
                        float s[1] = {0.f};
#pragma unroll
                        for (int e = 0; e < kPiece; ++e) s[0] += z[e];
                        row_sum.sum(s);
                        mean = s[0] * inv_dim;
                    }
                    float q[1] = {0.f};
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) {
                        z[e] = e < cnt ? z[e] - mean : 0.f;
                        q[0] += z[e] * z[e];
                    }
                    row_sum.sum(q);
                    const float rstd = 1.f / sqrtf(q[0] * inv_dim + a.post.eps);
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) z[e] = z[e] * rstd * w1[e] + b1[e];
                    if (a.stats && sub == 0 && live) {
                        a.stats[row] = mean;
                        a.stats[a.rows + row] = rstd;
                    }
                }
                if (mask.threshold) {
                    const uint32_t keep = keep8(mask, (uint64_t)row * a.dim + c);
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) z[e] = keep >> e & 1 ? z[e] * mask.inv : 0.f;
                }
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    const float k = a.gate_kind == P3D_GATE_FULL ? g[e] * gs[e] : tok * gs[e];
                    v[e] = e < cnt ? a.alpha * v[e] + k * z[e] : 0.f;
                }
                if (live) store8(reinterpret_cast<TX*>(a.out) + row * a.dim + c, cnt, v);
            }
            if (a.next.kind) {
                float mean = 0.f;
                if (a.next.kind == P3D_NORM_LAYER) {
                    float s[1] = {0.f};
#pragma unroll
                    for (int e = 0; e < kPiece; ++e) s[0] += v[e];
                    row_sum.sum(s);
                    mean = s[0] * inv_dim;
                }
                float q[1] = {0.f};
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    v[e] = e < cnt ? v[e] - mean : 0.f;
                    q[0] += v[e] * v[e];
                }
                row_sum.sum(q);
                const float rstd = 1.f / sqrtf(q[0] * inv_dim + a.next.eps);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) v[e] = v[e] * rstd * w2[e] + b2[e];
                if (live) store8(reinterpret_cast<TY*>(a.n) + row * a.dim + c, cnt, v);
                if (a.stats && sub == 0 && live) {
                    a.stats[2 * a.rows + row] = mean;
                    a.stats[3 * a.rows + row] = rstd;
                }
            }
        }
    }
}

bool known(int dtype) { return dtype >= P3D_F32 && dtype <= P3D_BF16; }

template <typename TX, typename TY>
int launch_fwd(const BlockDev& a, unsigned grid, hipStream_t s) {
    switch (threads_per_row(a.dim)) {
#define CASE(T) \
    case T: k_block_fwd<TX, TY, T><<<grid, block_threads(T), 0, s>>>(a); break;
        CASE(8) CASE(16) CASE(32) CASE(64) CASE(128) CASE(256) CASE(512) CASE(1024)
#undef CASE
        default: return fail(P3D_EUNSUPPORTED, "dim too large for the block kernels");
    }
    return check_launch("p3d_block_fwd");
}

}  // namespace

// Checks what both directions need and fills in the device's view of it.
int block_dev(const p3d_block_args* args, BlockDev& a) {
    P3D_REQUIRE(args, "null args");
    const p3d_block_args& g = *args;
    P3D_REQUIRE(g.samples >= 1 && g.tokens >= 1 && g.tokens < (1LL << 31) && g.samples * g.tokens < (1LL << 31),
                "row count out of range");
    P3D_REQUIRE(g.dim >= 1 && g.dim <= 8192, "dim must be 1 to 8192");
    P3D_REQUIRE(g.splits >= 1 && g.splits <= g.tokens && (int64_t)g.splits * g.samples < (1LL << 31),
                "splits out of range");
    P3D_REQUIRE(g.grid >= 1 && g.grid <= (int64_t)g.splits * g.samples, "grid out of range");
    P3D_REQUIRE(known(g.outer) && known(g.inner) && known(g.param) && known(g.gate_dtype), "unknown dtype");
    P3D_REQUIRE(g.outer == P3D_F32 || g.outer == g.inner, "a 16-bit stream takes blocks of its own type");
    P3D_REQUIRE(g.x, "null pointer argument");
    P3D_REQUIRE(g.post.kind >= 0 && g.post.kind <= P3D_NORM_RMS && g.next.kind >= 0 && g.next.kind <= P3D_NORM_RMS,
                "unknown norm kind");
    P3D_REQUIRE(g.gate_kind >= 0 && g.gate_kind <= P3D_GATE_FULL, "unknown gate kind");
    P3D_REQUIRE((g.gate_kind != 0) == (g.gate != nullptr), "gate and its kind disagree");
    P3D_REQUIRE(g.y || (!g.post.kind && !g.gate_kind && !g.scale && !g.dropout.threshold && g.alpha == 1.f),
                "without y there is only the next norm");
    P3D_REQUIRE(g.y || g.next.kind, "nothing to compute");
    P3D_REQUIRE(mask_ok(g.dropout), "threshold must be in [0, 65535]");
    a = BlockDev{};
    a.rows = (int64_t)g.samples * g.tokens;
    a.tokens = g.tokens;
    a.samples = g.samples;
    a.splits = g.splits;
    a.dim = g.dim;
    a.param = g.param;
    a.gate_dtype = g.gate_dtype;
    a.gate_kind = g.gate_kind;
    a.x = g.x;
    a.y = g.y;
    a.x_stride = g.x_stride;
    a.y_stride = g.y_stride;
    a.gate = g.gate;
    a.gate_stride = g.gate_stride;
    a.scale = g.scale;
    a.alpha = g.alpha;
    a.post = NormDev{g.post.weight, g.post.bias, g.post.kind, g.post.eps};
    a.next = NormDev{g.next.weight, g.next.bias, g.next.kind, g.next.eps};
    a.mask = mask_dev(g.dropout);
    a.out = g.out;
    a.n = g.n;
    a.stats = g.stats;
    a.dout = g.dout;
    a.dn = g.dn;
    a.dout_stride = g.dout_stride;
    a.dn_stride = g.dn_stride;
    a.dx = g.dx;
    a.dy = g.dy;
    a.dgate = g.dgate;
    a.dgate_part = g.dgate_part;
    a.part = g.part;
    return P3D_OK;
}

}  // namespace p3d

using namespace p3d;

extern "C" int p3d_block_fwd(const p3d_block_args* args, void* stream) {
    BlockDev a;
    if (const int rc = block_dev(args, a)) return rc;
    P3D_REQUIRE((!a.y || a.out) && (!a.next.kind || a.n), "null output");
    hipStream_t s = as_stream(stream);
    const unsigned grid = (unsigned)args->grid;
    if (args->outer == P3D_F16) return launch_fwd<_Float16, _Float16>(a, grid, s);
    if (args->outer == P3D_BF16) return launch_fwd<__bf16, __bf16>(a, grid, s);
    if (args->inner == P3D_F16) return launch_fwd<float, _Float16>(a, grid, s);
    if (args->inner == P3D_BF16) return launch_fwd<float, __bf16>(a, grid, s);
    return launch_fwd<float, float>(a, grid, s);
}
