// The entry points of what surrounds a block: checks, and the launch for the types.
#include "block.hpp"

namespace p3d {

extern template int launch_block<float, float>(const BlockDev&, const BlockLaunch&);
extern template int launch_block<_Float16, _Float16>(const BlockDev&, const BlockLaunch&);
extern template int launch_block<__bf16, __bf16>(const BlockDev&, const BlockLaunch&);
extern template int launch_block<float, _Float16>(const BlockDev&, const BlockLaunch&);
extern template int launch_block<float, __bf16>(const BlockDev&, const BlockLaunch&);

namespace {

bool known(int dtype) { return dtype >= P3D_F32 && dtype <= P3D_BF16; }

// Bytes between rows of a stride in elements; kernels multiply rows by them in 32 bits.
bool stride_ok(int64_t stride) { return stride >= 0 && stride < (1LL << 29); }

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
    P3D_REQUIRE(stride_ok(g.x_stride) && stride_ok(g.y_stride) && stride_ok(g.gate_stride) && stride_ok(g.dout_stride) &&
                    stride_ok(g.dn_stride),
                "row strides must be in [0, 2^29)");
    P3D_REQUIRE(mask_ok(g.dropout), "threshold must be in [0, 65535]");
    const uint32_t outer = dtype_size(g.outer), inner = dtype_size(g.inner);
    a = BlockDev{};
    a.rows = (int)(g.samples * g.tokens);
    a.tokens = g.tokens;
    a.samples = g.samples;
    a.splits = g.splits;
    a.dim = g.dim;
    a.param = g.param;
    a.gate_dtype = g.gate_dtype;
    a.gate_kind = g.gate_kind;
    a.x = g.x;
    a.y = g.y;
    a.x_stride = (uint32_t)g.x_stride * outer;
    a.y_stride = (uint32_t)g.y_stride * inner;
    a.gate = g.gate;
    a.gate_stride = (uint32_t)g.gate_stride * dtype_size(g.gate_dtype);
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
    a.dout_stride = (uint32_t)g.dout_stride * outer;
    a.dn_stride = (uint32_t)g.dn_stride * inner;
    a.dx = g.dx;
    a.dy = g.dy;
    a.dgate = g.dgate;
    return P3D_OK;
}

int launch(const p3d_block_args& g, const BlockDev& a, const BlockLaunch& l) {
    if (g.outer == P3D_F16) return launch_block<_Float16, _Float16>(a, l);
    if (g.outer == P3D_BF16) return launch_block<__bf16, __bf16>(a, l);
    if (g.inner == P3D_F16) return launch_block<float, _Float16>(a, l);
    if (g.inner == P3D_BF16) return launch_block<float, __bf16>(a, l);
    return launch_block<float, float>(a, l);
}

}  // namespace

int resident_workgroups(const void* kernel, int threads, int32_t* count) {
    int dev = 0, cus = 0, per_cu = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess) e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev);
    if (e == hipSuccess) e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, threads, 0);
    if (e != hipSuccess) return fail(P3D_EHIP, std::string("p3d_block_resident: ") + hipGetErrorString(e));
    *count = (cus > 0 ? cus : 1) * (per_cu > 0 ? per_cu : 1);
    return P3D_OK;
}

}  // namespace p3d

using namespace p3d;

extern "C" int p3d_block_resident(const p3d_block_args* args, int32_t backward, int32_t* count) {
    BlockDev a;
    if (const int rc = block_dev(args, a)) return rc;
    P3D_REQUIRE(count, "null pointer argument");
    return launch(*args, a, BlockLaunch{backward != 0, 0, nullptr, count});
}

extern "C" int p3d_block_fwd(const p3d_block_args* args, void* stream) {
    BlockDev a;
    if (const int rc = block_dev(args, a)) return rc;
    P3D_REQUIRE((!a.y || a.out) && (!a.next.kind || a.n), "null output");
    return launch(*args, a, BlockLaunch{false, (unsigned)args->grid, as_stream(stream), nullptr});
}

extern "C" int p3d_block_bwd(const p3d_block_args* args, void* stream) {
    BlockDev a;
    if (const int rc = block_dev(args, a)) return rc;
    P3D_REQUIRE(a.y ? a.dout != nullptr : a.dn != nullptr, "the upstream gradient is missing");
    P3D_REQUIRE(!a.dn || a.next.kind, "a gradient of n needs the next norm");
    P3D_REQUIRE((!a.post.kind && !a.dn) || a.stats, "the norms' statistics are missing");
    const p3d_block_args& g = *args;
    const bool gated = a.gate_kind == P3D_GATE_TOKEN || a.gate_kind == P3D_GATE_FULL;
    P3D_REQUIRE((!a.y || a.dy) && (!a.dn || a.dx) && (!gated || a.dgate), "null output");
    P3D_REQUIRE(a.gate_kind || !a.dgate, "dgate without a gate");
    // Where the sums over rows go: a row of the five parameters' a workgroup, a row of
    // the gate's a unit.
    p3d_sum_job jobs[6];
    int count = 0;
    const void* params[5] = {a.post.weight, a.post.bias, a.scale, a.next.weight, a.next.bias};
    float* part = g.work;
    for (int i = 0; i < 5; ++i) {
        if (!g.d_param[i]) continue;
        P3D_REQUIRE(params[i] && known(g.d_param_dtype[i]) && (i < 3 || a.dn), "d_param without its parameter or gradient");
        jobs[count++] = p3d_sum_job{part + (int64_t)i * a.dim, g.d_param[i], g.grid, 5 * (int64_t)a.dim, a.dim,
                                    g.d_param_dtype[i]};
    }
    if (count) a.part = part;
    if (a.gate_kind == P3D_GATE_SAMPLE && a.dgate) {
        P3D_REQUIRE((int64_t)a.samples * a.dim < (1LL << 31), "samples * dim out of range");
        a.dgate_part = part + (count ? (int64_t)g.grid * 5 * a.dim : 0);
        const int64_t cols = (int64_t)a.samples * a.dim;
        jobs[count++] = p3d_sum_job{a.dgate_part, a.dgate, a.splits, cols, (int32_t)cols, a.gate_dtype};
    }
    P3D_REQUIRE(!count || g.work, "work is missing");
    if (const int rc = launch(g, a, BlockLaunch{true, (unsigned)g.grid, as_stream(stream), nullptr})) return rc;
    return count ? p3d_sum_rows(jobs, count, stream) : P3D_OK;
}
