// The host side of the operators around a block (block.py, dropout.py, rotary.py), built
// as pack3d_amd/_torch_ops.so: checks, outputs and workspaces from torch's allocator, one
// call of the C ABI on the device's current stream, and the autograd nodes.
//
// These operators take 3 to 100 us on the GPU, and a model calls them several times a
// layer, so their host time counts.  In Python a training step of block_residual took
// 110 to 210 us of it (two thirds in the interpreter, part of that on the autograd
// engine's thread, which has to take the interpreter's lock), a single-token call 17.
//
// The entry points' addresses come from the loaded library (bind_library), so that this
// module takes the build that _lib loaded.
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <array>
#include <cmath>
#include <mutex>
#include <optional>
#include <unordered_map>

#include "../../include/pack3d_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

// --------------------------------------------------------- the C ABI
struct Library {
    decltype(&p3d_block_fwd) block_fwd = nullptr;
    decltype(&p3d_block_bwd) block_bwd = nullptr;
    decltype(&p3d_block_resident) block_resident = nullptr;
    decltype(&p3d_dropout_apply) dropout_apply = nullptr;
    decltype(&p3d_rotary) rotary = nullptr;
    decltype(&p3d_last_error) last_error = nullptr;
} lib;

void bind_library(int64_t block_fwd, int64_t block_bwd, int64_t block_resident, int64_t dropout_apply, int64_t rotary,
                  int64_t last_error) {
    lib.block_fwd = reinterpret_cast<decltype(lib.block_fwd)>(block_fwd);
    lib.block_bwd = reinterpret_cast<decltype(lib.block_bwd)>(block_bwd);
    lib.block_resident = reinterpret_cast<decltype(lib.block_resident)>(block_resident);
    lib.dropout_apply = reinterpret_cast<decltype(lib.dropout_apply)>(dropout_apply);
    lib.rotary = reinterpret_cast<decltype(lib.rotary)>(rotary);
    lib.last_error = reinterpret_cast<decltype(lib.last_error)>(last_error);
}

// Calls entry(args..., stream) with the tensor's device current, on its current stream.
template <typename Entry, typename... Args>
void launch(const char* name, const Tensor& on, Entry entry, Args... args) {
    const c10::OptionalDeviceGuard guard(on.device());
    void* stream = c10::hip::getCurrentHIPStream(on.device().index()).stream();
    const int rc = entry(args..., stream);
    TORCH_CHECK(rc == 0, name, " failed (", rc, "): ", lib.last_error());
}

int dtype_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return P3D_F32;
        case at::kHalf: return P3D_F16;
        case at::kBFloat16: return P3D_BF16;
        default: return -1;
    }
}

void require_device(const Tensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.is_cuda(), "the hip backend requires ", what, " on a HIP device; no CPU fallback exists");
}

// Contiguous, of t's shape.
Tensor empty_as(const Tensor& t, at::ScalarType dtype) {
    return at::empty(t.sizes(), t.options().dtype(dtype).requires_grad(false));
}

// --------------------------------------------------- autograd, in common
// Gradients of first order: a graph through them would be silently constant in `inputs`
// (what they were computed from), so what create_graph makes raises when it is
// differentiated.
variable_list first_order(variable_list&& grads, bool create_graph, const variable_list& inputs, const char* name) {
    if (!create_graph) return std::move(grads);
    const c10::AutoGradMode on(true);
    if (!torch::autograd::any_variable_requires_grad(inputs)) return std::move(grads);
    auto error = std::shared_ptr<torch::autograd::Error>(
        new torch::autograd::Error(
            std::string("trying to differentiate twice ") + name + ", whose gradient is of first order",
            torch::autograd::collect_next_edges(inputs)),
        torch::autograd::deleteNode);
    for (Tensor& g : grads)
        if (g.defined()) {
            g = g.detach();
            torch::autograd::set_history(g, error);
        }
    return std::move(grads);
}

// A backward that is captured must not hand a gradient to a node of the default stream: a
// leaf keeps the stream of its first use for as long as a graph of that use is alive, and
// autograd would make the default stream wait on the capture, which ends the process.
void refuse_default_stream(const Node& node) {
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (size_t i = 0; i < node.num_outputs(); ++i) {
        if (!node.task_should_compute_output(i)) continue;
        const auto stream = node.next_edge(i).function->stream();
        TORCH_CHECK(!stream || *stream != c10::Stream(c10::Stream::DEFAULT, stream->device()),
                    "a backward pass is captured into a graph while an eager graph of the same tensors, made on the "
                    "default stream, is alive: drop its outputs first, or make it on another stream");
    }
}

void no_forward_mode(const MaybeTensor& t) {
    TORCH_CHECK(!torch::autograd::isFwGradDefined(t), "forward-mode differentiation is not implemented");
}

Tensor or_undefined(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

// ------------------------------------------------------------- the block
constexpr int64_t kMaxDim = 8192;
constexpr int64_t kMaxStride = 1LL << 29;  // elements between rows

int64_t row_threads(int64_t dim) {
    int64_t threads = dim < 4 ? 4 : 2;
    while (threads < 1024 && dim > threads * 8) threads *= 2;
    return threads;
}

// Ranges that a sample's rows are cut into, and workgroups.  round: the workgroups that
// the backward is to have; 0 for the forward.
std::pair<int64_t, int64_t> block_split(int64_t samples, int64_t tokens, int64_t dim, int64_t round) {
    const int64_t threads = row_threads(dim);
    const int64_t rows = threads <= 64 ? 256 / threads : 1;  // that a workgroup holds at a time
    const int64_t per_sample = (tokens + rows - 1) / rows, steps = per_sample * samples;
    int64_t wanted = round;
    if (!round && threads > 64) {
        // Rows of 2 and 4 waves: several rounds, as below; of 8 and 16, whose workgroups fill
        // a CU by two or one: one (fp32 over bf16, two norms, dropout, a gate per token: 1,000
        // channels 106 us in 2,048 workgroups, 89 in 4,096; 6,144 channels 105 in 512, 99 in 256).
        wanted = (threads <= 256 ? 1 << 19 : 1 << 18) / threads;
    } else if (!round) {
        // Several rounds, of at least four steps each once every CU has work: a workgroup
        // begins by loading the parameters (4,913 x 3 rows of 327: 21 us in 921, 25 in 3,685).
        wanted = std::max(std::min<int64_t>(1024, steps), std::min<int64_t>(4096, steps / 4));
    }
    const int64_t splits = std::max<int64_t>(1, std::min(wanted / samples, per_sample));
    return {splits, std::min(splits * samples, wanted)};
}

struct NormSpec {
    int kind = P3D_NORM_NONE;
    float eps = 0.f;
};

// What a call computes, apart from its tensors.
struct BlockSpec {
    NormSpec post, next;
    float alpha = 1.f;
    p3d_dropout mask{};
    int gate_kind = P3D_GATE_NONE;
    at::ScalarType inner = at::kFloat;
};

// The tensors of a call: x, y, gate, scale, post weight and bias, next weight and bias.
enum { kX, kY, kGate, kScale, kPostWeight, kPostBias, kNextWeight, kNextBias, kInputs };
typedef std::array<Tensor, kInputs> Inputs;

// t as rows of dim channels with unit channel stride (a copy, kept in `keep`, where it
// does not lie so): the address and the stride between rows.
std::pair<const void*, int64_t> rows_of(const Tensor& t, int64_t dim, variable_list& keep) {
    if (t.is_contiguous()) return {t.const_data_ptr(), dim};
    Tensor r = t.reshape({-1, dim});
    if ((dim > 1 && r.stride(1) != 1) || r.stride(0) >= kMaxStride) r = r.clone(at::MemoryFormat::Contiguous);
    keep.push_back(r);
    return {r.const_data_ptr(), r.stride(0)};
}

// The argument block of both directions, without outputs; `keep` holds what it points
// into besides the inputs.
p3d_block_args bind_block(const BlockSpec& spec, const Inputs& in, variable_list& keep) {
    p3d_block_args a{};
    const Tensor& x = in[kX];
    a.dim = (int32_t)x.size(-1);
    a.alpha = spec.alpha;
    a.dropout = spec.mask;
    a.outer = dtype_of(x.scalar_type());
    a.inner = dtype_of(spec.inner);
    std::tie(a.x, a.x_stride) = rows_of(x, a.dim, keep);
    if (in[kY].defined()) std::tie(a.y, a.y_stride) = rows_of(in[kY], a.dim, keep);
    a.samples = 1;  // runs of rows that share a gate vector; a gate of batch 1 is shared by all of them
    if (in[kGate].defined()) {
        const Tensor& gate = in[kGate];
        if (spec.gate_kind == P3D_GATE_SAMPLE && x.dim() == 3) a.samples = (int32_t)gate.size(0);
        std::tie(a.gate, a.gate_stride) = rows_of(gate, gate.size(-1), keep);
        a.gate_dtype = dtype_of(gate.scalar_type());
        a.gate_kind = spec.gate_kind;
    }
    a.tokens = a.samples ? x.numel() / a.dim / a.samples : 0;
    // One type for all parameters: their own, or fp32, which holds each of them exactly.
    at::ScalarType type = at::kFloat;
    bool any = false;
    for (int i = kScale; i < kInputs; ++i) {
        if (!in[i].defined()) continue;
        const at::ScalarType t = in[i].scalar_type();
        type = (!any || t == type) && dtype_of(t) >= 0 ? t : at::kFloat;
        if (any && t != type) {
            type = at::kFloat;
            break;
        }
        any = true;
    }
    a.param = dtype_of(type);
    const void* at[kInputs] = {};
    for (int i = kScale; i < kInputs; ++i) {
        if (!in[i].defined()) continue;
        if (in[i].scalar_type() == type && in[i].is_contiguous()) {
            at[i] = in[i].const_data_ptr();
        } else {
            keep.push_back(in[i].to(type).contiguous());
            at[i] = keep.back().const_data_ptr();
        }
    }
    a.scale = at[kScale];
    a.post = p3d_norm{at[kPostWeight], at[kPostBias], spec.post.kind, spec.post.eps};
    a.next = p3d_norm{at[kNextWeight], at[kNextBias], spec.next.kind, spec.next.eps};
    return a;
}

// Workgroups of the backward: one round, since each leaves a row of partial parameter
// gradients and a second round waits on a few.  A lone norm takes two waves a SIMD
// (32,000 rows of 1,000, forward and backward: 109 us; 111 with three, 128 with the four
// that run at a time).  An end takes what the GPU runs of its kernel at a time, three at
// most, asked once for each kind of call (gated, without a next norm, rows of 192 and
// 1,024: 114 and 106 us with three, 132 and 118 with two).
int64_t backward_round(const Tensor& x, const p3d_block_args& args) {
    static std::mutex mutex;
    static std::unordered_map<uint64_t, int32_t> known;
    const int64_t threads = row_threads(args.dim);
    const int64_t simd_waves = 64 * 1024 / (threads > 64 ? threads : 256);  // workgroups that are a wave on each
    if (!args.y) return std::max<int64_t>(256, 2 * simd_waves);
    const int gated = args.gate_kind == P3D_GATE_TOKEN || args.gate_kind == P3D_GATE_FULL;
    const uint64_t key = (((((uint64_t)x.device().index() << 16 | (uint64_t)args.dim) << 2 | (uint64_t)args.outer) << 2 |
                           (uint64_t)args.inner) << 1 | gated) << 1 | (args.dn ? 1 : 0);
    std::lock_guard<std::mutex> lock(mutex);
    int32_t& count = known[key];
    if (!count) {
        const c10::OptionalDeviceGuard guard(x.device());
        p3d_block_args a = args;
        a.splits = a.grid = 1;
        const int rc = lib.block_resident(&a, 1, &count);
        TORCH_CHECK(rc == 0, "p3d_block_resident failed (", rc, "): ", lib.last_error());
    }
    return std::min(std::max<int64_t>(256, 3 * simd_waves), (int64_t)count);
}

struct BlockOutputs {
    Tensor out, n, stats;
};

BlockOutputs block_forward(const BlockSpec& spec, const Inputs& in, bool save) {
    const c10::AutoGradMode off(false);
    variable_list keep;
    p3d_block_args a = bind_block(spec, in, keep);
    const Tensor& x = in[kX];
    const int64_t rows = a.samples * a.tokens;
    BlockOutputs o;
    if (in[kY].defined()) o.out = empty_as(x, x.scalar_type());
    if (spec.next.kind) o.n = empty_as(x, spec.inner);
    if (save) o.stats = at::empty({4, rows}, x.options().dtype(at::kFloat).requires_grad(false));
    if (rows) {
        a.out = o.out.defined() ? o.out.data_ptr() : nullptr;
        a.n = o.n.defined() ? o.n.data_ptr() : nullptr;
        a.stats = save ? static_cast<float*>(o.stats.data_ptr()) : nullptr;
        const auto [splits, grid] = block_split(a.samples, a.tokens, a.dim, 0);
        a.splits = (int32_t)splits;
        a.grid = (int32_t)grid;
        launch("p3d_block_fwd", x, lib.block_fwd, &a);
    }
    return o;
}

// The forward saves its inputs and the rows' statistics; the backward forms out again
// from x and y.
struct BlockBackward : public Node {
    BlockSpec spec;
    std::array<SavedVariable, kInputs> saved;
    SavedVariable state;  // the dropout's seed, so that a change of it is noticed
    Tensor stats;

    std::string name() const override { return "Pack3DBlockBackward"; }

    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        for (auto& s : saved) s.reset_data();
        state.reset_data();
        stats.reset();
    }

    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        refuse_default_stream(*this);
        const bool create_graph = c10::GradMode::is_enabled();
        const c10::AutoGradMode off(false);
        auto self = shared_from_this();
        Inputs in;
        for (int i = 0; i < kInputs; ++i) in[i] = saved[i].unpack(self);
        const Tensor seed = state.unpack(self);
        const Tensor &x = in[kX], &y = in[kY], &gate = in[kGate];
        Tensor dout, dn;
        if (!y.defined()) dn = grads[0];
        else dout = grads[0];
        if (y.defined() && grads.size() == 2) dn = grads[1];
        variable_list result(kInputs);
        if (!dout.defined() && !dn.defined()) return result;
        variable_list keep;
        p3d_block_args a = bind_block(spec, in, keep);
        if (seed.defined()) a.dropout.state = static_cast<const int64_t*>(seed.const_data_ptr());
        const int64_t dim = a.dim, rows = a.samples * a.tokens;
        auto need = [&](int i) { return in[i].defined() && task_should_compute_output(i); };
        // Without a gradient through the next norm dx is alpha dout: dout itself for 1.
        const bool through = !dn.defined() && spec.alpha == 1.f;
        Tensor dx, dy, dgate;
        if (!through && (need(kX) || dn.defined())) {
            dx = empty_as(x, x.scalar_type());
            a.dx = dx.data_ptr();
        }
        if (y.defined()) {
            dy = empty_as(y, y.scalar_type());
            a.dy = dy.data_ptr();
        }
        if (gate.defined() && (need(kGate) || spec.gate_kind != P3D_GATE_SAMPLE)) {
            dgate = empty_as(gate, gate.scalar_type());
            a.dgate = dgate.data_ptr();
        }
        static constexpr int kParams[5] = {kPostWeight, kPostBias, kScale, kNextWeight, kNextBias};
        for (int i = 0; i < 5; ++i) {
            const Tensor& p = in[kParams[i]];
            if (!need(kParams[i])) continue;
            if (!rows || (i >= 3 && !dn.defined())) {
                result[kParams[i]] = at::zeros(p.sizes(), p.options().requires_grad(false));
                continue;
            }
            const at::ScalarType type = dtype_of(p.scalar_type()) >= 0 ? p.scalar_type() : at::kFloat;
            Tensor g = empty_as(p, type);
            a.d_param[i] = g.data_ptr();
            a.d_param_dtype[i] = dtype_of(type);
            result[kParams[i]] = g;
        }
        if (rows) {
            if (y.defined()) {
                // Only n was used: a row of zeros, for every row.
                if (!dout.defined()) dout = at::zeros({1, dim}, x.options().requires_grad(false)).expand({rows, dim});
                dout = dout.to(x.scalar_type());
                std::tie(a.dout, a.dout_stride) = rows_of(dout, dim, keep);
            }
            if (dn.defined()) {
                dn = dn.to(spec.inner);
                std::tie(a.dn, a.dn_stride) = rows_of(dn, dim, keep);
            }
            const auto [splits, grid] = block_split(a.samples, a.tokens, dim, backward_round(x, a));
            a.splits = (int32_t)splits;
            a.grid = (int32_t)grid;
            const int64_t sums = grid * 5 + (spec.gate_kind == P3D_GATE_SAMPLE ? splits * a.samples : 0);
            const Tensor work = at::empty({sums * dim}, x.options().dtype(at::kFloat).requires_grad(false));
            a.stats = static_cast<float*>(stats.data_ptr());
            a.work = static_cast<float*>(work.data_ptr());
            launch("p3d_block_bwd", x, lib.block_bwd, &a);
            for (const int i : kParams)
                if (result[i].defined() && result[i].scalar_type() != in[i].scalar_type())
                    result[i] = result[i].to(in[i].scalar_type());
        } else if (dgate.defined()) {
            dgate.zero_();
        }
        if (need(kX)) result[kX] = through ? grads[0] : dx;
        if (need(kY)) result[kY] = dy;
        if (need(kGate)) result[kGate] = dgate;
        variable_list from(in.begin(), in.end());
        from.insert(from.end(), grads.begin(), grads.end());
        return first_order(std::move(result), create_graph, from, "the end of a block");
    }
};

void check_param(const char* what, const MaybeTensor& t, const Tensor& x) {
    if (t)
        TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1) && t->device() == x.device() && t->is_floating_point(),
                          what, ": parameters must be floating point [dim] on the input's device");
}

NormSpec check_norm(const char* what, int64_t kind, double eps, const MaybeTensor& weight, const MaybeTensor& bias,
                    const Tensor& x) {
    if (!kind) return NormSpec{};
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), what, ": eps must be finite and not negative");
    check_param(what, weight, x);
    check_param(what, bias, x);
    return NormSpec{(int)kind, (float)eps};
}

// How the gate spreads over x [batch, tokens, dim] or [tokens, dim].
int gate_kind_of(const Tensor& gate, const Tensor& x) {
    TORCH_CHECK_VALUE(gate.dim() == x.dim() && gate.device() == x.device() && dtype_of(gate.scalar_type()) >= 0,
                      "gate must be fp32, fp16 or bf16 with x's number of dimensions, on its device");
    const int64_t r = x.dim(), n = x.size(r - 2), dim = x.size(r - 1), gn = gate.size(r - 2), gdim = gate.size(r - 1);
    const bool lead = r == 2 || gate.size(0) == x.size(0), one = r == 2 || gate.size(0) == 1;
    if (lead && gn == n && gdim == dim) return P3D_GATE_FULL;
    if (lead && gn == n && gdim == 1) return P3D_GATE_TOKEN;
    TORCH_CHECK_VALUE((lead || one) && gn == 1 && gdim == dim,
                      "gate must be [batch or 1, 1, dim], [batch, tokens, 1] or [batch, tokens, dim]");
    return P3D_GATE_SAMPLE;
}

py::object block(const Tensor& x, const MaybeTensor& y, const MaybeTensor& gate, const MaybeTensor& scale,
                 int64_t post_kind, const MaybeTensor& post_weight, const MaybeTensor& post_bias, double post_eps,
                 int64_t next_kind, const MaybeTensor& next_weight, const MaybeTensor& next_bias, double next_eps,
                 double alpha, int64_t threshold, const MaybeTensor& state, int64_t seed, int64_t offset,
                 std::optional<at::ScalarType> inner) {
    require_device(x, "x");
    const at::ScalarType outer = x.scalar_type();
    TORCH_CHECK_VALUE(dtype_of(outer) >= 0, "x must be fp32, fp16 or bf16");
    TORCH_CHECK_VALUE((x.dim() == 2 || x.dim() == 3) && x.size(-1) >= 1 && x.size(-1) <= kMaxDim,
                      "x must be [batch, tokens, dim] or [tokens, dim] with dim 1 to 8192");
    TORCH_CHECK_VALUE(x.numel() / x.size(-1) < (1LL << 31), "x has too many rows");
    BlockSpec spec;
    if (y) {
        TORCH_CHECK_VALUE(y->sizes() == x.sizes() && y->device() == x.device(), "y must have x's shape and device");
        spec.inner = y->scalar_type();
        TORCH_CHECK_VALUE(dtype_of(spec.inner) >= 0 && (outer == at::kFloat || spec.inner == outer),
                          "y must have x's type, or fp16 or bf16 over an fp32 x");
    } else {
        spec.inner = inner.value_or(outer);
        TORCH_CHECK_VALUE(dtype_of(spec.inner) >= 0 && (outer == at::kFloat || spec.inner == outer),
                          "dtype must be x's, or fp16 or bf16 for an fp32 x");
    }
    spec.post = check_norm("post_norm", post_kind, post_eps, post_weight, post_bias, x);
    spec.next = check_norm(y ? "next_norm" : "norm", next_kind, next_eps, next_weight, next_bias, x);
    check_param("scale", scale, x);
    TORCH_CHECK_VALUE(std::isfinite(alpha), "alpha must be finite");
    spec.alpha = (float)alpha;
    if (threshold) {
        spec.mask.threshold = (int32_t)threshold;
        spec.mask.state = state ? static_cast<const int64_t*>(state->const_data_ptr()) : nullptr;
        spec.mask.seed = seed;
        spec.mask.offset = offset;
    }
    if (gate) spec.gate_kind = gate_kind_of(*gate, x);
    const Inputs in = {x, or_undefined(y), or_undefined(gate), or_undefined(scale), or_undefined(post_weight),
                       or_undefined(post_bias), or_undefined(next_weight), or_undefined(next_bias)};
    for (const Tensor& t : in) no_forward_mode(t);
    const bool grad = torch::autograd::compute_requires_grad(in[0], in[1], in[2], in[3], in[4], in[5], in[6], in[7]);
    std::shared_ptr<BlockBackward> node;
    if (grad) {
        node = std::shared_ptr<BlockBackward>(new BlockBackward(), torch::autograd::deleteNode);
        node->set_next_edges(
            torch::autograd::collect_next_edges(in[0], in[1], in[2], in[3], in[4], in[5], in[6], in[7]));
        node->spec = spec;
        for (int i = 0; i < kInputs; ++i)
            if (in[i].defined()) node->saved[i] = SavedVariable(in[i], false);
        if (threshold && state) node->state = SavedVariable(*state, false);
    }
    BlockOutputs o = [&] {
        const py::gil_scoped_release free;
        return block_forward(spec, in, grad);
    }();
    if (grad) {
        node->stats = o.stats;
        if (o.out.defined()) torch::autograd::set_history(o.out, node);
        if (o.n.defined()) torch::autograd::set_history(o.n, node);
    }
    if (!o.n.defined()) return py::cast(o.out);
    if (!o.out.defined()) return py::cast(o.n);
    return py::make_tuple(o.out, o.n);
}

// --------------------------------------------------------------- dropout
Tensor dropout_pass(const Tensor& x, const p3d_dropout& mask) {
    const c10::AutoGradMode off(false);
    const Tensor c = x.contiguous();
    Tensor y = empty_as(c, c.scalar_type());
    if (c.numel())
        launch("p3d_dropout_apply", c, lib.dropout_apply, c.const_data_ptr(), y.data_ptr(), c.numel(),
               (int32_t)dtype_of(c.scalar_type()), &mask);
    return y;
}

struct DropoutBackward : public Node {
    p3d_dropout mask{};
    SavedVariable state;
    std::string name() const override { return "Pack3DDropoutBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        state.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        refuse_default_stream(*this);
        const Tensor seed = state.unpack(shared_from_this());
        if (!grads[0].defined()) return {Tensor()};
        if (seed.defined()) mask.state = static_cast<const int64_t*>(seed.const_data_ptr());
        return first_order({dropout_pass(grads[0], mask)}, c10::GradMode::is_enabled(), grads, "dropout");
    }
};

Tensor dropout(const Tensor& x, int64_t threshold, const MaybeTensor& state, int64_t seed, int64_t offset) {
    require_device(x, "x");
    TORCH_CHECK_VALUE(dtype_of(x.scalar_type()) >= 0, "counter_dropout takes fp32, fp16 or bf16");
    no_forward_mode(x);
    p3d_dropout mask{};
    mask.threshold = (int32_t)threshold;
    mask.state = state ? static_cast<const int64_t*>(state->const_data_ptr()) : nullptr;
    mask.seed = seed;
    mask.offset = offset;
    Tensor y = [&] {
        const py::gil_scoped_release free;
        return dropout_pass(x, mask);
    }();
    if (torch::autograd::compute_requires_grad(x)) {
        auto node = std::shared_ptr<DropoutBackward>(new DropoutBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x));
        node->mask = mask;
        if (state) node->state = SavedVariable(*state, false);
        torch::autograd::set_history(y, node);
    }
    return y;
}

// ---------------------------------------------------------------- rotary
constexpr size_t kMaxTensors = 4;

// The tensors turned, dense, with their dimensions in memory in the order of the inputs'.
variable_list turn(p3d_rotary_args a, const variable_list& tensors, bool inverse) {
    const c10::AutoGradMode off(false);
    variable_list outs, keep;
    a.count = (int32_t)tensors.size();
    a.inverse = inverse;
    for (size_t i = 0; i < tensors.size(); ++i) {
        Tensor t = tensors[i];
        if (t.stride(3) != 1) {
            t = t.contiguous();
            keep.push_back(t);
        }
        Tensor out = at::empty_like(t, t.options().requires_grad(false));
        if (out.stride(3) != 1) out = empty_as(t, t.scalar_type());
        a.x[i] = p3d_view{const_cast<void*>(t.const_data_ptr()), t.stride(0), t.stride(1), t.stride(2)};
        a.y[i] = p3d_view{out.data_ptr(), out.stride(0), out.stride(1), out.stride(2)};
        a.heads[i] = (int32_t)t.size(1);
        outs.push_back(std::move(out));
    }
    if (tensors[0].numel()) launch("p3d_rotary", tensors[0], lib.rotary, &a);
    return outs;
}

struct RotaryBackward : public Node {
    p3d_rotary_args args{};
    SavedVariable positions, freqs;
    std::string name() const override { return "Pack3DRotaryBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        positions.reset_data();
        freqs.reset_data();
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        refuse_default_stream(*this);
        const bool create_graph = c10::GradMode::is_enabled();
        const Tensor p = positions.unpack(shared_from_this()), f = freqs.unpack(shared_from_this());
        args.positions = p.const_data_ptr();
        args.freqs = static_cast<const double*>(f.const_data_ptr());
        variable_list result(grads.size()), given;
        std::vector<size_t> which;
        for (size_t i = 0; i < grads.size(); ++i)
            if (grads[i].defined() && task_should_compute_output(i)) {
                which.push_back(i);
                given.push_back(grads[i]);
            }
        if (given.empty()) return result;
        variable_list back = turn(args, given, true);
        for (size_t k = 0; k < which.size(); ++k) result[which[k]] = std::move(back[k]);
        return first_order(std::move(result), create_graph, grads, "rotary positions");
    }
};

variable_list rotary(const variable_list& tensors, const Tensor& positions, const Tensor& freqs,
                     const std::optional<std::vector<int64_t>>& pairs, bool half, double magnitude) {
    TORCH_CHECK_VALUE(!tensors.empty() && tensors.size() <= kMaxTensors, "apply_rotary takes one to four tensors");
    const Tensor& first = tensors[0];
    TORCH_CHECK_VALUE(first.dim() == 4, "tensors must be [batch, heads, tokens, head_dim]");
    const int64_t b = first.size(0), n = first.size(2), d = first.size(3);
    for (const Tensor& t : tensors) {
        TORCH_CHECK_VALUE(t.dim() == 4 && t.scalar_type() == first.scalar_type() && t.device() == first.device() &&
                              t.size(0) == b && t.size(2) == n && t.size(3) == d,
                          "tensors must be [batch, heads, tokens, head_dim] of one type, alike but for the heads");
        TORCH_CHECK_VALUE(t.size(1) >= 1 && t.size(1) * (d / 8 + 2) <= 8192,
                          "heads must be at least 1, heads * (head_dim / 8 + 2) at most 8192");
        no_forward_mode(t);
    }
    require_device(first, "q and k");
    TORCH_CHECK_VALUE(dtype_of(first.scalar_type()) >= 0, "apply_rotary takes fp32, fp16 or bf16");
    TORCH_CHECK_VALUE(b < (1LL << 31), "batch out of range");
    TORCH_CHECK_VALUE(freqs.scalar_type() == at::kDouble && freqs.dim() == 1 && freqs.device() == first.device(),
                      "freqs must be float64 [pairs] on the tensors' device (rotary_frequencies)");
    const int64_t count = freqs.size(0);
    TORCH_CHECK_VALUE(count >= 1 && count <= d / 2 && d <= 1024,
                      "freqs must have 1 to head_dim / 2 pairs, head_dim at most 1024");
    p3d_rotary_args a{};
    int64_t axes = 1;
    a.axis_pairs[0] = (int32_t)count;
    if (pairs) {
        axes = (int64_t)pairs->size();
        int64_t sum = 0;
        bool counts = true;
        for (const int64_t c : *pairs) {
            counts = counts && c >= 0 && c <= count;
            sum += c;
        }
        TORCH_CHECK_VALUE(axes >= 1 && axes <= 3 && counts && sum == count,
                          "pairs must give each of one to three axes its count of freqs");
        for (int64_t i = 0; i < axes; ++i) a.axis_pairs[i] = (int32_t)(*pairs)[i];
    }
    TORCH_CHECK_VALUE(std::isfinite(magnitude), "magnitude must be finite");
    TORCH_CHECK_VALUE((positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong) &&
                          positions.device() == first.device(),
                      "positions must be int32 or int64 on the tensors' device");
    // [tokens] or [batch, tokens], and an axis dimension last for several axes.
    const int64_t extra = axes > 1 ? 1 : 0, r = positions.dim() - extra;
    TORCH_CHECK_VALUE((r == 1 || r == 2) && positions.size(r - 1) == n && (!extra || positions.size(r) == axes) &&
                          (r == 1 || positions.size(0) == 1 || positions.size(0) == b),
                      "positions must be [tokens] or [batch, tokens], with an axis dimension last for several axes");
    a.tokens = n;
    a.batch = (int32_t)b;
    a.head_dim = (int32_t)d;
    a.pairs = (int32_t)count;
    a.axes = (int32_t)axes;
    a.positions = positions.const_data_ptr();
    a.pos_sb = r == 2 && positions.size(0) != 1 ? positions.stride(0) : 0;
    a.pos_sn = positions.stride(r - 1);
    a.pos_sa = extra ? positions.stride(r) : 1;
    a.pos_is64 = positions.scalar_type() == at::kLong;
    const Tensor f = freqs.contiguous();
    a.freqs = static_cast<const double*>(f.const_data_ptr());
    a.half = half;
    a.dtype = dtype_of(first.scalar_type());
    a.magnitude = (float)magnitude;
    variable_list outs = [&] {
        const py::gil_scoped_release free;
        return turn(a, tensors, false);
    }();
    bool grad = false;
    for (const Tensor& t : tensors) grad = grad || torch::autograd::compute_requires_grad(t);
    if (grad) {
        auto node = std::shared_ptr<RotaryBackward>(new RotaryBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(tensors));
        node->args = a;
        node->positions = SavedVariable(positions, false);
        node->freqs = SavedVariable(f, false);
        torch::autograd::set_history(outs, node);
    }
    return outs;
}

// f with torch's errors as Python's, whatever compiler torch itself was built by.
template <typename R, typename... A>
auto python_errors(R (*f)(A...)) {
    return [f](A... args) -> R {
        try {
            return f(static_cast<A>(args)...);
        } catch (const c10::ValueError& e) {
            throw py::value_error(e.what_without_backtrace());
        } catch (const c10::OutOfMemoryError&) {
            throw;
        } catch (const c10::Error& e) {
            throw std::runtime_error(e.what_without_backtrace());
        }
    };
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("abi_version", [] { return P3D_ABI_VERSION; });
    m.def("bind_library", &bind_library);
    m.def("block_split", &block_split);
    m.def("block", python_errors(&block));
    m.def("dropout", python_errors(&dropout));
    m.def("rotary", python_errors(&rotary));
}
