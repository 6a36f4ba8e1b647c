// The norm before a block and the end of a block in one pass over its rows, forward
// and backward.  Per row of dim channels, all in fp32, each output rounded once:
//   b = norm1(y) w1 + b1 (or y),  z = keep ? b / (1 - p) : 0,
//   out = alpha x + scale gate z,  n = norm2(out) w2 + b2,
// with norm(v) = (v - mean) rstd (LayerNorm, biased variance from the centred values)
// or v rstd (RMSNorm).  Without y, out is x: the norm before a block.  With go the
// gradient of out,
//   go = dout + rstd2 (g2 - [layer] mean(g2) - xh2 mean(g2 xh2)),  g2 = dn w2,
//   dx = alpha go,  dscale = sum gate z go,  dgate = sum scale z go,
//   db = keep scale gate go / (1 - p),  g1 = db w1,
//   dy = rstd1 (g1 - [layer] mean(g1) - xh1 mean(g1 xh1)),
// and the norms' weight and bias gradients sum xh and 1 times dn (next) and db
// (post) over the rows.  The backward forms out again from x and y (the same bytes as
// reading it, and not rounded); the statistics come from the forward.
//
// Both are bound by memory: x and y (and dout and dn) are read, out and n (dx and dy)
// written once.  262,144 rows of 192, fp32 x over bf16 y, with a post norm, dropout, a
// gate per sample, scale and the next norm: forward 604 MB in 122 us, backward 906 MB in
// 194 (4.9 and 4.7 TB/s; a large copy reaches 5.4), and 8 us for the partial sums.
// 8,192 rows of 4,096 in bf16 with a gate per token and two RMSNorms: 56 and 91 us for
// 268 and 403 MB (4.8 and 4.4).
//
// TPR threads share a row and hold E consecutive channels each, so a row is read
// once into registers whatever its width.  Rows of up to 512 channels lie within a
// wave, several to a wave below that; wider ones take a workgroup.  The next row's
// loads are issued before the present one is worked on (where registers allow).
//
// Where E does not divide the width, the row's last lane holds its last E channels
// and shares some with its neighbour: both compute and store the same bits, and sums
// leave the shared ones out.  Lanes past the row do the same work on the last channels
// and store nothing.
//
// Rows are dealt out in units: `tokens` rows that share a gate vector (a sample), cut
// into `splits` ranges.  A workgroup takes units blockIdx.x, + gridDim.x, ..., so the
// gate and the parameters stay in registers over a unit's rows.
//
// Sums over rows are held in registers over all rows of a workgroup, then added over
// its row groups in LDS in a fixed order; a workgroup writes one row of partials, which
// p3d_sum_rows adds.  No atomics.
#pragma once

#include "block.hpp"

namespace p3d {
namespace {

// The rows of unit u: `count` rows from `first` on.
struct Unit {
    int sample, first, count;
};
__device__ __forceinline__ Unit unit_of(const BlockDev& a, int u) {
    const int split = u / a.samples, sample = u - split * a.samples;
    const int64_t per = (a.tokens + a.splits - 1) / a.splits;
    const int64_t at = min(split * per, a.tokens), end = min(at + per, a.tokens);
    return Unit{sample, (int)(sample * a.tokens + at), (int)(end - at)};
}

constexpr int block_threads(int tpr) { return tpr <= 64 ? 256 : tpr; }

// Where a thread is in its row.
template <int TPR, int E>
struct Place {
    int sub, grp;
    int c;    // first channel
    int dup;  // leading channels that the lane before holds too; E or more: past the row
    __device__ __forceinline__ explicit Place(int dim) {
        sub = threadIdx.x % TPR;
        grp = threadIdx.x / TPR;
        c = min(sub * E, dim - E);
        dup = sub * E - c;
    }
    __device__ __forceinline__ bool in_row() const { return dup < E; }
    // Sum over the thread's own channels.
    __device__ __forceinline__ float own(const float (&v)[E]) const {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += v[e];
        if (dup) {
            s = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) s += e >= dup ? v[e] : 0.f;
        }
        return s;
    }
};

// E values of a tensor of a runtime dtype, as bits until they are used, so that the
// loads of several are in flight together.
template <int E>
struct AnyRun {
    uint32_t raw[E];
    __device__ __forceinline__ void load(const void* p, int dtype, int64_t c) {
        if (dtype == P3D_F32) __builtin_memcpy(raw, reinterpret_cast<const float*>(p) + c, 4 * E);
        else __builtin_memcpy(raw, reinterpret_cast<const uint16_t*>(p) + c, 2 * E);
    }
    __device__ __forceinline__ float one(int dtype, int e) const {
        if (dtype == P3D_F32) return __uint_as_float(raw[e]);
        const uint32_t word = raw[e >> 1];
        const uint16_t half = (uint16_t)(e & 1 ? word >> 16 : word);
        if (dtype == P3D_BF16) return __uint_as_float((uint32_t)half << 16);
        return (float)__builtin_bit_cast(_Float16, half);
    }
    __device__ __forceinline__ void to(int dtype, float (&v)[E]) const {
        if (dtype == P3D_F32) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = one(P3D_F32, e);
        } else if (dtype == P3D_F16) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = one(P3D_F16, e);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = one(P3D_BF16, e);
        }
    }
};

// Parameters of a run of channels: all loads, then all values, `missing` where one is
// not there.
template <int E, int N>
__device__ __forceinline__ void load_params(const void* const (&p)[N], int dtype, int64_t c, const float (&missing)[N],
                                            float (&v)[N][E]) {
    AnyRun<E> r[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (p[k]) r[k].load(p[k], dtype, c);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (p[k]) {
            r[k].to(dtype, v[k]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] = missing[k];
        }
    }
}
template <int E>
__device__ __forceinline__ void load_param(const void* p, int dtype, int64_t c, float missing, float (&v)[E]) {
    float one[1][E];
    load_params<E, 1>({p}, dtype, c, {missing}, one);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = one[0][e];
}

// A gate of one value a token or an element.
template <int E>
struct GateRun {
    AnyRun<E> r;
    __device__ __forceinline__ void load(const BlockDev& a, uint32_t row, int c) {
        const char* at = row_address(reinterpret_cast<const char*>(a.gate), row, a.gate_stride);
        if (a.gate_kind == P3D_GATE_TOKEN) {
            r.raw[0] = a.gate_dtype == P3D_F32 ? *reinterpret_cast<const uint32_t*>(at)
                                               : (uint32_t)*reinterpret_cast<const uint16_t*>(at);
        } else {
            r.load(at, a.gate_dtype, c);
        }
    }
    __device__ __forceinline__ void to(const BlockDev& a, float (&g)[E]) const {
        if (a.gate_kind == P3D_GATE_TOKEN) {
            const float t = r.one(a.gate_dtype, 0);
#pragma unroll
            for (int e = 0; e < E; ++e) g[e] = t;
        } else {
            r.to(a.gate_dtype, g);
        }
    }
};

// v -> (v - mean) rstd over the row.
template <int TPR, int E>
__device__ __forceinline__ void normalise(RowSum<TPR>& row_sum, const Place<TPR, E>& at, int kind, float eps,
                                          float inv_dim, float (&v)[E], float& mean, float& rstd) {
    mean = 0.f;
    if (kind == P3D_NORM_LAYER) {
        float s[1] = {at.own(v)};
        row_sum.sum(s);
        mean = s[0] * inv_dim;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] -= mean;
    }
    float q[E], s[1];
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = v[e] * v[e];
    s[0] = at.own(q);
    row_sum.sum(s);
    rstd = 1.f / sqrtf(s[0] * inv_dim + eps);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= rstd;
}

// What a kernel is made for: the norm before a block; the end of one, with no gate or a
// gate per sample; the end of one with a gate per token or element.
enum Form { kNorm, kEnd, kEndGated };

template <typename TX, typename TY, int TPR, int E, int FORM>
__global__ __launch_bounds__(block_threads(TPR)) void k_block_fwd(BlockDev a) {
    constexpr int GROUPS = TPR > 64 ? 1 : 256 / TPR;
    constexpr bool HAS_Y = FORM != kNorm, GATED = FORM == kEndGated;
    __shared__ float lds[RowSum<TPR>::LDS];
    RowSum<TPR> row_sum{lds};
    const Place<TPR, E> at(a.dim);
    const int c = at.c;
    const float inv_dim = 1.f / (float)a.dim;
    MaskDev mask = a.mask;
    mask_begin(mask);
    const char* px = reinterpret_cast<const char*>(a.x) + c * sizeof(TX);
    const char* py = reinterpret_cast<const char*>(a.y) + c * sizeof(TY);
    char* pout = reinterpret_cast<char*>(a.out) + c * sizeof(TX);
    char* pn = reinterpret_cast<char*>(a.n) + c * sizeof(TY);
    float par[4][E];
    load_params<E, 4>({a.next.weight, a.next.bias, HAS_Y ? a.post.weight : nullptr, HAS_Y ? a.post.bias : nullptr}, a.param,
                      c, {1.f, 0.f, 1.f, 0.f}, par);
    const float(&w2)[E] = par[0], (&b2)[E] = par[1], (&w1)[E] = par[2], (&b1)[E] = par[3];
    const int units = a.samples * a.splits;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit unit = unit_of(a, u);
        if (unit.count <= 0) continue;
        float ks[E];  // scale, gate of the sample and 1 / (1 - p)
        if constexpr (HAS_Y) {
            float gs[E];
            load_param(a.scale, a.param, c, 1.f, ks);
            load_param(a.gate_kind == P3D_GATE_SAMPLE ? a.gate : nullptr, a.gate_dtype,
                       (int64_t)unit.sample * (a.gate_stride / (a.gate_dtype == P3D_F32 ? 4 : 2)) + c, 1.f, gs);
#pragma unroll
            for (int e = 0; e < E; ++e) ks[e] *= gs[e] * mask.inv;
        }
        Run<TX, E> xr;
        Run<TY, E> yr;
        GateRun<E> gr;
        auto fetch = [&](uint32_t row) {
            xr.load(row_address(px, row, a.x_stride));
            if constexpr (HAS_Y) yr.load(row_address(py, row, a.y_stride));
            if constexpr (GATED) gr.load(a, row, c);
        };
        const int last = unit.count - 1;
        fetch(unit.first + min(at.grp, last));
        for (int i = at.grp; i <= last; i += GROUPS) {
            const uint32_t row = unit.first + i;
            float v[E], z[E], g[E];
            xr.to(v);
            if constexpr (HAS_Y) yr.to(z);
            if constexpr (GATED) gr.to(a, g);
            fetch(unit.first + min(i + GROUPS, last));
            float mean, rstd;
            if constexpr (HAS_Y) {
                if (a.post.kind) {
                    normalise(row_sum, at, a.post.kind, a.post.eps, inv_dim, z, mean, rstd);
#pragma unroll
                    for (int e = 0; e < E; ++e) z[e] = z[e] * w1[e] + b1[e];
                    if (a.stats && at.sub == 0) {
                        a.stats[row] = mean;
                        a.stats[a.rows + row] = rstd;
                    }
                }
                if (mask.threshold) {
                    uint32_t bits = 0;
                    if (TPR <= 64 || at.in_row()) bits = keep_run<TPR, E>(mask, row, a.dim, c, at.sub);
#pragma unroll
                    for (int e = 0; e < E; ++e) z[e] = and_word(z[e], bit_word(bits, e));
                }
                if constexpr (GATED) {
#pragma unroll
                    for (int e = 0; e < E; ++e) z[e] *= g[e];
                }
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = a.alpha * v[e] + ks[e] * z[e];
                if (at.in_row()) {
                    Run<TX, E> o;
                    o.from(v);
                    o.store(row_address(pout, row, a.dim * (uint32_t)sizeof(TX)));
                }
            }
            if (a.next.kind) {
                normalise(row_sum, at, a.next.kind, a.next.eps, inv_dim, v, mean, rstd);
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = v[e] * w2[e] + b2[e];
                if (at.in_row()) {
                    Run<TY, E> o;
                    o.from(v);
                    o.store(row_address(pn, row, a.dim * (uint32_t)sizeof(TY)));
                }
                if (a.stats && at.sub == 0) {
                    a.stats[2 * (int64_t)a.rows + row] = mean;
                    a.stats[3 * (int64_t)a.rows + row] = rstd;
                }
            }
        }
    }
}

// NEXT: with a gradient of n.  Every load and store of a row but the gate's is made on
// every path, by every lane (those past the row store their neighbour's bits): the wait
// for the next row's loads then knows how many stores came after them, and does not wait
// for the stores.
template <typename TX, typename TY, int TPR, int E, int FORM, bool NEXT>
__global__ __launch_bounds__(block_threads(TPR)) void k_block_bwd(BlockDev a) {
    constexpr int GROUPS = TPR > 64 ? 1 : 256 / TPR;
    constexpr bool HAS_Y = FORM != kNorm, GATED = FORM == kEndGated;
    // Rows of 1,024 threads leave 128 registers a thread: the next row's loads would be
    // spilled (5,333 rows of 6,144 forward and backward 255 us with, 173 without).
    constexpr bool AHEAD = TPR <= 512 || FORM == kNorm;
    __shared__ float lds[TPR > 64 ? RowSum<TPR>::LDS : 4 * TPR * E];
    RowSum<TPR> row_sum{lds};
    const Place<TPR, E> at(a.dim);
    const int c = at.c;
    const float inv_dim = 1.f / (float)a.dim;
    const bool layer1 = a.post.kind == P3D_NORM_LAYER, layer2 = a.next.kind == P3D_NORM_LAYER;
    const bool has_post = HAS_Y && a.post.kind;
    const bool per_sample = a.gate_kind == P3D_GATE_SAMPLE;
    MaskDev mask = a.mask;
    mask_begin(mask);
    const char* px = reinterpret_cast<const char*>(a.x) + c * sizeof(TX);
    const char* py = reinterpret_cast<const char*>(a.y) + c * sizeof(TY);
    const char* pdout = reinterpret_cast<const char*>(a.dout) + c * sizeof(TX);
    const char* pdn = reinterpret_cast<const char*>(a.dn) + c * sizeof(TY);
    char* pdx = reinterpret_cast<char*>(a.dx) + c * sizeof(TX);
    char* pdy = reinterpret_cast<char*>(a.dy) + c * sizeof(TY);
    // Next weight, post weight and bias, and scale, gate of the sample and 1 / (1 - p).
    // Rows of 1,024 threads hold them in LDS, each thread its own (3,906 bf16 rows of 8,192
    // with a gate per sample, a post and a next norm, forward and backward: 174 us, 282
    // with all of them in registers, of which 68 a thread were spilled).
    enum { kW2, kW1, kB1, kKs };
    constexpr bool STAGED = TPR > 512 && HAS_Y;
    __shared__ float staged[STAGED ? 4 : 1][STAGED ? E : 1][STAGED ? TPR : 1];
    float par[4][E];
    {
        float w[3][E];
        load_params<E, 3>({a.next.weight, HAS_Y ? a.post.weight : nullptr, HAS_Y ? a.post.bias : nullptr}, a.param, c,
                          {1.f, 1.f, 0.f}, w);
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (STAGED) staged[k][e][threadIdx.x] = w[k][e];
                else par[k][e] = w[k][e];
            }
    }
    auto param = [&](int k, int e) {
        if constexpr (STAGED) return staged[k][e][threadIdx.x];
        else return par[k][e];
    };
    // Sums over this thread's rows: dw1, db1, dscale (1 - p), dw2, db2.
    float dw1[E], db1[E], dsc[E], dw2[E], db2[E];
#pragma unroll
    for (int e = 0; e < E; ++e) dw1[e] = db1[e] = dsc[e] = dw2[e] = db2[e] = 0.f;

    // Sum over the workgroup's row groups, in a fixed order; group 0 stores it.
    auto gather = [&](float(&v)[E], float* to) {
        if constexpr (GROUPS > 1) {
            // The groups of a wave by lanes, then the four waves in order.
#pragma unroll
            for (int o = TPR; o < 64; o *= 2)
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] += __shfl_xor(v[e], o);
            __syncthreads();
            if ((threadIdx.x & 63) < TPR) {
#pragma unroll
                for (int e = 0; e < E; ++e) lds[((threadIdx.x >> 6) * E + e) * TPR + at.sub] = v[e];
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] = (lds[e * TPR + at.sub] + lds[(E + e) * TPR + at.sub]) +
                       (lds[(2 * E + e) * TPR + at.sub] + lds[(3 * E + e) * TPR + at.sub]);
        }
        if (at.grp == 0 && at.in_row()) {
            Run<float, E> o;
            o.from(v);
            o.store(to + c);
        }
    };

    const int units = a.samples * a.splits;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const Unit unit = unit_of(a, u);
        const int64_t gate_at = (int64_t)unit.sample * (a.gate_stride / (a.gate_dtype == P3D_F32 ? 4 : 2)) + c;
        float unit_acc[E];  // sum of gate keep b go
        if constexpr (HAS_Y) {
            float gs[E], ks[E];
            load_param(a.scale, a.param, c, 1.f, ks);
            load_param(per_sample ? a.gate : nullptr, a.gate_dtype, gate_at, 1.f, gs);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (STAGED) staged[kKs][e][threadIdx.x] = ks[e] * gs[e] * mask.inv;
                else par[kKs][e] = ks[e] * gs[e] * mask.inv;
                unit_acc[e] = 0.f;
            }
        }
        if (unit.count > 0) {
            Run<TX, E> xr, dor;
            Run<TY, E> yr, dnr;
            GateRun<E> gr;
            float st[4];  // the row's statistics
            auto fetch = [&](uint32_t row) {
                if (has_post) {
                    st[0] = a.stats[row];
                    st[1] = a.stats[a.rows + row];
                }
                if constexpr (NEXT) {
                    st[2] = a.stats[2 * (int64_t)a.rows + row];
                    st[3] = a.stats[3 * (int64_t)a.rows + row];
                }
                if constexpr (GATED) gr.load(a, row, c);
                if constexpr (HAS_Y) {
                    yr.load(row_address(py, row, a.y_stride));
                    dor.load(row_address(pdout, row, a.dout_stride));
                }
                if constexpr (NEXT) {
                    xr.load(row_address(px, row, a.x_stride));
                    dnr.load(row_address(pdn, row, a.dn_stride));
                }
            };
            const int last = unit.count - 1;
            if constexpr (AHEAD) fetch(unit.first + min(at.grp, last));
            for (int i = at.grp; i <= last; i += GROUPS) {
                const uint32_t row = unit.first + i;
                if constexpr (!AHEAD) fetch(row);
                float go[E], xh2[E], g2[E], xh1[E], g[E];
                if constexpr (HAS_Y) {
                    yr.to(xh1);
                    dor.to(go);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e) go[e] = 0.f;
                }
                if constexpr (NEXT) {
                    xr.to(xh2);
                    dnr.to(g2);
                }
                if constexpr (GATED) gr.to(a, g);
                const float mean1 = st[0], rstd1 = st[1], mean2 = st[2], rstd2 = st[3];
                if constexpr (AHEAD) fetch(unit.first + min(i + GROUPS, last));
                uint32_t bits = 0xffffffffu;
                float b[E];  // keep b
                if constexpr (HAS_Y) {
                    if (has_post) {
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            xh1[e] = (xh1[e] - mean1) * rstd1;
                            b[e] = xh1[e] * param(kW1, e) + param(kB1, e);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < E; ++e) b[e] = xh1[e];
                    }
                    if (mask.threshold) {
                        bits = keep_run<TPR, E>(mask, row, a.dim, c, at.sub);
#pragma unroll
                        for (int e = 0; e < E; ++e) b[e] = and_word(b[e], bit_word(bits, e));
                    }
                }
                if constexpr (NEXT) {
                    float p[E], s[2];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float out = xh2[e];
                        if constexpr (HAS_Y) out = a.alpha * out + param(kKs, e) * (GATED ? g[e] * b[e] : b[e]);
                        xh2[e] = (out - mean2) * rstd2;
                        dw2[e] += g2[e] * xh2[e];
                        db2[e] += g2[e];
                        g2[e] *= param(kW2, e);
                        p[e] = g2[e] * xh2[e];
                    }
                    s[0] = layer2 ? at.own(g2) : 0.f;
                    s[1] = at.own(p);
                    row_sum.sum(s);
                    const float m0 = s[0] * inv_dim, m1 = s[1] * inv_dim;
#pragma unroll
                    for (int e = 0; e < E; ++e) go[e] += rstd2 * (g2[e] - m0 - xh2[e] * m1);
                }
                if (NEXT || a.dx) {
                    float v[E];
                    Run<TX, E> o;
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = a.alpha * go[e];
                    o.from(v);
                    o.store(row_address(pdx, row, a.dim * (uint32_t)sizeof(TX)));
                }
                if constexpr (HAS_Y) {
                    float db[E], dg[E], s[GATED ? 3 : 2];
                    s[0] = s[1] = 0.f;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if constexpr (GATED) {
                            const float bg = b[e] * go[e];
                            unit_acc[e] += g[e] * bg;
                            dg[e] = param(kKs, e) * bg;
                            db[e] = param(kKs, e) * g[e] * go[e];
                        } else {
                            unit_acc[e] += b[e] * go[e];
                            db[e] = param(kKs, e) * go[e];
                        }
                    }
                    if (mask.threshold) {
#pragma unroll
                        for (int e = 0; e < E; ++e) db[e] = and_word(db[e], bit_word(bits, e));
                    }
                    const bool token_sum = GATED && a.gate_kind == P3D_GATE_TOKEN;
                    if constexpr (GATED) s[2] = token_sum ? at.own(dg) : 0.f;
                    if (has_post) {
                        float p[E];
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            dw1[e] += db[e] * xh1[e];
                            db1[e] += db[e];
                            db[e] *= param(kW1, e);
                            p[e] = db[e] * xh1[e];
                        }
                        if (layer1) s[0] = at.own(db);
                        s[1] = at.own(p);
                    }
                    if (has_post || token_sum) row_sum.sum(s);
                    if (has_post) {
                        const float m0 = s[0] * inv_dim, m1 = s[1] * inv_dim;
#pragma unroll
                        for (int e = 0; e < E; ++e) db[e] = rstd1 * (db[e] - m0 - xh1[e] * m1);
                    }
                    Run<TY, E> o;
                    o.from(db);
                    o.store(row_address(pdy, row, a.dim * (uint32_t)sizeof(TY)));
                    if constexpr (GATED) {
                        if (token_sum) {
                            store_any(a.dgate, row, a.gate_dtype, s[2]);
                        } else {
                            const int64_t to = (int64_t)row * a.dim + c;
                            if (a.gate_dtype == P3D_F32) {
                                Run<float, E> o;
                                o.from(dg);
                                o.store(reinterpret_cast<float*>(a.dgate) + to);
                            } else if (a.gate_dtype == P3D_F16) {
                                Run<_Float16, E> o;
                                o.from(dg);
                                o.store(reinterpret_cast<_Float16*>(a.dgate) + to);
                            } else {
                                Run<__bf16, E> o;
                                o.from(dg);
                                o.store(reinterpret_cast<__bf16*>(a.dgate) + to);
                            }
                        }
                    }
                }
            }
        }
        if constexpr (HAS_Y) {
            // gate keep b go over the unit's rows gives dscale times (1 - p), the gate
            // of a sample still to be multiplied in, and its gradient, the scale likewise.
            float gs[E], sc[E];
            load_param(per_sample ? a.gate : nullptr, a.gate_dtype, gate_at, 1.f, gs);
#pragma unroll
            for (int e = 0; e < E; ++e) dsc[e] += gs[e] * unit_acc[e];
            if (a.dgate_part) {
                load_param(a.scale, a.param, c, 1.f, sc);
#pragma unroll
                for (int e = 0; e < E; ++e) unit_acc[e] *= sc[e] * mask.inv;
                gather(unit_acc, a.dgate_part + (int64_t)u * a.dim);
            }
        }
    }
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 5 * a.dim;
    if constexpr (HAS_Y) {
        if (a.post.weight) gather(dw1, part);
        if (a.post.bias) gather(db1, part + a.dim);
        if (a.scale) {
#pragma unroll
            for (int e = 0; e < E; ++e) dsc[e] *= mask.inv;
            gather(dsc, part + 2 * a.dim);
        }
    }
    if (NEXT && a.next.weight) gather(dw2, part + 3 * (int64_t)a.dim);
    if (NEXT && a.next.bias) gather(db2, part + 4 * (int64_t)a.dim);
}

// Launches a kernel, or counts the workgroups of it that the GPU runs at a time.
template <typename K>
int launch_kernel(K kernel, int threads, const BlockDev& a, const BlockLaunch& l, const char* what) {
    if (l.resident) return resident_workgroups(reinterpret_cast<const void*>(kernel), threads, l.resident);
    kernel<<<l.grid, threads, 0, l.stream>>>(a);
    return check_launch(what);
}

template <typename TX, typename TY, int TPR, int E, int FORM>
int launch_form(const BlockDev& a, const BlockLaunch& l) {
    constexpr int threads = block_threads(TPR);
    if (!l.backward) return launch_kernel(k_block_fwd<TX, TY, TPR, E, FORM>, threads, a, l, "p3d_block_fwd");
    if (FORM == kNorm || a.dn)
        return launch_kernel(k_block_bwd<TX, TY, TPR, E, FORM, true>, threads, a, l, "p3d_block_bwd");
    return launch_kernel(k_block_bwd<TX, TY, TPR, E, FORM, FORM == kNorm>, threads, a, l, "p3d_block_bwd");
}

template <typename TX, typename TY, int TPR, int E>
int launch_as(const BlockDev& a, const BlockLaunch& l) {
    if (!a.y) return launch_form<TX, TY, TPR, E, kNorm>(a, l);
    if (a.gate_kind == P3D_GATE_TOKEN || a.gate_kind == P3D_GATE_FULL)
        return launch_form<TX, TY, TPR, E, kEndGated>(a, l);
    return launch_form<TX, TY, TPR, E, kEnd>(a, l);
}

}  // namespace

// Threads of a row and channels a thread: eight channels (16 bytes of a 16-bit type)
// over the fewest threads, a power of two, that cover the row; six where those cover it
// too (160 channels: 27 lanes of 32 hold six, 20 hold eight; 200,000 rows forward and
// backward 160 against 169 us).  Rows of 3, 5 or 7 waves fill fewer of a CU's wave slots:
// 25,000 rows of 1,280 took 215 us in three waves, 170 in four of which two have no
// channels.  block_split in binding/torch_ops.cpp deals out rows by the same widths.
template <typename TX, typename TY>
int launch_block(const BlockDev& a, const BlockLaunch& l) {
    const int d = a.dim;
    if (d < 4) return launch_as<TX, TY, 4, 1>(a, l);
    if (d < 8) return launch_as<TX, TY, 2, 4>(a, l);
    if (d <= 16) return launch_as<TX, TY, 2, 8>(a, l);
    if (d <= 32) return launch_as<TX, TY, 4, 8>(a, l);
    if (d <= 64) return launch_as<TX, TY, 8, 8>(a, l);
    if (d <= 96) return launch_as<TX, TY, 16, 6>(a, l);
    if (d <= 128) return launch_as<TX, TY, 16, 8>(a, l);
    if (d <= 192) return launch_as<TX, TY, 32, 6>(a, l);
    if (d <= 256) return launch_as<TX, TY, 32, 8>(a, l);
    if (d <= 384) return launch_as<TX, TY, 64, 6>(a, l);
    if (d <= 512) return launch_as<TX, TY, 64, 8>(a, l);
    if (d <= 128 * 6) return launch_as<TX, TY, 128, 6>(a, l);
    if (d <= 128 * 8) return launch_as<TX, TY, 128, 8>(a, l);
    if (d <= 256 * 6) return launch_as<TX, TY, 256, 6>(a, l);
    if (d <= 256 * 8) return launch_as<TX, TY, 256, 8>(a, l);
    if (d <= 512 * 6) return launch_as<TX, TY, 512, 6>(a, l);
    if (d <= 512 * 8) return launch_as<TX, TY, 512, 8>(a, l);
    if (d <= 1024 * 6) return launch_as<TX, TY, 1024, 6>(a, l);
    return launch_as<TX, TY, 1024, 8>(a, l);
}

}  // namespace p3d
