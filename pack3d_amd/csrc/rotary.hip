// Rotary positions of up to four tensors of heads in one launch.
//
// Pair j of a token at position p on the pair's axis turns by theta = p f_j: (a, b)
// -> m (a cos - b sin, a sin + b cos); channels 2j and 2j + 1 (interleaved) or j and
// P + j (half) for j < P, the channels from 2P on are copied.  The gradient turns
// back by -theta.  theta goes through 64 bits: in 32 the angle of position 10^6 is
// off by 0.03 radians.  It is formed in turns, p (f / 2 pi), and only its
// distance from the nearest whole turn is rounded to 32 bits, an error of at most
// 2^-26 turns.
//
// A block takes a run of tokens: first (cos, sin) of each of their pairs into LDS,
// once for all heads of all tensors, then the heads, 8 pairs (32 bytes of a 16-bit
// type) a thread and step.  Bound by memory: 4 bytes an element in 16 bits.
#include "elements.hpp"

namespace p3d {
namespace {

constexpr int kPiece = 8;
constexpr int kThreads = 256;
constexpr int kMaxTensors = 4;
constexpr int kMaxTable = 4096;  // (cos, sin) of a block: 32 KiB

struct RotaryDev {
    p3d_view x[kMaxTensors], y[kMaxTensors];
    uint32_t items[kMaxTensors];        // heads * chunks of a token
    uint32_t items_inv[kMaxTensors];    // ceil(2^32 / items)
    int count;
    int64_t tokens, tiles;              // tiles of a batch entry
    int run;                            // tokens of a tile
    int head_dim, pairs, chunks, turned;  // chunks of a head, of which `turned` hold pairs
    uint32_t chunks_inv;
    const void* positions;
    int64_t pb, pn, pa;                 // strides of the positions
    int pos64, axes, end0, end1;        // pairs below end0 are on axis 0, below end1 on axis 1
    const double* freqs;
    int half;
    float sign, magnitude;
};

// v = the first `count` of eight elements at p, zero past them.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int count, float (&v)[kPiece]) {
    if (count >= kPiece) {
        Run<T, kPiece> r;
        r.load(p);
        r.to(v);
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e) v[e] = e < count ? to_f32(p[e]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int count, const float (&v)[kPiece]) {
    if (count >= kPiece) {
        Run<T, kPiece> r;
        r.from(v);
        r.store(p);
    } else {
#pragma unroll
        for (int e = 0; e < kPiece; ++e)
            if (e < count) p[e] = from_f32<T>(v[e]);
    }
}

// a / d for a < 2^32 / d, with inv = ceil(2^32 / d); d = 1 has inv = 0.
__device__ __forceinline__ uint32_t quotient(uint32_t a, uint32_t inv) { return inv ? __umulhi(a, inv) : a; }

template <typename T>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryDev a) {
    __shared__ float2 table[kMaxTable];
    const int64_t b = blockIdx.x / a.tiles, first = (blockIdx.x - b * a.tiles) * a.run;
    const int live = (int)min((int64_t)a.run, a.tokens - first);
    for (int i = threadIdx.x; i < live * a.pairs; i += kThreads) {
        const int t = i / a.pairs, j = i - t * a.pairs;
        const int axis = j < a.end0 ? 0 : (j < a.end1 ? 1 : 2);
        const int64_t at = b * a.pb + (first + t) * a.pn + axis * a.pa;
        const int64_t pos = a.pos64 ? reinterpret_cast<const int64_t*>(a.positions)[at]
                                    : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[at];
        const double turns = (double)pos * (a.freqs[j] * 0.15915494309189533577);  // 1 / (2 pi)
        const float r = (float)(turns - rint(turns));
        float s, c;
        sincospif(2.f * r, &s, &c);
        table[i] = float2{c * a.magnitude, s * a.magnitude * a.sign};
    }
    __syncthreads();
    for (int k = 0; k < a.count; ++k) {
        const uint32_t items = a.items[k], all = (uint32_t)live * items;
        const T* xb = reinterpret_cast<const T*>(a.x[k].data) + b * a.x[k].sb;
        T* yb = reinterpret_cast<T*>(a.y[k].data) + b * a.y[k].sb;
        for (uint32_t i = threadIdx.x; i < all; i += kThreads) {
            const uint32_t t = quotient(i, a.items_inv[k]), r = i - t * items;
            const uint32_t h = quotient(r, a.chunks_inv), c = r - h * a.chunks;
            const T* xr = xb + (int64_t)h * a.x[k].sh + (first + t) * a.x[k].sn;
            T* yr = yb + (int64_t)h * a.y[k].sh + (first + t) * a.y[k].sn;
            if ((int)c >= a.turned) {
                const int at = 2 * a.pairs + ((int)c - a.turned) * kPiece, n = min(kPiece, a.head_dim - at);
                float v[kPiece];
                load8(xr + at, n, v);
                store8(yr + at, n, v);
                continue;
            }
            const int j = (int)c * kPiece, n = min(kPiece, a.pairs - j);
            const float2* cs = table + t * a.pairs + j;
            float u[kPiece], v[kPiece];
            if (a.half) {
                load8(xr + j, n, u);
                load8(xr + a.pairs + j, n, v);
#pragma unroll
                for (int e = 0; e < kPiece; ++e) {
                    const float2 w = cs[e < n ? e : 0];
                    const float p = u[e] * w.x - v[e] * w.y, q = u[e] * w.y + v[e] * w.x;
                    u[e] = p;
                    v[e] = q;
                }
                store8(yr + j, n, u);
                store8(yr + a.pairs + j, n, v);
            } else {
                load8(xr + 2 * j, min(2 * n, kPiece), u);
                load8(xr + 2 * j + kPiece, 2 * n - kPiece, v);
#pragma unroll
                for (int e = 0; e < kPiece / 2; ++e) {
                    const float2 w = cs[e < n ? e : 0], z = cs[e + kPiece / 2 < n ? e + kPiece / 2 : 0];
                    const float p = u[2 * e] * w.x - u[2 * e + 1] * w.y, q = u[2 * e] * w.y + u[2 * e + 1] * w.x;
                    const float f = v[2 * e] * z.x - v[2 * e + 1] * z.y, g = v[2 * e] * z.y + v[2 * e + 1] * z.x;
                    u[2 * e] = p;
                    u[2 * e + 1] = q;
                    v[2 * e] = f;
                    v[2 * e + 1] = g;
                }
                store8(yr + 2 * j, min(2 * n, kPiece), u);
                store8(yr + 2 * j + kPiece, 2 * n - kPiece, v);
            }
        }
    }
}

inline uint32_t inverse_of(uint32_t d) { return d == 1 ? 0 : (uint32_t)(((1ULL << 32) + d - 1) / d); }

}  // namespace
}  // namespace p3d

using namespace p3d;

extern "C" int p3d_rotary(const p3d_rotary_args* args, void* stream) {
    P3D_REQUIRE(args, "null args");
    const p3d_rotary_args& g = *args;
    P3D_REQUIRE(g.count >= 1 && g.count <= kMaxTensors, "need 1 to 4 tensors");
    P3D_REQUIRE(g.dtype >= P3D_F32 && g.dtype <= P3D_BF16, "unknown dtype");
    P3D_REQUIRE(g.batch >= 1 && g.tokens >= 1 && g.head_dim >= 2 && g.head_dim <= 1024, "bad sizes");
    P3D_REQUIRE(g.pairs >= 1 && 2 * g.pairs <= g.head_dim, "pairs must be 1 to head_dim / 2");
    P3D_REQUIRE(g.positions && g.freqs, "null pointer argument");
    P3D_REQUIRE(g.axes >= 1 && g.axes <= 3, "need 1 to 3 axes");
    const int axes = g.axes;
    int sum = 0;
    for (int i = 0; i < axes; ++i) {
        P3D_REQUIRE(g.axis_pairs[i] >= 0, "axis pairs must not be negative");
        sum += g.axis_pairs[i];
    }
    P3D_REQUIRE(sum == g.pairs, "axis pairs must add up to pairs");
    RotaryDev a{};
    a.count = g.count;
    a.tokens = g.tokens;
    a.head_dim = g.head_dim;
    a.pairs = g.pairs;
    a.turned = (int)cdiv(g.pairs, kPiece);
    a.chunks = a.turned + (int)cdiv(g.head_dim - 2 * g.pairs, kPiece);
    a.chunks_inv = inverse_of(a.chunks);
    uint32_t per_token = 0;
    for (int k = 0; k < g.count; ++k) {
        P3D_REQUIRE(g.x[k].data && g.y[k].data && g.heads[k] >= 1, "null tensor or no heads");
        P3D_REQUIRE((int64_t)g.heads[k] * a.chunks <= 8192, "heads * head_dim too large");
        a.x[k] = g.x[k];
        a.y[k] = g.y[k];
        a.items[k] = (uint32_t)(g.heads[k] * a.chunks);
        a.items_inv[k] = inverse_of(a.items[k]);
        per_token += a.items[k];
    }
    a.positions = g.positions;
    a.pb = g.pos_sb;
    a.pn = g.pos_sn;
    a.pa = g.pos_sa;
    a.pos64 = g.pos_is64;
    a.axes = axes;
    a.end0 = axes > 1 ? g.axis_pairs[0] : g.pairs;
    a.end1 = axes > 2 ? g.axis_pairs[0] + g.axis_pairs[1] : g.pairs;
    a.freqs = g.freqs;
    a.half = g.half;
    a.sign = g.inverse ? -1.f : 1.f;
    a.magnitude = g.magnitude;
    // Tokens of a block: about four steps of its threads, within the table, and
    // fewer where that leaves CUs without a block.
    int64_t run = cdiv(4 * kThreads, per_token);
    run = run < kMaxTable / g.pairs ? run : kMaxTable / g.pairs;
    while (run > 1 && g.batch * cdiv(g.tokens, run) < 512) run = (run + 1) / 2;
    a.run = (int)run;
    a.tiles = cdiv(g.tokens, run);
    P3D_REQUIRE(g.batch * a.tiles < (1LL << 31), "launch grid too large");
    const unsigned blocks = (unsigned)(g.batch * a.tiles);
    hipStream_t s = as_stream(stream);
    switch (g.dtype) {
        case P3D_F32: k_rotary<float><<<blocks, kThreads, 0, s>>>(a); break;
        case P3D_F16: k_rotary<_Float16><<<blocks, kThreads, 0, s>>>(a); break;
        default: k_rotary<__bf16><<<blocks, kThreads, 0, s>>>(a); break;
    }
    return check_launch("p3d_rotary");
}
