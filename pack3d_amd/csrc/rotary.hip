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
// A block takes a run of tokens: (cos, sin) of each of their pairs into LDS, once for
// all heads of all tensors, then the heads, 32 bytes a thread and step, the first step's
// loads issued before the angles are worked out.  A block takes the tokens of one step a
// thread: more blocks with smaller tables measured faster than steps ahead within one
// (three bf16 tensors of 262,144 x 4 x 48: one step 124 us, two a thread 126, four 136,
// their loads together 140), and the angles cost nothing next to the memory (138 and 139
// us without and with them; these figures before 16-byte runs, the same tensors now take
// 120 us).  Bound by memory: 4 bytes an element in 16 bits, 5.1 TB/s.
#include "elements.hpp"

namespace p3d {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTensors = 4;
constexpr int kMaxTable = 4096;  // (cos, sin) of a block: 32 KiB

struct RotaryDev {
    p3d_view x[kMaxTensors], y[kMaxTensors];
    uint32_t steps[kMaxTensors];        // of a token
    uint32_t steps_inv[kMaxTensors];    // ceil(2^32 / steps)
    int count;
    int64_t tokens;
    uint32_t tiles;                     // of a batch entry
    int run;                            // tokens of a tile
    int head_dim, pairs;
    uint32_t chunks, turned, chunks_inv;  // steps of a head, of which `turned` hold pairs
    int copied;                         // first channel of the steps that copy
    const void* positions;
    int64_t pb, pn, pa;                 // strides of the positions
    int pos64, end0, end1;              // pairs below end0 are on axis 0, below end1 on axis 1
    const double* freqs;
    float sign, magnitude;
};

// a / d for a < 2^32 / d, with inv = ceil(2^32 / d); d = 1 has inv = 0.
__device__ __forceinline__ uint32_t quotient(uint32_t a, uint32_t inv) { return inv ? __umulhi(a, inv) : a; }

// One step: two runs of N channels, 16 bytes each: N pairs (apart by the pairs, or
// adjacent), or 2N channels that are copied.  Where N does not divide the pairs, or 2N the
// copied channels, the last two steps overlap and store the same bits twice.  Heads with
// fewer than N pairs have one step of them, which reads whole runs all the same: adjacent,
// it copies the channels behind the pairs too; apart, it stores what is the pairs' (30M
// bf16 channels in heads of 16 with 3 pairs: 26 and 58 us; whole heads 27).  Fewer than 2N
// copied channels: the step reads the head's last 2N and stores what is theirs.  Heads of
// fewer than 2N channels go an element at a time.
enum Form { kWhole, kFew, kSmall };  // N pairs or more; fewer; heads of fewer than 2N channels

template <typename T, bool HALF, int FORM>
struct Step {
    static constexpr int N = Piece<T>::N;
    static constexpr bool FEW = FORM == kFew, SMALL = FORM == kSmall;
    const char* src;
    char* dst;
    uint32_t at;  // of the (cos, sin) of its first pair
    int count;    // pairs, or minus the channels to copy
    int gap;      // bytes from the first run to the second
    Run<T, N> u, v;

    // k: the tensor, the same for the whole launch's step.
    __device__ __forceinline__ void place(const RotaryDev& a, int k, int64_t b, int64_t first, uint32_t i) {
        const uint32_t t = quotient(i, a.steps_inv[k]), r = i - t * a.steps[k];
        const uint32_t h = quotient(r, a.chunks_inv), c = r - h * a.chunks;
        const p3d_view &x = a.x[k], &y = a.y[k];
        const int P = a.pairs;
        int channel;
        if (c < a.turned) {
            const int j = SMALL ? (int)c * N : (FEW ? 0 : min((int)c * N, P - N));
            at = t * P + j;
            count = SMALL ? min(N, P - j) : (FEW ? P : N);
            channel = HALF ? j : 2 * j;
            gap = (HALF ? P : N) * (int)sizeof(T);
        } else {
            const int j = a.copied + (int)(c - a.turned) * 2 * N, left = a.head_dim - a.copied;
            at = 0;
            count = SMALL ? -min(2 * N, a.head_dim - j) : -min(2 * N, left);
            channel = SMALL ? j : min(j, a.head_dim - 2 * N);
            gap = N * (int)sizeof(T);
        }
        src = reinterpret_cast<const char*>(reinterpret_cast<const T*>(x.data) + b * x.sb + (int64_t)h * x.sh +
                                            (first + t) * x.sn + channel);
        dst = reinterpret_cast<char*>(reinterpret_cast<T*>(y.data) + b * y.sb + (int64_t)h * y.sh +
                                      (first + t) * y.sn + channel);
    }
    // Elements low to high - 1 of a run.
    __device__ __forceinline__ static void load_some(Run<T, N>& r, const char* p, int high) {
#pragma unroll
        for (int e = 0; e < N; ++e) r.v[e] = e < high ? reinterpret_cast<const T*>(p)[e] : from_f32<T>(0.f);
    }
    __device__ __forceinline__ static void store_some(const Run<T, N>& r, char* p, int low, int high) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e >= low && e < high) reinterpret_cast<T*>(p)[e] = r.v[e];
    }
    // Channels of the two runs together where they are adjacent, of each where apart.
    __device__ __forceinline__ int channels() const { return count < 0 ? -count : (HALF ? count : 2 * count); }
    __device__ __forceinline__ int second() const { return HALF && count > 0 ? count : channels() - N; }
    __device__ __forceinline__ void load(const RotaryDev& a) {
        if constexpr (SMALL) {
            load_some(u, src, channels());
            load_some(v, src + gap, second());
        } else {
            u.load(src);
            v.load(src + gap);
        }
    }
    __device__ __forceinline__ void turn(const RotaryDev& a, const float2* table) {
        if (count > 0) {
            float f[N], g[N];
            u.to(f);
            v.to(g);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const bool real = SMALL ? e < count : (!FEW || e < a.pairs);
                const float2 w = table[at + (real ? e : 0)];
                float& p = HALF ? f[e] : (e < N / 2 ? f[(2 * e) % N] : g[(2 * e) % N]);
                float& q = HALF ? g[e] : (e < N / 2 ? f[(2 * e + 1) % N] : g[(2 * e + 1) % N]);
                const float s = p * w.x - q * w.y, t = p * w.y + q * w.x;
                p = real ? s : p;
                q = real ? t : q;
            }
            u.from(f);
            v.from(g);
        }
        if constexpr (SMALL) {
            store_some(u, dst, 0, channels());
            store_some(v, dst + gap, 0, second());
        } else if (FEW && HALF && count > 0) {
            store_some(u, dst, 0, a.pairs);
            store_some(v, dst + gap, 0, a.pairs);
        } else if (count > 0 || count == -2 * N) {
            u.store(dst);
            v.store(dst + gap);
        } else {
            store_some(u, dst, 2 * N + count, N);
            store_some(v, dst + gap, N + count, N);
        }
    }
};

template <typename T, bool HALF, int FORM>
__global__ __launch_bounds__(kThreads) void k_rotary(RotaryDev a) {
    extern __shared__ float2 table[];  // [run][pairs]
    const uint32_t entry = blockIdx.x / a.tiles;
    const int64_t b = entry, first = (int64_t)(blockIdx.x - entry * a.tiles) * a.run;
    const int live = (int)min((int64_t)a.run, a.tokens - first);
    Step<T, HALF, FORM> s;
    auto fetch = [&](int k, uint32_t i, uint32_t all) {
        s.place(a, k, b, first, min(i, all - 1));  // past the end: the last step once more
        s.load(a);
    };
    fetch(0, threadIdx.x, (uint32_t)live * a.steps[0]);
    for (int i = threadIdx.x; i < live * a.pairs; i += kThreads) {
        const int t = i / a.pairs, j = i - t * a.pairs;
        const int axis = j < a.end0 ? 0 : (j < a.end1 ? 1 : 2);
        const int64_t at = b * a.pb + (first + t) * a.pn + axis * a.pa;
        const int64_t pos = a.pos64 ? reinterpret_cast<const int64_t*>(a.positions)[at]
                                    : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[at];
        const double turns = (double)pos * (a.freqs[j] * 0.15915494309189533577);  // 1 / (2 pi)
        const float r = (float)(turns - rint(turns));
        float sn, cs;
        sincospif(2.f * r, &sn, &cs);
        table[i] = float2{cs * a.magnitude, sn * a.magnitude * a.sign};
    }
    __syncthreads();
    for (int k = 0; k < a.count; ++k) {
        const uint32_t all = (uint32_t)live * a.steps[k];
        if (k) fetch(k, threadIdx.x, all);
        for (uint32_t i = threadIdx.x;;) {
            if (i < all) s.turn(a, table);
            i += kThreads;
            if (i >= all) break;
            fetch(k, i, all);
        }
    }
}

inline uint32_t inverse_of(uint32_t d) { return d == 1 ? 0 : (uint32_t)(((1ULL << 32) + d - 1) / d); }

template <typename T, bool HALF>
void launch(const RotaryDev& a, int form, unsigned blocks, hipStream_t s) {
    const size_t lds = (size_t)a.run * a.pairs * sizeof(float2);
    switch (form) {
        case kWhole: k_rotary<T, HALF, kWhole><<<blocks, kThreads, lds, s>>>(a); break;
        case kFew: k_rotary<T, HALF, kFew><<<blocks, kThreads, lds, s>>>(a); break;
        default: k_rotary<T, HALF, kSmall><<<blocks, kThreads, lds, s>>>(a); break;
    }
}

template <typename T>
void launch(const RotaryDev& a, bool half, int form, unsigned blocks, hipStream_t s) {
    if (half) launch<T, true>(a, form, blocks, s);
    else launch<T, false>(a, form, blocks, s);
}

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
        P3D_REQUIRE(g.axis_pairs[i] >= 0 && g.axis_pairs[i] <= g.pairs, "axis pairs must add up to pairs");
        sum += g.axis_pairs[i];
    }
    P3D_REQUIRE(sum == g.pairs, "axis pairs must add up to pairs");
    RotaryDev a{};
    a.tokens = g.tokens;
    a.head_dim = g.head_dim;
    a.pairs = g.pairs;
    const int piece = 16 / dtype_size(g.dtype);
    a.turned = (uint32_t)cdiv(g.pairs, piece);
    const int form = g.head_dim < 2 * piece ? kSmall : (g.pairs < piece ? kFew : kWhole);
    a.copied = form == kFew && !g.half ? 2 * piece : 2 * g.pairs;
    a.chunks = a.turned + (uint32_t)cdiv(g.head_dim - a.copied, 2 * piece);
    a.chunks_inv = inverse_of(a.chunks);
    a.count = g.count;
    uint32_t most = 0;
    for (int k = 0; k < g.count; ++k) {
        P3D_REQUIRE(g.x[k].data && g.y[k].data && g.heads[k] >= 1, "null tensor or no heads");
        P3D_REQUIRE((int64_t)g.heads[k] * a.chunks <= 8192, "heads * head_dim too large");
        a.x[k] = g.x[k];
        a.y[k] = g.y[k];
        a.steps[k] = (uint32_t)g.heads[k] * a.chunks;
        a.steps_inv[k] = inverse_of(a.steps[k]);
        most = most > a.steps[k] ? most : a.steps[k];
    }
    a.positions = g.positions;
    a.pb = g.pos_sb;
    a.pn = g.pos_sn;
    a.pa = g.pos_sa;
    a.pos64 = g.pos_is64;
    a.end0 = axes > 1 ? g.axis_pairs[0] : g.pairs;
    a.end1 = axes > 2 ? g.axis_pairs[0] + g.axis_pairs[1] : g.pairs;
    a.freqs = g.freqs;
    a.sign = g.inverse ? -1.f : 1.f;
    a.magnitude = g.magnitude;
    // Tokens of a block: a step a thread of the tensor with most heads, within the table,
    // and fewer where that leaves CUs without a block.
    int64_t run = kThreads / most;
    run = run < 1 ? 1 : run;
    run = run < kMaxTable / g.pairs ? run : kMaxTable / g.pairs;
    while (run > 1 && g.batch * cdiv(g.tokens, run) < 512) run = (run + 1) / 2;
    a.run = (int)run;
    P3D_REQUIRE(g.batch * cdiv(g.tokens, run) < (1LL << 31), "launch grid too large");
    a.tiles = (uint32_t)cdiv(g.tokens, run);
    const unsigned blocks = (unsigned)g.batch * a.tiles;
    hipStream_t s = as_stream(stream);
    switch (g.dtype) {
        case P3D_F32: launch<float>(a, g.half, form, blocks, s); break;
        case P3D_F16: launch<_Float16>(a, g.half, form, blocks, s); break;
        default: launch<__bf16>(a, g.half, form, blocks, s); break;
    }
    return check_launch("p3d_rotary");
}
