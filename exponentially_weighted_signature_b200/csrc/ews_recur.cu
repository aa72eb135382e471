// Gated linear recurrence over a sequence, channel by channel, with its gradients and the single-token form.
//
//     r = sigmoid(decay),  a = exp(-rate r),  m = sqrt(1 - a^2),  i = sigmoid(gate)
//     h_t = a_t h_{t-1} + m_t i_t x_t
//     g_t = dh_t + a_{t+1} g_{t+1}
//     dx = g m i,  dgate = g m x i (1 - i),  dl = g (a h_{t-1} - (a^2 / m) i x)   (l = log a)
//     ddecay = -rate r (1 - r) dl,  drate = -sum r dl,  dh_0 = a_1 g_1
//
// (the flow exp(-dtheta lambda) of a diagonal generator at depth one with a clock step of each token and channel, and
// the input scaled so that unit inputs give a unit state.)
//
// Both directions are a scan of maps h -> A h + H. A tile is 64 tokens (or 32: see Back) by 32 V channels (128 bytes a token);
// its warps take 8 or 16 consecutive tokens each, with a and b of them in registers, so that the streams are read once. The
// warps' maps are joined in shared memory, the tiles' by a decoupled look-back in ticket order (a tile publishes its map, then
// its state): a tile folds the maps of up to as many tiles as it has warps onto a published state, always from the state
// upwards, so that the sum has one order and the results do not depend on timing. The backward reads no states: the forward
// leaves one for each of its tiles (float32), from which the tile runs the recurrence again. So the gradient of the rates, a
// float32 sum over all tokens, does not see the rounding of the stored states, and a stream less is read.
//
// Measured, 8 x 2,048 tokens of 2,048 channels: bfloat16 77 us forwards (four streams, 3.5 TB/s) and 137 back (seven, 3.4),
// float32 108 and 175 us (5.0 and 5.4 TB/s); with rates up to 4, so that decays take the exponent unit, 83 and 147 us, and 106 and 177.
// bfloat16 is bound by latency, no unit is saturated: four warps a scheduler (128 registers)
// issue in 46 % of the cycles forwards and 54 % back, the exponent unit works in 49 and 32 %, DRAM at a third of its rate, and a warp waits
// for the tile's barriers, for what it loads and for its own arithmetic about as long each. (Of an earlier build: without the gates'
// arithmetic 60 and 134 us, without the look-back too 56 and 116.) One sample of 17,984 tokens: 112 and 187 us; an earlier build's 111
// and 181 were 79 and 146 without the look-back: 32 chains of tiles, 18 of each in work at a time, wait for one another's maps
// and states (folding 12 or 16 tiles at once instead of 4 changed nothing).
#include <float.h>

#include <type_traits>

#include "ews_tc.cuh"

namespace ews {
namespace recur {

using namespace token;
using tc5::add2;
using tc5::fma2;
using tc5::mul2;
using tc5::pair;
using tc5::unpair;

constexpr int SMS = 148;
constexpr int TILE = 64;                           // tokens a tile
// Tokens a warp, warps a tile and CTAs an SM, of V channels a lane: what the registers of a token's values allow. (333 channels
// of float32, 16 x 1,440 tokens: 8 tokens a warp took 44 and 93 us forwards and back, 16 take 40 and 69.)
template <int V>
struct Shape {
    static constexpr int FL = V == 1 ? 16 : 8, FW = TILE / FL, FCTAS = V == 1 ? 8 : 3;  // forward
    static constexpr int BL = V == 1 ? 16 : 8, BW = TILE / BL, BCTAS = V == 1 ? 4 : 2;  // backward
};
constexpr int PL = 16, PW = TILE / PL, PCTAS = 4;  // the same where TMA brings the tiles
// And backwards, in tiles of ROWS tokens: TILE or, of bfloat16 where the chains (of 64 channels a sample) fill the GPU, HALF. Then
// more tiles are in work and fewer threads wait at a barrier; a chain of few passes through twice as many states. Tiles of 64
// tokens and of 32, 2,048 channels, us: 256 chains x 2,048 tokens 140 and 132, 160 x 2,048 99 and 93, 128 x 4,096 144 and 147,
// 64 x 8,192 151 and 163, 32 x 16,384 167 and 192. One tile is better than two: 8,192 chains x 40 tokens 121 and 126.
// (float32 has a token's 32 channels a tile, and enough tiles: 8 x 2,048 x 1,024 95 and 105. All before the choices of `open`, which added
// two or three to either.)
template <int V, int ROWS>
struct Back {
    static constexpr int QL = V == 1 ? 16 : 8, QW = ROWS / QL, QCTAS = V == 1 ? 3 : ROWS == TILE ? 2 : 4;
};
constexpr int HALF = TILE / 2;
constexpr int PSTAGES = 2, QSTAGES = 2;
constexpr int kPipedFrom = 33;            // steps from which it does: below, most of a tile would be empty
constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
struct Stream {
    const T* p;
    long sb, st;
};

template <typename T>
struct Params {
    int batch, steps, channels;
    int tiles, blocks;  // along the steps and the channels
    long total;         // tiles in all
    Stream<T> x, decay, gate, dout;
    const float* rate;
    const int* lengths;
    const float *initial, *dfinal;
    T* out;
    float* final_state;
    float* carry;  // (batch, carries, channels): the state in front of every `apart` tokens, for the backward
    int carries, apart;
    T *dx, *ddecay, *dgate;
    float *drate_part, *dinitial;
    // look-back
    DeviceStatus* st;
    uint2* slots;  // (batch, tiles, 2, channels): a value and what it is, see publish
    int* status;
};

// V floats, as one packed operand where there are two: the kernels are bound by their instructions, and one handles a pair.
template <int V>
struct F;
template <>
struct F<1> {
    float r;
    __device__ __forceinline__ F() {}
    __device__ __forceinline__ F(float x) : r(x) {}
    __device__ __forceinline__ float get(int) const { return r; }
    template <typename Fn>
    __device__ __forceinline__ F each(Fn f) const { return F(f(r)); }
    template <typename Fn>
    __device__ __forceinline__ static F make(Fn f) { return F(f(0)); }
};
template <>
struct F<2> {
    uint64_t r;
    __device__ __forceinline__ F() {}
    __device__ __forceinline__ F(float x) : r(pair(x, x)) {}
    __device__ __forceinline__ F(float x, float y) : r(pair(x, y)) {}
    __device__ __forceinline__ float get(int j) const {
        float x, y;
        unpair(r, x, y);
        return j ? y : x;
    }
    template <typename Fn>
    __device__ __forceinline__ F each(Fn f) const { return F(f(get(0)), f(get(1))); }
    template <typename Fn>
    __device__ __forceinline__ static F make(Fn f) { return F(f(0), f(1)); }
};
// rounded as the packed ones are
__device__ __forceinline__ F<1> operator*(F<1> a, F<1> b) { return F<1>(__fmul_rn(a.r, b.r)); }
__device__ __forceinline__ F<1> operator+(F<1> a, F<1> b) { return F<1>(__fadd_rn(a.r, b.r)); }
__device__ __forceinline__ F<1> fma(F<1> a, F<1> b, F<1> c) { return F<1>(fmaf(a.r, b.r, c.r)); }
__device__ __forceinline__ F<2> operator*(F<2> a, F<2> b) {
    F<2> o;
    o.r = mul2(a.r, b.r);
    return o;
}
__device__ __forceinline__ F<2> operator+(F<2> a, F<2> b) {
    F<2> o;
    o.r = add2(a.r, b.r);
    return o;
}
__device__ __forceinline__ F<2> fma(F<2> a, F<2> b, F<2> c) {
    F<2> o;
    o.r = fma2(a.r, b.r, c.r);
    return o;
}

// V elements of a stream.
template <typename T, int V>
struct Word;
template <>
struct Word<float, 1> {
    float w;
    __device__ __forceinline__ void load(const float* p) { w = __ldg(p); }
    __device__ __forceinline__ void fill(float x) { w = x; }
    __device__ __forceinline__ F<1> get() const { return F<1>(w); }
    __device__ __forceinline__ void put(F<1> v) { w = v.r; }
    __device__ static __forceinline__ void store(float* p, F<1> v) { *p = v.r; }
};
template <>
struct Word<bf16, 1> {
    bf16 w;
    __device__ __forceinline__ void load(const bf16* p) { w = __ldg(p); }
    __device__ __forceinline__ void fill(float x) { w = __float2bfloat16_rn(x); }
    __device__ __forceinline__ F<1> get() const { return F<1>(__bfloat162float(w)); }
    __device__ static __forceinline__ void store(bf16* p, F<1> v) { *p = __float2bfloat16_rn(v.r); }
};
template <>
struct Word<bf16, 2> {
    uint32_t w;
    __device__ __forceinline__ void load(const bf16* p) { w = __ldg(reinterpret_cast<const uint32_t*>(p)); }
    __device__ __forceinline__ void fill(float x) { w = pack_bf16(x, x); }
    __device__ __forceinline__ F<2> get() const { return F<2>(bf16_lo(w), bf16_hi(w)); }
    __device__ __forceinline__ void put(F<2> v) { w = pack_bf16(v.get(0), v.get(1)); }
    __device__ static __forceinline__ void store(bf16* p, F<2> v) { *reinterpret_cast<uint32_t*>(p) = pack_bf16(v.get(0), v.get(1)); }
};

// The exponent unit's own instructions; what lies below the normal range counts as zero (a sigmoid of less than -87, say),
// which spares their corrections, a third of the kernels' instructions. A sigmoid's exponent is rounded before it: 2^-24 of |x| log2(e) comes
// to 1e-6 of a sigmoid at x = -20 and 5e-6 at -87, in float32 too, where the states' own roundings are of that size over some ten tokens.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float root(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float inverse_root(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int V>
__device__ __forceinline__ F<V> sigmoid(F<V> x) {
    const F<V> e = (x * F<V>(-kLog2e)).each([](float t) { return ex2(t); });
    return (e + F<V>(1.f)).each([](float t) { return rcp(t); });
}

// a = exp(-p) and w = 1 - a^2, by way of q = 1 - a, whose series has no cancellation: a = 1 - q then has no error but its rounding,
// where the exponent unit's 2^-22 would add up over the hundreds of tokens that an a near one remembers, and w = q (2 - q).
// The series to the sixth power up to 0.175 (the first dropped term is 2^-27 of q there).
constexpr float kSeries = 0.175f;
template <int V>
__device__ __forceinline__ F<V> decay_loss(F<V> p) {
    F<V> q = fma(p, F<V>(-1.f / 720.f), F<V>(1.f / 120.f));
    q = fma(p, q, F<V>(-1.f / 24.f));
    q = fma(p, q, F<V>(1.f / 6.f));
    q = fma(p, q, F<V>(-0.5f));
    return fma(p * p, q, p);
}
// What a token keeps of its decay, and a and w of it. NEAR, where no rate of the warp exceeds 1.4, and with it no p: q, from the
// series at p / 8 and 1 - exp(-2 t) = q (2 - q) three times over, without the exponent unit, whose 16 results a clock bound the
// bfloat16 kernels. Else a: 1 - q up to 0.175, exp(-p) beyond, where a state forgets within some six tokens.
constexpr float kNear = 8.f * kSeries;
template <bool NEAR, int V>
struct Decay {
    F<V> k;
    __device__ __forceinline__ Decay() {}
    __device__ __forceinline__ explicit Decay(F<V> p) {
        if constexpr (NEAR) {
            k = decay_loss(p * F<V>(0.125f));
#pragma unroll
            for (int i = 0; i < 3; ++i) k = fma(k * F<V>(-1.f), k, k + k);
        } else {
            const F<V> near = fma(decay_loss(p), F<V>(-1.f), F<V>(1.f));
            const F<V> e = (p * F<V>(-kLog2e)).each([](float t) { return ex2(t); });
            k = F<V>::make([&](int j) { return p.get(j) < kSeries ? near.get(j) : e.get(j); });
        }
    }
    __device__ __forceinline__ static Decay of(F<V> kept) {
        Decay d;
        d.k = kept;
        return d;
    }
    __device__ __forceinline__ F<V> a() const { return NEAR ? fma(k, F<V>(-1.f), F<V>(1.f)) : k; }
    __device__ __forceinline__ F<V> w(F<V> p) const {
        if constexpr (NEAR) return fma(k, a(), k);
        const F<V> q = decay_loss(p), near = fma(q, fma(q, F<V>(-1.f), F<V>(1.f)), q);
        return F<V>::make([&](int j) { return p.get(j) < kSeries ? near.get(j) : fmaf(-k.get(j), k.get(j), 1.f); });
    }
};
template <int V>
__device__ __forceinline__ bool is_near(F<V> rate) {
    bool near = true;
#pragma unroll
    for (int j = 0; j < V; ++j) near = near && rate.get(j) <= kNear;
    return __all_sync(kFull, near);
}
// v where the clock moves (w = 1 - a^2 in the normal range, or NaN), zero where it does not: such a token takes no input, and may hold
// anything, which a product with the zero root would let through. (Forwards the choices cost nothing, backwards 134 -> 137 us for
// 8 x 2,048 tokens of 2,048 channels. Looking for NaN in a warp's sums, and forming them once more where there is one, took registers from
// both ways: 77 -> 95 us forwards.)
template <int V>
__device__ __forceinline__ F<V> open(F<V> w, F<V> v) {
    return F<V>::make([&](int j) { return fabsf(w.get(j)) < FLT_MIN ? 0.f : v.get(j); });
}
// What a token brings into the state.
template <int V>
__device__ __forceinline__ F<V> input(F<V> w, F<V> i, F<V> x) {
    return open(w, w.each([](float t) { return root(t); }) * i * x);
}

// A channel's rate; an infinite one as float32's largest, so that a shut gate's product with it is zero.
__device__ __forceinline__ float rate_at(const float* p) {
    const float r = __ldg(p);
    return r > FLT_MAX ? FLT_MAX : r;
}

struct Tile {
    int b, tt, c0;  // sample, tile along the steps, first channel
};

// Tiles are given out by the steps first, so that a tile only waits on lower tickets.
template <typename T>
__device__ __forceinline__ Tile tile_of(const Params<T>& a, int ticket, bool down, int width) {
    const unsigned per = (unsigned)(a.batch * a.blocks);
    Tile t;
    t.tt = (int)((unsigned)ticket / per);
    const unsigned rest = (unsigned)ticket - t.tt * per;
    if (down) t.tt = a.tiles - 1 - t.tt;
    t.b = (int)(rest / (unsigned)a.blocks);
    t.c0 = (int)(rest - t.b * (unsigned)a.blocks) * width;
    return t;
}

template <int V, int WARPS, bool BACK>
struct Shared {
    F<V> A[WARPS][32], H[WARPS][32], D[BACK ? WARPS : 1][32];  // the warps' maps of the tile
    F<V> before_a[WARPS][32], before_h[WARPS][32];             // the tiles' that a look-back folds
    unsigned kind[WARPS][32];
    F<V> sum[BACK ? 2 : 1][BACK ? WARPS : 1][32];  // the rate's gradient, of this tile and of the last
    int ticket;
};

// The maps of the warps in front of this one (h -> pa h + ph), and of those behind it. All are read at once, those that
// do not count as the identity: one after the other, each would wait for shared memory (a prompt of 17,984 tokens: 118 -> 111 us).
template <int V, int WARPS, bool BACK>
__device__ __forceinline__ void fold_front(const Shared<V, WARPS, BACK>& sh, int warp, int lane, F<V>* pa, F<V>* ph) {
    F<V> A[WARPS], H[WARPS];
#pragma unroll
    for (int w = 0; w < WARPS - 1; ++w) {
        A[w] = F<V>(1.f), H[w] = F<V>(0.f);
        if (w < warp) A[w] = sh.A[w][lane], H[w] = sh.H[w][lane];
    }
    F<V> a(1.f), h(0.f);
#pragma unroll
    for (int w = 0; w < WARPS - 1; ++w) a = a * A[w], h = fma(A[w], h, H[w]);
    *pa = a, *ph = h;
}
template <int V, int WARPS, bool BACK>
__device__ __forceinline__ void fold_behind(const Shared<V, WARPS, BACK>& sh, int warp, int lane, F<V>* pa, F<V>* pd) {
    F<V> A[WARPS], D[WARPS];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
        A[w] = F<V>(1.f), D[w] = F<V>(0.f);
        if (w > warp) A[w] = sh.A[w][lane], D[w] = sh.D[w][lane];
    }
    F<V> a(1.f), d(0.f);
#pragma unroll
    for (int w = WARPS - 1; w > 0; --w) a = a * A[w], d = fma(A[w], d, D[w]);
    *pa = a, *pd = d;
}

// V consecutive floats of the lane's channels; what lies beyond the last is not touched.
template <int V>
__device__ __forceinline__ F<V> load_channels(const float* p, int c, int channels) {
    return F<V>::make([&](int j) { return c + j < channels ? __ldcg(p + c + j) : 0.f; });
}
template <int V>
__device__ __forceinline__ void store_channels(float* p, int c, int channels, F<V> v) {
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (c + j < channels) __stcg(p + c + j, v.get(j));
}

// What a tile publishes is a value and its kind in one word of 64 bits, so that a reader needs no flag beside it and a writer no
// fence: a reader polls the values themselves (a flag with release and acquire took a hop from tile to tile from under one
// to some three microseconds). Two words a channel: A, and H until the state at the tile's end takes its place.
constexpr unsigned kMap = 1, kState = 2;

template <int V>
__device__ __forceinline__ void publish(uint2* p, F<V> v, unsigned kind) {
    if constexpr (V == 2)
        asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(p), "l"(((uint64_t)kind << 32) | __float_as_uint(v.get(0))),
                     "l"(((uint64_t)kind << 32) | __float_as_uint(v.get(1)))
                     : "memory");
    else
        asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(p), "l"(((uint64_t)kind << 32) | __float_as_uint(v.get(0))) : "memory");
}

// The words of the lane's channels once all are of at least the kind `want`; zero where the wait ran out.
template <int V>
__device__ __forceinline__ unsigned await(const uint2* p, unsigned want, DeviceStatus* st, F<V>* v) {
#pragma unroll 1
    for (int it = 0; it < kDefaultSpinLimit; ++it) {
        uint64_t x, y;
        if constexpr (V == 2) asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(x), "=l"(y) : "l"(p) : "memory");
        else asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(x) : "l"(p) : "memory");
        if constexpr (V == 1) y = x;
        const unsigned kind = (unsigned)(x >> 32);
        if (kind >= want && kind == (unsigned)(y >> 32)) {
            if constexpr (V == 2) *v = F<2>(__uint_as_float((unsigned)x), __uint_as_float((unsigned)y));
            else *v = F<1>(__uint_as_float((unsigned)x));
            return kind;
        }
        if (it > 16) __nanosleep(32);
        if ((it & 63) == 63 && *((volatile int*)&st->error) != 0) return 0;
    }
    atomicCAS(&st->error, 0, EWS_ERR_LOOKBACK_TIMEOUT);
    return 0;
}

template <typename T>
__device__ __forceinline__ uint2* slot_of(const Params<T>& a, const Tile& t, int tt, int c) {
    return a.slots + (((long)t.b * a.tiles + tt) * 2) * a.channels + c;
}

// The state that comes into the tile from the tiles before it (down: behind it). Every thread of the CTA calls it, after the
// tile's own map was published; false when a wait ran out. AT_ONCE: as fold_front, where there are registers for it.
template <bool AT_ONCE, typename T, int V, int WARPS, bool BACK>
__device__ __forceinline__ bool look_back(const Params<T>& a, const Tile& t, bool down, Shared<V, WARPS, BACK>& sh, int warp, int lane, int warps, F<V>* state) {
    const int before = down ? a.tiles - 1 - t.tt : t.tt;  // how many there are
    const int window = before < warps ? before : warps;
    bool ok = true;
    if (warp < window) {
        const int c = t.c0 + lane * V;
        const uint2* p = slot_of(a, t, down ? t.tt + 1 + warp : t.tt - 1 - warp, c);
        unsigned kind = kState;
        F<V> A(0.f), H(0.f);
        if (c < a.channels) {
            // the last of the window has to have its state: nothing further back is folded
            kind = await<V>(p + a.channels, warp == window - 1 ? kState : kMap, a.st, &H);
            ok = kind != 0 && (kind == kState || await<V>(p, kMap, a.st, &A) != 0);
        }
        sh.before_a[warp][lane] = A, sh.before_h[warp][lane] = H, sh.kind[warp][lane] = kind;
    }
    if (!__syncthreads_and(ok)) return false;
    // from the furthest state on; where a nearer tile has its own already, that is the same number
    F<V> h(0.f);
    if constexpr (AT_ONCE) {
        F<V> A[WARPS], H[WARPS];
        unsigned kind[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            kind[w] = kMap, A[w] = F<V>(1.f), H[w] = F<V>(0.f);
            if (w < window) kind[w] = sh.kind[w][lane], A[w] = sh.before_a[w][lane], H[w] = sh.before_h[w][lane];
        }
#pragma unroll
        for (int w = WARPS - 1; w >= 0; --w) {
            const F<V> n = fma(A[w], h, H[w]);
            h = kind[w] == kState ? H[w] : n;
        }
    } else {
        for (int w = window - 1; w >= 0; --w) {
            const F<V> A = sh.before_a[w][lane], H = sh.before_h[w][lane];
            h = sh.kind[w][lane] == kState ? H : fma(A, h, H);
        }
    }
    *state = h;
    return true;
}

template <typename T, int V>
__device__ __forceinline__ void publish_map(const Params<T>& a, const Tile& t, int lane, F<V> A, F<V> H) {
    const int c = t.c0 + lane * V;
    if (c >= a.channels) return;
    uint2* p = slot_of(a, t, t.tt, c);
    publish<V>(p, A, kMap);
    publish<V>(p + a.channels, H, kMap);
}
template <typename T, int V>
__device__ __forceinline__ void publish_end(const Params<T>& a, const Tile& t, int lane, F<V> h) {
    const int c = t.c0 + lane * V;
    if (c < a.channels) publish<V>(slot_of(a, t, t.tt, c) + a.channels, h, kState);
}

template <typename T, int V, int WARPS, bool BACK>
__device__ __forceinline__ Tile take_tile(const Params<T>& a, bool down, Shared<V, WARPS, BACK>& sh) {
    int ticket = blockIdx.x;
    if (a.tiles > 1) {
        if (threadIdx.x == 0) sh.ticket = atomicAdd(&a.st->ticket, 1);
        __syncthreads();
        ticket = sh.ticket;
    }
    return tile_of(a, ticket, down, 32 * V);
}

template <typename T, int V>
__global__ void __launch_bounds__(Shape<V>::FW * 32, Shape<V>::FCTAS) forward_kernel(const __grid_constant__ Params<T> a) {
    constexpr int FL = Shape<V>::FL, FW = Shape<V>::FW;
    __shared__ Shared<V, FW, false> sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const Tile t = take_tile(a, false, sh);
    const int c = t.c0 + lane * V;
    const bool in = c < a.channels;
    const int len = a.lengths ? min(max(__ldg(a.lengths + t.b), 0), a.steps) : a.steps;
    const int from = t.tt * TILE + warp * FL;
    const int live = in ? min(max(len - from, 0), FL) : 0, rows = in ? min(max(a.steps - from, 0), FL) : 0;

    Word<T, V> wx[FL], wr[FL], wi[FL];
    {
        const T* px = a.x.p + t.b * a.x.sb + (long)from * a.x.st + c;
        const T* pr = a.decay.p + t.b * a.decay.sb + (long)from * a.decay.st + c;
        const T* pi = a.gate.p + t.b * a.gate.sb + (long)from * a.gate.st + c;
#pragma unroll
        for (int l = 0; l < FL; ++l) {
            wx[l].fill(0.f), wr[l].fill(-INFINITY), wi[l].fill(0.f);  // where there is no token: a = 1, b = 0
            if (l < live) wx[l].load(px), wr[l].load(pr), wi[l].load(pi);
            px += a.x.st, pr += a.decay.st, pi += a.gate.st;
        }
    }
    const F<V> rate = F<V>::make([&](int j) { return in ? rate_at(a.rate + c + j) : 0.f; });
    F<V> av[FL], bv[FL], A(1.f), H(0.f);
    auto gates = [&](auto near) {
#pragma unroll
        for (int l = 0; l < FL; ++l) {
            const F<V> p = rate * sigmoid(wr[l].get());
            const Decay<decltype(near)::value, V> d(p);
            av[l] = d.a();
            bv[l] = input(d.w(p), sigmoid(wi[l].get()), wx[l].get());
            A = A * av[l];
            H = fma(av[l], H, bv[l]);
        }
    };
    if (is_near(rate)) gates(std::true_type());
    else gates(std::false_type());
    // the warps' maps in front of this one
    F<V> pa(1.f), ph(0.f), h(0.f);
    sh.A[warp][lane] = A, sh.H[warp][lane] = H;
    __syncthreads();
    for (int w = 0; w < warp; ++w) pa = pa * sh.A[w][lane], ph = fma(sh.A[w][lane], ph, sh.H[w][lane]);
    const bool last = warp == warps - 1;
    const F<V> ta = A * pa, th = fma(A, ph, H);
    if (t.tt == 0) {
        if (a.initial) h = load_channels<V>(a.initial + (long)t.b * a.channels, c, a.channels);
    } else {
        if (last) publish_map<T, V>(a, t, lane, ta, th);
        if (!look_back<false>(a, t, false, sh, warp, lane, warps, &h)) {
            if (threadIdx.x == 0) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
            return;
        }
    }
    if (last) {
        const F<V> end = fma(ta, h, th);
        if (t.tt < a.tiles - 1) publish_end<T, V>(a, t, lane, end);
        else if (a.final_state) store_channels<V>(a.final_state + (long)t.b * a.channels, c, a.channels, end);
    }
    h = fma(pa, h, ph);
    if (a.carry && (from & (a.apart - 1)) == 0 && from < a.steps)
        store_channels<V>(a.carry + ((long)t.b * a.carries + (from >> (a.apart == TILE ? 6 : 5))) * a.channels, c, a.channels, h);
    T* po = a.out + ((long)t.b * a.steps + from) * a.channels + c;
#pragma unroll
    for (int l = 0; l < FL; ++l) {
        h = fma(av[l], h, bv[l]);
        if (l < rows) Word<T, V>::store(po, l < live ? h : F<V>(0.f));
        po += a.channels;
    }
}

// One token's gradients: `g` comes in as what flows into its state from behind and leaves as what flows on, `sum` collects the
// rate's.
template <int V>
struct Slopes {
    F<V> x, decay, gate;
};
template <bool NEAR, int V>
__device__ __forceinline__ Slopes<V> slopes_of(F<V> rate, Decay<NEAR, V> d, F<V> r, F<V> gate, F<V> before, F<V> x, F<V> dout, F<V>* g, F<V>* sum) {
    const F<V> minus(-1.f), one(1.f);
    const F<V> a = d.a(), w = d.w(rate * r);  // formed again: kept, they would take too many registers
    const F<V> i = open(w, gate);
    // no step of the clock: the state passes, whatever the input
    const F<V> inv = w.each([](float t) { return fabsf(t) < FLT_MIN ? 0.f : inverse_root(t); });
    *g = *g + dout;
    const F<V> ix = open(w, gate * x), gm = *g * (w * inv);
    const F<V> rd = r * *g * fma(a * a * inv * ix, minus, a * before);
    *sum = fma(rd, minus, *sum);
    *g = a * *g;
    return Slopes<V>{gm * i, rate * rd * fma(r, one, minus), gm * ix * fma(i, minus, one)};
}

template <typename T, int V>
__global__ void __launch_bounds__(Shape<V>::BW * 32, Shape<V>::BCTAS) backward_kernel(const __grid_constant__ Params<T> a) {
    constexpr int BL = Shape<V>::BL, BW = Shape<V>::BW;
    __shared__ Shared<V, BW, true> sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const Tile t = take_tile(a, true, sh);
    const int c = t.c0 + lane * V;
    const bool in = c < a.channels;
    const int len = a.lengths ? min(max(__ldg(a.lengths + t.b), 0), a.steps) : a.steps;
    const int from = t.tt * TILE + warp * BL;
    const int live = in ? min(max(len - from, 0), BL) : 0, rows = in ? min(max(a.steps - from, 0), BL) : 0;

    Word<T, V> wx[BL], wg[BL];
    F<V> kv[BL], rv[BL], iv[BL], hb[BL];  // hb: the state in front of each token, at first from zero at the warp's start
    F<V> A(1.f), H(0.f), D(0.f), h(0.f);
    const F<V> rate = F<V>::make([&](int j) { return in ? rate_at(a.rate + c + j) : 0.f; });
    const bool near = is_near(rate);
    {
        Word<T, V> wr[BL], wi[BL];
        const T* px = a.x.p + t.b * a.x.sb + (long)from * a.x.st + c;
        const T* pr = a.decay.p + t.b * a.decay.sb + (long)from * a.decay.st + c;
        const T* pi = a.gate.p + t.b * a.gate.sb + (long)from * a.gate.st + c;
        const T* pg = a.dout.p + t.b * a.dout.sb + (long)from * a.dout.st + c;
#pragma unroll
        for (int l = 0; l < BL; ++l) {
            wx[l].fill(0.f), wr[l].fill(-INFINITY), wi[l].fill(0.f), wg[l].fill(0.f);
            if (l < live) wx[l].load(px), wr[l].load(pr), wi[l].load(pi);
            if (l < live && a.dout.p) wg[l].load(pg);
            px += a.x.st, pr += a.decay.st, pi += a.gate.st, pg += a.dout.st;
        }
        if (t.tt > 0) h = load_channels<V>(a.carry + ((long)t.b * a.carries + t.tt * (TILE / a.apart)) * a.channels, c, a.channels);
        else if (a.initial) h = load_channels<V>(a.initial + (long)t.b * a.channels, c, a.channels);
        auto gates = [&](auto near) {
            using K = Decay<decltype(near)::value, V>;
#pragma unroll
            for (int l = 0; l < BL; ++l) {
                rv[l] = sigmoid(wr[l].get()), iv[l] = sigmoid(wi[l].get());
                const K d(rate * rv[l]);
                kv[l] = d.k;
                hb[l] = H;
                H = fma(d.a(), H, input(d.w(rate * rv[l]), iv[l], wx[l].get()));
                A = A * d.a();
            }
#pragma unroll
            for (int l = BL - 1; l >= 0; --l) D = K::of(kv[l]).a() * (wg[l].get() + D);
        };
        if (near) gates(std::true_type());
        else gates(std::false_type());
    }
    // the states by the maps of the warps in front, the gradients by those of the warps behind
    F<V> pa(1.f), pd(0.f), g(0.f);
    sh.A[warp][lane] = A, sh.H[warp][lane] = H, sh.D[warp][lane] = D;
    __syncthreads();
    for (int w = 0; w < warp; ++w) h = fma(sh.A[w][lane], h, sh.H[w][lane]);
    for (int w = warps - 1; w > warp; --w) pa = pa * sh.A[w][lane], pd = fma(sh.A[w][lane], pd, sh.D[w][lane]);
    const F<V> ta = A * pa, td = fma(A, pd, D);
    if (t.tt == a.tiles - 1) {
        if (a.dfinal) g = load_channels<V>(a.dfinal + (long)t.b * a.channels, c, a.channels);
    } else {
        if (warp == 0) publish_map<T, V>(a, t, lane, ta, td);
        if (!look_back<false>(a, t, true, sh, warp, lane, warps, &g)) {
            if (threadIdx.x == 0) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
            return;
        }
    }
    if (warp == 0) {
        const F<V> end = fma(ta, g, td);
        if (t.tt > 0) publish_end<T, V>(a, t, lane, end);
        else if (a.dinitial) store_channels<V>(a.dinitial + (long)t.b * a.channels, c, a.channels, end);
    }
    g = fma(pa, g, pd);
    F<V> sum(0.f);
    const long at = ((long)t.b * a.steps + from + BL - 1) * a.channels + c;
    T *ox = a.dx + at, *od = a.ddecay + at, *oi = a.dgate + at;
    auto slopes = [&](auto near) {
        using K = Decay<decltype(near)::value, V>;
#pragma unroll
        for (int l = 0; l < BL; ++l) {
            hb[l] = hb[l] + h;
            h = K::of(kv[l]).a() * h;
        }
#pragma unroll
        for (int l = BL - 1; l >= 0; --l) {
            const Slopes<V> o = slopes_of(rate, K::of(kv[l]), rv[l], iv[l], hb[l], wx[l].get(), wg[l].get(), &g, &sum);
            if (l < rows) {
                const bool there = l < live;
                Word<T, V>::store(ox, there ? o.x : F<V>(0.f));
                Word<T, V>::store(oi, there ? o.gate : F<V>(0.f));
                Word<T, V>::store(od, there ? o.decay : F<V>(0.f));
            }
            ox -= a.channels, od -= a.channels, oi -= a.channels;
        }
    };
    if (near) slopes(std::true_type());
    else slopes(std::false_type());
    if (a.drate_part) {  // of the tile, the warps in order
        sh.sum[0][warp][lane] = sum;
        __syncthreads();
        if (warp == 0) {
            F<V> s(0.f);
            for (int w = 0; w < warps; ++w) s = s + sh.sum[0][w][lane];
            store_channels<V>(a.drate_part + ((long)t.b * a.tiles + t.tt) * a.channels, c, a.channels, s);
        }
    }
}

// ---- the same on tiles that TMA brings --------------------------------------------------------------------------
//
// Persistent kernels: thread 0 takes the tickets, has two tiles loaded ahead of the one in work and the one behind it stored. Rows
// of 128 bytes, so that a warp's access to shared memory has no conflict and no address of its own; results go where what they
// replace was read from.

struct Maps {
    CUtensorMap in[4];   // x, decay, gate; backward: dout
    CUtensorMap out[3];  // h; backward: dx, ddecay, dgate
};

template <int IN, int OUTS, int STAGES, int ROWS>
struct Pipe {
    static constexpr int STREAM = ROWS * 128, STAGE = IN * STREAM;
    static constexpr size_t bytes = (size_t)STAGES * STAGE + 128;
    uint64_t full[STAGES];
    Tile tile[STAGES];  // b < 0: there is none left
    int failed;

    __device__ __forceinline__ void init() {
        if (threadIdx.x == 0) {
            for (int i = 0; i < STAGES; ++i) tc5::mbar_init(full + i, 1);
            failed = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    // Thread 0: the tile of the ticket on its way into stage s.
    template <typename T>
    __device__ __forceinline__ void load(const Params<T>& a, const Maps& maps, unsigned char* stage, int s, long ticket, bool down) {
        if (ticket >= a.total) {
            tile[s].b = -1;
            tc5::mbar_arrive(full + s);
            return;
        }
        const Tile t = tile_of(a, (int)ticket, down, 128 / (int)sizeof(T));
        tile[s] = t;
        tc5::mbar_expect(full + s, STAGE);
#pragma unroll
        for (int k = 0; k < IN; ++k) tc5::tma_load(&maps.in[k], full + s, stage + s * STAGE + k * STREAM, t.c0, t.tt * ROWS, t.b);
    }
    __device__ __forceinline__ void store(const Maps& maps, unsigned char* stage, int s) {
        const Tile t = tile[s];
#pragma unroll
        for (int k = 0; k < OUTS; ++k) tc5::tma_store(&maps.out[k], stage + s * STAGE + k * STREAM, t.c0, t.tt * ROWS, t.b);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    // All threads, at the top of a tile: its stage is there and everyone is done with the tile before. False when a wait ran out.
    __device__ __forceinline__ bool arrive(int s, uint32_t phase) {
        return __syncthreads_and(tc5::warp_wait(full + s, phase, &failed)) != 0;
    }
    // All threads, after the last tile (or a wait that ran out in stage s): what is in flight lands.
    __device__ __forceinline__ void finish(const Maps& maps, unsigned char* stage, int s, uint32_t phase, bool any, bool ok, int* status) {
        __syncthreads();
        if (threadIdx.x == 0) {
            if (ok && any) store(maps, stage, (s + STAGES - 1) % STAGES);
            if (!ok) {
                for (int k = 0; k < STAGES; ++k) {  // the stages from this one on, as far as they were filled
                    tc5::mbar_drain(full + s, phase);
                    if (++s == STAGES) s = 0, phase ^= 1u;
                }
                report(status, EWS_ERR_LOOKBACK_TIMEOUT);
            }
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        }
    }
};

template <typename T>
__device__ __forceinline__ long take_ticket(const Params<T>& a, int it) {
    return a.tiles > 1 ? (long)atomicAdd(&a.st->ticket, 1) : blockIdx.x + (long)it * gridDim.x;
}

template <typename T>
__global__ void __launch_bounds__(PW * 32, PCTAS) forward_tma_kernel(const __grid_constant__ Params<T> a, const __grid_constant__ Maps maps) {
    constexpr int V = 4 / sizeof(T);
    using P = Pipe<3, 1, PSTAGES, TILE>;
    using W = Word<T, V>;
    constexpr int STREAM = P::STREAM / 4;
    extern __shared__ __align__(128) unsigned char raw[];
    unsigned char* stage = raw + ((128 - (smem_addr(raw) & 127)) & 127);
    __shared__ Shared<V, PW, false> sh;
    __shared__ P pipe;
    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    pipe.init();
    if (threadIdx.x == 0)
        for (int k = 0; k < PSTAGES - 1; ++k) pipe.load(a, maps, stage, k, take_ticket(a, k), false);
    int s = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (;; ++it) {
        if (!(ok = pipe.arrive(s, phase))) break;
        const Tile t = pipe.tile[s];
        if (t.b < 0) break;
        long next = 0;
        if (threadIdx.x == 0) {
            if (it > 0) pipe.store(maps, stage, s == 0 ? PSTAGES - 1 : s - 1);
            next = take_ticket(a, it + PSTAGES - 1);
        }
        const int c = t.c0 + lane * V, from = t.tt * TILE + warp * PL;
        const int len = a.lengths ? min(max(__ldg(a.lengths + t.b), 0), a.steps) : a.steps;
        const int live = min(max(len - from, 0), PL);
        W* row = reinterpret_cast<W*>(stage + s * P::STAGE + warp * PL * 128) + lane;
        // where there is no token: a = 1, b = 0
        for (int l = live; l < PL; ++l) row[l * 32].fill(0.f), row[STREAM + l * 32].fill(-INFINITY), row[2 * STREAM + l * 32].fill(0.f);
        const F<V> rate = F<V>::make([&](int j) { return c + j < a.channels ? rate_at(a.rate + c + j) : 0.f; });
        F<V> av[PL], bv[PL], A(1.f), H(0.f);
        auto gates = [&](auto near) {
#pragma unroll
            for (int l = 0; l < PL; ++l) {
                const F<V> p = rate * sigmoid(row[STREAM + l * 32].get());
                const Decay<decltype(near)::value, V> d(p);
                av[l] = d.a();
                bv[l] = input(d.w(p), sigmoid(row[2 * STREAM + l * 32].get()), row[l * 32].get());
                A = A * av[l];
                H = fma(av[l], H, bv[l]);
            }
        };
        if (is_near(rate)) gates(std::true_type());
        else gates(std::false_type());
        F<V> pa, ph, h(0.f);
        sh.A[warp][lane] = A, sh.H[warp][lane] = H;
        if (threadIdx.x == 0) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            pipe.load(a, maps, stage, s == 0 ? PSTAGES - 1 : s - 1, next, false);
        }
        __syncthreads();
        fold_front(sh, warp, lane, &pa, &ph);
        const bool last = warp == PW - 1;
        const F<V> ta = A * pa, th = fma(A, ph, H);
        if (t.tt == 0) {
            if (a.initial) h = load_channels<V>(a.initial + (long)t.b * a.channels, c, a.channels);
        } else {
            if (last) publish_map<T, V>(a, t, lane, ta, th);
            if (!(ok = look_back<true>(a, t, false, sh, warp, lane, PW, &h))) break;
        }
        if (last) {
            const F<V> end = fma(ta, h, th);
            if (t.tt < a.tiles - 1) publish_end<T, V>(a, t, lane, end);
            else if (a.final_state) store_channels<V>(a.final_state + (long)t.b * a.channels, c, a.channels, end);
        }
        h = fma(pa, h, ph);
        if (a.carry && (from & (a.apart - 1)) == 0 && from < a.steps)
            store_channels<V>(a.carry + ((long)t.b * a.carries + (from >> (a.apart == TILE ? 6 : 5))) * a.channels, c, a.channels, h);
#pragma unroll
        for (int l = 0; l < PL; ++l) {
            h = fma(av[l], h, bv[l]);
            row[l * 32].put(h);
        }
        for (int l = live; l < PL; ++l) row[l * 32].fill(0.f);
        tc5::fence_async_smem();
        if (++s == PSTAGES) s = 0, phase ^= 1u;
    }
    pipe.finish(maps, stage, s, phase, it > 0, ok, a.status);
}

template <typename T, int ROWS>
__global__ void __launch_bounds__(Back<4 / sizeof(T), ROWS>::QW * 32, Back<4 / sizeof(T), ROWS>::QCTAS)
    backward_tma_kernel(const __grid_constant__ Params<T> a, const __grid_constant__ Maps maps) {
    constexpr int V = 4 / sizeof(T), QL = Back<V, ROWS>::QL, QW = Back<V, ROWS>::QW;
    using P = Pipe<4, 3, QSTAGES, ROWS>;
    using W = Word<T, V>;
    constexpr int STREAM = P::STREAM / 4;
    extern __shared__ __align__(128) unsigned char raw[];
    unsigned char* stage = raw + ((128 - (smem_addr(raw) & 127)) & 127);
    __shared__ Shared<V, QW, true> sh;
    __shared__ P pipe;
    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    pipe.init();
    if (threadIdx.x == 0)
        for (int k = 0; k < QSTAGES - 1; ++k) pipe.load(a, maps, stage, k, take_ticket(a, k), true);
    int s = 0, it = 0;
    uint32_t phase = 0;
    bool ok = true;
    Tile last{};
    for (;; ++it) {
        if (!(ok = pipe.arrive(s, phase))) break;
        if (it > 0 && warp == QW - 1 && a.drate_part) {  // the last tile's, the warps in order
            F<V> total(0.f);
#pragma unroll
            for (int w = 0; w < QW; ++w) total = total + sh.sum[(it - 1) & 1][w][lane];
            store_channels<V>(a.drate_part + ((long)last.b * a.tiles + last.tt) * a.channels, last.c0 + lane * V, a.channels, total);
        }
        const Tile t = pipe.tile[s];
        if (t.b < 0) break;
        long next = 0;
        if (threadIdx.x == 0) {
            if (it > 0) pipe.store(maps, stage, s == 0 ? QSTAGES - 1 : s - 1);
            next = take_ticket(a, it + QSTAGES - 1);
        }
        const int c = t.c0 + lane * V, from = t.tt * ROWS + warp * QL;
        const int len = a.lengths ? min(max(__ldg(a.lengths + t.b), 0), a.steps) : a.steps;
        const int live = min(max(len - from, 0), QL);
        W* row = reinterpret_cast<W*>(stage + s * P::STAGE + warp * QL * 128) + lane;
        for (int l = live; l < QL; ++l) {
            row[l * 32].fill(0.f), row[STREAM + l * 32].fill(-INFINITY);
            row[2 * STREAM + l * 32].fill(0.f), row[3 * STREAM + l * 32].fill(0.f);
        }
        const F<V> rate = F<V>::make([&](int j) { return c + j < a.channels ? rate_at(a.rate + c + j) : 0.f; });
        F<V> kv[QL], rv[QL], iv[QL], hb[QL];  // as in backward_kernel
        const bool near = is_near(rate);
        F<V> A(1.f), H(0.f), D(0.f), h(0.f);
        if (t.tt > 0) h = load_channels<V>(a.carry + ((long)t.b * a.carries + t.tt) * a.channels, c, a.channels);
        else if (a.initial) h = load_channels<V>(a.initial + (long)t.b * a.channels, c, a.channels);
        auto gates = [&](auto near) {
            using K = Decay<decltype(near)::value, V>;
#pragma unroll
            for (int l = 0; l < QL; ++l) {
                rv[l] = sigmoid(row[STREAM + l * 32].get()), iv[l] = sigmoid(row[2 * STREAM + l * 32].get());
                const K d(rate * rv[l]);
                kv[l] = d.k;
                hb[l] = H;
                H = fma(d.a(), H, input(d.w(rate * rv[l]), iv[l], row[l * 32].get()));
                A = A * d.a();
            }
#pragma unroll
            for (int l = QL - 1; l >= 0; --l) D = K::of(kv[l]).a() * (row[3 * STREAM + l * 32].get() + D);
        };
        if (near) gates(std::true_type());
        else gates(std::false_type());
        F<V> pa, pd, g(0.f);
        sh.A[warp][lane] = A, sh.H[warp][lane] = H, sh.D[warp][lane] = D;
        if (threadIdx.x == 0) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            pipe.load(a, maps, stage, s == 0 ? QSTAGES - 1 : s - 1, next, true);
        }
        __syncthreads();
        fold_front(sh, warp, lane, &pa, &pd);
        h = fma(pa, h, pd);
        fold_behind(sh, warp, lane, &pa, &pd);
        const F<V> ta = A * pa, td = fma(A, pd, D);
        if (t.tt == a.tiles - 1) {
            if (a.dfinal) g = load_channels<V>(a.dfinal + (long)t.b * a.channels, c, a.channels);
        } else {
            if (warp == 0) publish_map<T, V>(a, t, lane, ta, td);
            if (!(ok = look_back<true>(a, t, true, sh, warp, lane, QW, &g))) break;
        }
        if (warp == 0) {
            const F<V> end = fma(ta, g, td);
            if (t.tt > 0) publish_end<T, V>(a, t, lane, end);
            else if (a.dinitial) store_channels<V>(a.dinitial + (long)t.b * a.channels, c, a.channels, end);
        }
        g = fma(pa, g, pd);
        F<V> sum(0.f);
        auto slopes = [&](auto near) {
            using K = Decay<decltype(near)::value, V>;
#pragma unroll
            for (int l = 0; l < QL; ++l) {
                hb[l] = hb[l] + h;
                h = K::of(kv[l]).a() * h;
            }
#pragma unroll
            for (int l = QL - 1; l >= 0; --l) {
                const Slopes<V> o = slopes_of(rate, K::of(kv[l]), rv[l], iv[l], hb[l], row[l * 32].get(), row[3 * STREAM + l * 32].get(), &g, &sum);
                row[l * 32].put(o.x), row[STREAM + l * 32].put(o.decay), row[2 * STREAM + l * 32].put(o.gate);
            }
        };
        if (near) slopes(std::true_type());
        else slopes(std::false_type());
        for (int l = live; l < QL; ++l) row[l * 32].fill(0.f), row[STREAM + l * 32].fill(0.f), row[2 * STREAM + l * 32].fill(0.f);
        tc5::fence_async_smem();
        sh.sum[it & 1][warp][lane] = sum;
        last = t;
        if (++s == QSTAGES) s = 0, phase ^= 1u;
    }
    pipe.finish(maps, stage, s, phase, it > 0, ok, a.status);
}

// drate from the tiles' sums, in a fixed order: 32 channels by 32 groups of rows a CTA.
__global__ void __launch_bounds__(1024) rate_kernel(const float* __restrict__ part, long rows, int channels, float* __restrict__ out) {
    __shared__ float red[32][33];
    const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + l;
    float s = 0.f;
    if (c < channels) {
#pragma unroll 8
        for (long r = g; r < rows; r += 32) s += part[r * channels + c];
    }
    red[g][l] = s;
    __syncthreads();
    if (g == 0 && c < channels) {
        s = 0.f;
        for (int k = 0; k < 32; ++k) s += red[k][l];
        out[c] = s;
    }
}

// ---- one token a row ------------------------------------------------------------------------------------------

template <typename T>
struct Step {
    const T *x, *decay, *gate;
    long xb, db, gb;
    const float* rate;
    const int* slots;
    float* state;
    T* out;
    int batch, channels, pool;
    int* status;
};

// V channels a thread (4 where the rows allow vectors of 16 bytes of the state).
template <typename T, int V>
__global__ void __launch_bounds__(128) step_kernel(const __grid_constant__ Step<T> a) {
    const int per = (a.channels + V - 1) / V;
    const long e = (long)blockIdx.x * 128 + threadIdx.x;
    const long row = e / per;
    if (row >= a.batch) return;
    const int c = (int)(e - row * per) * V;
    const int slot = a.slots ? __ldg(a.slots + row) : (int)row;
    T* out = a.out + row * a.channels + c;
    float o[V];
    if (slot < 0 || slot >= a.pool) {
        if (slot >= a.pool) report(a.status, EWS_ERR_INDEX);
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = 0.f;
    } else {
        float* state = a.state + (long)slot * a.channels + c;
        float x[V], r[V], i[V], k[V], h[V];
        if constexpr (V == 4) {
            auto load = [](const T* p, float v[4]) {
                if constexpr (sizeof(T) == 4) {
                    Vec<float, true>::load(p, v);
                } else {
                    const uint2 q = *reinterpret_cast<const uint2*>(p);
                    v[0] = bf16_lo(q.x), v[1] = bf16_hi(q.x), v[2] = bf16_lo(q.y), v[3] = bf16_hi(q.y);
                }
            };
            load(a.x + row * a.xb + c, x), load(a.decay + row * a.db + c, r), load(a.gate + row * a.gb + c, i);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = rate_at(a.rate + c + j);
            Vec<float, true>::load(state, h);
        } else {
            x[0] = to_f(a.x[row * a.xb + c]), r[0] = to_f(a.decay[row * a.db + c]), i[0] = to_f(a.gate[row * a.gb + c]);
            k[0] = rate_at(a.rate + c), h[0] = *state;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const F<1> p = F<1>(k[j]) * sigmoid(F<1>(r[j]));
            const Decay<false, 1> d(p);
            o[j] = fma(d.a(), F<1>(h[j]), input(d.w(p), sigmoid(F<1>(i[j])), F<1>(x[j]))).r;
        }
        if constexpr (V == 4) Vec<float, true>::store(state, o);
        else *state = o[0];
    }
    if constexpr (V == 4) {
        if constexpr (sizeof(T) == 4) Vec<float, true>::store(out, o);
        else *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]));
    } else {
        *out = from_f<T>(o[0]);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------

int check(const ews_recur_args* a) {
    if (!a || a->batch < 0 || a->steps < 0 || a->channels <= 0) return EWS_ERR_INVALID_ARGUMENT;
    if (a->steps > 1 << 30 || a->channels > 1 << 30) return EWS_ERR_UNSUPPORTED;
    if (a->dtype != EWS_DTYPE_F32 && a->dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    return EWS_OK;
}

size_t up(size_t b) { return (b + 255) / 256 * 256; }
int tiles_of(int steps, int tile = TILE) { return (steps + tile - 1) / tile; }

struct Sizes {
    size_t slots, part, bytes;  // slots: behind the status block, both cleared by a call
};

// Tokens a tile of the backward that TMA feeds, and from one state that the forward leaves to the next: see Back.
int back_rows(const ews_recur_args* a) {
    const bool many = (long)a->batch * ((a->channels + 63) / 64) >= SMS;
    return a->dtype == EWS_DTYPE_BF16 && a->steps > TILE && many ? HALF : TILE;
}

Sizes sizes(const ews_recur_args* a, bool bwd) {
    Sizes z{};
    const size_t tiles = tiles_of(a->steps, bwd ? back_rows(a) : TILE), states = (size_t)a->batch * tiles * a->channels;
    if (tiles > 1) z.slots = up(sizeof(DeviceStatus) + 2 * sizeof(uint2) * states);
    if (bwd) z.part = up(sizeof(float) * states);
    z.bytes = z.slots + z.part;
    return z;
}

template <typename T>
Stream<T> stream_of(const void* p, const int64_t st[2]) {
    return Stream<T>{static_cast<const T*>(p), (long)st[0], (long)st[1]};
}

template <typename T>
bool even(const ews_recur_args* a, const Stream<T>& s) {
    return ((uintptr_t)s.p & 3u) == 0 && (a->batch == 1 || s.sb % 2 == 0) && (a->steps == 1 || s.st % 2 == 0);
}

// A stream (batch, steps, channels) for TMA: boxes of 128 bytes of channels by a tile's steps. False where it cannot be read so.
template <typename T>
bool make_map(tc5::EncodeFn enc, CUtensorMap* map, const ews_recur_args* a, const void* p, long sb, long st, int rows) {
    constexpr long E = 16 / sizeof(T);
    const long one = (a->channels + E - 1) / E * E;  // an axis of one has no stride to speak of
    if (a->steps == 1) st = one;
    if (a->batch == 1) sb = st * a->steps;
    if (!aligned16(p) || st <= 0 || sb <= 0 || st % E || sb % E || a->channels % E) return false;
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)a->channels, (cuuint64_t)a->steps, (cuuint64_t)a->batch};
    const cuuint64_t strides[2] = {(cuuint64_t)st * sizeof(T), (cuuint64_t)sb * sizeof(T)};
    const cuuint32_t box[3] = {128 / sizeof(T), (cuuint32_t)rows, 1}, es[3] = {1, 1, 1};
    return enc(map, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(p), dims, strides,
               box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <auto K, typename T>
int piped_launch(const Params<T>& p, const Maps& m, size_t bytes, int threads, int resident, cudaStream_t s) {
    if (!tc5::allow_shared<K>((int)bytes)) return EWS_ERR_LAUNCH;
    const long most = (long)SMS * resident;
    K<<<(unsigned)(p.total < most ? p.total : most), threads, bytes, s>>>(p, m);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T>
int run(const ews_recur_args* a, bool bwd, cudaStream_t s) {
    Params<T> p{};
    p.batch = a->batch, p.steps = a->steps, p.channels = a->channels, p.apart = back_rows(a), p.carries = tiles_of(a->steps, p.apart);
    p.x = stream_of<T>(a->x, a->x_stride), p.decay = stream_of<T>(a->decay, a->decay_stride), p.gate = stream_of<T>(a->gate, a->gate_stride);
    p.rate = a->rate, p.lengths = a->lengths, p.initial = a->initial, p.carry = a->carry, p.status = a->status;
    bool pairs = sizeof(T) == 2 && a->channels % 2 == 0 && even(a, p.x) && even(a, p.decay) && even(a, p.gate);
    if (bwd) {
        p.dout = stream_of<T>(a->dout, a->dout_stride), p.dfinal = a->dfinal;
        p.dx = static_cast<T*>(a->dx), p.ddecay = static_cast<T*>(a->ddecay), p.dgate = static_cast<T*>(a->dgate), p.dinitial = a->dinitial;
        pairs = pairs && even(a, p.dout) && (((uintptr_t)a->dx | (uintptr_t)a->ddecay | (uintptr_t)a->dgate) & 3u) == 0;
    } else {
        p.out = static_cast<T*>(a->out), p.final_state = a->final_state;
        pairs = pairs && ((uintptr_t)a->out & 3u) == 0;
    }
    Maps m{};
    const int rows = bwd ? p.apart : TILE;
    const long C = a->channels, whole = (long)a->steps * C;
    const tc5::EncodeFn enc = a->steps >= kPipedFrom ? tc5::encoder() : nullptr;
    bool piped = enc && make_map<T>(enc, &m.in[0], a, a->x, p.x.sb, p.x.st, rows) &&
                 make_map<T>(enc, &m.in[1], a, a->decay, p.decay.sb, p.decay.st, rows) && make_map<T>(enc, &m.in[2], a, a->gate, p.gate.sb, p.gate.st, rows);
    if (bwd)
        piped = piped && a->dout && make_map<T>(enc, &m.in[3], a, a->dout, p.dout.sb, p.dout.st, rows) && make_map<T>(enc, &m.out[0], a, a->dx, whole, C, rows) &&
                make_map<T>(enc, &m.out[1], a, a->ddecay, whole, C, rows) && make_map<T>(enc, &m.out[2], a, a->dgate, whole, C, rows);
    else
        piped = piped && make_map<T>(enc, &m.out[0], a, a->out, whole, C, rows);
    p.tiles = tiles_of(a->steps, piped ? rows : TILE);
    const int width = pairs ? 64 : 32;
    p.blocks = (a->channels + width - 1) / width;
    const Sizes z = sizes(a, bwd);
    char* w = static_cast<char*>(a->work);
    if (p.tiles > 1) {
        p.st = reinterpret_cast<DeviceStatus*>(w);
        p.slots = reinterpret_cast<uint2*>(w + sizeof(DeviceStatus));
        if (cudaMemsetAsync(w, 0, z.slots, s) != cudaSuccess) return EWS_ERR_LAUNCH;
    }
    if (bwd && a->drate) p.drate_part = reinterpret_cast<float*>(w + z.slots);
    const long ctas = (long)p.batch * p.blocks * p.tiles;
    if (ctas > 0x7FFFFFFFl - 65536) return EWS_ERR_UNSUPPORTED;  // the tickets count a little further
    p.total = ctas;
    using One = Shape<1>;
    using Two = Shape<2>;
    constexpr int V = 4 / sizeof(T);
    const int per = pairs ? (bwd ? Two::BL : Two::FL) : (bwd ? One::BL : One::FL);
    const int warps = (int)((p.tiles > 1 ? TILE : a->steps) + per - 1) / per;  // a short axis: as many as it has work for
    auto go = [&](auto* kernel) {
        kernel<<<(unsigned)ctas, warps * 32, 0, s>>>(p);
        return cudaGetLastError() == cudaSuccess ? (int)EWS_OK : (int)EWS_ERR_LAUNCH;
    };
    int rc;
    auto back = [&](auto of) {
        using B = decltype(of);
        constexpr int ROWS = B::QL * B::QW;
        return piped_launch<backward_tma_kernel<T, ROWS>>(p, m, Pipe<4, 3, QSTAGES, ROWS>::bytes, B::QW * 32, B::QCTAS, s);
    };
    if (piped && bwd) {
        if constexpr (V == 2) rc = rows == HALF ? back(Back<V, HALF>{}) : back(Back<V, TILE>{});
        else rc = back(Back<V, TILE>{});
    } else if (piped) {
        rc = piped_launch<forward_tma_kernel<T>>(p, m, Pipe<3, 1, PSTAGES, TILE>::bytes, PW * 32, PCTAS, s);
    } else if constexpr (sizeof(T) == 2) {
        if (pairs) rc = bwd ? go(backward_kernel<T, 2>) : go(forward_kernel<T, 2>);
        else rc = bwd ? go(backward_kernel<T, 1>) : go(forward_kernel<T, 1>);
    } else {
        rc = bwd ? go(backward_kernel<T, 1>) : go(forward_kernel<T, 1>);
    }
    if (rc != EWS_OK || !p.drate_part) return rc;
    rate_kernel<<<(unsigned)((a->channels + 31) / 32), 1024, 0, s>>>(p.drate_part, (long)p.batch * p.tiles, a->channels, a->drate);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

// No tokens: the state passes through.
int pass(const ews_recur_args* a, const float* from, float* to, cudaStream_t s) {
    if (!to || a->batch == 0) return EWS_OK;
    const size_t bytes = sizeof(float) * (size_t)a->batch * a->channels;
    const cudaError_t e = from ? cudaMemcpyAsync(to, from, bytes, cudaMemcpyDeviceToDevice, s) : cudaMemsetAsync(to, 0, bytes, s);
    return e == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T>
int step(const ews_recur_args* a, const int* slots, int pool, float* state, cudaStream_t s) {
    Step<T> p{};
    p.x = static_cast<const T*>(a->x), p.decay = static_cast<const T*>(a->decay), p.gate = static_cast<const T*>(a->gate);
    p.xb = a->x_stride[0], p.db = a->decay_stride[0], p.gb = a->gate_stride[0];
    p.rate = a->rate, p.slots = slots, p.state = state, p.out = static_cast<T*>(a->out);
    p.batch = a->batch, p.channels = a->channels, p.pool = pool, p.status = a->status;
    constexpr uintptr_t mask = sizeof(T) * 4 - 1;
    auto fits = [&](const void* q, long stride) { return ((uintptr_t)q & mask) == 0 && (a->batch == 1 || stride % 4 == 0); };
    const bool vec = a->channels % 4 == 0 && fits(p.x, p.xb) && fits(p.decay, p.db) && fits(p.gate, p.gb) && fits(p.out, 0) &&
                     aligned16(state);
    const long threads = (long)a->batch * (vec ? a->channels / 4 : a->channels), ctas = (threads + 127) / 128;
    if (ctas > 0x7FFFFFFFl) return EWS_ERR_UNSUPPORTED;
    if (vec) step_kernel<T, 4><<<(unsigned)ctas, 128, 0, s>>>(p);
    else step_kernel<T, 1><<<(unsigned)ctas, 128, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

}  // namespace recur
}  // namespace ews

using namespace ews::recur;

extern "C" size_t ews_recur_carry_size(const ews_recur_args* a) {
    return check(a) == EWS_OK ? sizeof(float) * (size_t)a->batch * tiles_of(a->steps, back_rows(a)) * a->channels : 0;
}

extern "C" size_t ews_recur_work_size(const ews_recur_args* a, int backward) {
    return check(a) == EWS_OK && a->batch > 0 && a->steps > 0 ? sizes(a, backward != 0).bytes : 0;
}

extern "C" int ews_recur_fwd(const ews_recur_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->batch == 0 || a->steps == 0) return pass(a, a->initial, a->final_state, s);
    if (!a->x || !a->decay || !a->gate || !a->rate || !a->out) return EWS_ERR_INVALID_ARGUMENT;
    const Sizes z = sizes(a, false);
    if (z.bytes && (!a->work || !ews::token::aligned16(a->work) || a->work_bytes < z.bytes)) return EWS_ERR_WORKSPACE;
    return a->dtype == EWS_DTYPE_BF16 ? run<ews::token::bf16>(a, false, s) : run<float>(a, false, s);
}

extern "C" int ews_recur_bwd(const ews_recur_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (a->batch == 0 || a->steps == 0) {
        if (a->drate && cudaMemsetAsync(a->drate, 0, sizeof(float) * a->channels, s) != cudaSuccess) return EWS_ERR_LAUNCH;
        return pass(a, a->dfinal, a->dinitial, s);
    }
    if (!a->x || !a->decay || !a->gate || !a->rate || !a->dx || !a->ddecay || !a->dgate) return EWS_ERR_INVALID_ARGUMENT;
    if (a->steps > TILE && !a->carry) return EWS_ERR_INVALID_ARGUMENT;
    const Sizes z = sizes(a, true);
    if (z.bytes && (!a->work || !ews::token::aligned16(a->work) || a->work_bytes < z.bytes)) return EWS_ERR_WORKSPACE;
    return a->dtype == EWS_DTYPE_BF16 ? run<ews::token::bf16>(a, true, s) : run<float>(a, true, s);
}

extern "C" int ews_recur_step(const ews_recur_args* a, const int* slots, int pool, float* state, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    if (a->batch == 0) return EWS_OK;
    if (!a->x || !a->decay || !a->gate || !a->rate || !a->out || !state || pool < 0 || (!slots && pool < a->batch))
        return EWS_ERR_INVALID_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    return a->dtype == EWS_DTYPE_BF16 ? step<ews::token::bf16>(a, slots, pool, state, s) : step<float>(a, slots, pool, state, s);
}
