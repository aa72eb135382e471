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
// Both directions are a scan of maps h -> A h + H. A CTA takes a tile of 32 V channels by warps x L tokens, each warp L
// consecutive tokens with everything of them in registers: the streams are read once. The warps' maps are joined in shared
// memory, the tiles' by a decoupled look-back in ticket order (a tile publishes its map, then its state): a tile folds the
// maps of up to `warps` tiles onto the nearest published state, always from the state upwards, so that the sum has one order
// and the results do not depend on timing. The backward reads no states: the forward leaves one a tile of the backward
// (float32, 1 / 64 of the stream), from which the tile runs the recurrence again. So the gradient of the rates, a float32 sum
// over all tokens, does not see the rounding of the stored states, and a stream less is read.
#include <float.h>

#include "ews_tc.cuh"

namespace ews {
namespace recur {

using namespace token;
using tc5::add2;
using tc5::fma2;
using tc5::mul2;
using tc5::pair;
using tc5::unpair;

constexpr int kMaxWarps = 16;
constexpr int FL = 16, FW = 8, FCTAS = 2;  // forward: tokens a warp, warps a tile, CTAs an SM
constexpr int BL = 8, BW = 8, BCTAS = 2;   // backward
constexpr int FT = FL * FW, BT = BL * BW;
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
    Stream<T> x, decay, gate, dout;
    const float* rate;
    const int* lengths;
    const float *initial, *dfinal;
    T* out;
    float* final_state;
    float* carry;  // (batch, tiles of the backward, channels): the state in front of each of its tiles
    T *dx, *ddecay, *dgate;
    float *drate_part, *dinitial;
    // look-back
    DeviceStatus* st;
    int* flags;    // (batch, blocks, tiles)
    float *map_a, *map_h, *ends;  // (batch, tiles, channels)
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
// rounded as the packed ones are: whether a call's tensors allow pairs does not change its results
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
    __device__ static __forceinline__ void store(bf16* p, F<2> v) { *reinterpret_cast<uint32_t*>(p) = pack_bf16(v.get(0), v.get(1)); }
};

// The exponent unit's own instructions; what lies below the normal range counts as zero (a sigmoid of less than -87, say),
// which spares their corrections, a third of the kernels' instructions.
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

// a = exp(-p) and w = 1 - a^2. Up to p = 0.175 from q = 1 - exp(-p) by its series (the first dropped term is 2^-27 of q there):
// a = 1 - q then has no error but its rounding, where the exponent unit's 2^-22 would add up over the hundreds of tokens such
// an a remembers, and w = q (2 - q) loses nothing to cancellation. Beyond, a state forgets within some six tokens.
constexpr float kSeries = 0.175f;
template <int V>
__device__ __forceinline__ F<V> decay_loss(F<V> p) {
    F<V> q = fma(p, F<V>(-1.f / 720.f), F<V>(1.f / 120.f));
    q = fma(p, q, F<V>(-1.f / 24.f));
    q = fma(p, q, F<V>(1.f / 6.f));
    q = fma(p, q, F<V>(-0.5f));
    return fma(p * p, q, p);
}
template <int V>
struct Decay {
    F<V> a, w;
};
template <int V>
__device__ __forceinline__ Decay<V> decay_of(F<V> p) {
    const F<V> q = decay_loss(p), near = fma(q, F<V>(-1.f), F<V>(1.f)), w = fma(q, near, q);
    const F<V> e = (p * F<V>(-kLog2e)).each([](float t) { return ex2(t); });
    Decay<V> d;
    d.a = F<V>::make([&](int j) { return p.get(j) < kSeries ? near.get(j) : e.get(j); });
    d.w = F<V>::make([&](int j) { return p.get(j) < kSeries ? w.get(j) : fmaf(-e.get(j), e.get(j), 1.f); });
    return d;
}
// w once more where a is at hand.
template <int V>
__device__ __forceinline__ F<V> rest_of(F<V> p, F<V> a) {
    const F<V> q = decay_loss(p), w = fma(q, fma(q, F<V>(-1.f), F<V>(1.f)), q);
    return F<V>::make([&](int j) { return p.get(j) < kSeries ? w.get(j) : fmaf(-a.get(j), a.get(j), 1.f); });
}
template <int V>
__device__ __forceinline__ F<V> root(F<V> w) { return w.each([](float t) { return root(t); }); }

// A channel's rate; an infinite one as float32's largest, so that a shut gate's product with it is zero.
__device__ __forceinline__ float rate_at(const float* p) {
    const float r = __ldg(p);
    return r > FLT_MAX ? FLT_MAX : r;
}

struct Tile {
    int b, tt, c0;  // sample, tile along the steps, first channel
    int slot;       // of the flags
};

// Tiles are given out by the steps first, so that a tile only waits on lower tickets.
template <typename T>
__device__ __forceinline__ Tile tile_of(const Params<T>& a, long ticket, bool down, int width) {
    const long per = (long)a.batch * a.blocks;
    Tile t;
    t.tt = (int)(ticket / per);
    const int rest = (int)(ticket - t.tt * per);
    if (down) t.tt = a.tiles - 1 - t.tt;
    t.b = rest / a.blocks;
    const int cb = rest - t.b * a.blocks;
    t.c0 = cb * width;
    t.slot = rest * a.tiles;
    return t;
}

template <int V>
struct Shared {
    F<V> A[kMaxWarps][32], H[kMaxWarps][32];
    int flag[kMaxWarps];
    int ticket;
};

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

// The state that comes into the tile from the tiles before it (down: behind it). Every thread of the CTA calls it, after the
// tile's own map was published; false when a wait ran out.
template <typename T, int V>
__device__ __forceinline__ bool look_back(const Params<T>& a, const Tile& t, bool down, Shared<V>& sh, int warp, int lane, int warps, F<V>* state) {
    const int step = down ? 1 : -1;
    const int before = down ? a.tiles - 1 - t.tt : t.tt;  // how many there are
    const int window = before < warps ? before : warps;
    if (warp < window) {
        const int at = t.tt + step * (1 + warp);
        // the last of the window has to have its state: nothing further back is folded
        const int flag = wait_slot(a.flags + t.slot + at, a.st, kDefaultSpinLimit, t.slot + at, warp == window - 1 ? kFlagIncl : kFlagAgg);
        const long base = ((long)t.b * a.tiles + at) * a.channels;
        const int c = t.c0 + lane * V;
        if (flag == kFlagIncl) {
            sh.H[warp][lane] = load_channels<V>(a.ends + base, c, a.channels);
        } else if (flag == kFlagAgg) {
            sh.A[warp][lane] = load_channels<V>(a.map_a + base, c, a.channels);
            sh.H[warp][lane] = load_channels<V>(a.map_h + base, c, a.channels);
        }
        if (lane == 0) sh.flag[warp] = flag;
    }
    __syncthreads();
    int n = -1;
    bool ok = true;
    for (int w = window - 1; w >= 0; --w) {
        if (sh.flag[w] == kFlagIncl) n = w;
        if (sh.flag[w] < 0) ok = false;
    }
    if (!ok) return false;
    F<V> h = sh.H[n][lane];
    for (int w = n - 1; w >= 0; --w) h = fma(sh.A[w][lane], h, sh.H[w][lane]);
    *state = h;
    return true;
}

template <typename T, int V>
__device__ __forceinline__ void publish_map(const Params<T>& a, const Tile& t, int lane, F<V> A, F<V> H) {
    const long base = ((long)t.b * a.tiles + t.tt) * a.channels;
    store_channels<V>(a.map_a + base, t.c0 + lane * V, a.channels, A);
    store_channels<V>(a.map_h + base, t.c0 + lane * V, a.channels, H);
    publish(a.flags + t.slot + t.tt, kFlagAgg);
}
template <typename T, int V>
__device__ __forceinline__ void publish_end(const Params<T>& a, const Tile& t, int lane, F<V> h) {
    store_channels<V>(a.ends + ((long)t.b * a.tiles + t.tt) * a.channels, t.c0 + lane * V, a.channels, h);
    publish(a.flags + t.slot + t.tt, kFlagIncl);
}

template <typename T, int V>
__device__ __forceinline__ Tile take_tile(const Params<T>& a, bool down, Shared<V>& sh) {
    long ticket = blockIdx.x;
    if (a.tiles > 1) {
        if (threadIdx.x == 0) sh.ticket = atomicAdd(&a.st->ticket, 1);
        __syncthreads();
        ticket = sh.ticket;
    }
    return tile_of(a, ticket, down, 32 * V);
}

template <typename T, int V>
__global__ void __launch_bounds__(FW * 32, FCTAS) forward_kernel(const __grid_constant__ Params<T> a) {
    __shared__ Shared<V> sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const Tile t = take_tile(a, false, sh);
    const int c = t.c0 + lane * V;
    const bool in = c < a.channels;
    const int len = a.lengths ? min(max(__ldg(a.lengths + t.b), 0), a.steps) : a.steps;
    const int from = t.tt * warps * FL + warp * FL;
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
#pragma unroll
    for (int l = 0; l < FL; ++l) {
        const Decay<V> d = decay_of(rate * sigmoid(wr[l].get()));
        av[l] = d.a;
        bv[l] = root(d.w) * sigmoid(wi[l].get()) * wx[l].get();
        A = A * av[l];
        H = fma(av[l], H, bv[l]);
    }
    // the warps' maps in front of this one
    F<V> pa(1.f), ph(0.f), h(0.f);
    sh.A[warp][lane] = A, sh.H[warp][lane] = H;
    __syncthreads();
    for (int w = 0; w < warp; ++w) {
        const F<V> m = sh.A[w][lane];
        pa = pa * m;
        ph = fma(m, ph, sh.H[w][lane]);
    }
    const bool last = warp == warps - 1;
    const F<V> ta = A * pa, th = fma(A, ph, H);
    if (t.tt == 0) {
        if (a.initial) h = load_channels<V>(a.initial + (long)t.b * a.channels, c, a.channels);
    } else {
        if (last) publish_map<T, V>(a, t, lane, ta, th);
        __syncthreads();  // every warp has read the maps
        if (!look_back<T, V>(a, t, false, sh, warp, lane, warps, &h)) {
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
    if (a.carry && from % BT == 0 && from < a.steps)
        store_channels<V>(a.carry + ((long)t.b * ((a.steps + BT - 1) / BT) + from / BT) * a.channels, c, a.channels, h);
    T* po = a.out + ((long)t.b * a.steps + from) * a.channels + c;
#pragma unroll
    for (int l = 0; l < FL; ++l) {
        h = fma(av[l], h, bv[l]);
        if (l < rows) Word<T, V>::store(po, l < live ? h : F<V>(0.f));
        po += a.channels;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(BW * 32, BCTAS) backward_kernel(const __grid_constant__ Params<T> a) {
    __shared__ Shared<V> sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const Tile t = take_tile(a, true, sh);
    const int c = t.c0 + lane * V;
    const bool in = c < a.channels;
    const int len = a.lengths ? min(max(__ldg(a.lengths + t.b), 0), a.steps) : a.steps;
    const int from = t.tt * BT + warp * BL;
    const int live = in ? min(max(len - from, 0), BL) : 0, rows = in ? min(max(a.steps - from, 0), BL) : 0;

    Word<T, V> wx[BL], wg[BL];
    F<V> av[BL], rv[BL], iv[BL], hb[BL];  // hb: the state in front of each token, at first from zero at the warp's start
    F<V> A(1.f), H(0.f), D(0.f), h(0.f);
    const F<V> rate = F<V>::make([&](int j) { return in ? rate_at(a.rate + c + j) : 0.f; });
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
        if (t.tt > 0) h = load_channels<V>(a.carry + ((long)t.b * a.tiles + t.tt) * a.channels, c, a.channels);
        else if (a.initial) h = load_channels<V>(a.initial + (long)t.b * a.channels, c, a.channels);
#pragma unroll
        for (int l = 0; l < BL; ++l) {
            rv[l] = sigmoid(wr[l].get()), iv[l] = sigmoid(wi[l].get());
            const Decay<V> d = decay_of(rate * rv[l]);
            av[l] = d.a;
            hb[l] = H;
            H = fma(av[l], H, root(d.w) * iv[l] * wx[l].get());
            A = A * av[l];
        }
    }
#pragma unroll
    for (int l = BL - 1; l >= 0; --l) D = av[l] * (wg[l].get() + D);
    // the states: maps of the warps in front
    sh.A[warp][lane] = A, sh.H[warp][lane] = H;
    __syncthreads();
    for (int w = 0; w < warp; ++w) h = fma(sh.A[w][lane], h, sh.H[w][lane]);
    __syncthreads();
    // the gradients: maps of the warps behind
    F<V> pa(1.f), pd(0.f), g(0.f);
    sh.H[warp][lane] = D;
    __syncthreads();
    for (int w = warps - 1; w > warp; --w) {
        const F<V> m = sh.A[w][lane];
        pa = pa * m;
        pd = fma(m, pd, sh.H[w][lane]);
    }
    const F<V> ta = A * pa, td = fma(A, pd, D);
    if (t.tt == a.tiles - 1) {
        if (a.dfinal) g = load_channels<V>(a.dfinal + (long)t.b * a.channels, c, a.channels);
    } else {
        if (warp == 0) publish_map<T, V>(a, t, lane, ta, td);
        __syncthreads();
        if (!look_back<T, V>(a, t, true, sh, warp, lane, warps, &g)) {
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
#pragma unroll
    for (int l = 0; l < BL; ++l) {
        hb[l] = hb[l] + h;
        h = av[l] * h;
    }
    F<V> sum(0.f);
    const F<V> minus(-1.f), one(1.f);
    const long at = ((long)t.b * a.steps + from + BL - 1) * a.channels + c;
    T *ox = a.dx + at, *od = a.ddecay + at, *oi = a.dgate + at;
#pragma unroll
    for (int l = BL - 1; l >= 0; --l) {
        const F<V> e = av[l], r = rv[l], i = iv[l];
        const F<V> w = rest_of(rate * r, e);  // formed again: kept, it would take too many registers
        // no step of the clock: the state passes, whatever the input
        const F<V> inv = w.each([](float x) { return fabsf(x) < FLT_MIN ? 0.f : inverse_root(x); });
        g = g + wg[l].get();
        const F<V> ix = i * wx[l].get(), gm = g * (w * inv);
        const F<V> rd = r * g * fma(e * e * inv * ix, minus, e * hb[l]);
        if (l < rows) {
            const bool there = l < live;
            Word<T, V>::store(ox, there ? gm * i : F<V>(0.f));
            Word<T, V>::store(oi, there ? gm * ix * fma(i, minus, one) : F<V>(0.f));
            Word<T, V>::store(od, there ? rate * rd * fma(r, one, minus) : F<V>(0.f));
        }
        ox -= a.channels, od -= a.channels, oi -= a.channels;
        sum = fma(rd, minus, sum);
        g = e * g;
    }
    if (a.drate_part) {  // of the tile, the warps in order
        __syncthreads();
        sh.H[warp][lane] = sum;
        __syncthreads();
        if (warp == 0) {
            F<V> s(0.f);
            for (int w = 0; w < warps; ++w) s = s + sh.H[w][lane];
            store_channels<V>(a.drate_part + ((long)t.b * a.tiles + t.tt) * a.channels, c, a.channels, s);
        }
    }
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
            const Decay<1> d = decay_of(F<1>(k[j]) * sigmoid(F<1>(r[j])));
            o[j] = fma(d.a, F<1>(h[j]), root(d.w) * sigmoid(F<1>(i[j])) * F<1>(x[j])).r;
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
    if (a->dtype != EWS_DTYPE_F32 && a->dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    return EWS_OK;
}

size_t up(size_t b) { return (b + 255) / 256 * 256; }
int tiles_of(int steps, bool bwd) { return (steps + (bwd ? BT : FT) - 1) / (bwd ? BT : FT); }

struct Sizes {
    size_t flags, maps, ends, part, bytes;
};

// The flags lie behind the status block, counted for one channel a lane (the narrowest tile).
Sizes sizes(const ews_recur_args* a, bool bwd) {
    Sizes z{};
    const size_t tiles = tiles_of(a->steps, bwd), states = (size_t)a->batch * tiles * a->channels;
    if (tiles > 1) {
        z.flags = up(sizeof(DeviceStatus) + sizeof(int) * (size_t)a->batch * tiles * ((a->channels + 31) / 32));
        z.maps = up(2 * sizeof(float) * states), z.ends = up(sizeof(float) * states);
    }
    if (bwd) z.part = up(sizeof(float) * states);
    z.bytes = z.flags + z.maps + z.ends + z.part;
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

template <typename T>
int run(const ews_recur_args* a, bool bwd, cudaStream_t s) {
    Params<T> p{};
    p.batch = a->batch, p.steps = a->steps, p.channels = a->channels, p.tiles = tiles_of(a->steps, bwd);
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
    const int width = pairs ? 64 : 32;
    p.blocks = (a->channels + width - 1) / width;
    const Sizes z = sizes(a, bwd);
    char* w = static_cast<char*>(a->work);
    if (p.tiles > 1) {
        p.st = reinterpret_cast<DeviceStatus*>(w);
        p.flags = reinterpret_cast<int*>(w + sizeof(DeviceStatus));
        p.map_a = reinterpret_cast<float*>(w + z.flags);
        p.map_h = p.map_a + (size_t)a->batch * p.tiles * a->channels;
        p.ends = reinterpret_cast<float*>(w + z.flags + z.maps);
        if (cudaMemsetAsync(w, 0, z.flags, s) != cudaSuccess) return EWS_ERR_LAUNCH;
    }
    if (bwd && a->drate) p.drate_part = reinterpret_cast<float*>(w + z.flags + z.maps + z.ends);
    const long ctas = (long)p.batch * p.blocks * p.tiles;
    if (ctas > 0x7FFFFFFFl) return EWS_ERR_UNSUPPORTED;
    const int per = bwd ? BL : FL;
    const int warps = p.tiles > 1 ? (bwd ? BW : FW) : (a->steps + per - 1) / per;  // a short axis: as many as it has work for
    auto go = [&](auto* kernel) {
        kernel<<<(unsigned)ctas, warps * 32, 0, s>>>(p);
        return cudaGetLastError() == cudaSuccess ? (int)EWS_OK : (int)EWS_ERR_LAUNCH;
    };
    int rc;
    if constexpr (sizeof(T) == 2) {
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
    return check(a) == EWS_OK ? sizeof(float) * (size_t)a->batch * tiles_of(a->steps, true) * a->channels : 0;
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
    if (tiles_of(a->steps, true) > 1 && !a->carry) return EWS_ERR_INVALID_ARGUMENT;
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
