// Linear attention with a decay per head: prompts and training (chunks), and single tokens (a state).
//
//     S_t = g S_{t-1} + k_t v_t^T,    o_t = scale q_t S_t,    g = exp(-rate_h),
//
// the depth-one exponentially weighted state of the pair (k, v) with a unit clock. Every product here is one and
// the same chain over three streams x, y (dx wide) and z (dz wide),
//
//     out_p = oscale x_p State_p,    State_p = g State_{p-1} + y_p z_p^T,
//
// run over the tokens forwards or backwards: forward (x, y, z) = (q, k, v); dq = (dout, v, k) with the transposed
// state; and from the end, with R_t = q_t dout_t^T + g R_{t+1}, dv = (k, q, dout) and dk = (v, dout, q).
// Backwards the carried value is E = g R of the token behind, so that the last state's gradient enters
// unweighted: a row's weight of the carry is g^i, not g^(i+1), an update's g^(n-j), not g^(n-1-j).
//
// Which form runs: bfloat16 streams that TMA can read (16-byte-aligned rows and strides) run in ews_decay_tc.cu, float32
// with x and y up to 64 wide in ews_decay_f32.cu, both on the 5th-generation tensor core; the rest (odd bfloat16 widths and
// strides, wide float32 heads) here, on warp-level matrix instructions. Both sides of each rule, forward and backward:
// bfloat16 B = 8, T = 2048, 16 heads of 128: 274 us there, 857 here; float32 B = 16, T = 1440, 8 heads of 64, shared in
// pairs, ragged: 517 us there, 1,717 here. What bounds this form is the legacy instructions' rate (2,048 operations a
// cycle and SM) and the splitting of float32 fragments, each of which four warps repeat.
//
// chain_kernel: a CTA of four warps owns a (sample, head, segment of the axis, slice of up to 64 columns of z); it walks
// its segment in chunks of 64 tokens with the state in registers (float32). Within a chunk out = P Z + diag(g^(i+1)) X State,
// P = (X Y^T) * g^(i-j) for j <= i: warp-level matrix instructions, P straight from the accumulators to operand
// fragments, the state rounded to the operand type for its product alone. The update (g^(n-1-j) y_j) z_j^T splits
// the weighted operand into `NS` bfloat16 pieces: the weight makes it inexact, and the state is a float32 result
// (three pieces: 2^-24) or feeds a rounded output (two: 2^-16). float32 operands run as 3xTF32.
// When (sample, head, slice) alone cannot fill the GPU, the axis is split: a state-only pass gives each
// segment's own state, join_kernel chains them, and the segments run side by side from their states.
// Rows at or beyond a sample's length are neither loaded nor multiplied; their outputs are zero.
#include <cfloat>

#include "ews_decay.cuh"

namespace ews {
namespace decay {

constexpr int C = 64;      // tokens of a chunk
constexpr int NT = 128;    // threads: four warps of 16 rows
constexpr int MAXD = 128;  // widest head

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void cp16(void* s, const void* g, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(s)), "l"(g), "r"(in ? 16 : 0) : "memory");
}

// ---- operand fragments -------------------------------------------------------------------------------------
// A: 16 x KS, B: KS x 16 (two instruction tiles of 8 columns). c = lane % 4, r = lane / 4.

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t r[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
__device__ __forceinline__ void mma_bf16(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T>
struct Tc;

template <>
struct Tc<bf16> {
    static constexpr int KS = 16, PAD = 8;
    struct A {
        uint32_t r[4];
    };
    struct B {
        uint32_t r[4];
    };
    template <int NS>
    struct AW {
        uint32_t r[NS][4];
    };
    // rows of a [m][k] tile
    __device__ static __forceinline__ A a_mk(const bf16* t, int ld, int m0, int k0) {
        const int l = threadIdx.x & 31;
        A a;
        ldsm4(a.r, smem_u32(t + (m0 + (l & 15)) * ld + k0 + (l >> 4) * 8));
        return a;
    }
    // 16 columns from a [n][k] tile
    __device__ static __forceinline__ B b_nk(const bf16* t, int ld, int n0, int k0) {
        const int l = threadIdx.x & 31;
        B b;
        ldsm4(b.r, smem_u32(t + (n0 + (l & 7) + ((l >> 4) << 3)) * ld + k0 + ((l >> 3) & 1) * 8));
        return b;
    }
    // 16 columns from a [k][n] tile
    __device__ static __forceinline__ B b_kn(const bf16* t, int ld, int k0, int n0) {
        const int l = threadIdx.x & 31;
        B b;
        ldsm4t(b.r, smem_u32(t + (k0 + (l & 7) + ((l >> 3) & 1) * 8) * ld + n0 + ((l >> 4) << 3)));
        return b;
    }
    // accumulator tiles (16 x 8 each) starting at column k0 as an operand
    __device__ static __forceinline__ A a_acc(const float (*p)[4], int k0) {
        const float* u = p[k0 / 8];
        const float* w = p[k0 / 8 + 1];
        A a;
        a.r[0] = pack_bf16(u[0], u[1]), a.r[1] = pack_bf16(u[2], u[3]);
        a.r[2] = pack_bf16(w[0], w[1]), a.r[3] = pack_bf16(w[2], w[3]);
        return a;
    }
    // the transpose of a [k][m] tile, row k weighted by wt[k], in NS pieces
    template <int NS>
    __device__ static __forceinline__ AW<NS> a_km(const bf16* t, int ld, int k0, int m0, const float* wt) {
        const int l = threadIdx.x & 31, c = l & 3;
        uint32_t raw[4];
        ldsm4t(raw, smem_u32(t + (k0 + (l & 7) + ((l >> 4) << 3)) * ld + m0 + ((l >> 3) & 1) * 8));
        AW<NS> a;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float* w = wt + k0 + 2 * c + (q >> 1) * 8;
            float f0 = bf16_lo(raw[q]) * w[0], f1 = bf16_hi(raw[q]) * w[1];
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const uint32_t u = pack_bf16(f0, f1);
                a.r[s][q] = u;
                f0 -= bf16_lo(u), f1 -= bf16_hi(u);
            }
        }
        return a;
    }
    static constexpr bool SMALL = false;
    __device__ static __forceinline__ void mma2(float d0[4], float d1[4], float*, float*, const A& a, const B& b) {
        mma_bf16(d0, a.r, b.r[0], b.r[1]);
        mma_bf16(d1, a.r, b.r[2], b.r[3]);
    }
    template <int NS>
    __device__ static __forceinline__ void mma2w(float d0[4], float d1[4], float*, float*, const AW<NS>& a, const B& b) {
#pragma unroll
        for (int s = NS - 1; s >= 0; --s) {
            mma_bf16(d0, a.r[s], b.r[0], b.r[1]);
            mma_bf16(d1, a.r[s], b.r[2], b.r[3]);
        }
    }
};

// float32 as 3xTF32: each operand in two tf32 pieces, the product of the two small ones left out (2^-22). An
// instruction's k columns c and c + 4 stand for the tile's columns 2c and 2c + 1 on both operands, so a lane's two
// values are neighbours and an accumulator tile is an operand as it stands.
template <>
struct Tc<float> {
    static constexpr int KS = 8, PAD = 4;
    struct A {
        uint32_t h[4], l[4];
    };
    using B = A;
    template <int NS>
    using AW = A;
    __device__ static __forceinline__ uint32_t tf32(float x) { return (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u; }
    __device__ static __forceinline__ void split(float x, uint32_t& h, uint32_t& l) {
        h = tf32(x);
        l = tf32(x - __uint_as_float(h));
        if (!(fabsf(x) < 3.0e38f)) h = __float_as_uint(x), l = 0;  // no rounding past the largest value, none of inf and NaN
    }
    __device__ static __forceinline__ A of(float a, float b, float c, float d) {
        A f;
        split(a, f.h[0], f.l[0]), split(b, f.h[1], f.l[1]), split(c, f.h[2], f.l[2]), split(d, f.h[3], f.l[3]);
        return f;
    }
    __device__ static __forceinline__ A a_mk(const float* t, int ld, int m0, int k0) {
        const int l = threadIdx.x & 31, c = l & 3, r = l >> 2;
        const float2 u = *reinterpret_cast<const float2*>(t + (m0 + r) * ld + k0 + 2 * c);
        const float2 w = *reinterpret_cast<const float2*>(t + (m0 + r + 8) * ld + k0 + 2 * c);
        return of(u.x, w.x, u.y, w.y);
    }
    __device__ static __forceinline__ B b_nk(const float* t, int ld, int n0, int k0) {
        const int l = threadIdx.x & 31, c = l & 3, r = l >> 2;
        const float2 u = *reinterpret_cast<const float2*>(t + (n0 + r) * ld + k0 + 2 * c);
        const float2 w = *reinterpret_cast<const float2*>(t + (n0 + r + 8) * ld + k0 + 2 * c);
        return of(u.x, u.y, w.x, w.y);
    }
    __device__ static __forceinline__ B b_kn(const float* t, int ld, int k0, int n0) {
        const int l = threadIdx.x & 31, c = l & 3, r = l >> 2;
        const float* a = t + (k0 + 2 * c) * ld + n0 + r;
        return of(a[0], a[ld], a[8], a[ld + 8]);
    }
    __device__ static __forceinline__ A a_acc(const float (*p)[4], int k0) {
        const float* u = p[k0 / 8];
        return of(u[0], u[2], u[1], u[3]);
    }
    template <int NS>
    __device__ static __forceinline__ A a_km(const float* t, int ld, int k0, int m0, const float* wt) {
        const int l = threadIdx.x & 31, c = l & 3, r = l >> 2;
        const float* a = t + (k0 + 2 * c) * ld + m0 + r;
        const float w0 = wt[k0 + 2 * c], w1 = wt[k0 + 2 * c + 1];
        return of(a[0] * w0, a[8] * w0, a[ld] * w1, a[ld + 8] * w1);
    }
    // The small products have an accumulator of their own: every addition to the large one truncates.
    static constexpr bool SMALL = true;
    __device__ static __forceinline__ void mma2(float d0[4], float d1[4], float c0[4], float c1[4], const A& a, const B& b) {
        mma_tf32(c0, a.l, b.h[0], b.h[1]);
        mma_tf32(c1, a.l, b.h[2], b.h[3]);
        mma_tf32(c0, a.h, b.l[0], b.l[1]);
        mma_tf32(c1, a.h, b.l[2], b.l[3]);
        mma_tf32(d0, a.h, b.h[0], b.h[1]);
        mma_tf32(d1, a.h, b.h[2], b.h[3]);
    }
    template <int NS>
    __device__ static __forceinline__ void mma2w(float d0[4], float d1[4], float c0[4], float c1[4], const A& a, const B& b) {
        mma2(d0, d1, c0, c1, a, b);
    }
};

// ---- shared memory ------------------------------------------------------------------------------------------

template <typename T, int DK, int DV, bool STATE>
struct Smem {
    static constexpr int PAD = Tc<T>::PAD, LK = DK + PAD, LV = DV + PAD;
    static constexpr int X = STATE ? 0 : C * LK, Y = C * LK, Z = C * LV, STAGE = X + Y + Z;
    static constexpr int ST = STATE ? 0 : DK * LV;
    static constexpr size_t bytes = sizeof(T) * (2 * STAGE + ST) + sizeof(float) * (C + 4 + C);
};

// 64 rows of a stream from processed position p0, columns [c0, c0 + W), into a [64][ld] tile; what lies at or
// beyond `len` or the stream's width becomes zero.
template <typename T, int W>
__device__ __forceinline__ void load_tile(T* tile, int ld, const Stream<T>& s, const T* base, long p0, long len, int rev, int c0) {
    constexpr int E = 16 / sizeof(T), PER = W / E;
    if (s.vec) {
#pragma unroll
        for (int i = 0; i < C * PER / NT; ++i) {
            const int e = i * NT + threadIdx.x, row = e / PER, col = (e % PER) * E;
            const long p = p0 + row;
            const bool in = p < len && c0 + col < s.width;
            const T* g = in ? base + (rev ? len - 1 - p : p) * s.st + c0 + col : base;
            cp16(tile + row * ld + col, g, in);
        }
    } else {
        for (int e = threadIdx.x; e < C * W; e += NT) {
            const int row = e / W, col = e % W;
            const long p = p0 + row;
            T v = from_f<T>(0.f);
            if (p < len && c0 + col < s.width) v = base[(rev ? len - 1 - p : p) * s.st + c0 + col];
            tile[row * ld + col] = v;
        }
    }
}

template <typename T, int DK, int DV, int NS, bool STATE>
__global__ void __launch_bounds__(NT) chain_kernel(const __grid_constant__ Chain<T> a) {
    using M = Tc<T>;
    using S = Smem<T, DK, DV, STATE>;
    constexpr int WM = DK >= 64 ? 4 : DK / 16, WN = 4 / WM, MT = DK / 16 / WM, NTL = DV / 8 / WN;
    extern __shared__ __align__(16) unsigned char raw[];
    T* stage = reinterpret_cast<T*>(raw);
    T* st = stage + 2 * S::STAGE;
    float* pw = reinterpret_cast<float*>(st + S::ST);  // g^0 .. g^64
    float* wt = pw + C + 4;                            // the update's weights
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = lane & 3, r = lane >> 2;

    long u = blockIdx.x;
    const int slice = (int)(u % a.slices);
    u /= a.slices;
    const int seg = (int)(u % a.segs);
    const long bh = u / a.segs;
    const int b = (int)(bh / a.heads), h = (int)(bh - (long)b * a.heads);
    const int c0 = slice * DV;
    if (STATE && !a.fin && seg == a.segs - 1) return;  // no segment starts from it
    const long len = a.lengths ? min(max(a.lengths[b], 0), a.steps) : a.steps;
    const long p0 = (long)seg * a.span, p1 = min(p0 + (long)a.span, (long)a.steps);
    const int dx = a.y.width, dz = a.z.width;
    const T* xb = STATE ? nullptr : a.x.p + b * a.x.sb + (h / a.x.group) * a.x.sh;
    const T* yb = a.y.p + b * a.y.sb + (h / a.y.group) * a.y.sh;
    const T* zb = a.z.p + b * a.z.sb + (h / a.z.group) * a.z.sh;
    const float rate = a.rate[h];
    if (tid <= C) pw[tid] = tid == 0 ? 1.f : expf(-rate * (float)tid);

    const long end = min(p1, len);  // this segment's tokens are [p0, end)
    // the state: rows (wm * MT + i) * 16 + r (+ 8), columns (wn * NTL + j) * 8 + 2 c (+ 1)
    const int wm = warp % WM, wn = warp / WM;
    float s[MT][NTL][4];
    const float* init = nullptr;
    long ir = 0, ic = 0;
    float iscale = 1.f;
    if (!STATE) {
        if (a.segs > 1) init = a.seg + (bh * a.segs + seg) * (long)dx * dz, ir = dz, ic = 1;
        else if (a.init) init = a.init + bh * (long)dx * dz, ir = a.init_r, ic = a.init_c, iscale = a.init_scale;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = (wm * MT + i) * 16 + r + (e >> 1) * 8, col = c0 + (wn * NTL + j) * 8 + 2 * c + (e & 1);
                s[i][j][e] = init && row < dx && col < dz ? init[row * ir + col * ic] * iscale : 0.f;
            }
    auto put_state = [&]() {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    T* q = st + ((wm * MT + i) * 16 + r + (e >> 1) * 8) * S::LV + (wn * NTL + j) * 8 + 2 * c;
                    q[0] = from_f<T>(s[i][j][e]), q[1] = from_f<T>(s[i][j][e + 1]);
                }
    };
    if (!STATE) put_state();

    auto fetch = [&](long p, int k) {
        T* t = stage + k * S::STAGE;
        if (!STATE) load_tile<T, DK>(t, S::LK, a.x, xb, p, len, a.rev, 0);
        load_tile<T, DK>(t + S::X, S::LK, a.y, yb, p, len, a.rev, 0);
        load_tile<T, DV>(t + S::X + S::Y, S::LV, a.z, zb, p, len, a.rev, c0);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int k = 0;
    if (p0 < end) fetch(p0, 0);
    for (long p = p0; p < end; p += C, k ^= 1) {
        const int n = (int)min((long)C, end - p);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the chunk and the state are in place, and the chunk before is done with its buffers
        if (p + C < end) fetch(p + C, k ^ 1);
        if (tid < C) wt[tid] = tid < n ? pw[n - 1 - tid + (a.rev ? 1 : 0)] : 0.f;
        const T* X = stage + k * S::STAGE;
        const T* Y = X + S::X;
        const T* Z = Y + S::Y;
        if (!STATE) {
            const int m0 = warp * 16;
            float o[DV / 8][4];
#pragma unroll
            for (int j = 0; j < DV / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            float pr[C / 8][4];
#pragma unroll
            for (int j = 0; j < C / 8; ++j) pr[j][0] = pr[j][1] = pr[j][2] = pr[j][3] = 0.f;
            float os[M::SMALL ? DV / 8 : 2][4] = {}, ps[M::SMALL ? C / 8 : 2][4] = {};  // the small products' sums
            constexpr int O1 = M::SMALL ? 1 : 0;
#pragma unroll
            for (int kk = 0; kk < DK; kk += M::KS) {
                const typename M::A xa = M::a_mk(X, S::LK, m0, kk);
#pragma unroll
                for (int j = 0; j < C / 16; ++j)
                    if (j <= warp) M::mma2(pr[2 * j], pr[2 * j + 1], ps[2 * j * O1], ps[2 * j * O1 + 1], xa, M::b_nk(Y, S::LK, 16 * j, kk));
#pragma unroll
                for (int j = 0; j < DV / 16; ++j)
                    M::mma2(o[2 * j], o[2 * j + 1], os[2 * j * O1], os[2 * j * O1 + 1], xa, M::b_kn(st, S::LV, kk, 16 * j));
            }
            const int shift = a.rev ? 0 : 1;
            const float w0 = pw[m0 + r + shift], w1 = pw[m0 + r + 8 + shift];
#pragma unroll
            for (int j = 0; j < DV / 8; ++j) {
                o[j][0] *= w0, o[j][1] *= w0, o[j][2] *= w1, o[j][3] *= w1;
                if constexpr (M::SMALL) os[j][0] *= w0, os[j][1] *= w0, os[j][2] *= w1, os[j][3] *= w1;
            }
#pragma unroll
            for (int j = 0; j < C / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int gap = m0 + r + (e >> 1) * 8 - (8 * j + 2 * c + (e & 1));
                    if constexpr (M::SMALL) pr[j][e] += ps[j][e];
                    pr[j][e] = gap >= 0 ? pr[j][e] * pw[gap] : 0.f;
                }
#pragma unroll
            for (int kk = 0; kk < C; kk += M::KS)
                if (kk < m0 + 16) {
                    const typename M::A pa = M::a_acc(pr, kk);
#pragma unroll
                    for (int j = 0; j < DV / 16; ++j)
                        M::mma2(o[2 * j], o[2 * j + 1], os[2 * j * O1], os[2 * j * O1 + 1], pa, M::b_kn(Z, S::LV, kk, 16 * j));
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = m0 + r + 8 * e;
                if (row >= n) continue;
                const long t = a.rev ? len - 1 - (p + row) : p + row;
                const long at = (((long)b * a.steps + t) * a.heads + h) * dz + c0;
#pragma unroll
                for (int j = 0; j < DV / 8; ++j)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int col = 8 * j + 2 * c + q;
                        if (c0 + col >= dz) continue;
                        const float val = (M::SMALL ? o[j][2 * e + q] + os[j * O1][2 * e + q] : o[j][2 * e + q]) * a.oscale;
                        if (a.out32) a.out32[at + col] = val;
                        else a.out[at + col] = from_f<T>(val);
                    }
            }
        }
        __syncthreads();  // the update's weights are in place, and the state's operand is free
        const float gn = pw[n];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            float add[NTL][4], as[M::SMALL ? NTL : 2][4] = {};
            constexpr int A1 = M::SMALL ? 1 : 0;
#pragma unroll
            for (int j = 0; j < NTL; ++j) add[j][0] = add[j][1] = add[j][2] = add[j][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < C; kk += M::KS) {
                const auto ya = M::template a_km<NS>(Y, S::LK, kk, (wm * MT + i) * 16, wt);
#pragma unroll
                for (int j = 0; j < NTL; j += 2)
                    M::template mma2w<NS>(add[j], add[j + 1], as[j * A1], as[j * A1 + 1], ya, M::b_kn(Z, S::LV, kk, (wn * NTL + j) * 8));
            }
#pragma unroll
            for (int j = 0; j < NTL; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i][j][e] = fmaf(gn, s[i][j][e], M::SMALL ? add[j][e] + as[j * A1][e] : add[j][e]);
        }
        if (!STATE) put_state();
    }
    float* fin = nullptr;
    long fr = 0, fc = 0;
    float fscale = 1.f;
    if (STATE) fin = a.seg + (bh * a.segs + seg) * (long)dx * dz, fr = dz, fc = 1;
    else if (a.segs == 1 && a.fin) fin = a.fin + bh * (long)dx * dz, fr = a.fin_r, fc = a.fin_c, fscale = a.fin_scale;
    if (fin) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = (wm * MT + i) * 16 + r + (e >> 1) * 8, col = c0 + (wn * NTL + j) * 8 + 2 * c + (e & 1);
                    if (row < dx && col < dz) fin[row * fr + col * fc] = s[i][j][e] * fscale;
                }
    }
    if (!STATE) {
        // positions without a token
        const int w = min(DV, dz - c0);
        for (long e = tid; e < (p1 - max(p0, end)) * w; e += NT) {
            const long t = max(p0, end) + e / w;
            const long at = (((long)b * a.steps + t) * a.heads + h) * dz + c0 + e % w;
            if (a.out32) a.out32[at] = 0.f;
            else a.out[at] = from_f<T>(0.f);
        }
    }
}

// Chains the segments' own states into their starting states, one thread per state entry: the tail of a reversed
// axis is a short last segment, so each segment's decay counts its own tokens.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Chain<T> a) {
    const int dx = a.y.width, dz = a.z.width;
    const long per = (long)dx * dz;
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    if (e >= per * a.batch * a.heads) return;
    const long bh = e / per, i = (e - bh * per) / dz, j = e % dz;
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    const long len = a.lengths ? min(max(a.lengths[b], 0), a.steps) : a.steps;
    const long span = a.span;
    const float rate = a.rate[h];
    float s = a.init ? a.init[bh * per + i * a.init_r + j * a.init_c] * a.init_scale : 0.f;
    float* p = a.seg + bh * a.segs * per + i * dz + j;
    const long step = a.down ? -per : per;
    p += a.down ? (a.segs - 1) * per : 0;
    float next = *p;
    for (int k = 0; k < a.segs; ++k, p += step) {
        const float own = next;
        if (k + 1 < a.segs) next = p[step];  // on its way while this one is chained
        *p = s;
        const int g = a.down ? a.segs - 1 - k : k;
        const long n = min(max(len - g * span, 0l), span);
        if (n > 0) s = fmaf(expf(-rate * (float)n), s, own);
    }
    if (a.fin) a.fin[bh * per + i * a.fin_r + j * a.fin_c] = s * a.fin_scale;
}

// Sums the float32 gradients of the query heads that share a key/value head, in head order: a thread a vector of one
// head, the vectors of a row side by side.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) group_kernel(const float* __restrict__ in, long rows, int kv, int group, int d,
                                                    T* __restrict__ out) {
    constexpr int W = VEC ? 4 : 1;
    const int per = d / W;
    const long total = rows * kv * per;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        const long rk = e / per;
        const int c = (int)(e - rk * per) * W;
        const float* p = in + rk * group * d + c;
        float s[W];
        Vec<float, VEC>::load(p, s);
        for (int g = 1; g < group; ++g) {
            float v[W];
            Vec<float, VEC>::load(p + (long)g * d, v);
#pragma unroll
            for (int j = 0; j < W; ++j) s[j] += v[j];
        }
        T* o = out + rk * d + c;
        if constexpr (VEC && sizeof(T) == 2) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
        else Vec<T, VEC>::store(o, s);
    }
}

// ---- one token per row ----------------------------------------------------------------------------------------
// A CTA owns 64 columns of one (row, head) state: 16 lanes of four columns by 16 groups of state rows; each thread
// reads, decays, updates and writes its part of the state once and sums its rows of q S; the groups' sums meet in
// shared memory. Bound by HBM (8 bytes a state entry) for full batches and by one trip to memory for few rows: 256 rows of
// 16 heads of 128 x 128 (530 MB) take 96 us, 5.5 TB/s (on 32 columns a CTA 110 us); 8 heads of 64 x 64 take 6 us.
constexpr int STEP_T = 256, STEP_COLS = 64;

template <typename T>
struct Step {
    const T *q, *k, *v;
    long qb, qh, kb, kh, vb, vh;  // element strides of rows and heads
    const float* rate;
    const int* slots;
    float* state;
    T* out;
    int batch, heads, group, dk, dv, pool, slices;
    float scale;
    int* status;
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(STEP_T) step_kernel(const __grid_constant__ Step<T> a) {
    constexpr int W = VEC ? 4 : 1, LANES = STEP_COLS / W, GROUPS = STEP_T / LANES;
    __shared__ float red[GROUPS][STEP_COLS + 1];
    long u = blockIdx.x;
    const int slice = (int)(u % a.slices);
    u /= a.slices;
    const int h = (int)(u % a.heads), b = (int)(u / a.heads);
    const int tid = threadIdx.x, g = tid / LANES, l = tid % LANES;
    const int col = slice * STEP_COLS + l * W;
    T* out = a.out + ((long)b * a.heads + h) * a.dv;
    int slot = a.slots ? a.slots[b] : b;
    if (slot < 0 || slot >= a.pool) {
        if (slot >= a.pool && tid == 0) report(a.status, EWS_ERR_INDEX);
        const int o = slice * STEP_COLS + tid;
        if (tid < STEP_COLS && o < a.dv) out[o] = from_f<T>(0.f);
        return;
    }
    const float decay = expf(-a.rate[h]);
    const T* q = a.q + b * a.qb + h * a.qh;
    const T* k = a.k + b * a.kb + (h / a.group) * a.kh;
    const T* v = a.v + b * a.vb + (h / a.group) * a.vh;
    float* st = a.state + ((long)slot * a.heads + h) * a.dk * a.dv + col;
    float vv[W], acc[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        acc[w] = 0.f;
        vv[w] = col + w < a.dv ? to_f(v[col + w]) : 0.f;
    }
    if (col < a.dv) {
#pragma unroll 4
        for (int i = g; i < a.dk; i += GROUPS) {
            float x[W];
            Vec<float, VEC>::load(st + (long)i * a.dv, x);
            const float ki = to_f(k[i]), qi = to_f(q[i]);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                x[w] = fmaf(decay, x[w], ki * vv[w]);
                acc[w] = fmaf(qi, x[w], acc[w]);
            }
            Vec<float, VEC>::store(st + (long)i * a.dv, x);
        }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) red[g][l * W + w] = acc[w];
    __syncthreads();
    if (tid < STEP_COLS && slice * STEP_COLS + tid < a.dv) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) s += red[i][tid];
        out[slice * STEP_COLS + tid] = from_f<T>(s * a.scale);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------

int pad_width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

// Segments of the axis: as many as two CTAs on each of 148 SMs, but none shorter than four chunks, since each
// costs a second reading of y and z and a state.
void plan(int batch, int steps, int heads, int dz, int width, int* slices, int* segs, int* span) {
    *slices = (dz + width - 1) / width;
    const long ctas = (long)batch * heads * *slices;
    const int chunks = steps > 0 ? (steps + C - 1) / C : 1;
    long want = ctas >= 148 ? 1 : (296 + ctas - 1) / ctas;
    if (want > chunks / 4) want = chunks / 4;
    if (want < 1) want = 1;
    const int per = (int)((chunks + want - 1) / want);
    *span = per * C;
    *segs = (chunks + per - 1) / per;
}

// Columns of z a CTA takes: the float32 form's two sums of a wide product leave room for 32.
constexpr int slice_width(bool f32) { return f32 ? 32 : 64; }

// The segments' states, for whichever form runs (a state in full precision needs its pass even over one segment).
size_t seg_bytes(const ews_decay_args* a, int dx, int dz) {
    const bool f32 = a->dtype == EWS_DTYPE_F32;
    int slices, segs, span;
    if (f32 && dx <= F32_WIDE) segs = tc_segments(a->batch, a->steps, a->heads * ((dz + 63) / 64), false, &span);
    else plan(a->batch, a->steps, a->heads, dz, slice_width(f32), &slices, &segs, &span);
    if (segs == 1) segs = 0;
    if (!f32) {
        const int t = tc_segments(a->batch, a->steps, a->heads, true, &span);
        if (t > segs) segs = t;
        const int f = tc_segments(a->batch, a->steps, a->heads, false, &span);
        if (f > segs) segs = f;
    }
    return sizeof(float) * (size_t)a->batch * a->heads * segs * dx * dz;
}

template <typename T, int DK, int DV, int NS, bool STATE>
int launch(const Chain<T>& a, cudaStream_t s) {
    using S = Smem<T, DK, DV, STATE>;
    if (a.y.width > DK || a.z.width > a.slices * DV) return EWS_ERR_UNSUPPORTED;  // the plan's slices and the kernel's
    auto* kern = chain_kernel<T, DK, DV, NS, STATE>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::bytes) != cudaSuccess)
        return EWS_ERR_LAUNCH;
    const long ctas = (long)a.batch * a.heads * a.segs * a.slices;
    if (ctas > 0x7FFFFFFFl) return EWS_ERR_UNSUPPORTED;
    kern<<<(unsigned)ctas, NT, S::bytes, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T, int NS, bool STATE>
int launch_d(const Chain<T>& a, cudaStream_t s) {
    [[maybe_unused]] const int dk = pad_width(a.y.width);
    if constexpr (sizeof(T) == 4) {  // narrower x and y run in ews_decay_f32.cu, whatever the axis's length
        return launch<T, 128, slice_width(true), NS, STATE>(a, s);
    } else {
        if (a.z.width <= 32) {
            if (dk == 32) return launch<T, 32, 32, NS, STATE>(a, s);
            if (dk == 64) return launch<T, 64, 32, NS, STATE>(a, s);
            return launch<T, 128, 32, NS, STATE>(a, s);
        }
        if (dk == 32) return launch<T, 32, slice_width(false), NS, STATE>(a, s);
        if (dk == 64) return launch<T, 64, slice_width(false), NS, STATE>(a, s);
        return launch<T, 128, slice_width(false), NS, STATE>(a, s);
    }
}

template <typename T>
int join(const Chain<T>& a, cudaStream_t s) {
    const long total = (long)a.batch * a.heads * a.y.width * a.z.width;
    join_kernel<T><<<(unsigned)((total + 255) / 256), 256, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

// bfloat16 streams that TMA can read run on the tensor core's 5th-generation form. There a state that leaves in
// float32 takes the state pass (three pieces of the weighted operand) whatever the split.
int run_tc(Chain<bf16> a, cudaStream_t s) {
    a.segs = tc_segments(a.batch, a.steps, a.heads, a.fin != nullptr, &a.span);
    if (a.segs > 1 || a.fin) {
        if (!a.seg) return EWS_ERR_WORKSPACE;
        int rc = tc_chain(a, true, a.fin != nullptr, s);
        if (rc != EWS_OK) return rc;
        Chain<bf16> j = a;
        j.down = a.rev;
        if ((rc = join<bf16>(j, s)) != EWS_OK) return rc;
        a.fin = nullptr;
    }
    return tc_chain(a, false, false, s);
}

int run_f32(Chain<float> a, cudaStream_t s) {
    a.slices = (a.z.width + 63) / 64;
    a.segs = tc_segments(a.batch, a.steps, a.heads * a.slices, false, &a.span);
    if (a.segs > 1) {
        if (!a.seg) return EWS_ERR_WORKSPACE;
        int rc = f32_chain(a, true, s);
        if (rc != EWS_OK) return rc;
        Chain<float> j = a;
        j.down = a.rev;
        if ((rc = join<float>(j, s)) != EWS_OK) return rc;
    }
    return f32_chain(a, false, s);
}

// NS for a state that leaves the kernel in float32 is three, for one that only feeds rounded outputs two.
template <typename T>
int run_chain(Chain<T> a, cudaStream_t s) {
    constexpr bool f32 = sizeof(T) == 4;
    if constexpr (!f32) {
        if (tc_fits(a)) return run_tc(a, s);
    } else {
        if (f32_fits(a)) return run_f32(a, s);
    }
    plan(a.batch, a.steps, a.heads, a.z.width, slice_width(f32), &a.slices, &a.segs, &a.span);
    const bool exact = a.fin != nullptr && !f32;
    int rc;
    if (a.segs > 1) {
        if (!a.seg) return EWS_ERR_WORKSPACE;
        rc = exact ? launch_d<T, f32 ? 1 : 3, true>(a, s) : launch_d<T, f32 ? 1 : 2, true>(a, s);
        if (rc != EWS_OK || (rc = join<T>(a, s)) != EWS_OK) return rc;
        return launch_d<T, f32 ? 1 : 2, false>(a, s);
    }
    return exact ? launch_d<T, f32 ? 1 : 3, false>(a, s) : launch_d<T, f32 ? 1 : 2, false>(a, s);
}

template <typename T>
Stream<T> stream_of(const ews_decay_args* a, const void* p, const int64_t st[3], int group, int width) {
    Stream<T> s{};
    s.p = static_cast<const T*>(p);
    s.sb = st[0], s.st = st[1], s.sh = st[2];
    s.group = group, s.width = width;
    constexpr int E = 16 / sizeof(T);
    // an axis of one has no stride to speak of
    s.vec = aligned16(p) && width % E == 0 && (a->batch == 1 || s.sb % E == 0) && (a->steps == 1 || s.st % E == 0) &&
            (a->heads == group || s.sh % E == 0);
    return s;
}

int check(const ews_decay_args* a) {
    if (!a) return EWS_ERR_INVALID_ARGUMENT;
    if (a->batch < 0 || a->steps < 0 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads || a->dk <= 0 || a->dv <= 0)
        return EWS_ERR_INVALID_ARGUMENT;
    if (a->dk > MAXD || a->dv > MAXD) return EWS_ERR_UNSUPPORTED;
    if (a->dtype != EWS_DTYPE_F32 && a->dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    return EWS_OK;
}

size_t up(size_t b) { return (b + 255) / 256 * 256; }

struct Sizes {
    size_t seg, part, total;
};

Sizes sizes(const ews_decay_args* a, bool bwd) {
    Sizes z{};
    z.seg = up(seg_bytes(a, a->dk, a->dv));
    if (bwd) {
        const size_t t = up(seg_bytes(a, a->dv, a->dk));
        if (t > z.seg) z.seg = t;
        const int d = a->dk > a->dv ? a->dk : a->dv;
        if (a->heads != a->kv_heads) z.part = up(sizeof(float) * (size_t)a->batch * a->steps * a->heads * d);
    }
    z.total = z.seg + z.part;
    return z;
}

template <typename T>
Chain<T> base(const ews_decay_args* a) {
    Chain<T> c{};
    c.rate = a->rate, c.lengths = a->lengths;
    c.batch = a->batch, c.steps = a->steps, c.heads = a->heads;
    c.oscale = a->scale, c.init_scale = c.fin_scale = 1.f;
    c.seg = static_cast<float*>(a->work), c.status = a->status;
    return c;
}

template <typename T>
int forward(const ews_decay_args* a, cudaStream_t s) {
    const int group = a->heads / a->kv_heads;
    Chain<T> c = base<T>(a);
    c.x = stream_of<T>(a, a->q, a->q_stride, 1, a->dk);
    c.y = stream_of<T>(a, a->k, a->k_stride, group, a->dk);
    c.z = stream_of<T>(a, a->v, a->v_stride, group, a->dv);
    c.out = static_cast<T*>(a->out);
    c.init = a->initial, c.fin = a->final_state;
    c.init_r = c.fin_r = a->dv, c.init_c = c.fin_c = 1;
    return run_chain<T>(c, s);
}

template <typename T>
int backward(const ews_decay_args* a, const Sizes& z, cudaStream_t s) {
    const int group = a->heads / a->kv_heads;
    const auto q = stream_of<T>(a, a->q, a->q_stride, 1, a->dk);
    const auto k = stream_of<T>(a, a->k, a->k_stride, group, a->dk);
    const auto v = stream_of<T>(a, a->v, a->v_stride, group, a->dv);
    const auto g = stream_of<T>(a, a->dout, a->dout_stride, 1, a->dv);
    float* part = group > 1 ? reinterpret_cast<float*>(static_cast<char*>(a->work) + z.seg) : nullptr;
    const long rows = (long)a->batch * a->steps;
    auto sum = [&](int d, void* out) {
        if (!part) return (int)EWS_OK;
        const bool vec = d % 4 == 0 && aligned16(out);
        const long blocks = (rows * a->kv_heads * d / (vec ? 4 : 1) + 255) / 256;
        const unsigned grid = (unsigned)(blocks < 1 ? 1 : blocks < 148 * 64 ? blocks : 148 * 64);
        if (vec) group_kernel<T, true><<<grid, 256, 0, s>>>(part, rows, a->kv_heads, group, d, static_cast<T*>(out));
        else group_kernel<T, false><<<grid, 256, 0, s>>>(part, rows, a->kv_heads, group, d, static_cast<T*>(out));
        return cudaGetLastError() == cudaSuccess ? (int)EWS_OK : (int)EWS_ERR_LAUNCH;
    };
    // dq: forwards, the state transposed
    Chain<T> c = base<T>(a);
    c.x = g, c.y = v, c.z = k, c.out = static_cast<T*>(a->dq);
    c.init = a->initial, c.init_r = 1, c.init_c = a->dv;
    int rc = run_chain<T>(c, s);
    if (rc != EWS_OK) return rc;
    // dk and dv: from the end; the carried state is R / scale
    c = base<T>(a);
    c.rev = 1, c.init = a->dfinal, c.init_scale = 1.f / a->scale;
    c.x = v, c.y = g, c.z = q, c.out = part ? nullptr : static_cast<T*>(a->dk_out), c.out32 = part;
    c.init_r = 1, c.init_c = a->dv;
    if ((rc = run_chain<T>(c, s)) != EWS_OK || (rc = sum(a->dk, a->dk_out)) != EWS_OK) return rc;
    c.x = k, c.y = q, c.z = g, c.out = part ? nullptr : static_cast<T*>(a->dv_out);
    c.init_r = a->dv, c.init_c = 1;
    c.fin = a->dinitial, c.fin_scale = a->scale, c.fin_r = a->dv, c.fin_c = 1;
    if ((rc = run_chain<T>(c, s)) != EWS_OK) return rc;
    return sum(a->dv, a->dv_out);
}

template <typename T>
int step(const ews_decay_args* a, const int* slots, int pool, float* state, cudaStream_t s) {
    Step<T> p{};
    p.q = static_cast<const T*>(a->q), p.k = static_cast<const T*>(a->k), p.v = static_cast<const T*>(a->v);
    p.qb = a->q_stride[0], p.qh = a->q_stride[2], p.kb = a->k_stride[0], p.kh = a->k_stride[2];
    p.vb = a->v_stride[0], p.vh = a->v_stride[2];
    p.rate = a->rate, p.slots = slots, p.state = state, p.out = static_cast<T*>(a->out);
    p.batch = a->batch, p.heads = a->heads, p.group = a->heads / a->kv_heads, p.dk = a->dk, p.dv = a->dv;
    p.pool = pool, p.scale = a->scale, p.status = a->status;
    p.slices = (a->dv + STEP_COLS - 1) / STEP_COLS;
    const long ctas = (long)a->batch * a->heads * p.slices;
    if (ctas > 0x7FFFFFFFl) return EWS_ERR_UNSUPPORTED;
    if (a->dv % 4 == 0 && aligned16(state)) step_kernel<T, true><<<(unsigned)ctas, STEP_T, 0, s>>>(p);
    else step_kernel<T, false><<<(unsigned)ctas, STEP_T, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

}  // namespace decay
}  // namespace ews

using namespace ews::decay;

extern "C" size_t ews_decay_work_size(const ews_decay_args* a, int backward_pass) {
    return check(a) == EWS_OK && a->batch > 0 ? sizes(a, backward_pass != 0).total : 0;
}

extern "C" int ews_decay_fwd(const ews_decay_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    if (a->batch == 0) return EWS_OK;
    if (!a->rate || (a->steps > 0 && (!a->q || !a->k || !a->v || !a->out))) return EWS_ERR_INVALID_ARGUMENT;
    const Sizes z = sizes(a, false);
    if (z.total && (!a->work || a->work_bytes < z.total)) return EWS_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    return a->dtype == EWS_DTYPE_BF16 ? forward<bf16>(a, s) : forward<float>(a, s);
}

extern "C" int ews_decay_bwd(const ews_decay_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    if (a->batch == 0) return EWS_OK;
    if (!(fabsf(a->scale) >= FLT_MIN && fabsf(a->scale) <= FLT_MAX)) return EWS_ERR_INVALID_ARGUMENT;  // 1 / scale is used too
    if (!a->rate || (a->steps > 0 && (!a->q || !a->k || !a->v || !a->dout || !a->dq || !a->dk_out || !a->dv_out)))
        return EWS_ERR_INVALID_ARGUMENT;
    const Sizes z = sizes(a, true);
    if (z.total && (!a->work || a->work_bytes < z.total)) return EWS_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    return a->dtype == EWS_DTYPE_BF16 ? backward<bf16>(a, z, s) : backward<float>(a, z, s);
}

extern "C" int ews_decay_step(const ews_decay_args* a, const int* slots, int pool, float* state, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    if (a->batch == 0) return EWS_OK;
    if (!a->rate || !a->q || !a->k || !a->v || !a->out || !state || pool < 0 || (!slots && pool < a->batch))
        return EWS_ERR_INVALID_ARGUMENT;
    cudaStream_t s = (cudaStream_t)stream;
    return a->dtype == EWS_DTYPE_BF16 ? step<bf16>(a, slots, pool, state, s)
                                      : step<float>(a, slots, pool, state, s);
}
