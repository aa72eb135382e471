// The decayed attention's chain on the 5th-generation tensor core for float32 streams (the mathematics is in
// ews_decay.cu, the division of a chunk's work in ews_decay_tc.cu).
//
// A float32 is the sum of three bfloat16 (8 bits each), and a product of two takes six tensor-core products of
// planes (what is left out is below 2^-24), smallest first. The planes of x, y, the weighted y and z (three tiles of
// 128 x 64 each) and of the state fill shared memory, so x and y are at most 64 wide; z is taken in slices of 64
// columns. Group B reads the float32 rows with plain loads (any stride and alignment, a chunk ahead in registers),
// weights y before it is split, and writes the planes; the decayed scores are split by group A into three planes in
// tensor memory. Six products of 128 x 128 x 64 and three like it a chunk are about as long as the chunk's trip
// through HBM: neither bounds alone, the chain P -> scores -> output of one chunk after the other does.
#include "ews_decay.cuh"
#include "ews_tc.cuh"

namespace ews {
namespace decay {

using namespace tc5;

namespace {

constexpr int FC = 128, FW = 64;       // tokens of a chunk, columns of a tile
constexpr int PLANE = FC * 128;        // bytes of a plane of a stream, 128-byte rows
constexpr int SPLANE = FW * 128;       // of the state
constexpr int FTHR = 32 * 13;          // warps: MMA, four of group A, eight of group B
constexpr uint32_t TP = 0, TPP = 128, TO1 = 320, TO2 = 384, TU = 448;  // tensor-memory columns
constexpr int LX = 0, LY = LX + 3 * PLANE, LW = LY + 3 * PLANE, LZ = LW + 3 * PLANE, LS = LZ + 3 * PLANE, LBAR = LS + 3 * SPLANE,
              LPA = LBAR + 128, LPB = LPA + 4 * (FC + 4), LEND = LPB + 4 * (FC + 4);

struct Place {
    int b, h, seg, c0, dz;
    long bh;
    int t0, t1, end, chunks;
};

// Four neighbouring values into the three planes of a tile, at (row, 4 col4).
__device__ __forceinline__ void put4(unsigned char* tile, int plane, int row, int col4, float4 v) {
    unsigned char* p = tile + row * 128 + (((col4 >> 1) ^ (row & 7)) << 4) + (col4 & 1) * 8;
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        const uint32_t a = pack_bf16(v.x, v.y), b = pack_bf16(v.z, v.w);
        *reinterpret_cast<uint2*>(p + s * plane) = make_uint2(a, b);
        v.x -= bf16_lo(a), v.y -= bf16_hi(a), v.z -= bf16_lo(b), v.w -= bf16_hi(b);
    }
}

template <bool STATE>
__global__ void __launch_bounds__(FTHR, 1) f32_kernel(const __grid_constant__ Chain<float> a, int items) {
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + LBAR);
    uint64_t *xy_ready = bars, *z_ready = bars + 1, *p_full = bars + 2, *p_ready = bars + 3, *u_full = bars + 4, *o_full = bars + 5,
             *o_free = bars + 6, *drained = bars + 7, *sync_a = bars + 8, *sync_b = bars + 9;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 10);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_at + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int dx = a.y.width;

    if (threadIdx.x == 0) {
        mbar_init(p_full, 1), mbar_init(u_full, 1), mbar_init(o_full, 1), mbar_init(drained, 1);
        mbar_init(xy_ready, 256), mbar_init(z_ready, 256), mbar_init(p_ready, 128), mbar_init(o_free, 128);
        mbar_init(sync_a, 128), mbar_init(sync_b, 256);
        *fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_at;

    auto place = [&](int w) {
        Place it;
        const int slice = w % a.slices;
        w /= a.slices;
        it.seg = w % a.segs;
        it.bh = w / a.segs;
        it.b = (int)(it.bh / a.heads), it.h = (int)(it.bh - (long)it.b * a.heads);
        it.c0 = slice * FW, it.dz = min(FW, a.z.width - it.c0);
        const int len = a.lengths ? min(max(a.lengths[it.b], 0), a.steps) : a.steps;
        it.t0 = it.seg * a.span;
        it.t1 = (int)min((long)it.t0 + a.span, (long)a.steps);
        it.end = max(it.t0, min(it.t1, len));
        it.chunks = (it.end - it.t0 + FC - 1) / FC;
        return it;
    };
    auto skip = [&](const Place& it) { return STATE && !a.fin && it.seg == (a.rev ? 0 : a.segs - 1); };
    auto chunk_at = [&](const Place& it, int c) { return it.t0 + (a.rev ? it.chunks - 1 - c : c) * FC; };

    if (warp == 0) {
        if (lane == 0) {
            constexpr uint32_t base = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(FC >> 4) << 24);
            constexpr uint32_t amn = 1u << 15, bmn = 1u << 16, np = (uint32_t)(FC >> 3) << 17;
            constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};  // smallest products first
            const int kx = (dx + 15) / 16;
            const uint32_t S = smem_u32(sm);
            long n = 0;
            bool ok = true;
            for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
                const Place it = place(w);
                if (skip(it)) continue;
                const uint32_t nz = (uint32_t)((it.dz + 15) / 16 * 2) << 17;
                for (int c = 0; ok && c < it.chunks; ++c, ++n) {
                    const uint32_t ph = (uint32_t)(n & 1);
                    if (!(ok = mbar_wait(xy_ready, ph, fail))) break;
                    fence_after();
                    if (!STATE) {
#pragma unroll
                        for (int p = 0; p < 6; ++p)
                            for (int q = 0; q < kx; ++q)
                                mma_bf16(tmem + TP, desc(S + LX + PA[p] * PLANE + q * 32, false), desc(S + LY + PB[p] * PLANE + q * 32, false),
                                         base | np, p > 0 || q > 0);
                        mma_commit(p_full);
                        if (!(ok = mbar_wait(o_free, ph ^ 1u, fail))) break;
                        fence_after();
#pragma unroll
                        for (int p = 0; p < 6; ++p)
                            for (int q = 0; q < kx; ++q)
                                mma_bf16(tmem + TO1, desc(S + LX + PA[p] * PLANE + q * 32, false), desc(S + LS + PB[p] * SPLANE + q * 2048, true),
                                         base | bmn | nz, p > 0 || q > 0);
                    }
                    if (!(ok = mbar_wait(z_ready, ph, fail))) break;
                    fence_after();
                    // the weighted y is one box of 64 columns; the accumulator's upper 64 rows repeat it and are not read
#pragma unroll
                    for (int p = 0; p < 6; ++p)
                        for (int q = 0; q < FC / 16; ++q)
                            mma_bf16(tmem + TU, desc(S + LW + PA[p] * PLANE + q * 2048, true, 0), desc(S + LZ + PB[p] * PLANE + q * 2048, true),
                                     base | amn | bmn | nz, p > 0 || q > 0);
                    mma_commit(u_full);
                    if (!STATE) {
                        if (!(ok = mbar_wait(p_ready, ph, fail))) break;
                        fence_after();
#pragma unroll
                        for (int p = 0; p < 6; ++p)
                            for (int q = 0; q < FC / 16; ++q)
                                mma_bf16_ta(tmem + TO2, tmem + TPP + PA[p] * 64 + q * 8, desc(S + LZ + PB[p] * PLANE + q * 2048, true),
                                            base | bmn | nz, p > 0 || q > 0);
                        mma_commit(o_full);
                    }
                }
            }
            if (!ok) {
                mma_commit(drained);
                mbar_drain(drained, 0);
            }
        }
    } else if (warp < 5) {
        if (!STATE) {  // group A
            float* pw = reinterpret_cast<float*>(sm + LPA);
            const int quarter = warp & 3, i = quarter * 32 + lane, tid = threadIdx.x - 32;
            const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
            float* out = a.out32 ? a.out32 : a.out;
            const int dz = a.z.width;
            const bool vec = dz % 4 == 0 && aligned16_dev(out);
            long n = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
                const Place it = place(w);
                if (!(ok = group_sync(sync_a, phase, fail))) break;
                const float rate = a.rate[it.h];
                pw[tid] = tid == 0 ? 1.f : expf(-rate * (float)tid);
                if (tid == 0) pw[FC] = expf(-rate * (float)FC);
                if (!(ok = group_sync(sync_a, phase, fail))) break;
                for (int c = 0; c < it.chunks; ++c, ++n) {
                    const int t = chunk_at(it, c), m = min(FC, it.end - t);
                    const uint32_t ph = (uint32_t)(n & 1);
                    if (!(ok = __all_sync(kFull, mbar_wait(p_full, ph, fail)))) break;
                    fence_after();
                    for (int cb = 0; cb < 4; ++cb) {
                        float v[32];
                        const bool on = a.rev ? cb >= quarter : cb <= quarter;
                        if (on) {
                            tmem_ld32(tmem + TP + lanes + cb * 32, v);
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const int col = cb * 32 + j, gap = a.rev ? col - i : i - col;
                                v[j] = gap >= 0 && col < m ? v[j] * pw[max(gap, 0)] : 0.f;
                            }
                        }
                        uint32_t packed[16];
#pragma unroll
                        for (int s = 0; s < 3; ++s) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                packed[j] = 0u;
                                if (on) {
                                    packed[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                                    v[2 * j] -= bf16_lo(packed[j]), v[2 * j + 1] -= bf16_hi(packed[j]);
                                }
                            }
                            tmem_st16(tmem + TPP + lanes + s * 64 + cb * 16, packed);
                        }
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    fence_before();
                    mbar_arrive(p_ready);

                    if (!(ok = __all_sync(kFull, mbar_wait(o_full, ph, fail)))) break;
                    fence_after();
                    const bool in = i < m;
                    const float wi = a.rev ? pw[max(m - 1 - i, 0)] : pw[i + 1];
                    float* o = out + (((long)it.b * a.steps + t + i) * a.heads + it.h) * dz + it.c0;
                    for (int cb = 0; cb * 32 < it.dz; ++cb) {
                        float u[32], v[32];
                        tmem_ld32(tmem + TO1 + lanes + cb * 32, u);
                        tmem_ld32(tmem + TO2 + lanes + cb * 32, v);
                        if (cb * 32 + 32 >= it.dz) {  // the accumulators are read: the next chunk's products may have them
                            fence_before();
                            mbar_arrive(o_free);
                        }
                        if (t + i < it.t1) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = in ? fmaf(wi, u[j], v[j]) * a.oscale : 0.f;
                            const int width = it.dz - cb * 32;
                            if (vec && width >= 32) {
#pragma unroll
                                for (int j = 0; j < 32; j += 4)
                                    *reinterpret_cast<float4*>(o + cb * 32 + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                            } else {
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (j < width) o[cb * 32 + j] = v[j];
                            }
                        }
                    }
                }
                if (!ok) break;
                const long first = it.t0 + (long)it.chunks * FC;  // positions without a token beyond the last chunk
                for (long e = tid; e < (it.t1 - first) * it.dz; e += 128)
                    out[(((long)it.b * a.steps + first + e / it.dz) * a.heads + it.h) * dz + it.c0 + e % it.dz] = 0.f;
            }
        }
    } else {  // group B
        float* pw = reinterpret_cast<float*>(sm + LPB);
        const int tid = threadIdx.x - 160, quarter = warp & 3, half = (warp - 5) >> 2, row = quarter * 32 + lane;
        const bool keeper = quarter < 2;  // the state has at most 64 rows: four warps keep it, 32 columns each
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        long n = 0;
        uint32_t phase = 0;
        bool ok = true;

        // a thread's eight groups of four values of a tile: rows tid / 16 + 16 k, columns 4 (tid % 16) on
        auto load = [&](const Stream<float>& s, const float* p, int t, int m, int c0, float4 v[8]) {
            const int col = c0 + (tid & 15) * 4;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = (tid >> 4) + 16 * k;
                float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < m) {
                    const float* at = p + (long)(t + r) * s.st + col;
                    if (s.vec) {
                        if (col < s.width) q = __ldg(reinterpret_cast<const float4*>(at));
                    } else {
                        if (col < s.width) q.x = at[0];
                        if (col + 1 < s.width) q.y = at[1];
                        if (col + 2 < s.width) q.z = at[2];
                        if (col + 3 < s.width) q.w = at[3];
                    }
                }
                v[k] = q;
            }
        };
        for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
            const Place it = place(w);
            if (skip(it)) continue;
            const float* xb = STATE ? nullptr : a.x.p + it.b * a.x.sb + (it.h / a.x.group) * a.x.sh;
            const float* yb = a.y.p + it.b * a.y.sb + (it.h / a.y.group) * a.y.sh;
            const float* zb = a.z.p + it.b * a.z.sb + (it.h / a.z.group) * a.z.sh;
            if (!(ok = group_sync(sync_b, phase, fail))) break;
            const float rate = a.rate[it.h];
            if (tid <= FC) pw[tid] = tid == 0 ? 1.f : expf(-rate * (float)tid);
            if (!(ok = group_sync(sync_b, phase, fail))) break;
            float s[32];
            const long per = (long)dx * a.z.width;
            const float* init = nullptr;
            long ir = 0, ic = 0;
            float scale = 1.f;
            if (!STATE) {
                if (a.segs > 1) init = a.seg + (it.bh * a.segs + it.seg) * per, ir = a.z.width, ic = 1;
                else if (a.init) init = a.init + it.bh * per, ir = a.init_r, ic = a.init_c, scale = a.init_scale;
            }
            if (keeper) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const int col = half * 32 + j;
                    s[j] = init && row < dx && col < it.dz ? init[row * ir + (it.c0 + col) * ic] * scale : 0.f;
                }
            }
            for (int c = 0; c < it.chunks; ++c, ++n) {
                const int t = chunk_at(it, c), m = min(FC, it.end - t);
                const uint32_t ph = (uint32_t)(n & 1);
                float4 y[8], x[8];
                load(a.y, yb, t, m, 0, y);
                if (!STATE) load(a.x, xb, t, m, 0, x);
                // the products of the chunk before that read these tiles are done (n > 0: its state update waited)
                if (!STATE && keeper) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4)
                        put4(sm + LS, SPLANE, row, half * 8 + j / 4, make_float4(s[j], s[j + 1], s[j + 2], s[j + 3]));
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int r = (tid >> 4) + 16 * k;
                    const float wt = r < m ? pw[a.rev ? r + 1 : m - 1 - r] : 0.f;
                    if (!STATE) {
                        put4(sm + LY, PLANE, r, tid & 15, y[k]);
                        put4(sm + LX, PLANE, r, tid & 15, x[k]);
                    }
                    if (r < m) y[k].x *= wt, y[k].y *= wt, y[k].z *= wt, y[k].w *= wt;
                    put4(sm + LW, PLANE, r, tid & 15, y[k]);
                }
                fence_async_smem();
                mbar_arrive(xy_ready);
                load(a.z, zb, t, m, it.c0, x);
                if (!STATE && !(ok = __all_sync(kFull, mbar_wait(o_full, ph ^ 1u, fail)))) break;
#pragma unroll
                for (int k = 0; k < 8; ++k) put4(sm + LZ, PLANE, (tid >> 4) + 16 * k, tid & 15, x[k]);
                fence_async_smem();
                mbar_arrive(z_ready);
                if (!(ok = __all_sync(kFull, mbar_wait(u_full, ph, fail)))) break;
                fence_after();
                if (keeper && half * 32 < it.dz) {
                    const float gn = pw[m];
                    float v[32];
                    tmem_ld32(tmem + TU + lanes + half * 32, v);
#pragma unroll
                    for (int j = 0; j < 32; ++j) s[j] = fmaf(gn, s[j], v[j]);
                }
                fence_before();
            }
            if (!ok) break;
            float* fin = nullptr;
            long fr = 0, fc = 0;
            float fscale = 1.f;
            if (STATE) fin = a.seg + (it.bh * a.segs + it.seg) * per, fr = a.z.width, fc = 1;
            else if (a.segs == 1 && a.fin) fin = a.fin + it.bh * per, fr = a.fin_r, fc = a.fin_c, fscale = a.fin_scale;
            if (fin && keeper && row < dx)
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (half * 32 + j < it.dz) fin[row * fr + (it.c0 + half * 32 + j) * fc] = s[j] * fscale;
        }
    }
    __syncthreads();
    fence_after();
    if (threadIdx.x == 0 && *fail) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

}  // namespace

bool f32_fits(const Chain<float>& a) { return a.steps > 0 && a.y.width <= FW; }

int f32_chain(const Chain<float>& a, bool state_only, cudaStream_t s) {
    const long items = (long)a.batch * a.heads * a.segs * a.slices;
    if (items > 0x7FFFFFFFl) return EWS_ERR_UNSUPPORTED;
    auto* kern = state_only ? f32_kernel<true> : f32_kernel<false>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, LEND + 1024) != cudaSuccess) return EWS_ERR_LAUNCH;
    kern<<<(unsigned)(items < 148 ? items : 148), FTHR, LEND + 1024, s>>>(a, (int)items);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

}  // namespace decay
}  // namespace ews
