// The decayed attention's chain on the 5th-generation tensor core for float32 streams (the mathematics is in
// ews_decay.cu, the division of a chunk's work in ews_decay_tc.cu).
//
// A float32 is the sum of three bfloat16 (8 bits each), and a product of two takes six tensor-core products of
// planes (what is left out is below 2^-24), smallest first. The planes of x, y, the weighted y and z (three tiles of
// 128 x 64 each) and of the state fill shared memory, so x and y are at most 64 wide; z is taken in slices of 64
// columns. Group B reads the float32 rows with plain loads (any stride and alignment, a chunk ahead in registers),
// weights y before it is split, and writes the planes; the decayed scores are split by group A into three planes in
// tensor memory. Six products of 128 x 128 x 64 and three like it a chunk are about as long as the chunk's trip
// through HBM: neither bounds alone. Measured: one chain over B = 16, T = 1440, 8 heads of 64 (189 MB at full length) 122
// us; a chunk takes 14,000 cycles of a CTA, of which group B's splitting of three tiles into planes is 9,400 and its wait
// for U 3,900. Splitting y and x of the next chunk before that wait was not faster (610 us for forward and backward
// instead of 584 at the time): group A's three-plane scores then wait for the issue slots.
#include "ews_decay.cuh"
#include "ews_tc.cuh"

namespace ews {
namespace decay {

using namespace tc5;

namespace {

constexpr int FC = 128, FW = F32_WIDE;  // tokens of a chunk, columns of a tile
constexpr int PLANE = FC * 128;        // bytes of a plane of a stream, 128-byte rows
constexpr int SPLANE = FW * 128;       // of the state
constexpr int FTHR = 32 * 13;          // warps: MMA, four of group A, eight of group B (at most 16: 128 registers)
constexpr uint32_t TP = 0, TPP = 128, TO1 = 320, TO2 = 384, TU = 448;  // tensor-memory columns
constexpr int LX = 0, LY = LX + 3 * PLANE, LW = LY + 3 * PLANE, LZ = LW + 3 * PLANE, LS = LZ + 3 * PLANE, LBAR = LS + 3 * SPLANE,
              LTAB = LBAR + 128, LEND = LTAB + DECAY_BYTES;

struct Place {
    int b, h, seg, c0, dz;
    long bh;
    int t0, t1, end, chunks;
};

__device__ __forceinline__ void prefetch_l2(const float* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Up to four values, from column `col` on, of a row that 16-byte loads cannot read.
__device__ __noinline__ float4 load_ragged(const float* row, int col, int left) {
    return make_float4(left > 0 ? row[col] : 0.f, left > 1 ? row[col + 1] : 0.f, left > 2 ? row[col + 2] : 0.f, left > 3 ? row[col + 3] : 0.f);
}

// Four neighbouring values into the three planes of a tile, at (row, 4 col4).
__device__ __forceinline__ void put4(unsigned char* tile, int plane, int row, int col4, uint64_t a, uint64_t b) {
    unsigned char* p = tile + row * 128 + (((col4 >> 1) ^ (row & 7)) << 4) + (col4 & 1) * 8;
    const uint64_t minus_one = pair(-1.f, -1.f);
#pragma unroll
    for (int s = 0; s < 3; ++s) {
        const uint32_t u = s == 2 ? round2(a) : round2(a, minus_one), w = s == 2 ? round2(b) : round2(b, minus_one);
        *reinterpret_cast<uint2*>(p + s * plane) = make_uint2(u, w);
    }
}

template <bool STATE>
__global__ void __launch_bounds__(FTHR, 1) f32_kernel(const __grid_constant__ Chain<float> a, int items) {
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + LBAR);
    uint64_t *xy_ready = bars, *z_ready = bars + 1, *p_full = bars + 2, *p_ready = bars + 3, *u_full = bars + 4, *o_full = bars + 5,
             *o_free = bars + 6, *drained = bars + 7, *sync_a = bars + 8;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 9);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_at + 1);
    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int dx = a.y.width;

    if (threadIdx.x == 0) {
        mbar_init(p_full, 1), mbar_init(u_full, 1), mbar_init(o_full, 1), mbar_init(drained, 1);
        mbar_init(xy_ready, 256), mbar_init(z_ready, 256), mbar_init(p_ready, 128), mbar_init(o_free, 128);
        mbar_init(sync_a, 128);
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
    const uint32_t tmem = __shfl_sync(kFull, *tmem_at, 0);

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
        constexpr uint32_t base = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(FC >> 4) << 24);
        constexpr uint32_t amn = 1u << 15, bmn = 1u << 16, np = (uint32_t)(FC >> 3) << 17;
        // planes of the six products, a nibble each, smallest products first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
        constexpr int PA = 0x001102, PB = 0x010120;
        // descriptors of the first planes' first k-step (columns of x and y beyond their width are zero)
        const uint32_t S = smem_u32(sm);
        const uint64_t dX = desc(S + LX, false), dY = desc(S + LY, false), dS = desc(S + LS, true), dW = desc(S + LW, true, 0),
                       dZ = desc(S + LZ, true);
        long n = 0;
        bool ok = true;
        for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
            const Place it = place(w);
            if (skip(it)) continue;
            const uint32_t nz = (uint32_t)((it.dz + 15) / 16 * 2) << 17;
            for (int c = 0; ok && c < it.chunks; ++c, ++n) {
                const uint32_t ph = (uint32_t)(n & 1);
                const int ksteps = (min(FC, it.end - chunk_at(it, c)) + 15) / 16;  // the tokens' steps: the rest holds none
                if (!(ok = warp_wait(xy_ready, ph, fail))) break;
                fence_after();
                if (!STATE) {
                    if (elect_one()) {
#pragma unroll 1
                        for (int p = 0; p < 6; ++p) {
                            const uint64_t da = dX + ((PA >> (4 * p)) & 3) * (PLANE / 16), db = dY + ((PB >> (4 * p)) & 3) * (PLANE / 16);
#pragma unroll
                            for (int q = 0; q < FW / 16; ++q) mma_bf16(tmem + TP, da + q * 2, db + q * 2, base | np, p > 0 || q > 0);
                        }
                        mma_commit(p_full);
                    }
                    __syncwarp();
                    if (!(ok = warp_wait(o_free, ph ^ 1u, fail))) break;
                    fence_after();
                    if (elect_one()) {
#pragma unroll 1
                        for (int p = 0; p < 6; ++p) {
                            const uint64_t da = dX + ((PA >> (4 * p)) & 3) * (PLANE / 16), db = dS + ((PB >> (4 * p)) & 3) * (SPLANE / 16);
#pragma unroll
                            for (int q = 0; q < FW / 16; ++q) mma_bf16(tmem + TO1, da + q * 2, db + q * 128, base | bmn | nz, p > 0 || q > 0);
                        }
                    }
                    __syncwarp();
                }
                if (!(ok = warp_wait(z_ready, ph, fail))) break;
                fence_after();
                // the weighted y is one box of 64 columns; the accumulator's upper 64 rows repeat it and are not read
                if (elect_one()) {
#pragma unroll 1
                    for (int p = 0; p < 6; ++p) {
                        const uint64_t da = dW + ((PA >> (4 * p)) & 3) * (PLANE / 16), db = dZ + ((PB >> (4 * p)) & 3) * (PLANE / 16);
#pragma unroll 2
                        for (int q = 0; q < ksteps; ++q) mma_bf16(tmem + TU, da + q * 128, db + q * 128, base | amn | bmn | nz, p > 0 || q > 0);
                    }
                    mma_commit(u_full);
                }
                __syncwarp();
                if (!STATE) {
                    if (!(ok = warp_wait(p_ready, ph, fail))) break;
                    fence_after();
                    if (elect_one()) {
#pragma unroll 1
                        for (int p = 0; p < 6; ++p) {
                            const uint32_t ta = tmem + TPP + ((PA >> (4 * p)) & 3) * 64;
                            const uint64_t db = dZ + ((PB >> (4 * p)) & 3) * (PLANE / 16);
#pragma unroll 2
                            for (int q = 0; q < ksteps; ++q) mma_bf16_ta(tmem + TO2, ta + q * 8, db + q * 128, base | bmn | nz, p > 0 || q > 0);
                        }
                        mma_commit(o_full);
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok) {
            if (elect_one()) mma_commit(drained);
            __syncwarp();
            mbar_drain(drained, 0);
        }
    } else if (warp < 5) {
        if (!STATE) {  // group A: a thread a row
            const int quarter = warp & 3, i = quarter * 32 + lane, tid = threadIdx.x - 32;
            const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
            float* out = a.out32 ? a.out32 : a.out;
            const int dz = a.z.width;
            const bool vec = dz % 4 == 0 && aligned16_dev(out);
            const uint64_t minus_one = pair(-1.f, -1.f);
            long n = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
                const Place it = place(w);
                if (!(ok = group_sync(sync_a, phase, fail))) break;
                const float rate = a.rate[it.h];
                put_decay(sm + LTAB, tid, 128, rate, a.rev);
                const float wfull = decay_of(rate, a.rev ? FC - 1 - i : i + 1) * a.oscale;  // the carry's weight, of a full chunk
                const uint32_t row_tab = smem_u32(sm + LTAB) + (i + 127) * 8;
                if (!(ok = group_sync(sync_a, phase, fail))) break;
                for (int c = 0; c < it.chunks; ++c, ++n) {
                    const int t = chunk_at(it, c), m = min(FC, it.end - t);
                    const uint32_t ph = (uint32_t)(n & 1);
                    if (!(ok = __all_sync(kFull, mbar_wait(p_full, ph, fail)))) break;
                    fence_after();
#pragma unroll 1
                    for (int cb = 0; cb * 32 < m; ++cb) {
                        uint64_t v[16];
                        if (a.rev ? cb >= quarter : cb <= quarter) {
                            float e[32];
                            tmem_ld32(tmem + TP + lanes + cb * 32, e);
                            if (m < FC || cb == quarter) {
                                // as two bounds: as bits the training case takes 534 us instead of 520
                                const Live live = live_scores(cb, quarter, lane, m, a.rev);
#pragma unroll
                                for (int j = 0; j < 32; ++j) e[j] = j >= live.from && j < live.to ? e[j] : 0.f;
                            }
                            const uint32_t g = row_tab - cb * 256;
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = mul2(pair(e[2 * j], e[2 * j + 1]), lds64(g - 16 * j));
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = 0ull;
                        }
#pragma unroll 1
                        for (int s = 0; s < 3; ++s) {
                            uint32_t packed[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) packed[j] = round2(v[j], minus_one);
                            tmem_st16(tmem + TPP + lanes + s * 64 + cb * 16, packed);
                        }
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    fence_before();
                    mbar_arrive(p_ready);

                    if (!(ok = __all_sync(kFull, mbar_wait(o_full, ph, fail)))) break;
                    fence_after();
                    const bool in = i < m;
                    const float wi = m == FC ? wfull : (a.rev ? decay_of(rate, m - 1 - i) * a.oscale : wfull);
                    const uint64_t wi2 = pair(wi, wi), os2 = pair(a.oscale, a.oscale);
                    float* o = out + (((long)it.b * a.steps + t + i) * a.heads + it.h) * dz + it.c0;
#pragma unroll 1
                    for (int c0 = 0; c0 < FW; c0 += 32) {
                        const int width = it.dz - c0;
                        float u[32], v[32];
                        if (width > 0) {
                            tmem_ld32(tmem + TO1 + lanes + c0, u);
                            tmem_ld32(tmem + TO2 + lanes + c0, v);
                        }
                        if (c0 + 32 == FW) {  // the accumulators are read
                            fence_before();
                            mbar_arrive(o_free);
                        }
                        if (width <= 0 || t + i >= it.t1) continue;
                        uint64_t r[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            r[j] = fma2(wi2, pair(u[2 * j], u[2 * j + 1]), mul2(os2, pair(v[2 * j], v[2 * j + 1])));
                        if (!in) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) r[j] = 0ull;
                        }
                        if (vec && width >= 32) {
#pragma unroll
                            for (int j = 0; j < 16; j += 2) *reinterpret_cast<ulonglong2*>(o + c0 + 2 * j) = make_ulonglong2(r[j], r[j + 1]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                float e0, e1;
                                unpair(r[j], e0, e1);
                                if (2 * j < width) o[c0 + 2 * j] = e0;
                                if (2 * j + 1 < width) o[c0 + 2 * j + 1] = e1;
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
        const int tid = threadIdx.x - 160, quarter = warp & 3, half = (warp - 5) >> 2, row = quarter * 32 + lane;
        const bool keeper = quarter < 2;  // the state has at most 64 rows: four warps keep it, 32 columns each
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        long n = 0;
        bool ok = true;

        for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
            const Place it = place(w);
            if (skip(it)) continue;
            const float* xb = STATE ? nullptr : a.x.p + it.b * a.x.sb + (it.h / a.x.group) * a.x.sh;
            const float* yb = a.y.p + it.b * a.y.sb + (it.h / a.y.group) * a.y.sh;
            const float* zb = a.z.p + it.b * a.z.sb + (it.h / a.z.group) * a.z.sh;
            const float rate = a.rate[it.h];
            const float gfull = decay_of(rate, FC);
            uint64_t s[16];
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
                for (int j = 0; j < 16; ++j) s[j] = 0ull;
                if (init) {
                    const float* from = init + min(row, dx - 1) * ir;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float e[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {  // from places that exist, all in flight at once
                            const int col = half * 32 + 2 * j + k;
                            e[k] = from[(it.c0 + min(col, it.dz - 1)) * ic] * scale;
                            if (row >= dx || col >= it.dz) e[k] = 0.f;
                        }
                        s[j] = pair(e[0], e[1]);
                    }
                }
            }
            for (int c = 0; c < it.chunks; ++c, ++n) {
                const int t = chunk_at(it, c), m = min(FC, it.end - t);
                const uint32_t ph = (uint32_t)(n & 1);
                // the products of the chunk before that read these tiles are done (n > 0: its state update waited)
                if (!STATE && keeper) {
#pragma unroll
                    for (int j = 0; j < 16; j += 2) put4(sm + LS, SPLANE, row, half * 8 + j / 2, s[j], s[j + 1]);
                }
                // y, x, z: a thread has rows tid / 16 + 16 k, columns 4 (tid % 16) on
#pragma unroll 1
                for (int part = 0; part < 3; ++part) {
                    if (STATE && part == 1) part = 2;
                    const Stream<float>& st = part == 0 ? a.y : part == 1 ? a.x : a.z;
                    const float* p = part == 0 ? yb : part == 1 ? xb : zb;
                    const int col = (part == 2 ? it.c0 : 0) + (tid & 15) * 4, left = st.width - col;
                    float4 v[8];
                    // every load is issued, from a row and a column that exist, and what does not count is dropped after: under
                    // a condition each, the loads would come one by one
                    if (st.vec) {
                        const float* from = p + (left > 0 ? col : 0);
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            v[k] = __ldg(reinterpret_cast<const float4*>(from + (long)(t + min((tid >> 4) + 16 * k, m - 1)) * st.st));
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = load_ragged(p + (long)(t + min((tid >> 4) + 16 * k, m - 1)) * st.st, col, left);
                    }
                    if (part == 2) {
                        if (!STATE && !(ok = __all_sync(kFull, mbar_wait(o_full, ph ^ 1u, fail)))) break;
                    }
                    unsigned char* tile = sm + (part == 0 ? LY : part == 1 ? LX : LZ);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int r = (tid >> 4) + 16 * k;
                        if (16 * k >= m) continue;
                        uint64_t lo = pair(v[k].x, v[k].y), hi = pair(v[k].z, v[k].w);
                        if (r >= m || left <= 0) lo = hi = 0ull;
                        if (!(STATE && part == 0)) put4(tile, PLANE, r, tid & 15, lo, hi);
                        if (part == 0) {
                            const float wt = decay_of(rate, a.rev ? r + 1 : m - 1 - r);
                            const uint64_t wt2 = pair(wt, wt);
                            put4(sm + LW, PLANE, r, tid & 15, mul2(lo, wt2), mul2(hi, wt2));
                        }
                    }
                    if (part == (STATE ? 0 : 1)) {
                        fence_async_smem();
                        mbar_arrive(xy_ready);
                    }
                }
                if (!ok) break;
                fence_async_smem();
                mbar_arrive(z_ready);
                if (c + 1 < it.chunks) {  // the next chunk's rows on their way to L2: two threads a row
                    const int t2 = chunk_at(it, c + 1), r = tid >> 1, half_row = (tid & 1) * 32;
                    if (t2 + r < it.end) {
                        if (!STATE && half_row < a.x.width) prefetch_l2(xb + (long)(t2 + r) * a.x.st + half_row);
                        if (half_row < a.y.width) prefetch_l2(yb + (long)(t2 + r) * a.y.st + half_row);
                        if (it.c0 + half_row < a.z.width) prefetch_l2(zb + (long)(t2 + r) * a.z.st + it.c0 + half_row);
                    }
                }
                if (!(ok = __all_sync(kFull, mbar_wait(u_full, ph, fail)))) break;
                fence_after();
                if (keeper && half * 32 < it.dz) {
                    const float gn = m == FC ? gfull : decay_of(rate, m);
                    const uint64_t gn2 = pair(gn, gn);
                    float v[32];
                    tmem_ld32(tmem + TU + lanes + half * 32, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = fma2(gn2, s[j], pair(v[2 * j], v[2 * j + 1]));
                }
                fence_before();
            }
            if (!ok) break;
            float* fin = nullptr;
            long fr = 0, fc = 0;
            float fscale = 1.f;
            if (STATE) fin = a.seg + (it.bh * a.segs + it.seg) * per, fr = a.z.width, fc = 1;
            else if (a.segs == 1 && a.fin) fin = a.fin + it.bh * per, fr = a.fin_r, fc = a.fin_c, fscale = a.fin_scale;
            if (fin && keeper && row < dx) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float e[2];
                    unpair(s[j], e[0], e[1]);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int col = half * 32 + 2 * j + k;
                        if (col < it.dz) fin[row * fr + (it.c0 + col) * fc] = e[k] * fscale;
                    }
                }
            }
        }
    }
    __syncthreads();
    fence_after();
    if (threadIdx.x == 0 && *fail) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

}  // namespace

// An axis of no tokens is one item without a chunk: its state goes from where it starts to where it ends.
bool f32_fits(const Chain<float>& a) { return a.y.width <= FW; }

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
