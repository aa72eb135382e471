// The decayed attention's chain on the 5th-generation tensor core (bfloat16 streams; the mathematics is in
// ews_decay.cu). Chunks of 128 tokens, four products a chunk, all 128 rows of an accumulator in tensor memory:
//
//     P  = X Y^T            (tokens x tokens)      -> * decay, causal, to bfloat16 in tensor memory
//     O1 = X State          (tokens x dz)
//     U  = (w Y)^T Z        (dx x dz)              -> State = g^n State + U, float32 in registers
//     O2 = P Z              (tokens x dz)          -> out = g^(i+1) O1 + O2
//
// One persistent CTA per SM walks (sample, head, segment) items. Warp 0 fetches tiles by TMA, warp 1 issues the
// products, warps 2-5 (A) turn P into an operand and write the output, warps 6-13 (B) weight Y (in place, and its
// rounding residue beside it: the weighted operand is inexact, two bfloat16 pieces carry it to 2^-16, three to 2^-24),
// keep the state and write its bfloat16 copy. The only chain from chunk to chunk is U -> State -> O1; the loads, P and the
// output of neighbouring chunks run beside it.
// X, whose last product of a chunk (O1) is issued a chunk ahead, has one buffer, Y and Z two.
// Why 128 tokens: the accumulator has 128 rows; the waste of the upper half of P is 1/10 of a chunk's products.
//
// Measured: one chain over B = 8, T = 2048, 16 heads of 128 (268 MB of streams) 62 us, 4.3 TB/s, two thirds of the copy
// bandwidth, on 128 of the 148 SMs; a chunk takes 5,400 cycles of a CTA, of which its products are 2,600 and its traffic
// 4,800 at the copy bandwidth. What bounds it is group A: its scores (1,500), the wait for O2 (1,100) and the output
// (2,300) follow one another, and a role's instructions come slowly (its code runs once a chunk, and the roles' code
// together is larger than the inner instruction cache: unrolled loops lost more than they gained). A third group for
// the output took 96 registers a thread and spilled: 329 us for the training case instead of 290 at the time.
// Rounded to bfloat16 on the way are the decayed scores (the operand of O2 comes from tensor memory in that type) and the
// state's copy for O1; the state itself stays in float32. For random inputs the output is then 2.3e-3 from the exact one
// (norm over norm) where its own rounding alone leaves 1.7e-3.
// The states' pass over 17,984 tokens of 16 heads (three pieces) takes 62 us, the outputs' 74 us.
//
// Reversed chains keep the rows' order and walk the chunks down: decays are then g^(j-i) for j >= i, a row's weight of
// the carry g^(n-1-i), an update's g^(j+1).
#include "ews_decay.cuh"
#include "ews_tc.cuh"

namespace ews {
namespace decay {

using namespace tc5;

namespace {

constexpr int TC = 128;                  // tokens of a chunk
constexpr int BOX = TC * 128;            // bytes of 64 columns of a tile
constexpr int TILE = 2 * BOX;
constexpr int NTHR = 32 * 14;  // at most 16 warps: 128 registers a thread
constexpr uint32_t TP = 0, TO1 = 128, TO2 = 256, TU = 384;  // tensor-memory columns

struct Maps {
    CUtensorMap x, y, z;
};

template <bool STATE, int NS>
struct Lay {
    static constexpr int X = 0, Y = X + (STATE ? 0 : TILE), Z = Y + 2 * TILE, S = Z + 2 * TILE, LO = S + (STATE ? 0 : TILE),
                         BARS = LO + (NS - 1) * TILE, TAB = BARS + 256, END = TAB + DECAY_BYTES;
    static constexpr size_t bytes = END;
};

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }
__device__ __forceinline__ void tma_load4(const CUtensorMap* map, uint64_t* bar, void* dst, int x, int t, int h, int b) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(t), "r"(h), "r"(b)
        : "memory");
}
// An item's place: sample, head, its tokens [t0, t1), of which [t0, end) exist, and its chunks.
struct Item {
    int b, h, seg;
    long bh;
    int t0, t1, end, chunks;
};

template <bool STATE, int NS>
__global__ void __launch_bounds__(NTHR, 1) tc_kernel(const __grid_constant__ Chain<bf16> a, const __grid_constant__ Maps maps, int items) {
    using L = Lay<STATE, NS>;
    // the tiles' swizzle wants 1,024-byte boundaries; there is no room to round up
    extern __shared__ __align__(1024) unsigned char sm[];
    if (smem_u32(sm) & 1023) {
        report(a.status, EWS_ERR_LAUNCH);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(sm + L::BARS);
    uint64_t *x_full = bars, *y_full = bars + 2, *z_full = bars + 4, *x_empty = bars + 6, *y_empty = bars + 8, *z_empty = bars + 10;
    uint64_t *p_full = bars + 12, *p_ready = bars + 13, *o_full = bars + 14, *o_free = bars + 15, *s_ready = bars + 16,
             *yw_ready = bars + 17, *u_full = bars + 18, *xs_done = bars + 19, *drained = bars + 20, *sync_a = bars + 21;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(bars + 22);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_at + 1);
    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int dx = a.y.width, dz = a.z.width;
    const int dx16 = (dx + 15) & ~15, dz16 = (dz + 15) & ~15;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 12; ++i) mbar_init(bars + i, 1);
        mbar_init(p_full, 1), mbar_init(o_full, 1), mbar_init(u_full, 1), mbar_init(xs_done, 1), mbar_init(drained, 1);
        mbar_init(p_ready, 128), mbar_init(o_free, 128), mbar_init(s_ready, 256), mbar_init(yw_ready, 256);
        mbar_init(sync_a, 128);
        *fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 0) {  // the maps on their way before their first use
        prefetch_map(&maps.y), prefetch_map(&maps.z);
        if (!STATE) prefetch_map(&maps.x);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(kFull, *tmem_at, 0);

    auto place = [&](int w) {
        Item it;
        it.seg = w % a.segs;
        it.bh = w / a.segs;
        it.b = (int)(it.bh / a.heads), it.h = (int)(it.bh - (long)it.b * a.heads);
        const int len = a.lengths ? min(max(a.lengths[it.b], 0), a.steps) : a.steps;
        it.t0 = it.seg * a.span;
        it.t1 = (int)min((long)it.t0 + a.span, (long)a.steps);
        it.end = max(it.t0, min(it.t1, len));
        it.chunks = (it.end - it.t0 + TC - 1) / TC;
        return it;
    };
    auto skip = [&](const Item& it) {  // a state that no segment starts from
        return STATE && !a.fin && it.seg == (a.rev ? 0 : a.segs - 1);
    };

    if (warp == 0) {
        if (lane == 0) {
            long n = 0;
            bool ok = true;
            for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
                const Item it = place(w);
                if (skip(it)) continue;
                for (int c = 0; c < it.chunks; ++c, ++n) {
                    const int t = it.t0 + (a.rev ? it.chunks - 1 - c : c) * TC, s = (int)(n & 1);
                    const uint32_t two = (uint32_t)((n >> 1) & 1) ^ 1u;
                    if (!(ok = mbar_wait(y_empty + s, two, fail))) break;
                    const int bx = dx > 64 ? 2 : 1, bz = dz > 64 ? 2 : 1;
                    mbar_expect(y_full + s, bx * BOX);
                    for (int j = 0; j < bx; ++j)
                        tma_load4(&maps.y, y_full + s, sm + L::Y + s * TILE + j * BOX, j * 64, t, it.h / a.y.group, it.b);
                    if (!STATE) {
                        if (!(ok = mbar_wait(x_empty, (uint32_t)(n & 1) ^ 1u, fail))) break;
                        mbar_expect(x_full, bx * BOX);
                        for (int j = 0; j < bx; ++j)
                            tma_load4(&maps.x, x_full, sm + L::X + j * BOX, j * 64, t, it.h / a.x.group, it.b);
                    }
                    if (!(ok = mbar_wait(z_empty + s, two, fail))) break;
                    mbar_expect(z_full + s, bz * BOX);
                    for (int j = 0; j < bz; ++j)
                        tma_load4(&maps.z, z_full + s, sm + L::Z + s * TILE + j * BOX, j * 64, t, it.h / a.z.group, it.b);
                }
            }
            if (!ok) {  // what was asked for lands before the CTA leaves: at most the last two chunks' loads
                for (long j = n > 1 ? n - 2 : 0; j <= n; ++j) {
                    const uint32_t two = (uint32_t)((j >> 1) & 1);
                    mbar_drain(y_full + (j & 1), two);
                    if (!STATE) mbar_drain(x_full, (uint32_t)(j & 1));
                    mbar_drain(z_full + (j & 1), two);
                }
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t base = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TC >> 4) << 24);
        constexpr uint32_t amn = 1u << 15, bmn = 1u << 16;
        const uint32_t nz = (uint32_t)(dz16 >> 3) << 17, np = (uint32_t)(TC >> 3) << 17;
        const int kx = dx16 / 16;
        // descriptors of the tiles' first k-step
        const uint64_t dS = desc(smem_u32(sm + L::S), true, BOX);
        const uint64_t dLO = desc(smem_u32(sm + L::LO), true, BOX);
        long total = 0;  // chunks of this CTA, whichever items they belong to
        for (int w = blockIdx.x; w < items; w += gridDim.x) {
            const Item it = place(w);
            if (!skip(it)) total += it.chunks;
        }
        auto scores = [&](long n) {  // P of chunk n
            const int s = (int)(n & 1);
            const uint32_t two = (uint32_t)((n >> 1) & 1);
            if (!(warp_wait(x_full, (uint32_t)(n & 1), fail) && warp_wait(y_full + s, two, fail))) return false;
            fence_after();
            if (elect_one()) {
                const uint64_t dX = desc(smem_u32(sm + L::X), false), dY = desc(smem_u32(sm + L::Y + s * TILE), false);
                for (int q = 0; q < kx; ++q) {
                    const int off = (q >> 2) * (BOX >> 4) + (q & 3) * 2;
                    mma_bf16(tmem + TP, dX + off, dY + off, base | np, q > 0);
                }
                mma_commit(p_full);
            }
            __syncwarp();
            return true;
        };
        auto carried = [&](long n) {  // O1 of chunk n
            const uint32_t ph = (uint32_t)(n & 1);
            if (!(warp_wait(s_ready, ph, fail) && warp_wait(o_free, ph ^ 1u, fail))) return false;
            fence_after();
            if (elect_one()) {
                const uint64_t dX = desc(smem_u32(sm + L::X), false);
                for (int q = 0; q < kx; ++q)
                    mma_bf16(tmem + TO1, dX + (q >> 2) * (BOX >> 4) + (q & 3) * 2, dS + q * 128, base | bmn | nz, q > 0);
                mma_commit(xs_done);
                mma_commit(x_empty);
            }
            __syncwarp();
            return true;
        };
        // In the order in which the others' parts come free: O2 for group A's output, U for group B's state, then, while
        // they work, the next chunk's P, and O1 from the new state.
        bool ok = STATE || total == 0 || (scores(0) && carried(0));
        for (long n = 0; ok && n < total; ++n) {
            const int s = (int)(n & 1);
            const uint32_t ph = (uint32_t)(n & 1), two = (uint32_t)((n >> 1) & 1);
            const uint64_t dYw = desc(smem_u32(sm + L::Y + s * TILE), true, BOX), dZ = desc(smem_u32(sm + L::Z + s * TILE), true, BOX);
            if (!(ok = warp_wait(z_full + s, two, fail))) break;
            if (!STATE) {
                if (!(ok = warp_wait(p_ready, ph, fail))) break;
                fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int q = 0; q < TC / 16; ++q)
                        mma_bf16_ta(tmem + TO2, tmem + TP + q * 8, dZ + q * 128, base | bmn | nz, q > 0);
                    mma_commit(o_full);
                }
                __syncwarp();
            }
            if (!(ok = warp_wait(yw_ready, ph, fail))) break;
            fence_after();
            if (elect_one()) {
#pragma unroll
                for (int p = NS - 1; p >= 0; --p) {  // the smallest piece first
                    const uint64_t dW = p == 0 ? dYw : dLO + (p > 0 ? p - 1 : 0) * (TILE >> 4);
#pragma unroll
                    for (int q = 0; q < TC / 16; ++q)
                        mma_bf16(tmem + TU, dW + q * 128, dZ + q * 128, base | amn | bmn | nz, p < NS - 1 || q > 0);
                }
                mma_commit(u_full);
                mma_commit(y_empty + s);
                mma_commit(z_empty + s);
            }
            __syncwarp();
            if (!STATE && n + 1 < total) ok = scores(n + 1) && carried(n + 1);
        }
        if (!ok) {
            if (elect_one()) mma_commit(drained);
            __syncwarp();
            mbar_drain(drained, 0);
        }
    } else if (warp < 6) {
        if (!STATE) {  // group A: a thread a row
            const int quarter = warp & 3, i = quarter * 32 + lane, tid = threadIdx.x - 64;
            const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
            const bool wide = a.out && dz % 16 == 0 && ((uintptr_t)a.out & 31u) == 0;  // every row starts on a sector
            long n = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
                const Item it = place(w);
                if (!(ok = group_sync(sync_a, phase, fail))) break;
                const float rate = a.rate[it.h];
                put_decay(sm + L::TAB, tid, 128, rate, a.rev);
                const float ofull = decay_of(rate, a.rev ? TC - 1 - i : i + 1) * a.oscale;  // the carry's weight here, of a full chunk
                const uint32_t row_tab = smem_u32(sm + L::TAB) + (i + 127) * 8;
                if (!(ok = group_sync(sync_a, phase, fail))) break;
                for (int c = 0; c < it.chunks; ++c, ++n) {
                    const int t = it.t0 + (a.rev ? it.chunks - 1 - c : c) * TC, m = min(TC, it.end - t);
                    const uint32_t ph = (uint32_t)(n & 1);
                    if (!(ok = __all_sync(kFull, mbar_wait(p_full, ph, fail)))) break;
                    fence_after();
                    // 32 columns at a time; their 16 packed columns go where scores have been read already
#pragma unroll 1
                    for (int cb = 0; cb < 4; ++cb) {
                        uint32_t packed[16];
                        if (a.rev ? cb >= quarter : cb <= quarter) {
                            float v[32];
                            tmem_ld32(tmem + TP + lanes + cb * 32, v);
                            if (m < TC || cb == quarter) {
                                // as bits: as two bounds a score the training case takes 285 us instead of 274
                                const uint32_t live = live_scores(cb, quarter, lane, m, a.rev).bits();
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[j] = live & (1u << j) ? v[j] : 0.f;
                            }
                            const uint32_t g = row_tab - cb * 256;
#pragma unroll
                            for (int j = 0; j < 16; ++j) packed[j] = round2(mul2(pair(v[2 * j], v[2 * j + 1]), lds64(g - 16 * j)));
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; ++j) packed[j] = 0u;
                        }
                        tmem_st16(tmem + TP + lanes + cb * 16, packed);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    fence_before();
                    mbar_arrive(p_ready);

                    if (!(ok = __all_sync(kFull, mbar_wait(o_full, ph, fail)))) break;
                    fence_after();
                    const float wi = m == TC || !a.rev ? ofull : decay_of(rate, m - 1 - i) * a.oscale;
                    const uint64_t wi2 = pair(wi, wi), os2 = pair(a.oscale, a.oscale);
                    const long at = (((long)it.b * a.steps + t + i) * a.heads + it.h) * dz;
#pragma unroll 1
                    for (int c0 = 0; c0 < dz; c0 += 32) {
                        uint32_t u[32], v[32];
                        tmem_ld32x2(tmem + TO1 + lanes + c0, tmem + TO2 + lanes + c0, u, v);
                        uint64_t o[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            o[j] = fma2(wi2, pair(__uint_as_float(u[2 * j]), __uint_as_float(u[2 * j + 1])),
                                        mul2(os2, pair(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]))));
                        if (m < TC && i >= m) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = 0ull;
                        }
                        if (t + i >= it.t1) {
                        } else if (a.out32) {
                            float* to = a.out32 + at + c0;
#pragma unroll
                            for (int j = 0; j < 16; j += 2)
                                if (c0 + 2 * j < dz) *reinterpret_cast<ulonglong2*>(to + 2 * j) = make_ulonglong2(o[j], o[j + 1]);
                        } else {
                            uint32_t q[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) q[j] = round2(o[j]);
                            bf16* to = a.out + at + c0;
                            if (wide) {
                                store32(to, q);
                                if (c0 + 16 < dz) store32(to + 16, q + 8);
                            } else {
#pragma unroll
                                for (int j = 0; j < 16; j += 4)
                                    if (c0 + 2 * j < dz) *reinterpret_cast<uint4*>(to + 2 * j) = make_uint4(q[j], q[j + 1], q[j + 2], q[j + 3]);
                            }
                        }
                    }
                    fence_before();
                    mbar_arrive(o_free);
                }
                if (!ok) break;
                // positions without a token beyond the last chunk
                const long first = it.t0 + (long)it.chunks * TC;
                for (long e = tid; e < (it.t1 - first) * dz; e += 128) {
                    const long at = (((long)it.b * a.steps + first + e / dz) * a.heads + it.h) * dz + e % dz;
                    if (a.out32) a.out32[at] = 0.f;
                    else a.out[at] = from_f<bf16>(0.f);
                }
            }
        }
    } else {  // group B
        const int quarter = warp & 3, half = (warp - 6) >> 2, row = quarter * 32 + lane, tid = threadIdx.x - 192;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        long n = 0;
        bool ok = true;
        for (int w = blockIdx.x; ok && w < items; w += gridDim.x) {
            const Item it = place(w);
            if (skip(it)) continue;
            const float rate = a.rate[it.h];
            // a full chunk's weights of the four tokens that this thread weights, and of the carry
            const float gfull = decay_of(rate, TC);
            float wfull[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) wfull[k] = decay_of(rate, a.rev ? (tid >> 3) + 32 * k + 1 : TC - 1 - (tid >> 3) - 32 * k);
            uint64_t s[32];
            const long per = (long)dx * dz;
            const float* init = nullptr;
            long ir = 0, ic = 0;
            float scale = 1.f;
            if (!STATE) {
                if (a.segs > 1) init = a.seg + (it.bh * a.segs + it.seg) * per, ir = dz, ic = 1;
                else if (a.init) init = a.init + it.bh * per, ir = a.init_r, ic = a.init_c, scale = a.init_scale;
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j] = 0ull;
            if (init) {
                const float* from = init + min(row, dx - 1) * ir;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float e[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {  // from places that exist, all in flight at once
                        const int col = half * 64 + 2 * j + k;
                        e[k] = from[min(col, dz - 1) * ic] * scale;
                        if (row >= dx || col >= dz) e[k] = 0.f;
                    }
                    s[j] = pair(e[0], e[1]);
                }
            }
#pragma unroll 1
            for (int c = 0; c < it.chunks; ++c, ++n) {
                const int t = it.t0 + (a.rev ? it.chunks - 1 - c : c) * TC, m = min(TC, it.end - t);
                const int st = (int)(n & 1);
                const uint32_t ph = (uint32_t)(n & 1), two = (uint32_t)((n >> 1) & 1);
                if (m < TC) {  // a short chunk: rows of Z that are no tokens must not reach a product, the first of which follows O1
                    if (!(ok = __all_sync(kFull, mbar_wait(z_full + st, two, fail)))) break;
                    unsigned char* Z = sm + L::Z + st * TILE;
                    for (int e = tid; e < TILE / 16; e += 256)
                        if (((e >> 3) & (TC - 1)) >= m) *reinterpret_cast<uint4*>(Z + e * 16) = make_uint4(0, 0, 0, 0);
                }
                if (!STATE) {
                    if (!(ok = __all_sync(kFull, mbar_wait(xs_done, ph ^ 1u, fail)))) break;
                    if (half * 64 < dz) {
                        unsigned char* p = sm + L::S + half * BOX + row * 128;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            *reinterpret_cast<uint4*>(p + ((j ^ (row & 7)) * 16)) =
                                make_uint4(round2(s[4 * j]), round2(s[4 * j + 1]), round2(s[4 * j + 2]), round2(s[4 * j + 3]));
                    }
                    fence_async_smem();
                    mbar_arrive(s_ready);
                }
                if (!(ok = __all_sync(kFull, mbar_wait(y_full + st, two, fail) && mbar_wait(z_full + st, two, fail) &&
                                                 (STATE || mbar_wait(p_full, ph, fail)))))
                    break;
                unsigned char* Y = sm + L::Y + st * TILE;
                const uint64_t minus_one = pair(-1.f, -1.f);
                const int rounds = dx > 64 ? 2 : 1;
#pragma unroll 1
                for (int r = 0; r < rounds; ++r) {  // a box of 64 columns: 1,024 vectors of 16 bytes, four a thread
                    uint4 q[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) q[k] = *reinterpret_cast<const uint4*>(Y + r * BOX + (tid + 256 * k) * 16);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int e = tid + 256 * k, tok = e >> 3;
                        const bool live = tok < m;
                        const float wt = m == TC ? wfull[k] : decay_of(rate, a.rev ? tok + 1 : m - 1 - tok);
                        const uint64_t wt2 = pair(wt, wt);
                        const uint32_t in[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
                        uint32_t piece[NS][4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint64_t f = mul2(pair(bf16_lo(in[j]), bf16_hi(in[j])), wt2);
                            if (!live) f = 0ull;
#pragma unroll
                            for (int p = 0; p < NS; ++p) piece[p][j] = p == NS - 1 ? round2(f) : round2(f, minus_one);
                        }
                        *reinterpret_cast<uint4*>(Y + r * BOX + e * 16) = make_uint4(piece[0][0], piece[0][1], piece[0][2], piece[0][3]);
#pragma unroll
                        for (int p = 1; p < NS; ++p)
                            *reinterpret_cast<uint4*>(sm + L::LO + (p - 1) * TILE + r * BOX + e * 16) =
                                make_uint4(piece[p][0], piece[p][1], piece[p][2], piece[p][3]);
                    }
                }
                fence_async_smem();
                mbar_arrive(yw_ready);
                if (!(ok = __all_sync(kFull, mbar_wait(u_full, ph, fail)))) break;
                fence_after();
                const float gn = m == TC ? gfull : decay_of(rate, m);
                const uint64_t gn2 = pair(gn, gn);
                if (half * 64 < dz) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float v[32];
                        tmem_ld32(tmem + TU + lanes + half * 64 + q * 32, v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) s[q * 16 + j] = fma2(gn2, s[q * 16 + j], pair(v[2 * j], v[2 * j + 1]));
                    }
                }
                fence_before();
            }
            if (!ok) break;
            float* fin = nullptr;
            long fr = 0, fc = 0;
            float fscale = 1.f;
            if (STATE) fin = a.seg + (it.bh * a.segs + it.seg) * per, fr = dz, fc = 1;
            else if (a.segs == 1 && a.fin) fin = a.fin + it.bh * per, fr = a.fin_r, fc = a.fin_c, fscale = a.fin_scale;
            if (fin && row < dx) {
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const int col = half * 64 + 2 * j;
                    float e[2];
                    unpair(s[j], e[0], e[1]);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (col + k < dz) fin[row * fr + (col + k) * fc] = e[k] * fscale;
                }
            }
        }
    }
    __syncthreads();
    fence_after();
    if (threadIdx.x == 0 && *fail) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

bool map_of(CUtensorMap* m, const bf16* p, int width, int steps, int heads, int batch, long st, long sh, long sb) {
    EncodeFn enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)steps, (cuuint64_t)heads, (cuuint64_t)batch};
    // an axis of one has no stride to speak of
    const cuuint64_t strides[3] = {(cuuint64_t)(steps > 1 ? st * 2 : 16), (cuuint64_t)(heads > 1 ? sh * 2 : 16),
                                   (cuuint64_t)(batch > 1 ? sb * 2 : 16)};
    const cuuint32_t box[4] = {64, TC, 1, 1}, es[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<bf16*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool mappable(const Stream<bf16>& s, int steps, int heads, int batch) {
    const long most = 1l << 38;
    return s.vec && (steps == 1 || (s.st > 0 && s.st < most)) && (heads == 1 || (s.sh > 0 && s.sh < most)) &&
           (batch == 1 || (s.sb > 0 && s.sb < most));
}

template <bool STATE, int NS>
int go(const Chain<bf16>& a, const Maps& m, cudaStream_t s) {
    auto* kern = tc_kernel<STATE, NS>;
    using L = Lay<STATE, NS>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::bytes) != cudaSuccess) return EWS_ERR_LAUNCH;
    const long items = (long)a.batch * a.heads * a.segs;
    if (items > 0x7FFFFFFFl) return EWS_ERR_UNSUPPORTED;
    kern<<<(unsigned)(items < 148 ? items : 148), NTHR, L::bytes, s>>>(a, m, (int)items);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

}  // namespace

// The split of the axis that the cost model prefers, in chunks walked by the busiest CTA: a split walks each
// chunk once more for the states alone, at about 0.6 of a chunk's time, and costs two launches (about two chunks).
int tc_segments(int batch, int steps, int heads, bool state, int* span) {
    const int chunks = (steps + TC - 1) / TC < 1 ? 1 : (steps + TC - 1) / TC;
    const long rows = (long)batch * heads;
    double best = 0;
    int pick = 1;
    for (int s = 1; s <= 64 && (s == 1 || s * 2 <= chunks); ++s) {
        const int per = (chunks + s - 1) / s;
        const double waves = (double)((rows * s + 147) / 148);
        const double cost = waves * per * (s > 1 || state ? 1.6 : 1.0) + (s > 1 ? 2.0 : 0.0);
        if (s == 1 || cost < best) best = cost, pick = s;
    }
    const int per = (chunks + pick - 1) / pick;
    *span = per * TC;
    return (chunks + per - 1) / per;
}

bool tc_fits(const Chain<bf16>& a) {
    const int batch = a.batch, steps = a.steps;
    return steps > 0 && a.z.width % 8 == 0 && mappable(a.x, steps, a.heads / a.x.group, batch) &&
           mappable(a.y, steps, a.heads / a.y.group, batch) && mappable(a.z, steps, a.heads / a.z.group, batch) &&
           (a.out32 ? aligned16(a.out32) : aligned16(a.out));
}

int tc_chain(const Chain<bf16>& a, bool state_only, bool exact, cudaStream_t s) {
    Maps m{};
    auto in = [&](CUtensorMap* map, const Stream<bf16>& t) {
        return map_of(map, t.p, t.width, a.steps, a.heads / t.group, a.batch, t.st, t.sh, t.sb);
    };
    if (!in(&m.y, a.y) || !in(&m.z, a.z)) return EWS_ERR_LAUNCH;
    if (state_only) return exact ? go<true, 3>(a, m, s) : go<true, 2>(a, m, s);
    if (!in(&m.x, a.x)) return EWS_ERR_LAUNCH;
    return go<false, 2>(a, m, s);
}

}  // namespace decay
}  // namespace ews
