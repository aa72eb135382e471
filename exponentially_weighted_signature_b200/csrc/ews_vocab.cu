// Softmax cross entropy over a large vocabulary without keeping the logits, with its gradients.
//
//     loss_n = logsumexp_v z_nv - z_{n, t_n},    z = H W^T,
//     G = dloss_n (softmax(z)_nv - [v = t_n]),   dH = G W,   dW = G^T H.
//
// All four products run on one persistent GEMM kernel on the 5th-generation tensor core (gemm_kernel): operands
// by TMA into 128-byte-swizzled shared-memory tiles (K-major or MN-major as they lie in memory, so nothing is
// transposed), tcgen05.mma of 128 x BN x 16 issued by one thread, the accumulator in tensor memory, two deep, so
// that an output tile's epilogue runs under the next tile's products. What differs is the epilogue:
//   LSE   each row's maximum and sum of exponentials over the tile's columns, and the target's logit: the
//         logits are never stored;
//   GRAD  the logits once more, turned into G for one piece of the vocabulary (bounded by kPieceElems entries);
//   OUT   a gradient: rounded and stored, or added to a float32 partial (pieces, split K).
// The backward walks the vocabulary in pieces: G of a piece, dH += G W_piece, dW_piece = G^T H. It forms the logits a
// second time: 8 N V D operations against 6 N V D, where keeping them would take N V values.
//
// Operands are bfloat16. float32 inputs are split into three bfloat16 planes (8 bits each) and each product runs
// over the six pairs of planes that matter (2^-24), smallest first, with the same kernel.
// Measured, bfloat16: LSE over 3,690 rows, V = 131,072, D = 2,048: 1.26 ms, 1.57 PFLOP/s, 0.96 of the library product's
// burst rate and above its rate under the power cap; for 7,370 rows, D = 1,024 a piece of 10,240 entries takes 122 us for
// GRAD (1.27 PFLOP/s) and 256 us for both gradients in one launch (1.21 PFLOP/s; as launches of their own, 116 and 119 us
// for 7,424 entries, each left a fifth of its last wave of tiles idle). What bounds them is the tensor pipe under the
// power cap. Pieces of 16, 32, 64 M entries of G took 3.95, 3.24, 3.16 ms for a step that took 3.02 ms with 128 M (2.80 now).
// Targets may also be distributions over a few entries of the vocabulary, a teacher's top logits (TOP): p = softmax(t / tau)
// over a row's entries, loss_n = sum_k p_k (log p_k - log q_{id_k}) with q = softmax(z / tau), G = (q - p) dloss_n / tau. A row's
// entries are sorted by their ids once, so that an epilogue lane, which has one row, finds its tile's by a binary search while
// the tile's products run, and then looks at one id a block of 32 columns.
// Rows without a target cost nothing: a first kernel lists the rows that have one, and everything after works on those
// rows alone, packed (their number stays on the device: the kernels read it).
#include <float.h>
#include <limits.h>

#include "ews_tc.cuh"

namespace ews {
namespace vocab {

using namespace token;
using namespace tc5;

constexpr int BM = 128, BK = 64;
constexpr int EPW = 8;                 // epilogue warps
constexpr int NTH = 64 + EPW * 32;     // and one each for TMA and MMA
constexpr int SMS = 148;
constexpr long kPieceElems = 1l << 27; // entries of G (times planes) at a time: 256 MB
// Every addition to the tensor core's accumulator truncates (2^-24 of the sum, always towards zero), and a gradient's sum
// is long: for float32 a tile's sum leaves the accumulator every 256 of K and is added, rounded, to the float32 partial.
constexpr int kRun = 4;
constexpr float kLog2e = 1.4426950408889634f;
// Rounded to bfloat16 once, a teacher's G takes the gradients from 1.7e-3 of the exact ones, which is their own rounding, to 2.3e-3.
// Up to this many multiplications a product (of tiles, which are BM wide or more) G is kept in two planes, 16 bits: 2 us more for ten rows, 10 to 13 at a width of 1,024 (2,048 rows of
// 1,024: 57 -> 68 us), 34 at 127 (4,096 rows of 4,096: 82 -> 116). Beyond, a second plane would cost a second product. (Counted by the width
// itself, narrow rows had two planes of any length: 8,192 rows of 12,000, width 16, 421 us, so 248.)
constexpr long kTwoPlanes = 1l << 31;

// 2^x: the exponent unit's own instruction, results below the normal range to zero.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// G is kept in the inputs' type between the two products. The rows' loss gradients are most often one number, 1 / N,
// and where the softmax is small beside the target's 1 its rounding is then the same in every row's largest entry, so
// that it does not average out in the sums. The first row's mantissa, a number in [1, 2), is therefore left out of G and
// multiplied into the float32 sums: a common loss gradient becomes a power of two, which rounds nothing, and no entry
// changes its size by more than 2. Without it one random bfloat16 case in four had a gradient 1.5 times as far from
// the exact one as a float32 G rounded once at the end, with it one in a hundred. Loss gradients that differ from row to row,
// or a first row that differs from all others, leave the rounding as it is.
__device__ __forceinline__ float common_factor(const float* dloss, const int* row, int live, float inv_tau) {
    const float x = live > 0 ? fabsf(dloss[row[0]] * inv_tau) : 0.f;
    if (!(x > 1e-37f && x < 1e37f)) return 1.f;
    return __uint_as_float((__float_as_uint(x) & 0x007FFFFFu) | 0x3F800000u);
}

// ---- the GEMM --------------------------------------------------------------------------------------------------

enum Epilogue { LSE, GRAD, OUT };

// C (m, n) = sum over plane pairs of A_ia (m, k) B_ib (n, k)^T, in tiles and K splits.
struct Job {
    int m, n, k;
    int tiles_m, tiles_n, splits, blocks;  // k blocks of 64 a split, of every pair
    long units;
    bf16* out;            // OUT: rounded, rows n apart (bfloat16 inputs: dW of one split), or
    float* acc;           // (splits, m, n) float32 partials:
    int add;              // add to them (a later piece) rather than store
};

struct Gemm {
    Job job[2];           // OUT: dH (A = G, K-major) and dW (A = G, MN-major) in one launch; else job[0]
    int pairs;
    signed char ia[6], ib[6];
    int run;              // k blocks in one accumulator: the whole range, or few (float32 gradients, see kRun)
    int* status;          // the caller's word: a bounded wait that ran out
    const int* live;      // rows that have a target: the logits' m, dH's m, dW's k
    // LSE, GRAD (m = rows, n = the piece's part of the vocabulary from v0 on)
    const int *target, *row;  // of the packed rows: the target, and which row it was
    int v0;
    float2* part;         // (2 tiles_n of the whole vocabulary, rows): maximum, sum
    int part_tile0;
    float* picked;        // the target's logit
    const float *lse, *dloss;
    float inv_tau;        // 1 without TOP
    const int* ids;       // TOP, of the rows as they were given: (rows, top) ids in rising order, absent ones INT_MAX
    const float* prob;    // their probabilities
    const float* base;    // what a row's logits lose before they are scaled, see lse_kernel
    float* logit;         // their logits
    int top;
    bf16* g;              // (planes, rows, ldg)
    long ldg, g_plane;
    int planes;
};

struct Maps {
    CUtensorMap a[2], b[2], g;
};

// OUT: whether what a warp has goes to memory by way of shared memory: rows that start on no vector.
__host__ __device__ inline bool exchanged(const Job& j) {
    return j.n % (j.acc ? 4 : 8) || (!j.acc && ((uintptr_t)j.out & 15u));
}

// GRAD's epilogue stages its output, a box of 64 columns a warp at a time; OUT's passes what is exchanged through 16
// columns at a time, so that a store has neighbours of a row instead of 32 rows' single elements (dW of 123,911 x 158: 205 -> 90 us), with
// eight rows' partial sums in flight (both gradients of 3,000 rows, V = 5,001, D = 333, float32: 1,131 us one after the other, 503 so).
// A launch that exchanges nothing leaves that memory to the first-level cache, through which the partial sums are added to: taken from it,
// both gradients of 96 rows, V = 8,548, D = 800, float32, went from 613 to 685 us.
template <int EPI, int BN>
struct Tile {
    static constexpr int A = BM * BK * 2, B = BN * BK * 2, STAGE = A + B;
    static constexpr int OUTW = EPI == GRAD ? 4096 : 0;  // bytes a warp: 32 rows of 64 columns
    static constexpr int SHARE = 32 * 17 * 4;            // and behind all else where a launch needs it: of 16 columns and a pad
    static constexpr int STAGES = BN == 256 ? 4 : EPI == GRAD ? 5 : 6;
    static constexpr size_t bytes = (size_t)STAGES * STAGE + EPW * OUTW + 1024 + 256;
};

// The first of a row's entries at or behind `from`.
__device__ __forceinline__ int first_entry(const int* ids, int n, int from) {
    int lo = 0;
    while (n > 0) {
        const int half = n >> 1;
        if (__ldg(ids + lo + half) < from) lo += half + 1, n -= half + 1;
        else n = half;
    }
    return lo;
}

// v[k] from registers, by the bits of k (compared with each place, v went through local memory: 541 -> 660 us a pass).
__device__ __forceinline__ float element(const float v[32], int k) {
    float a[16], b[8];
    const bool k0 = k & 1, k1 = k & 2, k2 = k & 4, k3 = k & 8;
#pragma unroll
    for (int j = 0; j < 16; ++j) a[j] = k0 ? v[2 * j + 1] : v[2 * j];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = k1 ? a[2 * j + 1] : a[2 * j];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = k2 ? b[2 * j + 1] : b[2 * j];
    const float lo = k3 ? b[1] : b[0], hi = k3 ? b[3] : b[2];
    return k & 16 ? hi : lo;
}

template <int EPI, int BN, bool TOP>
__global__ void __launch_bounds__(NTH) gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Gemm a) {
    using TL = Tile<EPI, BN>;
    constexpr int S = TL::STAGES, HALF = BN / 2;
    constexpr bool BMN = EPI == OUT;
    extern __shared__ unsigned char raw[];
    unsigned char* tiles = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(tiles + S * TL::STAGE + EPW * TL::OUTW);
    uint64_t* empty = full + S;
    uint64_t* acc_full = empty + S;   // 2
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* drained = acc_empty + 2;
    uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* fail = reinterpret_cast<volatile int*>(tmem_at + 1);
    const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) mbar_init(full + i, 1), mbar_init(empty + i, 1);
        for (int i = 0; i < 2; ++i) mbar_init(acc_full + i, 1), mbar_init(acc_empty + i, EPW * 32);
        mbar_init(drained, 1);
        *fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_at)), "r"(2 * BN));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(kFull, *tmem_at, 0);
    const int live = __shfl_sync(kFull, *a.live, 0);
    const int m0 = min(a.job[0].m, live), tiles0 = (m0 + BM - 1) / BM;
    const int kb1 = (min(a.job[1].k, live) + BK - 1) / BK, blocks1 = EPI == OUT ? (kb1 + max(a.job[1].splits, 1) - 1) / max(a.job[1].splits, 1) : 0;
    const float factor = EPI == LSE ? 1.f : common_factor(a.dloss, a.row, live, a.inv_tau);
    const long units0 = (long)tiles0 * a.job[0].tiles_n * a.job[0].splits;
    const long units = units0 + (EPI == OUT ? a.job[1].units : 0);

    struct Unit {
        int job, tm, tn, sp, k0, k1;
    };
    auto unit = [&](long u) {
        Unit r;
        r.job = EPI == OUT && u >= units0 ? 1 : 0;
        if (r.job) u -= units0;
        const Job& j = a.job[r.job];
        const int tiles_m = r.job ? j.tiles_m : tiles0;
        const long per = (long)tiles_m * j.tiles_n;
        r.sp = (int)(u / per);
        const long t = u - r.sp * per;
        // neighbours share the larger operand's rows: a gradient's G, the logits' piece of the weight
        if (EPI == OUT) r.tn = (int)(t % j.tiles_n), r.tm = (int)(t / j.tiles_n);
        else r.tm = (int)(t % tiles_m), r.tn = (int)(t / tiles_m);
        const int blocks = r.job ? blocks1 : j.blocks;
        r.k0 = r.sp * blocks;
        r.k1 = min(r.k0 + blocks, r.job ? kb1 : (j.k + BK - 1) / BK);
        return r;
    };

    if (warp == 0) {
        if (lane == 0) {
            long it = 0;
            bool ok = true;
            for (long u = blockIdx.x; ok && u < units; u += gridDim.x) {
                const Unit r = unit(u);
                const CUtensorMap *ta = &maps.a[r.job], *tb = &maps.b[r.job];
                const bool amn = EPI == OUT && r.job == 1;
                for (int from = r.k0; ok && from < r.k1; from += a.run) {
                    for (int p = 0; ok && p < a.pairs; ++p)
                        for (int kb = from; kb < min(from + a.run, r.k1); ++kb, ++it) {
                            const int s = (int)(it % S);
                            if (!(ok = mbar_wait(empty + s, (uint32_t)((it / S) & 1) ^ 1u, fail))) break;
                            unsigned char* at = tiles + s * TL::STAGE;
                            mbar_expect(full + s, TL::STAGE);
                            if (amn) {
                                for (int j = 0; j < BM / 64; ++j)
                                    tma_load(ta, full + s, at + j * 8192, r.tm * BM + j * 64, kb * BK, a.ia[p]);
                            } else {
                                tma_load(ta, full + s, at, kb * BK, r.tm * BM, a.ia[p]);
                            }
                            if (BMN) {
                                for (int j = 0; j < BN / 64; ++j)
                                    tma_load(tb, full + s, at + TL::A + j * 8192, r.tn * BN + j * 64, kb * BK, a.ib[p]);
                            } else {
                                tma_load(tb, full + s, at + TL::A, kb * BK, r.tn * BN, a.ib[p]);
                            }
                        }
                }
            }
            if (!ok)
                for (long j = it > S ? it - S : 0; j < it; ++j) mbar_drain(full + j % S, (uint32_t)((j / S) & 1));
        }
    } else if (warp == 1) {
        int s = 0;
        uint32_t ph = 0;
        long tile = 0;
        bool ok = true;
        for (long u = blockIdx.x; ok && u < units; u += gridDim.x) {
            const Unit r = unit(u);
            const bool amn = EPI == OUT && r.job == 1;
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((amn ? 1u : 0u) << 15) | ((BMN ? 1u : 0u) << 16) |
                                   ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
            const uint32_t astep = amn ? 2048 >> 4 : 32 >> 4, bstep = BMN ? 2048 >> 4 : 32 >> 4;
            // a range of no blocks passes an empty accumulator on, once
            for (int from = r.k0; ok && (from == r.k0 || from < r.k1); from += a.run, ++tile) {
                const int buf = (int)(tile & 1);
                if (!(ok = warp_wait(acc_empty + buf, (uint32_t)((tile >> 1) & 1) ^ 1u, fail))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int steps = a.pairs * max(min(from + a.run, r.k1) - from, 0);
                const uint64_t ad0 = desc(smem_u32(tiles), amn), bd0 = desc(smem_u32(tiles) + TL::A, BMN);
                for (int i = 0; i < steps; ++i) {
                    if (!(ok = warp_wait(full + s, ph, fail))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
                        const uint64_t ad = ad0 + s * (TL::STAGE >> 4), bd = bd0 + s * (TL::STAGE >> 4);
#pragma unroll
                        for (int q = 0; q < BK / 16; ++q)
                            mma_bf16(tmem + buf * BN, ad + q * astep, bd + q * bstep, idesc, i > 0 || q > 0);
                        mma_commit(empty + s);
                        if (i == steps - 1) mma_commit(acc_full + buf);
                    }
                    __syncwarp();
                    if (++s == S) s = 0, ph ^= 1u;
                }
                if (ok && steps == 0) {
                    if (elect_one()) mma_commit(acc_full + buf);
                    __syncwarp();
                }
            }
        }
        if (!ok) {
            if (elect_one()) mma_commit(drained);
            __syncwarp();
            mbar_drain(drained, 0);
        }
    } else {
        // two warps share a quarter of the rows, each has half of the tile's columns
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        long tile = 0;
        bool ok = true;
        for (long u = blockIdx.x; ok && u < units; u += gridDim.x) {
            const Unit r = unit(u);
            const Job& job = a.job[r.job];
            const int* ids = nullptr;
            long entry0 = 0;
            int entry = 0, next = INT_MAX;  // the row's next entry, as a column of the tile
            if constexpr (TOP) {
                const int row = r.tm * BM + quarter * 32 + lane, col0 = a.v0 + r.tn * BN;
                if (row < m0) {
                    entry0 = (long)a.row[row] * a.top, ids = a.ids + entry0;
                    entry = first_entry(ids, a.top, col0 + half * HALF);
                    if (entry < a.top) next = __ldg(ids + entry) - col0;
                }
            }
            auto step_entry = [&] {
                ++entry;
                next = entry < a.top ? __ldg(ids + entry) - a.v0 - r.tn * BN : INT_MAX;
            };
            for (int from = r.k0; from == r.k0 || from < r.k1; from += a.run, ++tile) {
                const int buf = (int)(tile & 1);
                if (!(ok = __all_sync(kFull, mbar_wait(acc_full + buf, (uint32_t)((tile >> 1) & 1), fail)))) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t src = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
                const int row = r.tm * BM + quarter * 32 + lane;
                const bool in = row < (r.job ? job.m : m0);
                const int cols = min(half * HALF + HALF, job.n - r.tn * BN);
                const bool add = job.add || from > r.k0;
                if (EPI == LSE) {
                    const int pick = !TOP && in ? a.target[row] - a.v0 - r.tn * BN : -1;
                    const float scale = TOP ? kLog2e * a.inv_tau : kLog2e;
                    float mx = -INFINITY, sum = 0.f;
                    for (int c = half * HALF; c < cols; c += 32) {
                        float v[32];
                        tmem_ld32(src + c, v);
                        if (c + 32 > cols) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (c + j >= cols) v[j] = -INFINITY;
                        }
                        float top = v[0];
#pragma unroll
                        for (int j = 1; j < 32; ++j) top = fmaxf(top, v[j]);
                        const float was = mx;
                        mx = fmaxf(mx, top);
                        // the maximum leaves before the scaling: its own term is 1 and no other one exceeds it, where a rounded
                        // -mx * log2(e) put every exponent off by up to 2^-24 of the maximum
                        const float base = mx == -INFINITY ? 0.f : mx;
                        const uint64_t scale2 = pair(scale, scale), base2 = pair(-base, -base);
                        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float e0, e1;
                            unpair(mul2(add2(pair(v[j], v[j + 1]), base2), scale2), e0, e1);
                            part[j & 3] += ex2(e0), part[(j & 3) + 1] += ex2(e1);
                        }
                        sum = sum * exp2f((was - base) * scale) + ((part[0] + part[1]) + (part[2] + part[3]));
                        if constexpr (TOP) {
                            const int end = min(c + 32, cols);
                            while (next < end) {
                                a.logit[entry0 + entry] = element(v, next - c);
                                step_entry();
                            }
                        } else if ((unsigned)(pick - c) < 32u) {
                            float z = 0.f;
#pragma unroll
                            for (int j = 0; j < 32; ++j) z = pick - c == j ? v[j] : z;
                            a.picked[row] = z;
                        }
                    }
                    if (in) a.part[(long)((a.part_tile0 + r.tn) * 2 + half) * job.m + row] = make_float2(mx, sum);
                } else if (EPI == GRAD) {
                    const int t = in ? a.target[row] : -1;
                    const int pick = TOP || t < 0 ? -1 : t - a.v0 - r.tn * BN;
                    const float w = t < 0 ? 0.f : a.dloss[a.row[row]] * a.inv_tau / factor;
                    const float scale = TOP ? kLog2e * a.inv_tau : kLog2e;
                    const float lse = in ? a.lse[row] : 0.f, shift = -lse * kLog2e, base = TOP && in ? a.base[a.row[row]] : 0.f;
                    const uint64_t scale2 = pair(scale, scale), shift2 = pair(shift, shift);
                    for (int c = half * HALF; c < cols; c += 32) {
                        float v[32];
                        tmem_ld32(src + c, v);
                        if constexpr (TOP) {
#pragma unroll
                            for (int j = 0; j < 32; j += 2) unpair(add2(pair(v[j], v[j + 1]), pair(-base, -base)), v[j], v[j + 1]);
                        }
                        if (a.planes > 1) {  // float32: the scaled exponent's own rounding (2^-24 of some 15) would be the largest error
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = expf(TOP ? fmaf(v[j], a.inv_tau, -lse) : v[j] - lse);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                float e0, e1;
                                unpair(fma2(pair(v[j], v[j + 1]), scale2, shift2), e0, e1);
                                v[j] = ex2(e0), v[j + 1] = ex2(e1);
                            }
                        }
                        if constexpr (TOP) {
                            const int end = min(c + 32, cols);
                            while (next < end) {
                                const float p = __ldg(a.prob + entry0 + entry);
#pragma unroll
                                for (int j = 0; j < 32; ++j) v[j] -= next - c == j ? p : 0.f;
                                step_entry();
                            }
                        } else if ((unsigned)(pick - c) < 32u) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] -= pick - c == j ? 1.f : 0.f;
                        }
                        if (t >= 0) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] *= w;
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0.f;
                        }
                        if (c + 32 > cols) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (c + j >= cols) v[j] = 0.f;
                        }
                        if (a.planes == 1) {
                            // through shared memory (rows of 64 columns, swizzled) and out by TMA, which drops what lies
                            // beyond the matrix: stored from the registers, a warp's 32 rows at 16 bytes each took
                            // the logits' pass from 1.46 to 1.09 PFLOP/s
                            unsigned char* box = tiles + S * TL::STAGE + (warp - 2) * TL::OUTW;
                            if ((c & 32) == 0) {
                                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                                __syncwarp();
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                Vec<bf16, true>::store(reinterpret_cast<bf16*>(box + lane * 128 + (((c & 32) / 8 + j) ^ (lane & 7)) * 16), v + 8 * j);
                            if ((c & 32) || c + 32 >= cols) {
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                                __syncwarp();
                                if (lane == 0) {
                                    tma_store(&maps.g, box, r.tn * BN + (c & ~63), r.tm * BM + quarter * 32, 0);
                                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                                }
                            }
                            continue;
                        }
                        for (int s = 0; row < job.m && s < a.planes; ++s) {  // rows that are none: zeros
                            bf16* g = a.g + s * a.g_plane + (long)row * a.ldg + r.tn * BN + c;
#pragma unroll
                            for (int j = 0; j < 32; j += 8) {
                                uint32_t q[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    q[e] = pack_bf16(v[j + 2 * e], v[j + 2 * e + 1]);
                                    v[j + 2 * e] -= bf16_lo(q[e]), v[j + 2 * e + 1] -= bf16_hi(q[e]);
                                }
                                if (r.tn * BN + c + j < a.ldg) *reinterpret_cast<uint4*>(g + j) = make_uint4(q[0], q[1], q[2], q[3]);
                            }
                        }
                    }
                } else {
                    for (int c = half * HALF; c < cols; c += 32) {
                        float v[32];
                        tmem_ld32(src + c, v);
                        if (r.k0 >= r.k1) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] = 0.f;
                        }
                        const int col = r.tn * BN + c;
                        const int w = min(32, cols - c);
                        if (!job.acc) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[j] *= factor;
                        }
                        if (exchanged(job)) {
                            float* share = reinterpret_cast<float*>(tiles + S * TL::STAGE + 256 + (warp - 2) * TL::SHARE);
                            const int first = r.tm * BM + quarter * 32, there = min((r.job ? job.m : m0) - first, 32);
#pragma unroll
                            for (int h = 0; h < 32; h += 16) {
                                if (h >= w) break;
                                __syncwarp();
#pragma unroll
                                for (int j = 0; j < 16; ++j) share[lane * 17 + j] = v[h + j];
                                __syncwarp();
                                const int k = h + (lane & 15), rows = k < w ? there : 0;
                                if (job.acc) {  // eight rows' sums in flight
                                    for (int q0 = lane >> 4; q0 < rows; q0 += 16) {
                                        float* p = job.acc + ((long)r.sp * job.m + first + q0) * job.n + col + k;
                                        float o[8];
#pragma unroll
                                        for (int i = 0; i < 8; ++i) o[i] = add && q0 + 2 * i < rows ? p[(long)(2 * i) * job.n] : 0.f;
#pragma unroll
                                        for (int i = 0; i < 8; ++i) {
                                            const float x = share[(q0 + 2 * i) * 17 + (lane & 15)];
                                            if (q0 + 2 * i < rows) p[(long)(2 * i) * job.n] = add ? o[i] + x : x;
                                        }
                                    }
                                } else {
                                    for (int q = lane >> 4; q < rows; q += 2)
                                        job.out[(long)(first + q) * job.n + col + k] = from_f<bf16>(share[q * 17 + (lane & 15)]);
                                }
                            }
                        } else if (!in) {
                        } else if (job.acc) {
                            float* p = job.acc + ((long)r.sp * job.m + row) * job.n + col;
                            if (add) {
                                float4 o[8];
#pragma unroll
                                for (int j = 0; j < 32; j += 4)
                                    if (j < w) o[j / 4] = *reinterpret_cast<const float4*>(p + j);
#pragma unroll
                                for (int j = 0; j < 32; j += 4)
                                    if (j < w) v[j] += o[j / 4].x, v[j + 1] += o[j / 4].y, v[j + 2] += o[j / 4].z, v[j + 3] += o[j / 4].w;
                            }
#pragma unroll
                            for (int j = 0; j < 32; j += 4)
                                if (j < w) *reinterpret_cast<float4*>(p + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                        } else {
                            bf16* p = job.out + (long)row * job.n + col;
#pragma unroll
                            for (int j = 0; j < 32; j += 8)
                                if (j < w) Vec<bf16, true>::store(p + j, v + j);
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                mbar_arrive(acc_empty + buf);
            }
        }
        if (EPI == GRAD && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (threadIdx.x == 0 && *fail) report(a.status, EWS_ERR_LOOKBACK_TIMEOUT);
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN));
}

// ---- the passes around it ------------------------------------------------------------------------------------

// Rows as bfloat16 planes of `ld` columns, zero beyond `dim`.
template <typename T>
struct Pack {
    const T* in;
    long stride, rows;
    bf16* out;
    long plane;
};

// What the rows' targets say, for the forward and its backward: how many rows have one, which rows those are and their
// targets (by packed position), and each row's packed position (-1: no target).
struct RowPlan {
    int *live, *row, *target, *slot;
};

__host__ __device__ inline RowPlan row_plan(int* p, long rows) { return RowPlan{p, p + 4, p + 4 + rows, p + 4 + 2 * rows}; }

// One CTA: every thread counts its share of the rows, the CTA scans the counts, every thread lists its share.
__global__ void __launch_bounds__(1024) plan_kernel(const void* __restrict__ targets, int wide, long rows, long vocab, long ignore, RowPlan p,
                                                    float* __restrict__ loss, int* status) {
    __shared__ int warp_sum[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long per = (rows + 1023) / 1024, first = tid * per, last = first + per < rows ? first + per : rows;
    auto target = [&](long i) {
        const long t = wide ? __ldg(reinterpret_cast<const long long*>(targets) + i) : (long)__ldg(reinterpret_cast<const int*>(targets) + i);
        if (t == ignore) return -1;
        if (t >= 0 && t < vocab) return (int)t;
        report(status, EWS_ERR_INDEX);
        return -1;
    };
    int count = 0;
#pragma unroll 8
    for (long i = first; i < last; ++i) count += target(i) >= 0;
    int incl = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFull, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int at = incl - count;
    for (int w = 0; w < warp; ++w) at += warp_sum[w];
    if (tid == 1023) *p.live = at + count;
#pragma unroll 4
    for (long i = first; i < last; ++i) {
        const int t = target(i);
        p.slot[i] = t >= 0 ? at : -1;
        if (t >= 0) {
            p.row[at] = (int)i;
            p.target[at] = t;
            ++at;
        } else {
            loss[i] = 0.f;
        }
    }
}

// Packs the hidden rows that have a target (zeros up to the end of their last tile), and behind them the rows of a piece
// of the weight.
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Pack<T> h, const __grid_constant__ Pack<T> w, int dim, int ld,
                                                   int planes, const int* __restrict__ live_rows, const int* __restrict__ rows) {
    const int per = ld / 8;
    const int live = *live_rows;
    const long hidden_rows = h.rows ? min(h.rows, ((long)live + BM - 1) / BM * BM) : 0;
    const long total = (hidden_rows + w.rows) * per;
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < total; e += (long)gridDim.x * 256) {
        long row = e / per;
        const int col = (int)(e - row * per) * 8;
        const bool hidden = row < hidden_rows;
        if (!hidden) row -= hidden_rows;
        const T* in = hidden ? h.in : w.in;
        const long stride = hidden ? h.stride : w.stride;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
        if (!hidden || row < live) {
            const T* p = in + (hidden ? rows[row] : row) * stride + col;
            if (stride % (16 / (int)sizeof(T)) == 0 && dim % 8 == 0 && aligned16_dev(in)) {
#pragma unroll
                for (int j = 0; j < 8; j += Vec<T, true>::N) Vec<T, true>::load(p + j, v + j);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (col + j < dim) v[j] = to_f(p[j]);
            }
        }
        bf16* out = (hidden ? h.out : w.out) + row * ld + col;
        const long plane = hidden ? h.plane : w.plane;
        for (int s = 0; s < planes; ++s) {
            Vec<bf16, true>::store(out + s * plane, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] -= to_f(from_f<bf16>(v[j]));
        }
    }
}

// A distribution's targets: by row of the call, see the epilogues.
struct Entries {
    int *ids, *flag;             // flag: 0 where the row has a distribution, else -1: the row plan's targets
    float *prob, *self;          // self: sum p log p, in whose place the base is left for the backward
    float* base;
    int top;
    float inv_tau;
};

inline Entries entries_of(void* p, long rows, int top, float inv_tau) {
    int* at = static_cast<int*>(p);
    float* f = reinterpret_cast<float*>(at + rows * (top + 1));
    return Entries{at, at + rows * top, f, f + rows * top, f + rows * top, top, inv_tau};
}

constexpr int kMaxTop = 128;

// A warp a row: the probabilities of its entries, sorted by id (equal ids keep their order). Ids below zero and logits of -inf are
// absent, a row of which is left nothing has no target; an id beyond the vocabulary is absent and reported. The temperature comes
// after the row's maximum has been subtracted: before, a finite logit near its type's ends would overflow, and every logit would be
// rounded at its own size.
template <typename L>
__global__ void __launch_bounds__(256) entries_kernel(const void* __restrict__ ids, int wide, const L* __restrict__ logits, long rows, long vocab,
                                                      Entries e, int* status) {
    constexpr int E = kMaxTop / 32;
    __shared__ int keys[8][kMaxTop];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long row = (long)blockIdx.x * 8 + warp;
    if (row >= rows) return;
    int id[E];
    float t[E], top = -INFINITY;
    bool bad = false, any = false;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int i = k * 32 + lane;
        id[k] = INT_MAX, t[k] = -INFINITY;
        if (i < e.top) {
            const long at = row * e.top + i;
            const long v = wide ? (long)__ldg(static_cast<const long long*>(ids) + at) : (long)__ldg(static_cast<const int*>(ids) + at);
            if (v >= vocab) report(status, EWS_ERR_INDEX);
            const float x = to_f(logits[at]);
            if (v >= 0 && v < vocab && x != -INFINITY) id[k] = (int)v, t[k] = x, any = true, bad = bad || x != x, top = fmaxf(top, x);
            keys[warp][i] = id[k];
        }
    }
    __syncwarp();  // the keys
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    if (__any_sync(kFull, bad)) top = NAN;
    any = __any_sync(kFull, any);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        t[k] = (t[k] - top) * e.inv_tau;
        if (id[k] != INT_MAX) sum += expf(t[k]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    const float log_sum = logf(sum);
    float self = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        const int i = k * 32 + lane;
        if (i >= e.top) continue;
        float p = 0.f;
        if (id[k] != INT_MAX) {
            p = expf(t[k]) / sum;
            if (p != 0.f) self += p * (t[k] - log_sum);
        }
        int rank = 0;
        for (int j = 0; j < e.top; ++j) {
            const int other = keys[warp][j];
            rank += other < id[k] || (other == id[k] && j < i);
        }
        e.ids[row * e.top + rank] = id[k];
        e.prob[row * e.top + rank] = p;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) self += __shfl_xor_sync(kFull, self, o);
    if (lane == 0) e.self[row] = self, e.flag[row] = any ? 0 : -1;
}

// The row's logsumexp from the tiles' maxima and sums: 32 rows by 8 groups of tiles a CTA. TOP: `picked` are the entries' logits.
template <bool TOP>
__global__ void __launch_bounds__(256) lse_kernel(const float2* __restrict__ part, int tiles, long rows, RowPlan plan,
                                                  const float* __restrict__ picked, float* __restrict__ loss, float* __restrict__ lse, Entries e) {
    __shared__ float2 red[8][32];
    const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
    const long row = (long)blockIdx.x * 32 + l;
    const int live = *plan.live;
    const float scale = TOP ? kLog2e * e.inv_tau : kLog2e;
    float m = -INFINITY, s = 0.f;
    if (row < live)
        for (int t0 = g; t0 < tiles; t0 += 64) {
            float2 p[8];  // eight tiles in flight
#pragma unroll
            for (int k = 0; k < 8; ++k) p[k] = t0 + 8 * k < tiles ? part[(long)(t0 + 8 * k) * rows + row] : make_float2(-INFINITY, 0.f);
            float n = m;
#pragma unroll
            for (int k = 0; k < 8; ++k) n = fmaxf(n, p[k].x);
            const float base = n == -INFINITY ? 0.f : n;
            s *= exp2f((m - base) * scale);
#pragma unroll
            for (int k = 0; k < 8; ++k) s += p[k].y * exp2f((p[k].x - base) * scale);
            m = n;
        }
    red[g][l] = make_float2(m, s);
    __syncthreads();
    if (!TOP && (g > 0 || row >= live)) return;
    m = red[0][l].x, s = red[0][l].y;
    for (int j = 1; j < 8; ++j) {
        const float2 p = red[j][l];
        const float n = fmaxf(m, p.x);
        const float base = n == -INFINITY ? 0.f : n;
        s = s * exp2f((m - base) * scale) + p.y * exp2f((p.x - base) * scale);
        m = n;
    }
    if constexpr (TOP) {
        // sum p (m - z) / tau: what a student is sure of and right about cancels first; the groups take the entries in turn
        const long at = row < live ? (long)plan.row[row] * e.top : 0;
        float far = 0.f;
        bool twice = false;  // an id occurs twice: neighbours, the entries are sorted
        if (row < live)
            for (int k = g; k < e.top; k += 8) {
                const float p = e.prob[at + k];
                if (p != 0.f) far += p * ((m - picked[at + k]) * e.inv_tau);
                twice = twice || (k > 0 && e.ids[at + k] != INT_MAX && e.ids[at + k] == e.ids[at + k - 1]);
            }
        __shared__ float sums[8][32];
        __shared__ bool again[8][32];
        sums[g][l] = far, again[g][l] = twice;
        __syncthreads();
        if (g > 0 || row >= live) return;
        for (int j = 1; j < 8; ++j) far += sums[j][l], twice = twice || again[j][l];
        const float rest = logf(s), kl = far + rest + e.self[plan.row[row]];
        // For the gradient: q = exp((z - base) / tau - lse). A logsumexp is rounded at its own size, and q by as much relatively: beyond
        // 64 (2^-18 of q) the row's maximum stays apart, and what is rounded are differences from it.
        const float base = fabsf(m * e.inv_tau) > 64.f && fabsf(m) <= FLT_MAX ? m : 0.f;
        lse[row] = fmaf(m - base, e.inv_tau, rest);
        e.base[plan.row[row]] = base;
        // Of distinct ids the sum is never negative, its rounding may be. An id that is two entries can have more of the student's
        // probability than either of the teacher's.
        loss[plan.row[row]] = kl < 0.f && !twice ? 0.f : kl;
        return;
    }
    // The maximum and the target's logit cancel first, exactly where the target is the maximum: a sum rounded at the
    // logits' size would lose a confident row's loss, or turn it negative. With s >= 1 no loss is.
    const float rest = logf(s);
    lse[row] = m + rest;
    loss[plan.row[row]] = (m - picked[row]) + rest;
}

// A gradient from its float32 partials, summed in order and rounded once; with `slot` the rows of the result are taken
// from their packed positions, and a row without one is zero.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) reduce_kernel(const float* __restrict__ acc, int splits, long rows, int n, const int* __restrict__ slot,
                                                     const float* __restrict__ dloss, const int* __restrict__ live_rows,
                                                     const int* __restrict__ row_of, float inv_tau, T* __restrict__ out) {
    constexpr int W = VEC ? 4 : 1;
    const int per = n / W;
    const long total = rows * n;
    // a row's vectors to consecutive threads
    const int lanes = per < 256 ? per : 256, group = 256 / lanes, l = threadIdx.x % lanes, g = threadIdx.x / lanes;
    if (g >= group) return;
    const float factor = common_factor(dloss, row_of, *live_rows, inv_tau);
    for (long row = (long)blockIdx.x * group + g; row < rows; row += (long)gridDim.x * group) {
        const long at = slot ? slot[row] : row;
        for (int c = l; c < per; c += lanes) {
            float s[W];
#pragma unroll
            for (int j = 0; j < W; ++j) s[j] = 0.f;
            if (at >= 0) {
                const float* p = acc + at * n + c * W;
                Vec<float, VEC>::load(p, s);
                constexpr int AT_ONCE = VEC ? 4 : 8;  // in flight, added in order
                for (int k0 = 1; k0 < splits; k0 += AT_ONCE) {
                    float v[AT_ONCE][W];
#pragma unroll
                    for (int k = 0; k < AT_ONCE; ++k)
                        if (k0 + k < splits) Vec<float, VEC>::load(p + (k0 + k) * total, v[k]);
#pragma unroll
                    for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
                        for (int j = 0; j < W; ++j) s[j] = k0 + k < splits ? s[j] + v[k][j] : s[j];
                }
            }
#pragma unroll
            for (int j = 0; j < W; ++j) s[j] *= factor;
            T* o = out + row * n + c * W;
            if constexpr (VEC && sizeof(T) == 2) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(s[0], s[1]), pack_bf16(s[2], s[3]));
            else Vec<T, VEC>::store(o, s);
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------

// (planes, rows, cols) bfloat16 with rows `ld` apart; a box of 64 columns by `box_rows` rows.
struct Operand {
    const bf16* p;
    long rows, cols, ld, plane;
    int planes;
};

bool make_map(CUtensorMap* map, const Operand& o, int box_rows) {
    EncodeFn enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
    const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.planes > 1 ? o.plane : o.ld * o.rows) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(o.p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Column tiles of 256, or of 128 where a narrow output leaves half of a wide one empty.
int tile_n(long n) { return n <= 128 ? 128 : 256; }

// K splits of a gradient of (m, n): as many as leave no SM without a tile, none below eight k blocks.
int splits_of(long m, long n, long k, long other) {
    const long tiles = ((m + BM - 1) / BM) * ((n + tile_n(n) - 1) / tile_n(n));
    long want = (SMS - other > tiles ? SMS - other : tiles) / tiles;
    const long most = (k + BK * 8 - 1) / (BK * 8);
    if (want > most) want = most;
    return want < 1 ? 1 : (int)want;
}

Job job_of(long m, long n, long k, int splits) {
    Job j{};
    j.m = (int)m, j.n = (int)n, j.k = (int)k, j.splits = splits;
    j.tiles_m = (int)((m + BM - 1) / BM), j.tiles_n = (int)((n + tile_n(n) - 1) / tile_n(n));
    j.blocks = (int)(((k + BK - 1) / BK + splits - 1) / splits);
    j.units = (long)j.tiles_m * j.tiles_n * splits;
    return j;
}

template <int EPI, int BN, bool TOP>
int gemm_bn(const Maps& maps, const Gemm& g, cudaStream_t s) {
    auto* kern = gemm_kernel<EPI, BN, TOP>;
    size_t bytes = Tile<EPI, BN>::bytes;
    for (const Job& j : g.job)
        if (EPI == OUT && j.units && exchanged(j)) bytes = Tile<EPI, BN>::bytes + EPW * Tile<EPI, BN>::SHARE;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return EWS_ERR_LAUNCH;
    const long units = g.job[0].units + g.job[1].units;
    kern<<<(unsigned)(units < SMS ? units : SMS), NTH, bytes, s>>>(maps, g);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

// Operands of job[0], and of job[1] where it has units (OUT). Both jobs' n is the model's width, so they share BN.
template <int EPI>
int gemm(Gemm g, const Operand& a0, const Operand& b0, const Operand& a1, const Operand& b1, int planes, cudaStream_t s) {
    const int gplanes = EPI == LSE ? planes : g.planes;
    static const signed char pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};  // smallest products first
    g.pairs = planes == 1 ? 1 : 6;
    for (int i = 0; i < g.pairs; ++i) g.ia[i] = planes == 1 ? 0 : pa[i], g.ib[i] = planes == 1 ? 0 : pb[i];
    if (EPI == OUT && planes == 1)  // G's second plane first
        for (g.pairs = 0; g.pairs < gplanes; ++g.pairs) g.ia[g.pairs] = (signed char)(gplanes - 1 - g.pairs);
    Maps m{};
    if (EPI == GRAD && gplanes == 1 &&
        !make_map(&m.g, Operand{g.g, g.job[0].m, g.job[0].n, g.ldg, 0, 1}, 32))
        return EWS_ERR_LAUNCH;
    g.run = EPI == OUT && planes > 1 ? kRun : 1 << 28;
    const int bn = tile_n(g.job[0].units ? g.job[0].n : g.job[1].n);
    if (g.job[0].units && (!make_map(&m.a[0], a0, BM) || !make_map(&m.b[0], b0, EPI == OUT ? 64 : bn))) return EWS_ERR_LAUNCH;
    if (g.job[1].units && (!make_map(&m.a[1], a1, 64) || !make_map(&m.b[1], b1, 64))) return EWS_ERR_LAUNCH;
    if constexpr (EPI != OUT)
        if (g.top) return bn == 128 ? gemm_bn<EPI, 128, true>(m, g, s) : gemm_bn<EPI, 256, true>(m, g, s);
    return bn == 128 ? gemm_bn<EPI, 128, false>(m, g, s) : gemm_bn<EPI, 256, false>(m, g, s);
}

struct Plan {
    int planes, gplanes;   // planes of an operand, of G
    int ldd;               // padded dim
    bool pack_w;           // the weight is packed piece by piece
    long piece, pieces;    // vocabulary entries a piece
    int split_h, split_w;  // K splits of dhidden, dweight
    bool acc_w;
    size_t picked, part, h, w, g, ah, aw, bytes;
};

int check(const ews_vocab_args* a) {
    if (!a || a->rows < 0 || a->vocab <= 0 || a->dim <= 0) return EWS_ERR_INVALID_ARGUMENT;
    if (a->hidden_stride < a->dim || a->weight_stride < a->dim) return EWS_ERR_INVALID_ARGUMENT;
    if (a->dtype != EWS_DTYPE_F32 && a->dtype != EWS_DTYPE_BF16) return EWS_ERR_UNSUPPORTED;
    if (a->rows >= (1l << 30) || a->vocab >= (1l << 30) || a->dim >= (1l << 20)) return EWS_ERR_UNSUPPORTED;
    return EWS_OK;
}

long up(long n, long to) { return (n + to - 1) / to * to; }

// Pieces of the vocabulary: the fewest that keep G (and a packed weight) within kPieceElems, or up to four more
// where that fills the SMs' waves of tiles better (a launch whose last wave has a few tiles idles the rest).
void pick_pieces(Plan* p, long n, long v, long d, bool bwd) {
    long most = v;
    if (bwd) most = kPieceElems / (n * p->gplanes);
    if (p->pack_w && kPieceElems / ((long)p->ldd * p->planes) < most) most = kPieceElems / ((long)p->ldd * p->planes);
    if (most < 1024) most = 1024;
    const long least = (v + most - 1) / most;
    p->pieces = least;
    p->piece = least == 1 ? v : up((v + least - 1) / least, 256);
    if (!bwd || least == 1) {
        p->pieces = (v + p->piece - 1) / p->piece;
        return;
    }
    const long tm = (n + BM - 1) / BM, td = (d + tile_n(d) - 1) / tile_n(d);
    double best = 0;
    for (long c = least; c <= least + 4; ++c) {
        const long piece = up((v + c - 1) / c, 256), count = (v + piece - 1) / piece;
        auto waves = [](long tiles) { return (double)((tiles + SMS - 1) / SMS); };
        // a tile's time goes with its K: the width for the logits, the piece and the rows for the gradients
        const double kgrad = (piece * (double)(tm * td) + n * (double)(piece / BM * td)) / (tm * td + piece / BM * td);
        const double cost = count * (waves(tm * (piece / 256)) * d + waves(tm * td + piece / BM * td) * kgrad + 2000.0);
        if (c == least || cost < best) best = cost, p->piece = piece, p->pieces = count;
    }
}

// K splits of the gradients where one has few tiles and long sums: as many as bring a unit down to an SM's share of both products
// (96 rows, V = 8,548, D = 800, float32: 524 -> 78 us for both gradients), at least eight k blocks and at most 48 to a sum. For a teacher's
// loss alone: the loss against single targets keeps its splits, and with them the order of its sums and its results to the last bit.
void even_splits(Plan* p, long n, long d) {
    const long td = (d + tile_n(d) - 1) / tile_n(d), th = (n + BM - 1) / BM * td, tw = (p->piece + BM - 1) / BM * td;
    const long kh = (p->piece + BK - 1) / BK, kw = (n + BK - 1) / BK, all = th * kh + tw * kw;
    auto even = [&](long k, int split) {
        long want = k * SMS / all;
        if (want > k / 8) want = k / 8;
        if (want > 48) want = 48;
        return want > split ? (int)want : split;
    };
    p->split_h = even(kh, p->split_h), p->split_w = even(kw, p->split_w);
}

// top: entries a row of a teacher's logits; 0 for the loss against single targets.
Plan plan(const ews_vocab_args* a, bool bwd, int top = 0) {
    Plan p{};
    p.planes = p.gplanes = a->dtype == EWS_DTYPE_F32 ? 3 : 1;
    if (top && p.planes == 1 && a->rows * a->vocab <= kTwoPlanes / (a->dim < BM ? BM : a->dim)) p.gplanes = 2;
    p.ldd = (int)up(a->dim, 8);
    p.pack_w = p.planes > 1 || a->weight_stride % 8 || a->dim % 8 || !aligned16(a->weight);
    const long n = a->rows, v = a->vocab;
    pick_pieces(&p, n, v, a->dim, bwd);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    p.h = take(sizeof(bf16) * (size_t)p.planes * n * p.ldd);
    if (p.pack_w) p.w = take(sizeof(bf16) * (size_t)p.planes * p.piece * p.ldd);
    if (!bwd) {
        p.picked = take(sizeof(float) * n * (top ? top : 1));
        const long tiles = p.pieces * ((p.piece + tile_n(p.piece) - 1) / tile_n(p.piece));
        p.part = take(sizeof(float2) * 2 * tiles * n);
    } else {
        p.g = take(sizeof(bf16) * (size_t)p.gplanes * n * up(p.piece, 8));
        const long th = ((n + BM - 1) / BM) * ((a->dim + tile_n(a->dim) - 1) / tile_n(a->dim));
        const long tw = ((p.piece + BM - 1) / BM) * ((a->dim + tile_n(a->dim) - 1) / tile_n(a->dim));
        p.split_h = splits_of(n, a->dim, p.piece, tw);
        p.split_w = splits_of(p.piece, a->dim, n, th * p.split_h);
        if (top) even_splits(&p, n, a->dim);
        p.acc_w = p.split_w > 1 || p.planes > 1;
        p.ah = take(sizeof(float) * (size_t)p.split_h * n * a->dim);
        if (p.acc_w) p.aw = take(sizeof(float) * (size_t)p.split_w * p.piece * a->dim);
    }
    p.bytes = at;
    return p;
}

unsigned grid_of(long total) {
    const long b = (total + 255) / 256;
    return (unsigned)(b < 1 ? 1 : b < SMS * 32 ? b : SMS * 32);
}

template <typename T>
int reduce(const ews_vocab_args* a, const float* acc, int splits, long rows, const int* slot, float inv_tau, T* out, cudaStream_t s) {
    const RowPlan plan = row_plan(a->plan, a->rows);
    const long n = a->dim;
    const unsigned grid = grid_of(rows * n / 4 + 1);
    if (n % 4 == 0 && aligned16(out)) reduce_kernel<T, true><<<grid, 256, 0, s>>>(acc, splits, rows, (int)n, slot, a->dloss, plan.live, plan.row, inv_tau, out);
    else reduce_kernel<T, false><<<grid, 256, 0, s>>>(acc, splits, rows, (int)n, slot, a->dloss, plan.live, plan.row, inv_tau, out);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

// The operands of the piece [v0, v0 + n) of the vocabulary, packed where they cannot be read as they lie (hidden:
// with the first piece).
template <typename T>
int operands(const ews_vocab_args* a, const Plan& p, char* w, long v0, long n, Operand* h, Operand* o, cudaStream_t s) {
    Pack<T> ph{}, pw{};
    if (v0 == 0) {
        bf16* at = reinterpret_cast<bf16*>(w + p.h);
        h->p = at, h->rows = a->rows, h->cols = h->ld = p.ldd, h->planes = p.planes, h->plane = a->rows * p.ldd;
        ph.in = static_cast<const T*>(a->hidden), ph.stride = a->hidden_stride, ph.rows = a->rows, ph.out = at, ph.plane = h->plane;
    }
    const T* rows = static_cast<const T*>(a->weight) + v0 * a->weight_stride;
    o->rows = n, o->planes = p.planes;
    if (p.pack_w) {
        bf16* at = reinterpret_cast<bf16*>(w + p.w);
        o->p = at, o->cols = o->ld = p.ldd, o->plane = n * p.ldd;
        pw.in = rows, pw.stride = a->weight_stride, pw.rows = n, pw.out = at, pw.plane = o->plane;
    } else {
        o->p = reinterpret_cast<const bf16*>(rows), o->cols = a->dim, o->ld = a->weight_stride, o->plane = 0;
    }
    if (ph.rows + pw.rows == 0) return EWS_OK;
    const RowPlan plan = row_plan(a->plan, a->rows);
    pack_kernel<T><<<grid_of((ph.rows + pw.rows) * (p.ldd / 8)), 256, 0, s>>>(ph, pw, (int)a->dim, p.ldd, p.planes, plan.live, plan.row);
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

// The rows' distributions in a product's arguments; without any, the targets' own.
void targets(Gemm* g, const Entries* e) {
    g->inv_tau = e ? e->inv_tau : 1.f;
    if (e) g->ids = e->ids, g->prob = e->prob, g->base = e->base, g->top = e->top;
}

template <typename T>
int forward(const ews_vocab_args* a, const Plan& p, const Entries* e, cudaStream_t s) {
    char* w = static_cast<char*>(a->work);
    Operand h{}, wt{}, none{};
    int rc = EWS_OK;
    Gemm g{};
    const RowPlan plan = row_plan(a->plan, a->rows);
    if (e) plan_kernel<<<1, 1024, 0, s>>>(e->flag, 0, a->rows, a->vocab, -1, plan, a->loss, a->status);
    else plan_kernel<<<1, 1024, 0, s>>>(a->targets, a->targets_wide, a->rows, a->vocab, a->ignore, plan, a->loss, a->status);
    g.status = a->status;
    targets(&g, e);
    g.live = plan.live, g.target = plan.target, g.row = plan.row;
    g.part = reinterpret_cast<float2*>(w + p.part);
    g.picked = g.logit = reinterpret_cast<float*>(w + p.picked);
    for (long v0 = 0; rc == EWS_OK && v0 < a->vocab; v0 += p.piece) {
        const long n = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;
        if ((rc = operands<T>(a, p, w, v0, n, &h, &wt, s)) != EWS_OK) break;
        g.job[0] = job_of(a->rows, n, a->dim, 1), g.v0 = (int)v0;
        rc = gemm<LSE>(g, h, wt, none, none, p.planes, s);
        g.part_tile0 += g.job[0].tiles_n;
    }
    if (rc != EWS_OK) return rc;
    const unsigned grid = (unsigned)((a->rows + 31) / 32);
    if (e) lse_kernel<true><<<grid, 256, 0, s>>>(g.part, 2 * g.part_tile0, a->rows, plan, g.picked, a->loss, a->lse, *e);
    else lse_kernel<false><<<grid, 256, 0, s>>>(g.part, 2 * g.part_tile0, a->rows, plan, g.picked, a->loss, a->lse, Entries{});
    return cudaGetLastError() == cudaSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T>
int backward(const ews_vocab_args* a, const Plan& p, const Entries* e, cudaStream_t s) {
    char* w = static_cast<char*>(a->work);
    Operand h{}, wt{}, go{}, none{};
    int rc = EWS_OK;
    float* acc_h = reinterpret_cast<float*>(w + p.ah);
    const RowPlan plan = row_plan(a->plan, a->rows);
    float* acc_w = p.acc_w ? reinterpret_cast<float*>(w + p.aw) : nullptr;
    Gemm base{};
    base.status = a->status;
    targets(&base, e);
    base.live = plan.live, base.target = plan.target, base.row = plan.row, base.lse = a->lse, base.dloss = a->dloss;
    base.g = reinterpret_cast<bf16*>(w + p.g), base.planes = p.gplanes;
    for (long v0 = 0; rc == EWS_OK && v0 < a->vocab; v0 += p.piece) {
        const long n = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;
        if ((rc = operands<T>(a, p, w, v0, n, &h, &wt, s)) != EWS_OK) break;
        Gemm g = base;
        g.job[0] = job_of(a->rows, n, a->dim, 1), g.v0 = (int)v0;
        g.ldg = up(n, 8), g.g_plane = a->rows * g.ldg;
        if ((rc = gemm<GRAD>(g, h, wt, none, none, p.planes, s)) != EWS_OK) break;
        go.p = g.g, go.rows = a->rows, go.cols = n, go.ld = g.ldg, go.plane = g.g_plane, go.planes = p.gplanes;
        Gemm o = base;
        T* out = static_cast<T*>(a->dweight) + (a->dweight ? v0 * a->dim : 0);
        if (a->dhidden) {  // dH += G W: K is the piece of the vocabulary
            o.job[0] = job_of(a->rows, a->dim, n, p.split_h);
            o.job[0].acc = acc_h, o.job[0].add = v0 > 0;
        }
        if (a->dweight) {  // dW = G^T H: K is the rows
            o.job[1] = job_of(n, a->dim, a->rows, p.split_w);
            o.job[1].acc = acc_w;
            if constexpr (sizeof(T) == 2) o.job[1].out = out;  // read where there are no partials
        }
        if ((rc = gemm<OUT>(o, go, wt, go, h, p.planes, s)) != EWS_OK) break;
        if (a->dweight && acc_w) rc = reduce<T>(a, acc_w, p.split_w, n, nullptr, base.inv_tau, out, s);
    }
    if (rc == EWS_OK && a->dhidden) rc = reduce<T>(a, acc_h, p.split_h, a->rows, plan.slot, base.inv_tau, static_cast<T*>(a->dhidden), s);
    return rc;
}

}  // namespace vocab
}  // namespace ews

using namespace ews::vocab;

extern "C" size_t ews_vocab_work_size(const ews_vocab_args* a, int backward_pass) {
    return check(a) == EWS_OK && a->rows > 0 ? plan(a, backward_pass != 0).bytes : 0;
}

namespace ews {
namespace vocab {

int run_forward(const ews_vocab_args* a, const Entries* e, cudaStream_t s) {
    const Plan p = plan(a, false, e ? e->top : 0);
    if (!a->work || !aligned16(a->work) || a->work_bytes < p.bytes) return EWS_ERR_WORKSPACE;
    return a->dtype == EWS_DTYPE_BF16 ? forward<bf16>(a, p, e, s) : forward<float>(a, p, e, s);
}

int run_backward(const ews_vocab_args* a, const Entries* e, cudaStream_t s) {
    if (a->rows == 0) {
        const size_t size = a->dtype == EWS_DTYPE_BF16 ? 2 : 4;
        if (a->dweight && cudaMemsetAsync(a->dweight, 0, size * a->vocab * a->dim, s) != cudaSuccess) return EWS_ERR_LAUNCH;
        return EWS_OK;
    }
    if (!a->hidden || !a->weight || !a->dloss || !a->lse || !a->plan) return EWS_ERR_INVALID_ARGUMENT;
    if (!a->dhidden && !a->dweight) return EWS_OK;
    const Plan p = plan(a, true, e ? e->top : 0);
    if (!a->work || !aligned16(a->work) || a->work_bytes < p.bytes) return EWS_ERR_WORKSPACE;
    return a->dtype == EWS_DTYPE_BF16 ? backward<bf16>(a, p, e, s) : backward<float>(a, p, e, s);
}

int check_top(const ews_distill_args* a) {
    if (!a) return EWS_ERR_INVALID_ARGUMENT;
    const int rc = check(&a->v);
    if (rc != EWS_OK) return rc;
    if (a->top <= 0 || !(a->inv_temperature >= FLT_MIN && a->inv_temperature <= FLT_MAX)) return EWS_ERR_INVALID_ARGUMENT;
    if (a->top > kMaxTop || (a->logits_dtype != EWS_DTYPE_F32 && a->logits_dtype != EWS_DTYPE_BF16)) return EWS_ERR_UNSUPPORTED;
    return EWS_OK;
}

}  // namespace vocab
}  // namespace ews

extern "C" int ews_vocab_fwd(const ews_vocab_args* a, ews_stream_t stream) {
    const int rc = check(a);
    if (rc != EWS_OK) return rc;
    if (a->rows == 0) return EWS_OK;
    if (!a->hidden || !a->weight || !a->targets || !a->loss || !a->lse || !a->plan) return EWS_ERR_INVALID_ARGUMENT;
    return run_forward(a, nullptr, (cudaStream_t)stream);
}

extern "C" int ews_vocab_bwd(const ews_vocab_args* a, ews_stream_t stream) {
    const int rc = check(a);
    return rc != EWS_OK ? rc : run_backward(a, nullptr, (cudaStream_t)stream);
}

extern "C" size_t ews_distill_entries_size(int64_t rows, int top) {
    return rows > 0 && top > 0 ? sizeof(int) * 2 * (size_t)rows * ((size_t)top + 1) : 0;
}

extern "C" size_t ews_distill_work_size(const ews_distill_args* a, int backward_pass) {
    return check_top(a) == EWS_OK && a->v.rows > 0 ? plan(&a->v, backward_pass != 0, a->top).bytes : 0;
}

extern "C" int ews_distill_fwd(const ews_distill_args* a, ews_stream_t stream) {
    const int rc = check_top(a);
    if (rc != EWS_OK) return rc;
    const ews_vocab_args* v = &a->v;
    if (v->rows == 0) return EWS_OK;
    if (!v->hidden || !v->weight || !v->loss || !v->lse || !v->plan || !a->ids || !a->logits || !a->entries) return EWS_ERR_INVALID_ARGUMENT;
    const Plan p = plan(v, false, a->top);
    if (!v->work || !ews::token::aligned16(v->work) || v->work_bytes < p.bytes) return EWS_ERR_WORKSPACE;
    cudaStream_t s = (cudaStream_t)stream;
    const Entries e = entries_of(a->entries, v->rows, a->top, a->inv_temperature);
    const unsigned grid = (unsigned)((v->rows + 7) / 8);
    if (a->logits_dtype == EWS_DTYPE_BF16)
        entries_kernel<ews::token::bf16><<<grid, 256, 0, s>>>(a->ids, a->ids_wide, static_cast<const ews::token::bf16*>(a->logits), v->rows, v->vocab, e, v->status);
    else
        entries_kernel<float><<<grid, 256, 0, s>>>(a->ids, a->ids_wide, static_cast<const float*>(a->logits), v->rows, v->vocab, e, v->status);
    if (cudaGetLastError() != cudaSuccess) return EWS_ERR_LAUNCH;
    return run_forward(v, &e, s);
}

extern "C" int ews_distill_bwd(const ews_distill_args* a, ews_stream_t stream) {
    const int rc = check_top(a);
    if (rc != EWS_OK) return rc;
    if (a->v.rows > 0 && !a->entries) return EWS_ERR_INVALID_ARGUMENT;
    const Entries e = entries_of(a->entries, a->v.rows, a->top, a->inv_temperature);
    return run_backward(&a->v, &e, (cudaStream_t)stream);
}
